// group.cu -- contractions with 4-bit weights, a scale and a zero point per group of inputs.
//
//   w[j][i] = s[j][i / g] (q[j][i] - z[j][i / g]),   q and z in 0..15 (z = 8 where none are given)
//   Y[b][j] = sum_i w[j][i] X[b][i] + bias[j] * delta on the body       (transposed: sum over j)
//
// mod 2^64 over LWE ciphertexts.  |w| <= 128 * 15 = 1920.  X comes as rows of u64 words, or as the
// rounded words of a cache (cache.cu), whose limbs below the kept ones are zero.  The reference's
// Linear holds one integer per weight (runtime/src/ops/linear.rs:52-75).
#include <algorithm>
#include <atomic>

#include "pnb_keys.h"
#include "tc_tiles.cuh"

namespace pnb {

struct GroupWeights {
  const uint8_t* q;      // [M][ceil(K / 2)], low nibble first
  const int8_t* scales;  // [M][groups]
  const uint8_t* zeros;  // [M][groups] or null
  int M, K, group, groups;
  bool transposed;
  __device__ __forceinline__ int at(int j, int i) const {
    const int v = __ldg(q + (size_t)j * ((K + 1) / 2) + i / 2) >> (4 * (i & 1)) & 15;
    const size_t g = (size_t)j * groups + i / group;
    return __ldg(scales + g) * (v - (zeros ? __ldg(zeros + g) & 15 : 8));
  }
};

struct GroupArgs {
  GroupWeights w;
  const int64_t* bias;
  const int32_t* slots;   // of the cache; null: X holds the batch's rows
  const unsigned char* X;
  uint64_t* Y;
  uint64_t delta;
  size_t x_row;           // bytes between ciphertexts of X
  int batch, n_slots, n_in, n_out, L, ldy;
};

// ---- few products -------------------------------------------------------------------------------
// One thread per word, 16 outputs at a time, weights in shared memory as w + 2048 >= 0, so that a product
// is one 32 x 32 + 64 and one 32 x 32 + 32 bit multiply-add and sum w x = sum (w + 2048) x - 2048 sum x.
constexpr int GF_THREADS = 256, GF_OUT = 16, GF_IN = 64;
constexpr uint32_t GF_BIAS = 2048;
constexpr long long GF_MOST = 256;  // weights that go this way

// A word of X, of 8 bytes or the top 2, 3 or 4 of them.
template <int BYTES>
__device__ __forceinline__ uint64_t load_word(const unsigned char* row, int c) {
  if (BYTES == 8) return __ldg(reinterpret_cast<const unsigned long long*>(row) + c);
  if (BYTES == 4) return (uint64_t)__ldg(reinterpret_cast<const uint32_t*>(row) + c) << 32;
  if (BYTES == 2) return (uint64_t)__ldg(reinterpret_cast<const uint16_t*>(row) + c) << 48;
  const unsigned char* p = row + 3 * c;
  return (uint64_t)(__ldg(p) | (uint32_t)__ldg(p + 1) << 8 | (uint32_t)__ldg(p + 2) << 16) << 40;
}

template <int BYTES>
__global__ void __launch_bounds__(GF_THREADS) group_few_kernel(const __grid_constant__ GroupArgs a) {
  __shared__ __align__(16) uint32_t w_s[GF_IN][GF_OUT];
  const int c = blockIdx.x * GF_THREADS + threadIdx.x;
  const int j0 = blockIdx.y * GF_OUT;
  for (int b = blockIdx.z; b < a.batch; b += gridDim.z) {
    const int src = a.slots ? __ldg(a.slots + b) : b;
    if (a.slots && (src < 0 || src >= a.n_slots)) continue;
    const unsigned char* x = a.X + (size_t)src * a.n_in * a.x_row;
    uint64_t acc[GF_OUT] = {}, sum = 0;
    for (int k0 = 0; k0 < a.n_in; k0 += GF_IN) {
      const int n = min(GF_IN, a.n_in - k0);
      __syncthreads();  // the last chunk has been read
      for (int i = threadIdx.x; i < n * GF_OUT; i += GF_THREADS) {
        const int k = i / GF_OUT, j = j0 + i % GF_OUT;
        const int w = j >= a.n_out ? 0 : a.w.transposed ? a.w.at(k0 + k, j) : a.w.at(j, k0 + k);
        w_s[k][i % GF_OUT] = GF_BIAS + (uint32_t)w;
      }
      __syncthreads();
      if (c >= a.L) continue;
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const uint64_t v = load_word<BYTES>(x + (size_t)(k0 + k) * a.x_row, c);
        sum += v;
        const uint4* w4 = reinterpret_cast<const uint4*>(w_s[k]);
#pragma unroll
        for (int u = 0; u < GF_OUT / 4; ++u) {
          const uint4 w = w4[u];
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int h = 0; h < 4; ++h)
            acc[4 * u + h] += (uint64_t)(uint32_t)v * ws[h] +
                              ((uint64_t)((uint32_t)(v >> 32) * ws[h]) << 32);
        }
      }
    }
    if (c >= a.L) continue;
    uint64_t* y = a.Y + ((size_t)b * a.n_out + j0) * a.ldy + c;
#pragma unroll
    for (int u = 0; u < GF_OUT; ++u) {
      if (j0 + u >= a.n_out) break;
      uint64_t v = acc[u] - GF_BIAS * sum;
      if (a.bias && c == a.L - 1) v += (uint64_t)__ldg(a.bias + j0 + u) * a.delta;
      y[(size_t)u * a.ldy] = v;
    }
  }
}

// ---- weights as bytes ---------------------------------------------------------------------------
// Two rows of signed bytes per output, w = 256 hi + lo: row 2j holds the lo of output j, row 2j + 1 its
// hi.  Rows are padded by zeros to a multiple of 16 bytes.  A thread makes 16 bytes of both.
constexpr int GX_THREADS = 128;

__global__ void __launch_bounds__(GX_THREADS)
    group_expand_kernel(const __grid_constant__ GroupWeights w, int n_in, int n_out, int pitch,
                        int8_t* to) {
  asm volatile("griddepcontrol.launch_dependents;");
  // neighbouring threads read neighbouring bytes: along the inputs, or transposed along the outputs
  const int chunks = pitch / 16;
  const long long t = (long long)blockIdx.x * GX_THREADS + threadIdx.x;
  if (t >= (long long)chunks * n_out) return;
  const int o = (int)(w.transposed ? t % n_out : t / chunks);
  const int i0 = (int)(w.transposed ? t / n_out : t % chunks) * 16;
  union { int8_t b[16]; uint4 v; } lo, hi;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int v = i0 + i >= n_in ? 0 : w.transposed ? w.at(i0 + i, o) : w.at(o, i0 + i);
    lo.b[i] = (int8_t)v;
    hi.b[i] = (int8_t)((v - lo.b[i]) >> 8);
  }
  uint4* out = reinterpret_cast<uint4*>(to + (size_t)2 * o * pitch + i0);
  out[0] = lo.v;
  out[pitch / 16] = hi.v;
}

// ---- tensor cores -------------------------------------------------------------------------------
// Status word of the kernel: non-zero when one of its bounded waits ran out.
__device__ int g_gc_status;

int gc_status_read_and_clear(int* out) {
  int v = 0;
  PNB_CUDA(cudaMemcpyFromSymbol(&v, g_gc_status, sizeof(int)));
  const int zero = 0;
  PNB_CUDA(cudaMemcpyToSymbol(g_gc_status, &zero, sizeof(int)));
  *out = v;
  return PNB_OK;
}

constexpr int GC_BM = 128;       // weight rows per tile: 64 outputs
constexpr int GC_OUT = GC_BM / 2;
constexpr int GC_WK = 128;       // inputs per weight slot
constexpr int GC_XK = 64;        // inputs per X slot
constexpr int GC_KSTEP = 32;     // inputs per MMA
constexpr int GC_W_SLOT = GC_BM * GC_WK;  // 16 KB
constexpr int GC_X_SLOT = GC_XK * 256;    // 16 KB
constexpr int GC_EPI_WARPS = 8;  // two per TMEM lane quarter
constexpr int GC_COPY_WARPS = 4;
constexpr int GC_PART = 16;      // words staged at a time: rows of 128 bytes
constexpr int GC_STAGE = 16 * GC_PART * 8;  // of one warp: its 16 outputs
constexpr int GC_MAX_W = 12, GC_MAX_X = 12, GC_MAX_RAW = 16;
constexpr int GC_RAW_ROWS = 32, GC_RAW_PITCH = 256 + 16, GC_RAW_SLOT = GC_RAW_ROWS * GC_RAW_PITCH;
constexpr int GC_BARS = 2 * (GC_MAX_W + GC_MAX_X + GC_MAX_RAW) + 4;
constexpr int GC_BAR_BYTES = (8 * GC_BARS + 8 + 127) / 128 * 128;
constexpr int GC_SMEM = 227 * 1024;
constexpr uint32_t GC_WAIT_LIMIT = 1u << 24;

template <int BYTES, bool SHIFTED>
struct GcShape {
  // words of X per tile: 256 bytes (192 of the 256 that are loaded where words have three)
  static constexpr int WORDS = BYTES == 8 ? 32 : BYTES == 2 ? 128 : 64;
  static constexpr int BN = WORDS * BYTES;
  static constexpr int COPY = SHIFTED ? GC_COPY_WARPS : 0;
  static constexpr int MMA_WARP = 2 + COPY;  // warp 0 loads X, warp 1 the weights
  static constexpr int EPI_WARP = MMA_WARP + 1;
  static constexpr int THREADS = 32 * (EPI_WARP + GC_EPI_WARPS);
  static constexpr int EW = WORDS / 2;       // words per epilogue warp
  static constexpr int CW = BYTES == 8 ? 4 : BYTES == 2 ? 16 : 8;  // of which it fetches at a time
  static constexpr int COLS = CW * BYTES;
};

struct GcMaps {
  CUtensorMap W, Y;
  CUtensorMap X[2];  // shifted: rows 0, 2, .. and 1, 3, ..; else X[0]
};

struct GcArgs {
  GroupArgs g;
  int off0, off1;    // words by which rows 0, 2, .. / 1, 3, .. start past 16-byte alignment
  int n_tiles, m_tiles;
  long long total;   // tiles: outputs fastest, then words, then requests
  int keep_w;        // a block's tiles all have the same outputs, whose weights stay
  int w_slots, x_slots, raw_slots;
  int x_at, raw_at, out_at, bars_at;  // shared-memory offsets; weights at 0
  int plain_out;     // results leave by plain stores
};

// A block's tiles, one grid apart.  The next one's slot is on its way while one is worked on.
struct GcTile {
  int b, nt, m, src;
};
template <bool CACHED>
struct GcWalk {
  const GcArgs& a;
  long long t;
  int slot = 0;
  __device__ __forceinline__ explicit GcWalk(const GcArgs& args) : a(args), t(blockIdx.x) {
    if (CACHED && t < a.total) slot = __ldg(a.g.slots + t / a.m_tiles / a.n_tiles);
  }
  // the next tile that has something to do; false behind the last
  __device__ __forceinline__ bool next(GcTile& tile) {
    while (t < a.total) {
      const long long u = t / a.m_tiles, b = u / a.n_tiles;
      tile.m = (int)(t - u * a.m_tiles);
      tile.nt = (int)(u - b * a.n_tiles);
      tile.b = (int)b;
      tile.src = CACHED ? slot : (int)b;
      t += gridDim.x;
      if (!CACHED) return true;
      if (t < a.total) slot = __ldg(a.g.slots + t / a.m_tiles / a.n_tiles);
      if (tile.src >= 0 && tile.src < a.g.n_slots) return true;
    }
    return false;
  }
};

// Bounded wait that also gives up as soon as another role has flagged an abort.
__device__ __noinline__ bool gc_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_s) {
  for (uint32_t it = 0; it < GC_WAIT_LIMIT; it += 1024) {
    if (tc::mbar_wait(bar, parity, 1024)) return true;
    if (*abort_s) return false;
  }
  *abort_s = 1;
  atomicExch(&g_gc_status, 1);
  return false;
}
__device__ __forceinline__ bool gc_wait(uint32_t bar, uint32_t parity, volatile int* abort_s) {
  return tc::mbar_test(bar, parity & 1u) || gc_wait_slow(bar, parity & 1u, abort_s);
}

template <int COLS>
__device__ __forceinline__ void gc_tmem_ld(uint32_t at, uint32_t (&r)[COLS]) {
  if constexpr (COLS == 32) {
    tc::tmem_ld_32x32_nowait(at, r);
  } else {
    static_assert(COLS == 24, "16 and 8 columns");
    tc::tmem_ld_32x32_x16(at, *reinterpret_cast<uint32_t(*)[16]>(&r[0]));
    tc::tmem_ld_32x32_x8(at + 16, *reinterpret_cast<uint32_t(*)[8]>(&r[16]));
  }
}

// The word that the limb sums c stand for, mod 2^64; of a cache's word its high half, the low one is zero.
template <int BYTES>
__device__ __forceinline__ uint64_t gc_word(const uint32_t* c) {
  if constexpr (BYTES == 8) {
    return add_limbs(0, c);
  } else {
    uint32_t v = c[0];
#pragma unroll
    for (int b = 1; b < BYTES; ++b) v += c[b] << (8 * b);
    return (uint64_t)(v << (32 - 8 * BYTES)) << 32;
  }
}

template <int BYTES>
__device__ __forceinline__ uint64_t gc_other_lane(uint64_t v) {
  if (BYTES == 8) return shfl_xor_u64(v, 1);
  return (uint64_t)__shfl_xor_sync(0xffffffffu, (uint32_t)(v >> 32), 1) << 32;
}

template <int BYTES, bool SHIFTED>
__global__ void __launch_bounds__(GcShape<BYTES, SHIFTED>::THREADS, 1)
    group_kernel(const __grid_constant__ GcMaps tm, const __grid_constant__ GcArgs a) {
  using S = GcShape<BYTES, SHIFTED>;
  constexpr bool CACHED = BYTES != 8;
  extern __shared__ __align__(1024) unsigned char gc_raw[];  // the swizzles want 1024-byte boundaries
  const uint32_t base = tc::smem_u32(gc_raw);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(&g_gc_status, 1);
    return;
  }
  auto w_at = [&](int s) { return base + (uint32_t)(s * GC_W_SLOT); };
  auto x_at = [&](int s) { return base + (uint32_t)(a.x_at + s * GC_X_SLOT); };
  auto raw_at = [&](int s) { return base + (uint32_t)(a.raw_at + s * GC_RAW_SLOT); };
  const uint32_t bars = base + (uint32_t)a.bars_at;
  const uint32_t w_full = bars, w_empty = w_full + 8 * GC_MAX_W;
  const uint32_t x_full = w_empty + 8 * GC_MAX_W, x_empty = x_full + 8 * GC_MAX_X;
  const uint32_t r_full = x_empty + 8 * GC_MAX_X, r_empty = r_full + 8 * GC_MAX_RAW;
  const uint32_t acc_full = r_empty + 8 * GC_MAX_RAW, acc_empty = acc_full + 16;
  const uint32_t holder = bars + 8 * GC_BARS;
  volatile int* abort_s = reinterpret_cast<volatile int*>(gc_raw + (holder + 4 - base));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.w_slots; ++s) {
      tc::mbar_init(w_full + 8 * s, 1);
      tc::mbar_init(w_empty + 8 * s, 1);
    }
    for (int s = 0; s < a.x_slots; ++s) {
      tc::mbar_init(x_full + 8 * s, SHIFTED ? S::COPY : 1);
      tc::mbar_init(x_empty + 8 * s, 1);
    }
    for (int s = 0; s < a.raw_slots; ++s) {
      tc::mbar_init(r_full + 8 * s, 1);
      tc::mbar_init(r_empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(acc_full + 8 * s, 1);
      tc::mbar_init(acc_empty + 8 * s, GC_EPI_WARPS);
    }
    *abort_s = 0;
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tm.W);
    tc::prefetch_tmap(&tm.X[0]);
    if (SHIFTED) tc::prefetch_tmap(&tm.X[1]);
    if (!a.plain_out) tc::prefetch_tmap(&tm.Y);
  }
  if (warp == S::MMA_WARP) tc::tmem_alloc(holder, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gc_raw + (holder - base));

  const int kx_n = (a.g.n_in + GC_XK - 1) / GC_XK;  // X slots of one tile
  const int kb_n = (a.g.n_in + GC_WK - 1) / GC_WK;  // weight slots
  GcTile tile;

  if (warp == 0) {
    // ---------------- X loads (one lane) ---------------------------------------------------------
    // X was there before the weights' kernel began, so it need not be waited for.
    if (lane == 0) {
      TileRing ring;
      bool wrapped = false, ok = true;
      const int slots = SHIFTED ? a.raw_slots : a.x_slots;
      GcWalk<CACHED> walk(a);
      while (ok && walk.next(tile)) {
        for (int k = 0; k < a.g.n_in; k += SHIFTED ? GC_RAW_ROWS : GC_XK) {
          const int s = ring.slot;
          const uint32_t full = (SHIFTED ? r_full : x_full) + 8 * s;
          ok = gc_wait((SHIFTED ? r_empty : x_empty) + 8 * s, ring.phase ^ 1u, abort_s);
          if (!ok) break;
          if (SHIFTED) {
            const int row = tile.src * a.g.n_in + k;
            tc::mbar_expect_tx(full, GC_RAW_SLOT);  // the rows of either parity, in order
            tc::tma_load_2d(raw_at(s), &tm.X[row & 1], tile.nt * S::WORDS, row >> 1, full);
            tc::tma_load_2d(raw_at(s) + GC_RAW_SLOT / 2, &tm.X[(row + 1) & 1], tile.nt * S::WORDS,
                            (row + 1) >> 1, full);
          } else {
            tc::mbar_expect_tx(full, GC_X_SLOT);  // rows past the last input read as zeros
            tc::tma_load_3d(x_at(s), &tm.X[0], tile.nt * S::BN, k, tile.src, full);
            tc::tma_load_3d(x_at(s) + GC_X_SLOT / 2, &tm.X[0], tile.nt * S::BN + 128, k, tile.src,
                            full);
          }
          ring.advance(slots);
          wrapped |= ring.slot == 0;
        }
      }
      tile_drain(SHIFTED ? r_full : x_full, ring, wrapped, slots, GC_WAIT_LIMIT);
    }
  } else if (warp == 1) {
    // ---------------- weight loads (one lane) ----------------------------------------------------
    if (lane == 0) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the weights' kernel is done
      TileRing ring;
      bool wrapped = false, ok = true;
      GcWalk<CACHED> walk(a);
      while (ok && walk.next(tile)) {
        for (int k = 0; k < kb_n; ++k) {
          const int s = ring.slot;
          ok = gc_wait(w_empty + 8 * s, ring.phase ^ 1u, abort_s);
          if (!ok) break;
          tc::mbar_expect_tx(w_full + 8 * s, GC_W_SLOT);
          tc::tma_load_2d(w_at(s), &tm.W, k * GC_WK, tile.m * GC_BM, w_full + 8 * s);
          ring.advance(a.w_slots);
          wrapped |= ring.slot == 0;
        }
        if (a.keep_w) break;
      }
      tile_drain(w_full, ring, wrapped, a.w_slots, GC_WAIT_LIMIT);
    }
  } else if (SHIFTED && warp < S::MMA_WARP) {
    // ---------------- raw rows -> operand layout (shifted rows only) -----------------------------
    // Raw slot r is copied by warp r % 4 (their number is a multiple of 4).  Every warp waits for every
    // X slot's turn and answers it, also where it copies nothing: a parity tells only neighbouring
    // turns apart.
    const int cw = warp - 2;
    constexpr int BATCH = 16;  // rows whose words are on their way together
    const int box = lane >> 4, ch = (lane & 15) >> 1, half = lane & 1;
    TileRing xr, rr;
    bool ok = true;
    GcWalk<CACHED> walk(a);
    while (ok && walk.next(tile)) {
      const int parity = tile.src * a.g.n_in & 1;  // of the tile's first row
      const int off_e = parity ? a.off1 : a.off0, off_o = parity ? a.off0 : a.off1;
      for (int kx = 0; ok && kx < kx_n; ++kx) {
        ok = gc_wait(x_empty + 8 * xr.slot, xr.phase ^ 1u, abort_s);
        if (!ok) break;
        const int raws = min(2, (a.g.n_in - kx * GC_XK + GC_RAW_ROWS - 1) / GC_RAW_ROWS);
        for (int i = 0; i < raws; ++i) {
          if ((rr.slot & 3) == cw) {
            ok = gc_wait(r_full + 8 * rr.slot, rr.phase, abort_s);
            if (!ok) break;
            // row r of the slot: its parity's half, r / 2; one word further where it is shifted
            const unsigned char* from = gc_raw + (raw_at(rr.slot) - base) + lane * 8;
            unsigned char* to = gc_raw + (x_at(xr.slot) - base) + box * (GC_XK * 128) +
                                i * (GC_RAW_ROWS * 128) + half * 8;
#pragma unroll
            for (int r0 = 0; r0 < GC_RAW_ROWS; r0 += BATCH) {
              uint64_t v[BATCH];
#pragma unroll
              for (int j = 0; j < BATCH; ++j) {
                const int r = r0 + j;
                v[j] = *reinterpret_cast<const uint64_t*>(
                    from + (r & 1 ? GC_RAW_SLOT / 2 + off_o * 8 : off_e * 8) +
                    (r >> 1) * GC_RAW_PITCH);
              }
#pragma unroll
              for (int j = 0; j < BATCH; ++j) {
                const int r = r0 + j;
                *reinterpret_cast<uint64_t*>(to + r * 128 + ((ch ^ (r & 7)) << 4)) = v[j];
              }
            }
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(r_empty + 8 * rr.slot);
          }
          rr.advance(a.raw_slots);
        }
        if (!ok) break;
        if (lane == 0) tc::mbar_arrive(x_full + 8 * xr.slot);
        xr.advance(a.x_slots);
      }
    }
  } else if (warp == S::MMA_WARP) {
    // ---------------- products (one lane) --------------------------------------------------------
    if (lane == 0) {
      constexpr uint32_t IDESC = tc::idesc_i8(GC_BM, S::BN, true, false, false, true);
      const uint64_t wd = tc::smem_desc_sw128(w_at(0), 16u, 1024u);
      const uint64_t xd = tc::smem_desc_sw128(x_at(0), GC_XK * 128u, 1024u);
      const uint32_t w_hi = (uint32_t)(wd >> 32), x_hi = (uint32_t)(xd >> 32);
      const int steps = (a.g.n_in + GC_KSTEP - 1) / GC_KSTEP;
      TileRing x, w;
      int tt = 0;
      bool ok = true;
      GcWalk<CACHED> walk(a);
      while (ok && walk.next(tile)) {
        const int buf = tt & 1;
        const uint32_t d = tmem + (uint32_t)(buf * 256);
        ok = gc_wait(acc_empty + 8 * buf, (uint32_t)(tt >> 1) ^ 1u, abort_s);
        if (!ok) break;
        tc::tc_fence_after();
        const bool load = !a.keep_w || tt == 0;
        if (a.keep_w) w = TileRing{};
        uint32_t acc = 0;
        for (int left = steps, kx = 0; left > 0; left -= GC_XK / GC_KSTEP, ++kx) {
          if ((kx & 1) == 0 && load) {
            ok = gc_wait(w_full + 8 * w.slot, w.phase, abort_s);
            if (!ok) break;
          }
          ok = gc_wait(x_full + 8 * x.slot, x.phase, abort_s);
          if (!ok) break;
          const uint32_t x_lo = (uint32_t)xd + (uint32_t)(x.slot * (GC_X_SLOT / 16));
          const uint32_t w_lo = (uint32_t)wd + (uint32_t)(w.slot * (GC_W_SLOT / 16)) + 4u * (kx & 1);
#pragma unroll
          for (int k = 0; k < GC_XK / GC_KSTEP; ++k)
            if (k < left)
              tc::mma_i8_lo(d, w_lo + 2 * k, w_hi, x_lo + 256 * k, x_hi, IDESC, k ? 1u : acc);
          acc = 1;
          tc::mma_commit(x_empty + 8 * x.slot);
          x.advance(a.x_slots);
          if ((kx & 1) || left <= GC_XK / GC_KSTEP) {
            if (!a.keep_w) tc::mma_commit(w_empty + 8 * w.slot);
            w.advance(a.w_slots);
          }
        }
        if (!ok) break;
        tc::mma_commit(acc_full + 8 * buf);
        ++tt;
      }
    }
  } else {
    // ---------------- epilogue -------------------------------------------------------------------
    // Warp w reads TMEM lane quarter w % 4 and half eh of the tile's words.  An even lane has an output's
    // lo sums and the odd lane beside it the hi sums: of every two words each lane completes one, with
    // the other lane's share of it.  Words are staged in shared memory, 16 outputs x 16 words at a time with
    // the 16-byte chunks XORed by the row, and leave by TMA, or as row segments by plain stores.
    const int e_w = warp - S::EPI_WARP;
    const int q = warp & 3, eh = e_w >> 2;
    const bool odd = lane & 1;
    const uint32_t out_at = base + (uint32_t)(a.out_at + e_w * GC_STAGE);
    unsigned char* out = gc_raw + (out_at - base);
    const int row = lane >> 1;  // of the warp's 16 outputs
    unsigned char* out_row = out + row * 128 + odd * 8;
    int tt = 0;
    bool ok = true;
    GcWalk<CACHED> walk(a);
    while (walk.next(tile)) {
      const int buf = tt & 1;
      ok = gc_wait(acc_full + 8 * buf, (uint32_t)(tt >> 1), abort_s);
      if (!ok) break;
      tc::tc_fence_after();
      ++tt;
      const uint32_t c_tmem = tmem + (uint32_t)(buf * 256 + eh * (S::BN / 2)) +
                              ((uint32_t)(q * 32) << 16);
      const int row0 = tile.m * GC_OUT + q * 16, col0 = tile.nt * S::WORDS + eh * S::EW;
      if (row0 >= a.g.n_out || col0 >= a.g.L) {  // nothing of this warp's share is kept
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(acc_empty + 8 * buf);
        continue;
      }
      const int body = a.g.L - 1 - col0;  // the body among this warp's words
      const bool live = row0 + row < a.g.n_out;
      uint64_t bias = 0;
      if (a.g.bias && body < S::EW && live)
        bias = (uint64_t)__ldg(a.g.bias + row0 + row) * a.g.delta;
      constexpr int CHUNKS = S::EW / S::CW, PER_PART = GC_PART / S::CW;
      uint32_t c[2][S::COLS];
      gc_tmem_ld<S::COLS>(c_tmem, c[0]);
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        tc::tmem_ld_wait_pin(c[i & 1]);
        if (i + 1 < CHUNKS) {
          gc_tmem_ld<S::COLS>(c_tmem + (uint32_t)((i + 1) * S::COLS), c[(i + 1) & 1]);
        } else {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(acc_empty + 8 * buf);
        }
        const int w0 = i * S::CW / GC_PART * GC_PART;  // the part's first word
        if (i % PER_PART == 0 && !a.plain_out) {  // what was staged before has left
          if (lane == 0) tc::tma_store_wait_read();
          __syncwarp();
        }
#pragma unroll
        for (int u = 0; u < S::CW; u += 2) {
          uint64_t v0 = gc_word<BYTES>(c[i & 1] + u * BYTES);
          uint64_t v1 = gc_word<BYTES>(c[i & 1] + (u + 1) * BYTES);
          if (odd) {
            v0 <<= 8;
            v1 <<= 8;
          }
          const uint64_t keep = odd ? v1 : v0, give = odd ? v0 : v1;
          uint64_t y = keep + gc_other_lane<BYTES>(give);
          const int word = i * S::CW + u;
          if (body - word == (odd ? 1 : 0)) {
            y += bias;
            // tiled stores end on 16-byte boundaries, so the last word of an odd count goes alone
            if (!a.plain_out && (a.g.L & 1) && live)
              a.g.Y[((size_t)tile.b * a.g.n_out + row0 + row) * a.g.ldy + a.g.L - 1] = y;
          }
          const int chunk = (word - w0) >> 1;
          *reinterpret_cast<uint64_t*>(out_row + ((chunk ^ (row & 7)) << 4)) = y;
        }
        if ((i + 1) % PER_PART != 0) continue;
        if (!a.plain_out) {
          tc::fence_async_smem();
          __syncwarp();
          if (lane == 0 && col0 + w0 < (a.g.L & ~1))
            tc::tma_store_3d(&tm.Y, col0 + w0, row0, tile.b, out_at);
        } else {
          __syncwarp();
          const int wd = lane & 15, sub = lane >> 4;
          uint64_t* y = a.g.Y + ((size_t)tile.b * a.g.n_out + row0 + sub) * a.g.ldy + col0 + w0 + wd;
          const int left = col0 + w0 + wd < a.g.L ? a.g.n_out - row0 - sub : 0;
          uint64_t v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            v[j] = *reinterpret_cast<const uint64_t*>(
                out + (2 * j + sub) * 128 + (((wd >> 1) ^ ((2 * j + sub) & 7)) << 4) + (wd & 1) * 8);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (2 * j < left) y[(size_t)(2 * j) * a.g.ldy] = v[j];
          __syncwarp();
        }
      }
    }
    if (!a.plain_out && lane == 0) tc::tma_store_wait();
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == S::MMA_WARP) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// ---- launch -------------------------------------------------------------------------------------
// How one block's shared memory is shared out.  Weights stay when they leave X four slots (shifted rows:
// three, and 40 KB of raw ones) and the grid is a whole number of times the tiles of outputs without
// losing more than a sixteenth of the machine.
template <bool SHIFTED>
static unsigned gc_plan(GcArgs& a, int sms) {
  const int kb = (a.g.n_in + GC_WK - 1) / GC_WK;
  int room = GC_SMEM - GC_BAR_BYTES - GC_EPI_WARPS * GC_STAGE;
  const int raw_min = SHIFTED ? 40 * 1024 / GC_RAW_SLOT * GC_RAW_SLOT : 0;
  const int x_min = SHIFTED ? 3 : 4;
  const int w_most = std::min(GC_MAX_W, (room - raw_min - x_min * GC_X_SLOT) / GC_W_SLOT);
  unsigned grid = (unsigned)std::min<long long>(a.total, sms);
  const unsigned whole = grid / a.m_tiles * a.m_tiles;
  a.keep_w = kb <= w_most && whole && 16 * (grid - whole) <= grid;
  if (a.keep_w) grid = whole;
  a.w_slots = a.keep_w ? kb : 4;
  room -= a.w_slots * GC_W_SLOT;
  if (SHIFTED) {
    a.x_slots = x_min;
    a.raw_slots = std::min(GC_MAX_RAW, (room - a.x_slots * GC_X_SLOT) / GC_RAW_SLOT & ~3);
  } else {
    a.x_slots = std::min(GC_MAX_X, room / GC_X_SLOT);
    a.raw_slots = 0;
  }
  a.x_at = a.w_slots * GC_W_SLOT;
  a.out_at = a.x_at + a.x_slots * GC_X_SLOT;
  a.raw_at = a.out_at + GC_EPI_WARPS * GC_STAGE;
  a.bars_at = a.raw_at + a.raw_slots * GC_RAW_SLOT;
  return grid;
}

template <int BYTES, bool SHIFTED>
static int gc_launch(const GcMaps& tm, GcArgs& a, cudaStream_t st) {
  using S = GcShape<BYTES, SHIFTED>;
  static std::atomic<int> sm_count[64];  // per device, once the kernel's shared-memory limit is raised
  int dev = 0;
  PNB_CUDA(cudaGetDevice(&dev));
  int sms = dev < 64 ? sm_count[dev].load(std::memory_order_acquire) : 0;
  if (sms == 0) {
    PNB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    PNB_CUDA(cudaFuncSetAttribute(group_kernel<BYTES, SHIFTED>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, GC_SMEM));
    if (dev < 64) sm_count[dev].store(sms, std::memory_order_release);
  }
  const unsigned grid = gc_plan<SHIFTED>(a, sms);
  cudaLaunchAttribute attr;  // its set-up and its first loads of X run beside the weights' kernel
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = (size_t)(a.bars_at + GC_BAR_BYTES);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  PNB_CUDA(cudaLaunchKernelEx(&cfg, group_kernel<BYTES, SHIFTED>, tm, a));
  return PNB_OK;
}

static int gc_run(const GroupArgs& g, int bits, int8_t* ws, cudaStream_t st) {
  const char* name = g.slots ? "group_contract_cached" : "group_contract";
  const int bytes = bits / 8;
  GcArgs a{};
  a.g = g;
  const int words = bytes == 8 ? 32 : bytes == 2 ? 128 : 64;
  a.n_tiles = (g.L + words - 1) / words;
  a.m_tiles = (g.n_out + GC_OUT - 1) / GC_OUT;
  a.total = (long long)g.batch * a.n_tiles * a.m_tiles;
  const long long x_rows = (long long)(g.slots ? g.n_slots : g.batch) * g.n_in;
  if (bytes == 8 && x_rows > 0x7fffffffLL - GC_BM) {  // (TMA coordinates are 32-bit)
    set_error("%s: %lld ciphertexts exceed a 32-bit index", name, x_rows);
    return PNB_ERR_INVALID;
  }
  const uintptr_t xw = (uintptr_t)g.X / 8;
  const int ldx = (int)(g.x_row / 8);  // (words)
  a.off0 = bytes == 8 ? (int)(xw & 1) : 0;
  a.off1 = bytes == 8 ? (int)((xw + (uintptr_t)ldx) & 1) : 0;
  const bool shifted = a.off0 || a.off1;
  a.plain_out = g.ldy % 2 != 0 || ((uintptr_t)g.Y % 16) != 0;
  const int pitch = (g.n_in + 15) & ~15;
  const long long chunks = (long long)g.n_out * (pitch / 16);
  if ((chunks + GX_THREADS - 1) / GX_THREADS > 0x7fffffffLL) {
    set_error("%s: %d x %d weights exceed one launch", name, g.n_out, g.n_in);
    return PNB_ERR_INVALID;
  }
  GcMaps tm{};
  int rc = tile_map_bytes(&tm.W, ws, (uint64_t)pitch, 2 * (uint64_t)g.n_out, (uint64_t)pitch, GC_WK,
                          GC_BM);
  if (rc) return rc;
  if (!shifted) {
    const cuuint64_t dims[3] = {(cuuint64_t)g.L * bytes, (cuuint64_t)g.n_in,
                                (cuuint64_t)(g.slots ? g.n_slots : g.batch)};
    const cuuint64_t strides[2] = {g.x_row, g.x_row * g.n_in};
    const cuuint32_t box[3] = {128, GC_XK, 1};
    rc = tile_map(&tm.X[0], CU_TENSOR_MAP_DATA_TYPE_UINT8, g.X, 3, dims, strides, box,
                  CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    // rows p, p + 2, ..: from the 16-byte boundary at or before row p, at twice the pitch.  A row
    // off by one word has that word's 16 bytes inside its allocation (allocations start aligned).
    for (int p = 0; p < 2 && !rc; ++p) {
      // (a single row has no row 1: both maps are its own, and the second meets zero weights)
      const bool second = p && x_rows > 1;
      const int off = second ? a.off1 : a.off0;
      const cuuint64_t dims[2] = {(cuuint64_t)g.L + off,
                                  (cuuint64_t)std::max<long long>(1, (x_rows + 1 - p) / 2)};
      const cuuint64_t strides[1] = {g.x_row * 2};
      const cuuint32_t box[2] = {GC_RAW_PITCH / 8, GC_RAW_ROWS / 2};
      rc = tile_map(&tm.X[p], CU_TENSOR_MAP_DATA_TYPE_UINT64,
                    reinterpret_cast<const uint64_t*>(g.X) + (second ? ldx : 0) - off, 2, dims,
                    strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
  }
  if (!rc && !a.plain_out) {
    // writes end at word L (rounded down to 16 bytes) of the last output of each request
    const cuuint64_t dims[3] = {(cuuint64_t)std::max(2, g.L & ~1), (cuuint64_t)g.n_out,
                                (cuuint64_t)g.batch};
    const cuuint64_t strides[2] = {(cuuint64_t)g.ldy * 8, (cuuint64_t)g.ldy * 8 * g.n_out};
    const cuuint32_t box[3] = {GC_PART, 16, 1};
    rc = tile_map(&tm.Y, CU_TENSOR_MAP_DATA_TYPE_UINT64, g.Y, 3, dims, strides, box,
                  CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (rc) return rc;
  group_expand_kernel<<<(unsigned)((chunks + GX_THREADS - 1) / GX_THREADS), GX_THREADS, 0, st>>>(
      g.w, g.n_in, g.n_out, pitch, ws);
  PNB_CHECK_LAUNCH("group_expand_kernel");
  switch (bytes) {
    case 8: return shifted ? gc_launch<8, true>(tm, a, st) : gc_launch<8, false>(tm, a, st);
    case 4: return gc_launch<4, false>(tm, a, st);
    case 3: return gc_launch<3, false>(tm, a, st);
    default: return gc_launch<2, false>(tm, a, st);
  }
}

size_t group_workspace_bytes(int n_in, int n_out) {
  return (size_t)2 * n_out * (((size_t)n_in + 15) & ~(size_t)15);
}

static int few_run(const GroupArgs& a, int bits, cudaStream_t st) {
  const dim3 grid((a.L + GF_THREADS - 1) / GF_THREADS, (a.n_out + GF_OUT - 1) / GF_OUT,
                  std::min(65535, a.batch));
  if (bits == 64)
    group_few_kernel<8><<<grid, GF_THREADS, 0, st>>>(a);
  else if (bits == 32)
    group_few_kernel<4><<<grid, GF_THREADS, 0, st>>>(a);
  else if (bits == 24)
    group_few_kernel<3><<<grid, GF_THREADS, 0, st>>>(a);
  else
    group_few_kernel<2><<<grid, GF_THREADS, 0, st>>>(a);
  PNB_CHECK_LAUNCH("group_few_kernel");
  return PNB_OK;
}

static int group_run(const GroupArgs& a, int bits, void* ws, size_t ws_bytes, cudaStream_t st) {
  const size_t need = group_workspace_bytes(a.n_in, a.n_out);
  if (ws && (ws_bytes < need || ((uintptr_t)ws % 16) != 0)) {
    set_error("%s: workspace of %zu bytes at %p, %zu bytes 16-byte aligned are needed",
              a.slots ? "group_contract_cached" : "group_contract", ws_bytes, ws, need);
    return PNB_ERR_INVALID;
  }
  if ((long long)a.n_in * a.n_out <= GF_MOST) return few_run(a, bits, st);
  int8_t* own = nullptr;
  if (!ws) PNB_CUDA(cudaMallocAsync((void**)&own, need, st));
  int rc = gc_run(a, bits, own ? own : (int8_t*)ws, st);
  if (own) {
    const cudaError_t e = cudaFreeAsync(own, st);
    if (!rc && e != cudaSuccess) rc = cuda_status(e, "cudaFreeAsync(weights as bytes)");
  }
  return rc;
}

int group_contract(const uint8_t* W, const int8_t* scales, const uint8_t* zeros, int group,
                   const int64_t* bias, uint64_t delta, int M, int K, bool transposed,
                   const uint64_t* X, int ldx, uint64_t* Y, int ldy, int batch, int L, void* ws,
                   size_t ws_bytes, cudaStream_t st) {
  GroupArgs a{};
  a.w = {W, scales, zeros, M, K, group, (K - 1) / group + 1, transposed};
  a.bias = bias; a.delta = delta;
  a.X = (const unsigned char*)X; a.x_row = (size_t)ldx * 8;
  a.Y = Y; a.ldy = ldy; a.batch = batch; a.L = L;
  a.n_in = transposed ? M : K;
  a.n_out = transposed ? K : M;
  return group_run(a, 64, ws, ws_bytes, st);
}

int group_contract_cached(const uint8_t* W, const int8_t* scales, const uint8_t* zeros, int group,
                          const int64_t* bias, uint64_t delta, int M, int K, const int32_t* slots,
                          const void* cache, int n_slots, int bits, uint64_t* Y, int ldy,
                          int batch, int L, void* ws, size_t ws_bytes, cudaStream_t st) {
  GroupArgs a{};
  a.w = {W, scales, zeros, M, K, group, (K - 1) / group + 1, false};
  a.bias = bias; a.delta = delta;
  a.slots = slots; a.n_slots = n_slots;
  a.X = (const unsigned char*)cache; a.x_row = cache_row_bytes(L, bits);
  a.Y = Y; a.ldy = ldy; a.batch = batch; a.L = L;
  a.n_in = K; a.n_out = M;
  return group_run(a, bits, ws, ws_bytes, st);
}

}  // namespace pnb

// group.cu -- contractions with 4-bit weights, a scale and a zero point per group of inputs.
//
//   w[j][i] = s[j][i / g] (q[j][i] - z[j][i / g]),   q and z in 0..15 (z = 8 where none are given)
//   Y[b][j] = sum_i w[j][i] X[b][i] + bias[j] * delta on the body       (transposed: sum over j)
//
// mod 2^64 over LWE ciphertexts.  |w| <= 128 * 15 = 1920.  X comes as rows of u64 words, or as the
// rounded words of a cache (cache.cu), whose limbs below the kept ones are zero.  The reference's
// Linear holds one integer per weight (runtime/src/ops/linear.rs:52-75).
//
// On the tensor cores (calls of few products take plain multiply-adds, below).  A word is BYTES
// little-endian byte limbs (8, or the 2 to 4 that a cache keeps), so the inputs of a request are a u8
// matrix [n_in][BYTES L], which kind::i8 reads as an MN-major operand where it lies; a weight is two
// signed bytes, w = lo + 256 hi, however small its group, and
//     Y = sum_p (LO[p] + HI[p - 1]) << 8p,    LO[p] = sum_i lo_i x_i[p],  HI[p] = sum_i hi_i x_i[p].
// (Products by the bare nibbles with a scale per group in the epilogue would need half of the MMAs and
// read the accumulators once per group: 13 times at K = 784 in groups of 64, where this reads two.)
//
// The floor is HBM, X read once and Y written once, with the MMAs close behind: 256 requests 784->128
// need 585 us for 3.83 GB at the measured copy bandwidth and 513 us for the products at twice the
// measured bf16 rate (from a cache of 32 bits 333 and 257).  Then shared memory: an MMA of N columns reads
// 4 KB of weights and 32 N bytes of X in N / 2 cycles, at N = 128 all of its 128 bytes a cycle.  And the
// path from the end of a tile's MMAs to the next ones into the same accumulator (a commit, a wait, two
// loads of columns, the limb sums, an arrival, a wait), about 2000 cycles.  So there are three forms:
//
//   LONG (over 896 inputs, over 4736 outputs, odd pitches over 384, more tiles of outputs than the device
//     has blocks or pairs for): tiles of 128 outputs x 32 words (of 8 bytes), lo and hi in 256 columns each;
//     weights stream from L2.
//   SHORT (up to 384 inputs): tiles of 128 x 16, lo and hi in 128 columns each, twice, so that the
//     epilogue of a tile runs beside the MMAs of the next; weights stay in shared memory.
//   PAIR (between): a pair of blocks shares a tile of 128 x 32 by MMAs of M = 256 (cta_group::2), each with
//     half of X and half of the weights, which stay.  Lo and hi are neighbouring rows, so that either block
//     can finish its half of the outputs; the lanes exchange words, which makes the epilogue dearer.
//
// Each form made to take the layers of the others, us, calls one after the other under the power cap (rows of
// 2049 random words), and the floors by bytes and by MMAs:
//                                                          SHORT   PAIR   LONG   bytes   MMAs
//     64 x 300->300                                          241    258    286      96    115
//     64 x 400->128                                                 128    175      85     65
//     64 x 784->128                                                 216    255     146    128
//     32 x 512->512                                                 238    263      82    167
//     61 x 130->200                                           99    125    176      50     32
//     61 x 130->200, odd pitch                               111           182      50     32
//     64 x 784->128, odd pitch (a pair that copied: 301 where LONG took 238)
//                                                                          272     146    128
// Measured: 256 x 784->128 670 us as a call of its own (0.87 of the copy's rate), 790-925 one after the
// other, where the power cap takes the SM clock to about 1.2 GHz; from 32 bits 370 and 420-486, from 16 250.
// 96 x 128->784 transposed 414-472 (its share of the floor, 219, is the lowest of the batches: the path
// above, 1000 cycles a tile).  45 x 257->384 from 24 bits 97-110.  One request 784->128 9.2 us in a graph,
// 13.6 a call: the host's.
// Layers of few outputs pay for 128 rows: 256 x 64->10 119 us (floor 47), 128->10 137 (89).
#include <algorithm>
#include <atomic>

#include "group_plan.h"
#include "pnb_keys.h"
#include "tc_tiles.cuh"

namespace pnb {

constexpr uint32_t GROUP_BIAS = 2048;  // above every |w|

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
  // The weights of output o for the 16 inputs from `in` (a multiple of 16, below n_in) on as signed
  // bytes, w = lo + 256 hi, four to a word; zeros past the last input.
  //
  // Eight weights at a time: two nibbles in the halves of a word, times the scale and plus 2048 - scale *
  // zero in both halves, give u = w + 2048 > 0 twice without a borrow between them.  The low byte of u is
  // that of w, and hi = ((u + 128) >> 8) - 8.
  __device__ __forceinline__ void bytes(int o, int in, int n_in, uint32_t (&lo)[4],
                                        uint32_t (&hi)[4]) const {
    uint32_t u[8];  // the u of inputs 8 h + k in the low half of u[4 h + k], of 8 h + k + 4 in its high one
    const int pitch = (K + 1) / 2;
    if (!transposed && in + 16 <= n_in && in % group + 16 <= group) {  // one scale
      const uint8_t* p = q + (size_t)o * pitch + in / 2;
      uint32_t v[2] = {0, 0};
      if (((uintptr_t)q & 3) == 0 && (pitch & 3) == 0) {
        v[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        v[1] = __ldg(reinterpret_cast<const uint32_t*>(p) + 1);
      } else {
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t / 4] |= (uint32_t)__ldg(p + t) << (8 * (t % 4));
      }
      const size_t g = (size_t)o * groups + in / group;
      const int scale = __ldg(scales + g), zero = zeros ? __ldg(zeros + g) & 15 : 8;
      const uint32_t more = (uint32_t)((int)GROUP_BIAS - scale * zero) * 0x10001u;
#pragma unroll
      for (int t = 0; t < 8; ++t)
        u[t] = (v[t / 4] >> (4 * (t % 4)) & 0x000f000fu) * (uint32_t)scale + more;
    } else {
      // all loads on their way together
      const int n = min(16, n_in - in);
      int w[16], scale[16], zero[16];
      const uint8_t* p = transposed ? q + (size_t)in * pitch + o / 2 : q + (size_t)o * pitch + in / 2;
      const size_t g0 = transposed ? (size_t)in * groups + o / group : (size_t)o * groups;
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const size_t row = t < n ? t : 0;
        const size_t g = transposed ? g0 + row * groups : g0 + (in + (int)row) / group;
        w[t] = __ldg(p + (transposed ? row * pitch : row / 2));
        scale[t] = __ldg(scales + g);
        zero[t] = zeros ? __ldg(zeros + g) : 8;
      }
#pragma unroll
      for (int t = 0; t < 16; ++t)
        w[t] = t < n ? scale[t] * ((w[t] >> (4 * ((transposed ? o : t) & 1)) & 15) - (zero[t] & 15)) : 0;
#pragma unroll
      for (int t = 0; t < 8; ++t)
        u[t] = (uint32_t)(w[t / 4 * 8 + t % 4] + (int)GROUP_BIAS) |
               (uint32_t)(w[t / 4 * 8 + t % 4 + 4] + (int)GROUP_BIAS) << 16;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t* x = u + 4 * h;
      const uint32_t l01 = __byte_perm(x[0], x[1], 0x6240), l23 = __byte_perm(x[2], x[3], 0x6240);
      lo[2 * h] = __byte_perm(l01, l23, 0x5410);
      lo[2 * h + 1] = __byte_perm(l01, l23, 0x7632);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] += 0x00800080u;
      const uint32_t h01 = __byte_perm(x[0], x[1], 0x7351), h23 = __byte_perm(x[2], x[3], 0x7351);
#pragma unroll
      for (int k = 0; k < 2; ++k)  // each byte less 8
        hi[2 * h + k] = ((__byte_perm(h01, h23, k ? 0x7632 : 0x5410) | 0x80808080u) - 0x08080808u) ^
                        0x80808080u;
    }
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
// Most weights, outputs padded to 16, that go this way.  256 requests of 2049-word rows take 137 us on the
// tensor cores with 24->16 (161 at an odd pitch, 62 from 24 bits) and 75 (75, 64) here, with 10->4 136 and
// 31; 64->10 takes 118 there and 166 here.
constexpr long long GF_MOST = 384;

static bool gf_few(int n_in, int n_out) {
  return (long long)n_in * ((n_out + GF_OUT - 1) / GF_OUT * GF_OUT) <= GF_MOST;
}

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
        w_s[k][i % GF_OUT] = GROUP_BIAS + (uint32_t)w;
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
      uint64_t v = acc[u] - GROUP_BIAS * sum;
      if (a.bias && c == a.L - 1) v += (uint64_t)__ldg(a.bias + j0 + u) * a.delta;
      y[(size_t)u * a.ldy] = v;
    }
  }
}

// ---- weights as bytes ---------------------------------------------------------------------------
// Two matrices of signed bytes, w = lo + 256 hi, lo [n_out][pitch], then hi, rows padded by zeros to a
// multiple of 16 bytes.  A thread makes 16 bytes of both.  (Every block expanding for itself what stays in
// its shared memory costs more, as the code runs once and cold: 784 inputs 9 us against 2.)
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
  const int in = (int)(w.transposed ? t / n_out : t % chunks) * 16;
  int8_t* out = to + (size_t)o * pitch + in;
  uint32_t lo[4], hi[4];
  w.bytes(o, in, n_in, lo, hi);
  *reinterpret_cast<uint4*>(out) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  *reinterpret_cast<uint4*>(out + (size_t)n_out * pitch) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
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

constexpr uint32_t GC_WAIT_LIMIT = 1u << 24;

struct GcMaps {
  CUtensorMap W, W_tail, Y;
  CUtensorMap X[2];  // boxes of one slot's and of one MMA's rows; shifted: rows 0, 2, .. and 1, 3, ..
};

struct GcArgs : GcPlan {
  GroupArgs g;
  int off0, off1;    // words by which rows 0, 2, .. / 1, 3, .. start past 16-byte alignment
  int plain_out;     // results leave by plain stores
  int in_place;      // SHORT: the weights are expanded by every block for itself
};

// Every stride-th tile from `first` on.  The next one's slot is on its way while one is worked on.
template <bool CACHED>
struct GcWalk {
  const GcArgs& a;
  int b, nt, m, src, next_b, next_n, next_m, slot = 0;
  int step_m, step_n, step_b;
  int m_tiles;
  // (one_m: tiles of X)
  __device__ __forceinline__ GcWalk(const GcArgs& args, unsigned first, unsigned stride, bool one_m)
      : a(args), m_tiles(one_m ? 1 : args.m_tiles) {
    split(first, next_m, next_n, next_b);
    split(stride, step_m, step_n, step_b);
    if (CACHED && next_b < a.g.batch) slot = __ldg(a.g.slots + next_b);
  }
  __device__ __forceinline__ void split(unsigned t, int& m_of, int& n_of, int& b_of) const {
    const unsigned u = t / (unsigned)m_tiles;
    m_of = (int)(t - u * m_tiles);
    b_of = (int)(u / (unsigned)a.n_tiles);
    n_of = (int)(u - (unsigned)b_of * a.n_tiles);
  }
  // src: the place of the request's ciphertexts, or the number of slots where it has none
  __device__ __forceinline__ bool next() {
    if (next_b >= a.g.batch) return false;
    b = next_b, nt = next_n, m = next_m;
    src = !CACHED ? b : slot >= 0 && slot < a.g.n_slots ? slot : a.g.n_slots;
    next_m += step_m;
    const int carry_m = next_m >= m_tiles;
    next_m -= carry_m ? m_tiles : 0;
    next_n += step_n + carry_m;
    const int carry_n = next_n >= a.n_tiles;
    next_n -= carry_n ? a.n_tiles : 0;
    next_b += step_b + carry_n;
    if (CACHED && next_b < a.g.batch) slot = __ldg(a.g.slots + next_b);
    return true;
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
  } else if constexpr (COLS == 16) {
    tc::tmem_ld_32x32_x16(at, r);
  } else {
    static_assert(COLS == 24, "16 and 8 columns");
    tc::tmem_ld_32x32_x16(at, *reinterpret_cast<uint32_t(*)[16]>(&r[0]));
    tc::tmem_ld_32x32_x8(at + 16, *reinterpret_cast<uint32_t(*)[8]>(&r[16]));
  }
}

// sum_p t[p] << 8p: a word mod 2^64, or the high half of one from a cache, whose low half is zero.  NARROW:
// t[p] + 256 t[p+1] stays below 2^31, so two multiply-adds of 64 bits do for the low four.
template <int BYTES, bool NARROW = false>
__device__ __forceinline__ auto gc_limbs(const uint32_t* t) {
  if constexpr (BYTES == 8 && NARROW) {
    const int t01 = (int)(t[0] + (t[1] << 8)), t23 = (int)(t[2] + (t[3] << 8));
    const uint64_t s = (uint64_t)(t01 + (int64_t)t23 * 65536);
    const uint32_t hi = (uint32_t)(s >> 32) + t[4] + (t[5] << 8) + (t[6] << 16) + (t[7] << 24);
    return (uint64_t)hi << 32 | (uint32_t)s;
  } else if constexpr (BYTES == 8) {
    return add_limbs(0, t);
  } else {
    uint32_t v = t[0];
#pragma unroll
    for (int p = 1; p < BYTES; ++p) v += t[p] << (8 * p);
    return v << (32 - 8 * BYTES);
  }
}
// The word of limb sums by lo and by hi, sum_p (lo[p] + hi[p-1]) << 8p.  Sums of two stay below 2^31 for
// up to 61922 inputs ((128 + 8) * 255 each).
constexpr int GC_NARROW = 240;  // inputs: 257 * (128 + 8) * 255 * 240 < 2^31
template <int BYTES, bool NARROW>
__device__ __forceinline__ auto gc_word(const uint32_t* lo, const uint32_t* hi) {
  uint32_t t[BYTES];
  t[0] = lo[0];
#pragma unroll
  for (int p = 1; p < BYTES; ++p) t[p] = lo[p] + hi[p - 1];
  return gc_limbs<BYTES, NARROW>(t);
}
__device__ __forceinline__ uint64_t gc_whole(uint64_t v) { return v; }
__device__ __forceinline__ uint64_t gc_whole(uint32_t v) { return (uint64_t)v << 32; }
__device__ __forceinline__ uint64_t gc_other_lane(uint64_t v) { return shfl_xor_u64(v, 1); }
__device__ __forceinline__ uint32_t gc_other_lane(uint32_t v) {
  return __shfl_xor_sync(0xffffffffu, v, 1);
}

template <int BYTES, bool SHIFTED, GcMode MODE>
__global__ void __launch_bounds__(GcShape<BYTES, SHIFTED, MODE>::THREADS, 1)
    group_kernel(const __grid_constant__ GcMaps tm, const __grid_constant__ GcArgs a) {
  using S = GcShape<BYTES, SHIFTED, MODE>;
  constexpr bool CACHED = BYTES != 8;
  constexpr bool TWO = MODE == PAIR;
  static_assert(!(TWO && SHIFTED), "the copying warps answer their own block's barriers");
  constexpr int STAGES = S::STAGES;
  extern __shared__ __align__(1024) unsigned char gc_raw[];  // the swizzles want 1024-byte boundaries
  const uint32_t base = tc::smem_u32(gc_raw);
  if (base & 1023u) {
    if (threadIdx.x == 0) atomicExch(&g_gc_status, 1);
    return;
  }
  // slot s of the weights of the m-th tile of outputs that stay, or of the ring
  auto w_at = [&](int m, int s) { return base + (uint32_t)(m * a.w_tile + s * S::W_SLOT); };
  auto x_at = [&](int s) { return base + (uint32_t)(a.x_at + s * GC_X_SLOT); };
  auto raw_at = [&](int s) { return base + (uint32_t)(a.raw_at + s * S::RAW_SLOT); };
  const uint32_t bars = base + (uint32_t)a.bars_at;
  const uint32_t w_full = bars, w_empty = w_full + 8 * GC_MAX_W;
  const uint32_t x_full = w_empty + 8 * GC_MAX_W, x_empty = x_full + 8 * GC_MAX_X;
  const uint32_t r_full = x_empty + 8 * GC_MAX_X, r_empty = r_full + 8 * GC_MAX_RAW;
  const uint32_t acc_full = r_empty + 8 * GC_MAX_RAW, acc_empty = acc_full + 16;
  const uint32_t holder = bars + 8 * GC_BARS;
  volatile int* abort_s = reinterpret_cast<volatile int*>(gc_raw + (holder + 4 - base));
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Of a pair the first block issues the MMAs of both; it is told of both blocks' slots.
  const int rank = TWO ? (int)(blockIdx.x & 1u) : 0;
  unsigned first = TWO ? blockIdx.x >> 1 : blockIdx.x, grid = TWO ? gridDim.x >> 1 : gridDim.x;
  int m_first = 0, m_n = 1;  // SHORT: the block's tiles of outputs
  if (MODE == SHORT) {
    // All tiles of outputs, or one: then a run of neighbouring blocks has the same.  (Dealt out in turn,
    // seven tiles of outputs of 96 x 128->784 take 770 us instead of 430 when a launch writes more than L2
    // holds.)
    auto start = [&](int m) { return (unsigned)((long long)gridDim.x * m / a.m_tiles); };
    if (a.m_group > 1) {
      m_n = a.m_tiles;
    } else {
      while (blockIdx.x >= start(m_first + 1)) ++m_first;
      first = blockIdx.x - start(m_first);
      grid = start(m_first + 1) - start(m_first);
    }
  }
  auto leads = [&](uint32_t bar) { return TWO ? tc::cluster_address(bar, 0) : bar; };
  auto drained = [&](uint32_t bar) {  // the first block's: a warp's loads from tensor memory are done
    if (TWO)
      tc::mbar_arrive_cluster(leads(bar));
    else
      tc::mbar_arrive(bar);
  };
  auto commit = [&](uint32_t bar) {
    if (TWO)
      tc::mma_commit_pair(bar);  // on both blocks'
    else
      tc::mma_commit(bar);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.w_slots; ++s) {
      tc::mbar_init(w_full + 8 * s, MODE == SHORT && a.in_place ? GC_EPI_WARPS : 1);
      tc::mbar_init(w_empty + 8 * s, S::ISSUERS);
    }
    for (int s = 0; s < a.x_slots; ++s) {
      tc::mbar_init(x_full + 8 * s, SHIFTED ? S::COPY : 1);
      tc::mbar_init(x_empty + 8 * s, S::ISSUERS);
    }
    for (int s = 0; s < a.raw_slots; ++s) {
      tc::mbar_init(r_full + 8 * s, 1);
      tc::mbar_init(r_empty + 8 * s, 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(acc_full + 8 * s, S::ISSUERS);
      tc::mbar_init(acc_empty + 8 * s, (1 + TWO) * GC_EPI_WARPS / STAGES);
    }
    *abort_s = 0;
    tc::fence_mbar_init();
    if (!a.in_place) tc::prefetch_tmap(&tm.W);
    tc::prefetch_tmap(&tm.X[0]);
    tc::prefetch_tmap(&tm.X[1]);
    if (!a.plain_out) tc::prefetch_tmap(&tm.Y);
  }
  if (warp == S::MMA_WARP) {
    if (TWO)
      tc::tmem_alloc_pair(holder, 512);
    else
      tc::tmem_alloc(holder, 512);
  }
  tc::tc_fence_before();
  if (TWO)
    tc::cluster_sync();
  else
    __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gc_raw + (holder - base));

  const int kx_n = (a.g.n_in + S::XK - 1) / S::XK;  // X slots of one tile
  const int kb_n = (a.g.n_in + GC_WK - 1) / GC_WK;  // weight slots
  const long long x_tiles =
      ((long long)a.g.batch * a.n_tiles * (MODE == SHORT ? 1 : a.m_tiles) - first + grid - 1) / grid;

  if (warp == 0) {
    // ---------------- X loads (one lane) ---------------------------------------------------------
    // (X was there before the weights' kernel began, so it need not be waited for.)
    // Loads of X fill the memory's queues, so those of weights that are expanded here go first.
    if (MODE == SHORT && a.in_place)
      asm volatile("barrier.cta.sync 1, %0;" ::"n"(32 * GC_EPI_WARPS + 32) : "memory");
    if (lane == 0) {
      TileRing ring;
      bool wrapped = false, ok = true;
      const int slots = SHIFTED ? a.raw_slots : a.x_slots;
      GcWalk<CACHED> walk(a, first, grid, MODE == SHORT);
      while (ok && walk.next()) {
        const int word = walk.nt * S::TILE + rank * S::WORDS;
        for (int k = 0; k < a.g.n_in; k += SHIFTED ? S::RAW_ROWS : S::XK) {
          const int s = ring.slot;
          const uint32_t full = (SHIFTED ? r_full : x_full) + 8 * s;
          ok = gc_wait((SHIFTED ? r_empty : x_empty) + 8 * s, ring.phase ^ 1u, abort_s);
          if (!ok) break;
          if (SHIFTED) {
            const int row = walk.src * a.g.n_in + k;
            tc::mbar_expect_tx(full, S::RAW_SLOT);  // the rows of either parity, in order
            tc::tma_load_2d(raw_at(s), &tm.X[row & 1], word, row >> 1, full);
            tc::tma_load_2d(raw_at(s) + S::RAW_SLOT / 2, &tm.X[(row + 1) & 1], word, (row + 1) >> 1,
                            full);
          } else {
            // The last slot gets whole MMAs' rows only: a load takes its time also for rows past the last
            // input, which read as zeros (as do requests without a place).
            const int rows = min(S::XK, (a.g.n_in - k + GC_KSTEP - 1) / GC_KSTEP * GC_KSTEP);
            const int box = rows == S::XK ? S::XK : GC_KSTEP;
            const CUtensorMap* map = rows == S::XK ? &tm.X[0] : &tm.X[1];
            if (rank == 0) tc::mbar_expect_tx(full, (uint32_t)((1 + TWO) * rows * S::LOAD));
            for (int r = 0; r < rows; r += box)
#pragma unroll
              for (int b = 0; b < S::BOXES; ++b) {
                const uint32_t to = x_at(s) + (uint32_t)((b * S::XK + r) * 128);
                if (TWO)
                  tc::tma_load_3d_pair(to, map, word * BYTES, k + r, walk.src, leads(full));
                else
                  tc::tma_load_3d(to, map, word * BYTES + b * 128, k + r, walk.src, full);
              }
          }
          ring.advance(slots);
          wrapped |= ring.slot == 0;
        }
      }
      if (rank == 0) tile_drain(SHIFTED ? r_full : x_full, ring, wrapped, slots, GC_WAIT_LIMIT);
    }
  } else if (warp == 1) {
    // ---------------- weight loads (one lane) ----------------------------------------------------
    if (lane == 0 && !a.in_place) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the weights' kernel is done
      if (MODE == LONG) {
        TileRing ring;
        bool wrapped = false, ok = true;
        GcWalk<false> walk(a, first, grid, false);
        while (ok && walk.next()) {
          for (int k = 0; k < kb_n; ++k) {
            const int s = ring.slot;
            ok = gc_wait(w_empty + 8 * s, ring.phase ^ 1u, abort_s);
            if (!ok) break;
            tc::mbar_expect_tx(w_full + 8 * s, S::W_SLOT);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              tc::tma_load_3d(w_at(0, s) + h * GC_W_HALF, &tm.W, k * GC_WK, walk.m * GC_BM, h,
                              w_full + 8 * s);
            ring.advance(a.w_slots);
            wrapped |= ring.slot == 0;
          }
        }
        tile_drain(w_full, ring, wrapped, a.w_slots, GC_WAIT_LIMIT);
      } else {
        const int m0 = TWO ? (int)(first % (unsigned)a.m_tiles) : m_first;
        for (int m = 0; m < m_n; ++m)
          for (int k = 0; k < kb_n; ++k) {
            const int s = m * kb_n + k, row = (m0 + m) * GC_BM;
            const bool tail = MODE == SHORT && a.w_tail && k + 1 == kb_n;
            if (rank == 0)
              tc::mbar_expect_tx(w_full + 8 * s, (uint32_t)((1 + TWO) * (tail ? S::W_TAIL : S::W_SLOT)));
            if (TWO)  // rows of lo and of hi in turn
              tc::tma_load_3d_pair(w_at(m, k), &tm.W, k * GC_WK, 0, row + rank * 64, leads(w_full + 8 * s));
            else
#pragma unroll
              for (int h = 0; h < 2; ++h)
                tc::tma_load_3d(w_at(m, k) + h * (tail ? S::W_TAIL / 2 : GC_W_HALF),
                                tail ? &tm.W_tail : &tm.W, k * GC_WK, row, h, w_full + 8 * s);
          }
        if (rank == 0)
          for (int s = 0; s < m_n * kb_n; ++s) (void)tc::mbar_wait(w_full + 8 * s, 0, GC_WAIT_LIMIT);
      }
    }
  } else if (SHIFTED && warp < S::MMA_WARP) {
    // ---------------- raw rows -> operand layout (shifted rows only) -----------------------------
    // Raw slot r is copied by warp r % 4 (their number is a multiple of 4).  Every warp waits for every
    // X slot's turn and answers it, also where it copies nothing: a parity tells only neighbouring
    // turns apart.
    const int cw = warp - 2;
    constexpr int PER = SHIFTED ? 32 / S::WORDS : 1;  // rows per pass of a warp
    constexpr int BATCH = 16;                         // passes whose words are on their way together
    const int word = lane % S::WORDS, sub = lane / S::WORDS;
    const int box = word >> 4, ch = (word & 15) >> 1, half = word & 1;
    TileRing xr, rr;
    bool ok = true;
    GcWalk<CACHED> walk(a, first, grid, MODE == SHORT);
    while (ok && walk.next()) {
      const int parity = walk.src * a.g.n_in & 1;  // of the tile's first row
      const int off_e = parity ? a.off1 : a.off0, off_o = parity ? a.off0 : a.off1;
      for (int kx = 0; ok && kx < kx_n; ++kx) {
        ok = gc_wait(x_empty + 8 * xr.slot, xr.phase ^ 1u, abort_s);
        if (!ok) break;
        const int raws =
            min(S::XK, a.g.n_in - kx * S::XK + S::RAW_ROWS - 1) / S::RAW_ROWS;
        for (int i = 0; i < raws; ++i) {
          if ((rr.slot & 3) == cw) {
            ok = gc_wait(r_full + 8 * rr.slot, rr.phase, abort_s);
            if (!ok) break;
            // row r of the slot: its parity's half, r / 2; one word further where it is shifted
            const unsigned char* from = gc_raw + (raw_at(rr.slot) - base) + word * 8;
            unsigned char* to = gc_raw + (x_at(xr.slot) - base) + box * (S::XK * 128) +
                                i * (S::RAW_ROWS * 128) + half * 8;
#pragma unroll
            for (int b = 0; b < S::RAW_ROWS / PER; b += BATCH) {
              uint64_t v[BATCH];
#pragma unroll
              for (int j = 0; j < BATCH; ++j) {
                const int r = (b + j) * PER + sub;
                v[j] = *reinterpret_cast<const uint64_t*>(
                    from + (r & 1 ? S::RAW_SLOT / 2 + off_o * 8 : off_e * 8) +
                    (r >> 1) * S::RAW_PITCH);
              }
#pragma unroll
              for (int j = 0; j < BATCH; ++j) {
                const int r = (b + j) * PER + sub;
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
  } else if (warp < S::EPI_WARP) {
    // ---------------- products: one warp by lo, another by hi, or of a pair one for both -----------
    // The whole warp goes through the loop and one lane issues: what every lane knows stays in uniform
    // registers, which the MMAs take their operands from.
    if (rank == 0) {
      constexpr uint32_t IDESC = tc::idesc_i8(TWO ? 256 : 128, (1 + TWO) * S::BN, true, false, false, true);
      constexpr int STEPS = S::XK / GC_KSTEP, PER_W = GC_WK / S::XK;
      const bool one = tc::elect_one();
      const int hi = warp - S::MMA_WARP;
      const uint64_t wd = tc::smem_desc_sw128(w_at(0, 0) + hi * GC_W_HALF, 16u, 1024u);
      const uint64_t td = tc::smem_desc_sw32(w_at(0, kb_n - 1) + hi * (S::W_TAIL / 2), 16u, 256u);
      const uint64_t xd = tc::smem_desc_sw128(x_at(0), S::XK * 128u, 1024u);
      const uint32_t w_hi = (uint32_t)(wd >> 32), x_hi = (uint32_t)(xd >> 32);
      const int tail = MODE == SHORT ? a.w_tail : 0;
      const int steps = (a.g.n_in + GC_KSTEP - 1) / GC_KSTEP;
      TileRing x, w;
      bool ok = true;
      int buf = 0;
      uint32_t turn = 0;
      for (long long t = 0; ok && t < x_tiles; ++t) {
        const TileRing x0 = x;
        for (int m = 0; ok && m < m_n; ++m) {  // tiles of outputs that take turns at these X slots
          const uint32_t d = tmem + (uint32_t)(buf * 256 + hi * S::HI_AT);
          ok = gc_wait(acc_empty + 8 * buf, turn ^ 1u, abort_s);
          if (!ok) break;
          tc::tc_fence_after();
          uint32_t acc = 0;
          x = x0;
          if (MODE != LONG) w.slot = 0;
          const uint32_t w_m = (uint32_t)(m * (a.w_tile / 16));
          for (int left = steps - tail; ok && left > 0;) {  // one weight slot
            if (MODE == LONG || t == 0) {
              ok = gc_wait(w_full + 8 * (MODE == SHORT ? m * kb_n + w.slot : w.slot), w.phase, abort_s);
              if (!ok) break;
            }
            const uint32_t w_lo = (uint32_t)wd + w_m + (uint32_t)(w.slot * (S::W_SLOT / 16));
#pragma unroll
            for (int h = 0; h < PER_W; ++h) {
              if (left <= 0) break;
              if (m == 0) ok = gc_wait(x_full + 8 * x.slot, x.phase, abort_s);
              if (!ok) break;
              const uint32_t x_lo = (uint32_t)xd + (uint32_t)(x.slot * (GC_X_SLOT / 16));
              if (one) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k)
                  if (k < left) {
                    if (TWO)
                      tc::mma_i8_lo_pair(d, w_lo + 2 * (h * STEPS + k), w_hi, x_lo + 256 * k, x_hi,
                                         IDESC, k ? 1u : acc);
                    else
                      tc::mma_i8_lo(d, w_lo + 2 * (h * STEPS + k), w_hi, x_lo + 256 * k, x_hi, IDESC,
                                    k ? 1u : acc);
                  }
                if (m + 1 == m_n) commit(x_empty + 8 * x.slot);
              }
              acc = 1;
              left -= STEPS;
              x.advance(a.x_slots);
            }
            if (MODE == LONG) {
              if (one) commit(w_empty + 8 * w.slot);
              w.advance(a.w_slots);
            } else {
              ++w.slot;
            }
          }
          if (MODE == SHORT && tail && ok) {  // the last slot, of one MMA
            if (t == 0) ok = gc_wait(w_full + 8 * (m * kb_n + kb_n - 1), 0, abort_s);
            if (ok && m == 0) ok = gc_wait(x_full + 8 * x.slot, x.phase, abort_s);
            if (ok && one) {
              tc::mma_i8_lo(d, (uint32_t)td + w_m, (uint32_t)(td >> 32),
                            (uint32_t)xd + (uint32_t)(x.slot * (GC_X_SLOT / 16)), x_hi, IDESC, acc);
              if (m + 1 == m_n) commit(x_empty + 8 * x.slot);
            }
            x.advance(a.x_slots);
          }
          if (!ok) break;
          if (one) commit(acc_full + 8 * buf);
          if (++buf == STAGES) {
            buf = 0;
            turn ^= 1u;
          }
        }
      }
    }
  } else {
    // ---------------- weights that stay, then the epilogue ---------------------------------------
    const int e_w = warp - S::EPI_WARP;
    if (MODE == SHORT && a.in_place) {
      // 16 bytes of lo and of hi per thread and turn, of one output and 16 inputs, into the K-major operand
      // layout
      const int chunks = a.w_tail ? GC_KSTEP / 16 : GC_WK / 16;
#pragma unroll 1
      for (int i = (int)threadIdx.x - 32 * S::EPI_WARP; i < GC_BM * chunks; i += 32 * GC_EPI_WARPS) {
        const int o = i % GC_BM, c = i / GC_BM;
        uint32_t lo[4] = {}, hi[4] = {};
        if (o < a.g.n_out && 16 * c < a.g.n_in) a.g.w.bytes(o, 16 * c, a.g.n_in, lo, hi);
        unsigned char* to =
            gc_raw + (a.w_tail ? o * 32 + ((c ^ (o >> 2 & 1)) << 4) : o * 128 + ((c ^ (o & 7)) << 4));
        *reinterpret_cast<uint4*>(to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        *reinterpret_cast<uint4*>(to + (a.w_tail ? S::W_TAIL / 2 : GC_W_HALF)) =
            make_uint4(hi[0], hi[1], hi[2], hi[3]);
      }
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(w_full);
      asm volatile("barrier.cta.arrive 1, %0;" ::"n"(32 * GC_EPI_WARPS + 32) : "memory");
    }
    // Warp w reads TMEM lane quarter w % 4.  With two accumulators each group of eight warps has one of
    // them, and a warp half of its words; with one, a warp has a quarter.  A lane holds the sums of one
    // output, or of a pair an even lane those by lo and the odd lane beside it those by hi: of every two
    // words each then completes one, with the other's share of it.  Words are staged in shared memory
    // with the 16-byte chunks XORed by the row, and leave by TMA, or as row segments by plain stores.
    const int q = warp & 3, group = e_w >> 3, share = STAGES == 1 ? e_w >> 2 : (e_w >> 2) & 1;
    const uint32_t out_at = base + (uint32_t)(a.out_at + e_w * S::STAGE);
    unsigned char* out = gc_raw + (out_at - base);
    constexpr int PITCH = S::PART * 8;
    auto xored = [](int r) { return (r >> 1) & 3; };
    const int row = TWO ? lane >> 1 : lane, odd = TWO ? lane & 1 : 0;
    // chunk k of this lane's row, as XORed
    auto chunk = [&](int k) { return out + ((row * PITCH | xored(row) << 4) ^ (k << 4)); };
    const int buf = STAGES == 1 ? 0 : group;
    uint32_t turn = 0;
    // A group's tiles: every second one, or where several tiles of outputs take turns at one of X
    // every second turn.
    const bool turns = MODE == SHORT && m_n > 1, apart = STAGES == 2 && !turns;
    GcWalk<CACHED> walk(a, apart ? first + group * grid : first, apart ? 2 * grid : grid, MODE == SHORT);
    int m = turns ? group : 0;
    for (bool more = walk.next(); more; ++turn) {
      const int row0 = (MODE == SHORT ? m_first + m : walk.m) * GC_BM + rank * 64 + q * S::ROWS;
      const int col0 = walk.nt * S::TILE + share * S::EW;
      const int body = a.g.L - 1 - col0;  // the body among this warp's words
      const int b = walk.b, src = walk.src;
      // the next one
      if (turns && (m += 2) < m_n) {
        more = true;
      } else {
        m = turns ? m - m_n : 0;
        more = walk.next();
      }
      if (!gc_wait(acc_full + 8 * buf, turn, abort_s)) break;
      tc::tc_fence_after();
      const uint32_t c_tmem = tmem + (uint32_t)(buf * 256 + share * S::EW * BYTES) +
                              ((uint32_t)(q * 32) << 16);
      // nothing of this warp's share is kept
      if (row0 >= a.g.n_out || body < 0 || (CACHED && src == a.g.n_slots)) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) drained(acc_empty + 8 * buf);
        continue;
      }
      constexpr int FETCH = TWO ? 2 * S::CW : S::CW;  // words of one turn
#pragma unroll
      for (int i = 0; i < S::EW / FETCH; ++i) {
        // lo's sums and hi's, or of a pair the sums of two runs of words
        uint32_t c0[S::COLS], c1[S::COLS];
        gc_tmem_ld<S::COLS>(c_tmem + (uint32_t)(i * FETCH * BYTES), c0);
        gc_tmem_ld<S::COLS>(
            c_tmem + (uint32_t)(TWO ? i * FETCH * BYTES + S::COLS : S::HI_AT + i * S::COLS), c1);
        tc::tmem_ld_wait_pin(c0);
        tc::tmem_ld_wait_pin(c1);
        if (i + 1 == S::EW / FETCH) {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) drained(acc_empty + 8 * buf);
        }
        constexpr int N = FETCH < S::PART ? FETCH : S::PART;
#pragma unroll
        for (int u0 = 0; u0 < FETCH; u0 += N) {
          const int first_w = i * FETCH + u0;               // of this warp's words
          const int part = first_w / S::PART * S::PART;     // the first word staged with it
          uint64_t y[N];                                    // of a pair every other one: this lane's
          if constexpr (TWO) {
#pragma unroll
            for (int u = 0; u < N; u += 2) {
              auto at = [&](int w) { return w < S::CW ? c0 + w * BYTES : c1 + (w - S::CW) * BYTES; };
              const auto v0 = gc_limbs<BYTES>(at(u0 + u)) << (8 * odd);
              const auto v1 = gc_limbs<BYTES>(at(u0 + u + 1)) << (8 * odd);
              y[u] = gc_whole((odd ? v1 : v0) + gc_other_lane(odd ? v0 : v1));
            }
          } else if (BYTES == 8 && MODE == SHORT && a.g.n_in <= GC_NARROW) {
#pragma unroll
            for (int u = 0; u < N; ++u)
              y[u] = gc_whole(gc_word<BYTES, true>(c0 + (u0 + u) * BYTES, c1 + (u0 + u) * BYTES));
          } else {
#pragma unroll
            for (int u = 0; u < N; ++u)
              y[u] = gc_whole(gc_word<BYTES, false>(c0 + (u0 + u) * BYTES, c1 + (u0 + u) * BYTES));
          }
          if (first_w == part && !a.plain_out) {  // what was staged before has left
            if (lane == 0) tc::tma_store_wait_read();
            __syncwarp();
          }
#pragma unroll
          for (int u = 0; u < N; u += 2) {
            unsigned char* to = chunk((first_w - part + u) >> 1);
            if constexpr (TWO)
              *reinterpret_cast<uint64_t*>(to + 8 * odd) = y[u];
            else
              *reinterpret_cast<ulonglong2*>(to) = make_ulonglong2(y[u], y[u + 1]);
          }
          if (first_w + N != part + S::PART) continue;
          if (body >= part && body < part + S::PART && (!TWO || ((body - part) & 1) == odd) &&
              row0 + row < a.g.n_out) {
            uint64_t* p = reinterpret_cast<uint64_t*>(chunk((body - part) >> 1) + ((body - part) & 1) * 8);
            if (a.g.bias) *p += (uint64_t)__ldg(a.g.bias + row0 + row) * a.g.delta;
            // tiled stores end on 16-byte boundaries, so the last word of an odd count goes alone
            if (!a.plain_out && (a.g.L & 1))
              a.g.Y[((size_t)b * a.g.n_out + row0 + row) * a.g.ldy + a.g.L - 1] = *p;
          }
          if (!a.plain_out) {
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0 && col0 + part < (a.g.L & ~1))
              tc::tma_store_3d(&tm.Y, col0 + part, row0, b, out_at);
          } else {
            __syncwarp();
            constexpr int PER = 32 / S::PART;  // rows per instruction
            const int wd = lane % S::PART, sub = lane / S::PART;
            uint64_t* to =
                a.g.Y + ((size_t)b * a.g.n_out + row0 + sub) * a.g.ldy + col0 + part + wd;
            const int left = col0 + part + wd < a.g.L ? a.g.n_out - row0 - sub : 0;
            constexpr int TIMES = S::ROWS / PER;
            uint64_t v[TIMES];
#pragma unroll
            for (int j = 0; j < TIMES; ++j) {
              const int r = PER * j + sub;
              v[j] = *reinterpret_cast<const uint64_t*>(
                  out + r * PITCH + (((wd >> 1) ^ xored(r)) << 4) + (wd & 1) * 8);
            }
#pragma unroll
            for (int j = 0; j < TIMES; ++j)
              if (PER * j < left) to[(size_t)(PER * j) * a.g.ldy] = v[j];
            __syncwarp();
          }
        }
      }
    }
    if (!a.plain_out && lane == 0) tc::tma_store_wait();
  }
  tc::tc_fence_before();
  if (TWO)
    tc::cluster_sync();  // the other block's MMAs read this one's memory, and it arrives on its barriers
  else
    __syncthreads();
  if (warp == S::MMA_WARP) {
    tc::tc_fence_after();
    if (TWO)
      tc::tmem_dealloc_pair(tmem, 512);
    else
      tc::tmem_dealloc(tmem, 512);
  }
}

// ---- launch -------------------------------------------------------------------------------------
// Multiprocessors of the current device.
static int gc_sms(int* sms) {
  static std::atomic<int> count[64];
  int dev = 0;
  PNB_CUDA(cudaGetDevice(&dev));
  *sms = dev < 64 ? count[dev].load(std::memory_order_relaxed) : 0;
  if (*sms) return PNB_OK;
  PNB_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  if (dev < 64) count[dev].store(*sms, std::memory_order_relaxed);
  return PNB_OK;
}

template <int BYTES, bool SHIFTED, GcMode MODE>
static int gc_launch(GcArgs& a, int sms, int8_t* ws, cudaStream_t st) {
  using S = GcShape<BYTES, SHIFTED, MODE>;
  const GroupArgs& g = a.g;
  const char* name = g.slots ? "group_contract_cached" : "group_contract";
  static std::atomic<bool> raised[64];  // per device: the kernel's shared-memory limit
  auto kernel = group_kernel<BYTES, SHIFTED, MODE>;
  int dev = 0;
  PNB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !raised[dev].load(std::memory_order_acquire)) {
    PNB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GC_SMEM));
    if (dev < 64) raised[dev].store(true, std::memory_order_release);
  }
  const unsigned grid = gc_plan<BYTES, SHIFTED, MODE>(a, g.n_in, g.n_out, g.L, g.batch, sms);
  GcMaps tm{};
  int rc = PNB_OK;
  if (!SHIFTED) {
    const cuuint64_t dims[3] = {(cuuint64_t)g.L * BYTES, (cuuint64_t)g.n_in,
                                (cuuint64_t)(g.slots ? g.n_slots : g.batch)};
    const cuuint64_t strides[2] = {g.x_row, g.x_row * g.n_in};
    for (int i = 0; i < 2 && !rc; ++i) {
      const cuuint32_t box[3] = {128, (cuuint32_t)(i ? GC_KSTEP : S::XK), 1};
      rc = tile_map(&tm.X[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, g.X, 3, dims, strides, box,
                    CU_TENSOR_MAP_SWIZZLE_128B);
    }
  } else {
    // rows p, p + 2, ..: from the 16-byte boundary at or before row p, at twice the pitch.  A row
    // off by one word has that word's 16 bytes inside its allocation (allocations start aligned).
    const long long x_rows = (long long)g.batch * g.n_in;
    if (x_rows > 0x7fffffffLL - GC_WK) {  // coordinates are 32-bit
      set_error("%s: %lld ciphertexts exceed a 32-bit index", name, x_rows);
      return PNB_ERR_INVALID;
    }
    for (int p = 0; p < 2 && !rc; ++p) {
      // (a single row has no row 1: both maps are its own, and the second meets zero weights)
      const bool second = p && x_rows > 1;
      const int off = second ? a.off1 : a.off0;
      const cuuint64_t dims[2] = {(cuuint64_t)g.L + off,
                                  (cuuint64_t)std::max<long long>(1, (x_rows + 1 - p) / 2)};
      const cuuint64_t strides[1] = {g.x_row * 2};
      const cuuint32_t box[2] = {S::RAW_PITCH / 8, S::RAW_ROWS / 2};
      rc = tile_map(&tm.X[p], CU_TENSOR_MAP_DATA_TYPE_UINT64, g.X + (second ? g.x_row : 0) - 8 * off,
                    2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
  }
  if (!rc && !a.plain_out) {
    // writes end at word L (rounded down to 16 bytes) of the last output of each request
    const cuuint64_t dims[3] = {(cuuint64_t)std::max(2, g.L & ~1), (cuuint64_t)g.n_out,
                                (cuuint64_t)g.batch};
    const cuuint64_t strides[2] = {(cuuint64_t)g.ldy * 8, (cuuint64_t)g.ldy * 8 * g.n_out};
    const cuuint32_t box[3] = {S::PART, S::ROWS, 1};
    rc = tile_map(&tm.Y, CU_TENSOR_MAP_DATA_TYPE_UINT64, g.Y, 3, dims, strides, box,
                  tile_swizzle(8 * S::PART));
  }
  if (rc) return rc;
  cudaLaunchAttribute attrs[2]{};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = (size_t)(a.bars_at + GC_BAR_BYTES);
  cfg.stream = st;
  cfg.attrs = attrs;
  cfg.numAttrs = 0;
  if (MODE == PAIR) {
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim = {2, 1, 1};
    cfg.numAttrs = 1;
  }
  if (!a.in_place) {
    const int pitch = (g.n_in + 15) & ~15;
    const long long blocks = ((long long)g.n_out * (pitch / 16) + GX_THREADS - 1) / GX_THREADS;
    if (blocks > 0x7fffffffLL) {
      set_error("%s: %d x %d weights exceed one launch", name, g.n_out, g.n_in);
      return PNB_ERR_INVALID;
    }
    const cuuint64_t all = (cuuint64_t)pitch * g.n_out;
    cuuint64_t dims[3] = {(cuuint64_t)pitch, (cuuint64_t)g.n_out, 2};
    cuuint64_t strides[2] = {(cuuint64_t)pitch, all};
    cuuint32_t box[3] = {GC_WK, GC_BM, 1};
    if (MODE == PAIR) {
      std::swap(dims[1], dims[2]);
      std::swap(strides[0], strides[1]);
      box[1] = 2;
      box[2] = GC_BM / 2;
    }
    rc = tile_map(&tm.W, CU_TENSOR_MAP_DATA_TYPE_UINT8, ws, 3, dims, strides, box,
                  CU_TENSOR_MAP_SWIZZLE_128B);
    box[0] = GC_KSTEP;
    if (!rc && a.w_tail)
      rc = tile_map(&tm.W_tail, CU_TENSOR_MAP_DATA_TYPE_UINT8, ws, 3, dims, strides, box,
                    CU_TENSOR_MAP_SWIZZLE_32B);
    if (rc) return rc;
    group_expand_kernel<<<(unsigned)blocks, GX_THREADS, 0, st>>>(g.w, g.n_in, g.n_out, pitch, ws);
    PNB_CHECK_LAUNCH("group_expand_kernel");
    // this kernel's set-up and its first loads of X run beside that one
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  PNB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tm, a));
  return PNB_OK;
}

template <int BYTES, bool SHIFTED>
static int gc_run(GcArgs& a, int8_t* ws, cudaStream_t st) {
  int sms = 0;
  const int rc = gc_sms(&sms);
  if (rc) return rc;
  switch (gc_mode(a.g.n_in, a.g.n_out, SHIFTED, sms)) {
    case LONG: return gc_launch<BYTES, SHIFTED, LONG>(a, sms, ws, st);
    case SHORT: return gc_launch<BYTES, SHIFTED, SHORT>(a, sms, ws, st);
    default: return gc_launch<BYTES, SHIFTED, SHIFTED ? LONG : PAIR>(a, sms, ws, st);
  }
}

static int gc_run(const GroupArgs& g, int bits, int8_t* ws, cudaStream_t st) {
  GcArgs a{};
  a.g = g;
  a.in_place = gc_in_place(g.n_in, g.n_out);
  a.plain_out = g.ldy % 2 != 0 || ((uintptr_t)g.Y % 16) != 0;
  if (bits == 64) {
    a.off0 = (int)((uintptr_t)g.X / 8 & 1);
    a.off1 = (int)(((uintptr_t)g.X + g.x_row) / 8 & 1);
    return a.off0 || a.off1 ? gc_run<8, true>(a, ws, st) : gc_run<8, false>(a, ws, st);
  }
  return bits == 32 ? gc_run<4, false>(a, ws, st)
         : bits == 24 ? gc_run<3, false>(a, ws, st)
                      : gc_run<2, false>(a, ws, st);
}

size_t group_workspace_bytes(int n_in, int n_out) {
  if (gf_few(n_in, n_out) || gc_in_place(n_in, n_out)) return 0;
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
  if (need && ws && (ws_bytes < need || ((uintptr_t)ws % 16) != 0)) {
    set_error("%s: workspace of %zu bytes at %p, %zu bytes 16-byte aligned are needed",
              a.slots ? "group_contract_cached" : "group_contract", ws_bytes, ws, need);
    return PNB_ERR_INVALID;
  }
  if (gf_few(a.n_in, a.n_out)) return few_run(a, bits, st);
  int8_t* own = nullptr;
  if (need && !ws) PNB_CUDA(cudaMallocAsync((void**)&own, need, st));
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

// request.cu -- contractions whose cleartext weights differ from request to request.
//
//   expert:   Y[r][j] = sum_i W[e][j][i] X[src(r)][i] + bias[e][j] * delta on the body, e the
//             expert of row r, src(r) its token (or r itself for rows already sorted)
//   adapter:  Y[b][j] = 2^s sum_i W[j][i] X[b][i] + sum_q B[a][j][q] (sum_i A[a][q][i] X[b][i])
//             + bias[j] * delta on the body, a the adapter of request b (none outside its range)
//
// mod 2^64 over LWE ciphertexts, int8 weights.  Ciphertext x cleartext sums need no key, so the
// requests of one call may be encrypted under different clients' keys.  The reference has one W
// per Linear node (runtime/src/ops/linear.rs:52-75).
//
// One kernel for both, on the tensor cores.  A u64 word is 8 little-endian byte limbs, so the K
// ciphertexts of a row are a u8 matrix [K][8 ld], N-contiguous: kind::i8 reads it as an MN-major
// operand and the epilogue puts the limb sums together,
//     y = sum_b C[.][8c + b] << 8b  (mod 2^64),  |C| <= 128 * 255 * K < 2^31 for K < 65794.
// A tile is 128 output rows x 32 words (256 limb columns) of one ciphertext row; persistent
// blocks walk them.  Weights are picked per tile by the TMA coordinate, so rows of different
// experts share a launch; rows sorted by expert keep the weights of neighbouring tiles in L2.
//
// Adapters: the low-rank pair rides on the same pass over X.  While the K loop accumulates
// C = W X it also accumulates the transposed low product  L^T = X^T A^T  (the X tile as the M = 128
// operand, twice, and A's rows as N: rank/256 of the main product's work, where A as a padded
// M = 128 operand would double it).  The epilogue warps add up the limbs of t = A X mod 2^64
// across lanes, write t's bytes to shared memory as the next MN-major operand, and one short MMA
// makes D = B t.  y = (C << s) + D.  X is read once; t never leaves the SM.
//
// Rows that start 16-byte aligned (an even pitch) move by TMA straight into the operand layout, and
// results leave by TMA.  Other rows (contiguous [count][kN+1] ciphertexts) are off by one word
// every other row, which no tiled load can shift: they land unshifted in a ring of raw slots, and
// four warps copy them word by word into the operand layout.
#include <algorithm>

#include <cudaTypedefs.h>

#include "pnb_internal.cuh"
#include "pnb_keys.h"
#include "tc_primitives.cuh"

namespace pnb {

// Status word of the kernel: non-zero when one of its bounded waits ran out.
__device__ int g_rq_status;

int rq_status_read_and_clear(int* out) {
  int v = 0;
  PNB_CUDA(cudaMemcpyFromSymbol(&v, g_rq_status, sizeof(int)));
  const int zero = 0;
  PNB_CUDA(cudaMemcpyToSymbol(g_rq_status, &zero, sizeof(int)));
  *out = v;
  return PNB_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder();

constexpr int RQ_BM = 128;      // output rows per tile
constexpr int RQ_WORDS = 32;    // output words per tile
constexpr int RQ_BN = 8 * RQ_WORDS;
constexpr int RQ_BK = 128;      // K per stage
constexpr int RQ_KSTEP = 32;    // K per MMA; a ragged K costs at most 31 rows
constexpr int RQ_W_BYTES = RQ_BM * RQ_BK;              // 16 KB
constexpr int RQ_X_BYTES = RQ_BK * RQ_BN;              // 32 KB
constexpr int RQ_A_BYTES = PNB_MAX_RANK * RQ_BK;       // 8 KB
constexpr int RQ_T_BYTES = PNB_MAX_RANK * RQ_BN;       // 16 KB: t as bytes
constexpr int RQ_B_BYTES = RQ_BM * PNB_MAX_RANK;       // 8 KB: B rows of 64 bytes
constexpr int RQ_EPI_WARPS = 8;                        // two per TMEM lane quarter
constexpr int RQ_COPY_WARPS = 4;
constexpr int RQ_RAW_ROWS = 32;                        // rows per raw slot, half of each parity
constexpr int RQ_RAW_PITCH = 8 * (RQ_WORDS + 2);       // one word of shift, to 16 bytes
constexpr int RQ_RAW_BYTES = RQ_RAW_ROWS * RQ_RAW_PITCH;
constexpr uint32_t RQ_WAIT_LIMIT = 1u << 24;

template <bool SHIFTED, bool ADAPT>
struct RqShape {
  static constexpr int STAGE = RQ_W_BYTES + RQ_X_BYTES + (ADAPT ? RQ_A_BYTES : 0);
  // shifted rows wait in the raw ring, so two operand stages do
  static constexpr int STAGES = SHIFTED ? 2 : ADAPT ? 3 : 4;
  static constexpr int RAW = SHIFTED ? (ADAPT ? 8 : 12) : 0;  // raw slots
  static constexpr int COPY = SHIFTED ? RQ_COPY_WARPS : 0;
  static constexpr int MMA_WARP = 1 + COPY;  // warp 0 issues the loads
  static constexpr int THREADS = 32 * (2 + COPY + RQ_EPI_WARPS);
  // output staging of one epilogue warp: 32 rows x 16 words leaving by TMA, or x 8 by plain stores
  static constexpr int OUT = SHIFTED ? 32 * 64 : 32 * 128;
  static constexpr int RAW_AT = STAGES * STAGE;
  static constexpr int T_AT = RAW_AT + RAW * RQ_RAW_BYTES;
  static constexpr int B_AT = T_AT + (ADAPT ? RQ_T_BYTES : 0);
  static constexpr int OUT_AT = B_AT + (ADAPT ? RQ_B_BYTES : 0);
  static constexpr int BARS_AT = OUT_AT + RQ_EPI_WARPS * OUT;
  static constexpr int SMEM = 1024 + BARS_AT + 512;
  static_assert(SMEM <= 227 * 1024, "shared memory of one block");
  static_assert(8 * (2 * STAGES + 8 + 2 * RAW) + 16 <= 512, "barriers");
  static_assert(T_AT % 1024 == 0 && B_AT % 1024 == 0 && OUT_AT % 1024 == 0, "swizzle atoms");
};

struct RqMaps {
  CUtensorMap W, A, B, Y;
  CUtensorMap X[2];  // aligned: boxes of 128 and of 32 rows; shifted: rows 0, 2, .. and 1, 3, ..
};

struct RqArgs {
  const uint64_t* X;
  uint64_t* Y;
  const int64_t* bias;
  const int32_t* row_choice;  // null: row n reads X row group n
  const int32_t* which;       // expert or adapter of each row
  uint64_t delta;
  int rows, top_k, choices, n_which;
  int M, K, L, ldx, ldy;
  int shift, rank, rank16;    // adapters
  int off0, off1;             // words by which rows 0, 2, .. / 1, 3, .. start past 16-byte alignment
  int n_tiles, k_blocks, w_rows;
  int per_row;                // tiles of one row
  int step_n, step_r;         // the grid as whole rows and tiles
};

// A block's tiles (row n, 128 output rows, 32 words; words fastest), one grid apart.  What a row's
// tables hold is fetched one tile ahead of its use.
template <bool ADAPT>
struct RqWalk {
  int n, r, which, choice;
  __device__ __forceinline__ void fetch(const RqArgs& a) {
    which = choice = -1;
    if (n < a.rows) {
      which = __ldg(a.which + n);
      if (!ADAPT) choice = __ldg(a.row_choice + n);
    }
  }
  __device__ __forceinline__ void start(const RqArgs& a) {
    n = (int)blockIdx.x / a.per_row;
    r = (int)blockIdx.x - n * a.per_row;
    fetch(a);
  }
  __device__ __forceinline__ RqWalk next(const RqArgs& a) const {
    RqWalk o;
    o.n = n + a.step_n;
    o.r = r + a.step_r;
    if (o.r >= a.per_row) {
      o.r -= a.per_row;
      ++o.n;
    }
    o.fetch(a);
    return o;
  }
  __device__ __forceinline__ int mt(const RqArgs& a) const { return r / a.n_tiles; }
  // the row's expert or adapter, -1 when it has none
  __device__ __forceinline__ int weights(const RqArgs& a) const {
    return which >= 0 && which < a.n_which ? which : -1;
  }
  // the row's X group, -1 when the row is skipped
  __device__ __forceinline__ int source(const RqArgs& a) const {
    if (ADAPT) return n;
    if (weights(a) < 0 || choice < 0 || choice >= a.choices) return -1;
    return a.top_k > 0 ? choice / a.top_k : n;
  }
};

// Bounded wait that also gives up as soon as another role has flagged an abort.
__device__ __forceinline__ bool rq_wait(uint32_t bar, uint32_t parity, volatile int* abort_s) {
  for (uint32_t it = 0; it < RQ_WAIT_LIMIT; it += 1024) {
    if (tc::mbar_wait(bar, parity, 1024)) return true;
    if (*abort_s) return false;
  }
  *abort_s = 1;
  atomicExch(&g_rq_status, 1);
  return false;
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int m) {
  return (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)v, m);
}

// v + sum_b c[b] << 8b mod 2^64: the low four limb sums reach into the high word (one multiply-add
// of 32 x 32 + 64 bits each), the high four only live there.
__device__ __forceinline__ uint64_t add_limbs(uint64_t v, const uint32_t* c) {
  int64_t s = (int64_t)v;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    asm("mad.wide.s32 %0, %1, %2, %0;" : "+l"(s) : "r"((int)c[b]), "r"(1 << (8 * b)));
  uint32_t hi = (uint32_t)((uint64_t)s >> 32);
#pragma unroll
  for (int b = 0; b < 4; ++b) hi += c[4 + b] << (8 * b);
  return ((uint64_t)hi << 32) | (uint32_t)s;
}

template <bool SHIFTED, bool ADAPT>
__global__ void __launch_bounds__(RqShape<SHIFTED, ADAPT>::THREADS, 1)
    request_kernel(const __grid_constant__ RqMaps tm, RqArgs a) {
  using S = RqShape<SHIFTED, ADAPT>;
  constexpr int STAGES = S::STAGES, RAW = S::RAW;
  extern __shared__ unsigned char rq_raw[];
  const uint32_t raw = tc::smem_u32(rq_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  auto w_at = [&](int s) { return base + (uint32_t)(s * S::STAGE); };
  auto x_at = [&](int s) { return w_at(s) + RQ_W_BYTES; };
  auto a_at = [&](int s) { return x_at(s) + RQ_X_BYTES; };
  auto raw_at = [&](int r) { return base + (uint32_t)(S::RAW_AT + r * RQ_RAW_BYTES); };
  const uint32_t t_at = base + S::T_AT, b_at = base + S::B_AT;
  const uint32_t bars = base + S::BARS_AT;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (STAGES + s); };
  auto acc_full = [&](int b) { return bars + 8u * (2 * STAGES + b); };
  auto acc_empty = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
  const uint32_t low_full = bars + 8u * (2 * STAGES + 4), t_full = low_full + 8,
                 b_full = low_full + 16, b_empty = low_full + 24;
  auto raw_full = [&](int r) { return low_full + 32 + 8u * r; };
  auto raw_empty = [&](int r) { return low_full + 32 + 8u * (RAW + r); };
  const uint32_t holder = low_full + 32 + 16u * RAW;
  volatile int* abort_s = reinterpret_cast<volatile int*>(rq_raw + (holder + 8 - raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(full(s), 1 + S::COPY);
      tc::mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(acc_full(b), 1);
      tc::mbar_init(acc_empty(b), 32 * RQ_EPI_WARPS);
    }
    tc::mbar_init(low_full, 1);
    tc::mbar_init(t_full, 32 * RQ_EPI_WARPS);
    tc::mbar_init(b_full, 1);
    tc::mbar_init(b_empty, 1);
    for (int r = 0; r < RAW; ++r) {
      tc::mbar_init(raw_full(r), 1);
      tc::mbar_init(raw_empty(r), RQ_COPY_WARPS);
    }
    *abort_s = 0;
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tm.W);
    tc::prefetch_tmap(&tm.X[0]);
    tc::prefetch_tmap(&tm.X[1]);
    if (ADAPT) {
      tc::prefetch_tmap(&tm.A);
      tc::prefetch_tmap(&tm.B);
    }
    if (!SHIFTED) tc::prefetch_tmap(&tm.Y);
  }
  if (warp == S::MMA_WARP) tc::tmem_alloc(holder, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(rq_raw + (holder - raw));

  // K rows of block kb, rounded up to whole MMAs.  The rows past K belong to the next group (or lie
  // past the tensor and read as zeros) and meet zero weights.
  auto k_rows = [&](int kb) {
    return min(RQ_BK, ((a.K - kb * RQ_BK) + RQ_KSTEP - 1) / RQ_KSTEP * RQ_KSTEP);
  };

  // the weights of K block kb into stage s, which takes x_bytes of X by TMA besides
  auto load_weights = [&](int s, int kb, int mt, int w, uint32_t x_bytes) {
    const bool has = ADAPT && w >= 0;
    tc::mbar_expect_tx(full(s), (uint32_t)(a.w_rows + (has ? a.rank16 : 0)) * RQ_BK + x_bytes);
    tc::tma_load_2d(w_at(s), &tm.W, kb * RQ_BK, (ADAPT ? 0 : w * a.M) + mt * RQ_BM, full(s));
    if (has) tc::tma_load_2d(a_at(s), &tm.A, kb * RQ_BK, w * a.rank, full(s));
  };
  // no load may still be landing when the block exits: the last use of each stage completes when
  // its loads have landed (bounded; immediate unless a wait ran out)
  auto drain_stages = [&](int used) {
    for (int k = used > STAGES ? used - STAGES : 0; k < used; ++k)
      (void)tc::mbar_wait(full(k % STAGES), (uint32_t)(k / STAGES) & 1u, RQ_WAIT_LIMIT);
  };

  if (warp == 0) {
    // ---------------- loads (one lane) -----------------------------------------------------------
    if (lane == 0) {
      int kbg = 0, rawg = 0;
      RqWalk<ADAPT> at, ahead;
      for (at.start(a); at.n < a.rows && !*abort_s; at = ahead) {
        ahead = at.next(a);
        const int src = at.source(a), w = at.weights(a);
        if (src < 0) continue;
        const int mt = at.mt(a), nt = at.r - mt * a.n_tiles;
        bool ok = true;
        for (int kb = 0; kb < a.k_blocks && ok; ++kb, ++kbg) {
          const int s = kbg % STAGES;
          const int kr = k_rows(kb);
          const int row = src * a.K + kb * RQ_BK;
          if (SHIFTED) {
            for (int r = 0; r < kr; r += RQ_RAW_ROWS, ++rawg) {
              const int slot = rawg % RAW;
              const uint32_t use = (uint32_t)(rawg / RAW);
              if (use > 0 && !rq_wait(raw_empty(slot), (use - 1) & 1u, abort_s)) { ok = false; break; }
              tc::mbar_expect_tx(raw_full(slot), RQ_RAW_BYTES);
              const int first = row + r;  // its rows of either parity, in order
              tc::tma_load_2d(raw_at(slot), &tm.X[first & 1], nt * RQ_WORDS, first >> 1,
                              raw_full(slot));
              tc::tma_load_2d(raw_at(slot) + RQ_RAW_BYTES / 2, &tm.X[(first + 1) & 1],
                              nt * RQ_WORDS, (first + 1) >> 1, raw_full(slot));
            }
            if (!ok) break;
          }
          if (!SHIFTED) {
            const uint32_t use = (uint32_t)(kbg / STAGES);
            if (use > 0 && !rq_wait(empty(s), (use - 1) & 1u, abort_s)) { ok = false; break; }
            load_weights(s, kb, mt, w, (uint32_t)(kr * RQ_BN));
            const CUtensorMap* mx = kr == RQ_BK ? &tm.X[0] : &tm.X[1];
            const int step = kr == RQ_BK ? RQ_BK : RQ_KSTEP;
            for (int r = 0; r < kr; r += step) {
              tc::tma_load_2d(x_at(s) + r * 128, mx, nt * RQ_BN, row + r, full(s));
              tc::tma_load_2d(x_at(s) + RQ_BK * 128 + r * 128, mx, nt * RQ_BN + 128, row + r,
                              full(s));
            }
          }
        }
        if (!ok) break;
      }
      if (SHIFTED) {
        for (int k = rawg > RAW ? rawg - RAW : 0; k < rawg; ++k)
          (void)tc::mbar_wait(raw_full(k % RAW), (uint32_t)(k / RAW) & 1u, RQ_WAIT_LIMIT);
      } else {
        drain_stages(kbg);
      }
    }
  } else if (warp < S::MMA_WARP) {
    // ---------------- raw rows -> operand layout (shifted rows only) -----------------------------
    const int cw = warp - 1;
    constexpr int ROWS = RQ_RAW_ROWS / RQ_COPY_WARPS;  // rows of each slot per warp
    const int box = lane >> 4, ch = (lane & 15) >> 1, half = lane & 1;
    int kbg = 0, rawg = 0;
    RqWalk<ADAPT> at, ahead;
    for (at.start(a); at.n < a.rows && !*abort_s; at = ahead) {
      ahead = at.next(a);
      const int src = at.source(a), w = at.weights(a);
      if (src < 0) continue;
      const int mt = at.mt(a), nt = at.r - mt * a.n_tiles;
      bool ok = true;
      for (int kb = 0; kb < a.k_blocks && ok; ++kb, ++kbg) {
        const int s = kbg % STAGES;
        const uint32_t use = (uint32_t)(kbg / STAGES);
        if (use > 0 && !rq_wait(empty(s), (use - 1) & 1u, abort_s)) { ok = false; break; }
        if (cw == 0 && lane == 0) load_weights(s, kb, mt, w, 0u);
        const int kr = k_rows(kb);
        const int parity = (src * a.K + kb * RQ_BK) & 1;  // of the stage's first row
        for (int r0 = 0; r0 < kr; r0 += RQ_RAW_ROWS, ++rawg) {
          const int slot = rawg % RAW;
          if (!rq_wait(raw_full(slot), (uint32_t)(rawg / RAW) & 1u, abort_s)) { ok = false; break; }
          uint64_t v[ROWS];
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            const int r = cw * ROWS + i;
            const int off = ((parity + r) & 1) ? a.off1 : a.off0;
            v[i] = *reinterpret_cast<const uint64_t*>(
                rq_raw + (raw_at(slot) - raw) + (r & 1) * (RQ_RAW_BYTES / 2) +
                (r >> 1) * RQ_RAW_PITCH + (lane + off) * 8);
          }
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            const int r = r0 + cw * ROWS + i;
            *reinterpret_cast<uint64_t*>(rq_raw + (x_at(s) - raw) + box * (RQ_BK * 128) +
                                         (r >> 3) * 1024 + (r & 7) * 128 +
                                         ((ch ^ (r & 7)) << 4) + half * 8) = v[i];
          }
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(raw_empty(slot));
        }
        if (!ok) break;
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(full(s));
      }
      if (!ok) break;
    }
    if (cw == 0 && lane == 0) drain_stages(kbg);
  } else if (warp == S::MMA_WARP) {
    // ---------------- MMA issue (one lane) -------------------------------------------------------
    if (lane == 0) {
      constexpr uint32_t MAIN = tc::idesc_i8(RQ_BM, RQ_BN, true, false, false, true);
      const uint32_t LOW = tc::idesc_i8(128, a.rank16, false, true, true, false);
      int kbg = 0, tt = 0, has_n = 0, b_n = 0;
      auto load_b = [&](const RqWalk<ADAPT>& tile) {
        tc::mbar_expect_tx(b_full, RQ_B_BYTES);
        tc::tma_load_2d(b_at, &tm.B, 0, tile.weights(a) * a.M + tile.mt(a) * RQ_BM, b_full);
        ++b_n;
      };
      RqWalk<ADAPT> at, ahead;
      for (at.start(a); at.n < a.rows && !*abort_s; at = ahead) {
        ahead = at.next(a);
        if (at.source(a) < 0) continue;
        const bool has = ADAPT && at.weights(a) >= 0;
        if (has && b_n == has_n) load_b(at);
        // experts: two accumulators in turn; adapters: C in columns 0-255, L^T and then D in 256-511
        const int buf = ADAPT ? 0 : tt & 1;
        const int turn = ADAPT ? tt : tt >> 1;
        const uint32_t c_tmem = tmem + (uint32_t)(buf * 256);
        if (turn > 0 && !rq_wait(acc_empty(buf), (uint32_t)(turn - 1) & 1u, abort_s)) break;
        tc::tc_fence_after();
        bool ok = true;
        for (int kb = 0; kb < a.k_blocks; ++kb, ++kbg) {
          const int s = kbg % STAGES;
          if (!rq_wait(full(s), (uint32_t)(kbg / STAGES) & 1u, abort_s)) { ok = false; break; }
          tc::tc_fence_after();
          const int steps = k_rows(kb) / RQ_KSTEP;
          for (int k = 0; k < steps; ++k) {
            const uint32_t acc = (kb | k) != 0 ? 1u : 0u;
            const uint64_t wd = tc::smem_desc_sw128(w_at(s) + 32u * k, 16u, 1024u);
            const uint64_t xd = tc::smem_desc_sw128(x_at(s) + 4096u * k, RQ_BK * 128u, 1024u);
            tc::mma_i8(c_tmem, wd, xd, MAIN, acc);
            if (has) {
              const uint64_t ad = tc::smem_desc_sw128(a_at(s) + 32u * k, 16u, 1024u);
              const uint64_t x1 = tc::smem_desc_sw128(x_at(s) + RQ_BK * 128u + 4096u * k,
                                                      RQ_BK * 128u, 1024u);
              tc::mma_i8(tmem + 256u, xd, ad, LOW, acc);
              tc::mma_i8(tmem + 256u + PNB_MAX_RANK, x1, ad, LOW, acc);
            }
          }
          tc::mma_commit(empty(s));
        }
        if (!ok) break;
        if (has) {
          tc::mma_commit(low_full);
          if (!rq_wait(b_full, (uint32_t)has_n & 1u, abort_s)) break;
          if (!rq_wait(t_full, (uint32_t)has_n & 1u, abort_s)) break;
          tc::tc_fence_after();
          // columns of B past the rank are zero, so t's rows past it do not matter
          for (int k = 0; k < (a.rank + 31) / 32; ++k)
            tc::mma_i8(tmem + 256u, tc::smem_desc_sw64(b_at + 32u * k, 16u, 512u),
                       tc::smem_desc_sw128(t_at + 4096u * k, PNB_MAX_RANK * 128u, 1024u), MAIN,
                       k != 0 ? 1u : 0u);
          tc::mma_commit(b_empty);
          ++has_n;
        }
        tc::mma_commit(acc_full(buf));
        ++tt;
        if (ADAPT && ahead.n < a.rows && ahead.weights(a) >= 0) {
          // B of the next tile, once this one's has been read; the epilogue hides it
          if (has && !rq_wait(b_empty, (uint32_t)(has_n - 1) & 1u, abort_s)) break;
          load_b(ahead);
        }
      }
      if (b_n > 0) (void)tc::mbar_wait(b_full, (uint32_t)(b_n - 1) & 1u, RQ_WAIT_LIMIT);
    }
  } else {
    // ---------------- epilogue -------------------------------------------------------------------
    // Warp w reads TMEM lane quarter w % 4 (32 output rows, one per lane) and half eh of the tile's
    // words.  Limb sums become u64 words, staged in shared memory with their 16-byte chunks XORed by
    // the row, and leave as 32 rows x 16 words by TMA, or as 64-byte row segments by plain stores.
    const int e_w = warp - S::MMA_WARP - 1;
    const int q = warp & 3, eh = e_w >> 2;
    constexpr int EW = RQ_WORDS / 2;
    const uint32_t out_at = base + S::OUT_AT + (uint32_t)(e_w * S::OUT);
    unsigned char* out = rq_raw + (out_at - raw);
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    int tt = 0, has_n = 0;
    RqWalk<ADAPT> at, ahead;
    for (at.start(a); at.n < a.rows && !*abort_s; at = ahead) {
      ahead = at.next(a);
      const int src = at.source(a), w = at.weights(a);
      if (src < 0) continue;
      const int mt = at.mt(a), nt = at.r - mt * a.n_tiles;
      const bool has = ADAPT && w >= 0;
      if (has) {
        // t = A X: lane l of quarter q holds limb l % 8 of word eh*16 + q*4 + l/8 for every rank
        // row.  Eight lanes add up 16 rows at a time, halving the rows they keep at each step.
        if (!rq_wait(low_full, (uint32_t)has_n & 1u, abort_s)) break;
        tc::tc_fence_after();
        const int word = q * 4 + (lane >> 3);  // within the 16 words of half eh
        for (int r0 = 0; r0 < a.rank16; r0 += 16) {
          uint32_t c[16];
          tc::tmem_ld_32x32_x16(tmem + 256u + eh * PNB_MAX_RANK + lanes + r0, c);
          tc::tmem_ld_wait_for(c);
          uint64_t v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = (uint64_t)(int64_t)(int32_t)c[j] << (8 * (lane & 7));
#pragma unroll
          for (int half = 8; half >= 2; half >>= 1) {
            const bool up = (lane & (half >> 1)) != 0;
#pragma unroll
            for (int j = 0; j < half; ++j) {
              const uint64_t give = up ? v[j] : v[j + half];
              v[j] = (up ? v[j + half] : v[j]) + shfl_xor_u64(give, half >> 1);
            }
          }
          const int r = r0 + 2 * (lane & 7);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int rr = r + j;
            const uint32_t at = t_at + eh * (PNB_MAX_RANK * 128) + (rr >> 3) * 1024 +
                                (rr & 7) * 128 + (((word >> 1) ^ (rr & 7)) << 4) + (word & 1) * 8;
            *reinterpret_cast<uint64_t*>(rq_raw + (at - raw)) = v[j];
          }
        }
        tc::fence_async_smem();
        tc::tc_fence_before();
        tc::mbar_arrive(t_full);
        ++has_n;
      }
      const int buf = ADAPT ? 0 : tt & 1;
      const int turn = ADAPT ? tt : tt >> 1;
      const uint32_t c_tmem = tmem + (uint32_t)(buf * 256) + lanes + (uint32_t)(eh * EW * 8);
      const int row0 = mt * RQ_BM + q * 32, col0 = nt * RQ_WORDS + eh * EW;
      // C is complete with the low product; only D is still to come
      if (!has && !rq_wait(acc_full(buf), (uint32_t)turn & 1u, abort_s)) break;
      tc::tc_fence_after();
      if (row0 >= a.M || col0 >= a.L) {  // nothing of this warp's share is kept
        if (has && !rq_wait(acc_full(buf), (uint32_t)turn & 1u, abort_s)) break;
        tc::tc_fence_before();
        tc::mbar_arrive(acc_empty(buf));
        ++tt;
        continue;
      }
      // the word of this half that is the body, and its bias
      const int body = a.L - 1 - col0;
      uint64_t bias = 0;
      if (a.bias && body < EW && row0 + lane < a.M)
        bias = (uint64_t)__ldg(a.bias + (ADAPT ? (size_t)0 : (size_t)w * a.M) + row0 + lane) *
               a.delta;
      // 4 words (32 columns) at a time, the next columns on their way while these are added up
      constexpr int CHUNKS = EW / 4;
      uint32_t c[2][32], d[32];
      bool ok = true;
      tc::tmem_ld_32x32_nowait(c_tmem, c[0]);
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) {
        uint32_t(&ci)[32] = c[i & 1];
        tc::tmem_ld_wait_for(ci);
        if (has) {
          if (i == 0) {
            ok = rq_wait(acc_full(buf), (uint32_t)turn & 1u, abort_s);
            tc::tc_fence_after();
          }
          tc::tmem_ld_32x32_nowait(c_tmem + (uint32_t)(256 + i * 32), d);
        } else if (i + 1 < CHUNKS) {
          tc::tmem_ld_32x32_nowait(c_tmem + (uint32_t)((i + 1) * 32), c[(i + 1) & 1]);
        }
        uint64_t y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          y[u] = add_limbs(0, ci + 8 * u);
          if (ADAPT) y[u] <<= a.shift;
        }
        if (has) {
          tc::tmem_ld_wait_for(d);
          if (i + 1 < CHUNKS)
            tc::tmem_ld_32x32_nowait(c_tmem + (uint32_t)((i + 1) * 32), c[(i + 1) & 1]);
        }
        if (i + 1 == CHUNKS) {
          tc::tc_fence_before();
          tc::mbar_arrive(acc_empty(buf));
        }
        if (has) {
#pragma unroll
          for (int u = 0; u < 4; ++u) y[u] = add_limbs(y[u], d + 8 * u);
        }
        if (!SHIFTED && i == 0) {  // the staging rows of the previous tile have left
          if (lane == 0) tc::tma_store_wait_read();
          __syncwarp();
        }
        // lane's row, its 16-byte chunks XORed by the lane
        constexpr int PITCH = S::OUT / 32, SPAN = PITCH / 32;  // SPAN chunks of 4 words per row
        const int ch = (i % SPAN) * 2;
        const int x = SHIFTED ? (lane >> 1) & 3 : lane & 7;
        *reinterpret_cast<ulonglong2*>(out + lane * PITCH + ((ch ^ x) << 4)) =
            make_ulonglong2(y[0], y[1]);
        *reinterpret_cast<ulonglong2*>(out + lane * PITCH + (((ch + 1) ^ x) << 4)) =
            make_ulonglong2(y[2], y[3]);
        const int at_word = body - (i - i % SPAN) * 4;  // the body within the staged words
        if (body >= i * 4 && body < i * 4 + 4)
          *reinterpret_cast<uint64_t*>(out + lane * PITCH + (((at_word >> 1) ^ x) << 4) +
                                       (at_word & 1) * 8) += bias;
        if (SHIFTED && i % SPAN == SPAN - 1) {
          __syncwarp();
          // 4 rows per instruction, 8 lanes x 8 bytes = one 64-byte row segment each
          const int wd = lane & 7;
          const int col = col0 + (i - i % SPAN) * 4 + wd;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int rr = 4 * j + (lane >> 3);
            if (row0 + rr < a.M && col < a.L)
              a.Y[((size_t)at.n * a.M + row0 + rr) * a.ldy + col] =
                  *reinterpret_cast<const uint64_t*>(
                      out + rr * PITCH + (((wd >> 1) ^ ((rr >> 1) & 3)) << 4) + (wd & 1) * 8);
          }
          __syncwarp();
        }
      }
      if (!ok) break;
      if (!SHIFTED) {
        // tiled stores end on 16-byte boundaries, so the last word of an odd count goes alone
        if ((a.L & 1) && body < EW && row0 + lane < a.M)
          a.Y[((size_t)at.n * a.M + row0 + lane) * a.ldy + a.L - 1] =
              *reinterpret_cast<const uint64_t*>(out + lane * 128 +
                                                 (((body >> 1) ^ (lane & 7)) << 4) +
                                                 (body & 1) * 8);
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0 && col0 < (a.L & ~1))
          tc::tma_store_3d(&tm.Y, col0, row0, at.n, out_at);
      }
      ++tt;
    }
    if (!SHIFTED && lane == 0) tc::tma_store_wait();
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == S::MMA_WARP) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// ---- launch -------------------------------------------------------------------------------------
// TMA reads an int8 matrix [rows][cols] in place when its rows start 16-byte aligned; otherwise it
// is copied to the workspace with its rows padded by zeros to a multiple of 16.
struct RqMatrix {
  const int8_t* p;
  long long rows;
  int cols;
  int pitch() const { return (cols + 15) & ~15; }
  bool in_place() const { return cols % 16 == 0 && ((uintptr_t)p % 16) == 0; }
  size_t copy_bytes() const { return (size_t)rows * pitch(); }
};

__global__ void rq_pad_kernel(const int8_t* __restrict__ in, long long rows, int cols, int pitch,
                              int8_t* __restrict__ out) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= rows * pitch) return;
  const long long r = i / pitch;
  const int c = (int)(i - r * pitch);
  out[i] = c < cols ? in[r * cols + c] : (int8_t)0;
}

static int rq_place(RqMatrix& m, int8_t*& ws, cudaStream_t st) {
  if (m.in_place()) return PNB_OK;
  const size_t n = m.copy_bytes();
  rq_pad_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(m.p, m.rows, m.cols, m.pitch(), ws);
  PNB_CHECK_LAUNCH("rq_pad_kernel");
  m.p = ws;
  ws += n;
  return PNB_OK;
}

// A tiled map of `rank` dimensions (strides of all but the first, in bytes).
static int rq_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int rank,
                  const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                  CUtensorMapSwizzle swizzle) {
  auto fn = tmap_encoder();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled is unavailable from the driver");
    return PNB_ERR_CUDA;
  }
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = fn(map, type, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return PNB_OK;
  set_error("cuTensorMapEncodeTiled failed (%d): %llu x %llu, pitch %llu", (int)r,
            (unsigned long long)dims[0], (unsigned long long)dims[1],
            (unsigned long long)strides[0]);
  return PNB_ERR_CUDA;
}

// Byte matrix [rows][cols] at a pitch, in boxes of box_cols bytes (one swizzle span) x box_rows.
static int rq_map_bytes(CUtensorMap* map, const void* p, uint64_t cols, uint64_t rows,
                        uint64_t pitch, int box_cols, int box_rows) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  return rq_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, 2, dims, strides, box,
                box_cols == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}
static int rq_map_weights(CUtensorMap* map, const RqMatrix& m, int box_cols, int box_rows) {
  return rq_map_bytes(map, m.p, (uint64_t)m.pitch(), (uint64_t)m.rows, (uint64_t)m.pitch(), box_cols,
                      box_rows);
}

template <bool SHIFTED, bool ADAPT>
static int rq_launch(int grid, const RqMaps& tm, const RqArgs& a, cudaStream_t st) {
  using S = RqShape<SHIFTED, ADAPT>;
  PNB_CUDA(cudaFuncSetAttribute(request_kernel<SHIFTED, ADAPT>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
  request_kernel<SHIFTED, ADAPT><<<grid, S::THREADS, S::SMEM, st>>>(tm, a);
  PNB_CHECK_LAUNCH("request_kernel");
  return PNB_OK;
}

template <bool ADAPT>
static int rq_run(RqMatrix W, RqMatrix A, RqMatrix B, RqArgs a, int x_groups, cudaStream_t st) {
  const long long x_rows = (long long)x_groups * a.K;
  // TMA coordinates are 32-bit, and a tile reaches up to a stage past its first row
  constexpr long long MOST = 0x7fffffffLL - RQ_BK;
  if (x_rows > MOST || W.rows > MOST || A.rows > MOST || B.rows > MOST) {
    set_error("%s: %lld ciphertexts or %lld weight rows exceed a 32-bit index",
              ADAPT ? "adapter_contract" : "expert_contract", x_rows,
              std::max(W.rows, std::max(A.rows, B.rows)));
    return PNB_ERR_INVALID;
  }
  a.n_tiles = (a.L + RQ_WORDS - 1) / RQ_WORDS;
  const long long per_row = (long long)((a.M + RQ_BM - 1) / RQ_BM) * a.n_tiles;
  if (per_row > 1 << 30 || a.rows > 1 << 30) {
    set_error("%s: %d rows of %lld tiles exceed one launch",
              ADAPT ? "adapter_contract" : "expert_contract", a.rows, per_row);
    return PNB_ERR_INVALID;
  }
  a.per_row = (int)per_row;
  a.k_blocks = (a.K + RQ_BK - 1) / RQ_BK;
  a.w_rows = std::min(RQ_BM, (a.M + 7) & ~7);
  const uintptr_t xw = (uintptr_t)a.X / 8;
  a.off0 = (int)(xw & 1);
  a.off1 = (int)((xw + (uintptr_t)a.ldx) & 1);
  const bool shifted = a.off0 || a.off1 || a.ldy % 2 != 0 || ((uintptr_t)a.Y % 16) != 0;
  RqMaps tm{};
  int rc = PNB_OK;
  if (!shifted) {
    const uint64_t pitch = (uint64_t)a.ldx * 8;
    rc = rq_map_bytes(&tm.X[0], a.X, pitch, (uint64_t)x_rows, pitch, 128, RQ_BK);
    if (!rc) rc = rq_map_bytes(&tm.X[1], a.X, pitch, (uint64_t)x_rows, pitch, 128, RQ_KSTEP);
    // writes end at word L (rounded down to 16 bytes) of row M of each ciphertext row
    const cuuint64_t dims[3] = {(cuuint64_t)std::max(2, a.L & ~1), (cuuint64_t)a.M, (cuuint64_t)a.rows};
    const cuuint64_t strides[2] = {(cuuint64_t)a.ldy * 8, (cuuint64_t)a.M * a.ldy * 8};
    const cuuint32_t box[3] = {RQ_WORDS / 2, 32, 1};
    if (!rc)
      rc = rq_map(&tm.Y, CU_TENSOR_MAP_DATA_TYPE_UINT64, a.Y, 3, dims, strides, box,
                  CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    // rows p, p + 2, ..: from the 16-byte boundary at or before row p, at twice the pitch.  A row
    // off by one word has that word's 16 bytes inside its allocation (allocations start aligned).
    for (int p = 0; p < 2 && !rc; ++p) {
      // (a single row has no row 1: both maps are its own, and the second meets zero weights)
      const bool second = p && x_rows > 1;
      const int off = second ? a.off1 : a.off0;
      const cuuint64_t dims[2] = {(cuuint64_t)a.ldx + off,
                                  (cuuint64_t)std::max<long long>(1, (x_rows + 1 - p) / 2)};
      const cuuint64_t strides[1] = {(cuuint64_t)a.ldx * 16};
      const cuuint32_t box[2] = {RQ_WORDS + 2, RQ_RAW_ROWS / 2};
      const uint64_t* first = a.X + (second ? a.ldx : 0) - off;
      rc = rq_map(&tm.X[p], CU_TENSOR_MAP_DATA_TYPE_UINT64, first, 2, dims, strides, box,
                  CU_TENSOR_MAP_SWIZZLE_NONE);
    }
  }
  if (rc) return rc;
  size_t need = W.in_place() ? 0 : W.copy_bytes();
  if (ADAPT) need += (A.in_place() ? 0 : A.copy_bytes()) + (B.in_place() ? 0 : B.copy_bytes());
  int8_t* own = nullptr;
  if (need) PNB_CUDA(cudaMallocAsync((void**)&own, need, st));
  int8_t* ws = own;
  rc = rq_place(W, ws, st);
  if (ADAPT && !rc) rc = rq_place(A, ws, st);
  if (ADAPT && !rc) rc = rq_place(B, ws, st);
  if (!rc) rc = rq_map_weights(&tm.W, W, 128, a.w_rows);
  if (ADAPT && !rc) rc = rq_map_weights(&tm.A, A, 128, a.rank16);
  if (ADAPT && !rc) rc = rq_map_weights(&tm.B, B, PNB_MAX_RANK, RQ_BM);
  int dev = 0, sms = 0;
  if (!rc) {
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) rc = cuda_status(e, "cudaDeviceGetAttribute");
  }
  if (!rc) {
    const int grid = (int)std::min<long long>(a.rows * per_row, sms);
    a.step_n = grid / a.per_row;
    a.step_r = grid % a.per_row;
    rc = shifted ? rq_launch<true, ADAPT>(grid, tm, a, st) : rq_launch<false, ADAPT>(grid, tm, a, st);
  }
  if (own) {
    const cudaError_t e = cudaFreeAsync(own, st);
    if (!rc && e != cudaSuccess) rc = cuda_status(e, "cudaFreeAsync(padded weights)");
  }
  return rc;
}

int expert_contract(const int32_t* row_choice, const int32_t* row_expert, int tokens, int top_k,
                    int experts, bool sorted_rows, const int8_t* W, const int64_t* bias,
                    uint64_t delta, int M, int K, const uint64_t* X, int ldx, uint64_t* Y, int ldy,
                    int L, cudaStream_t st) {
  RqArgs a{};
  a.X = X; a.Y = Y; a.bias = bias; a.delta = delta;
  a.row_choice = row_choice; a.which = row_expert;
  a.rows = a.choices = tokens * top_k;
  a.top_k = sorted_rows ? 0 : top_k;
  a.n_which = experts;
  a.M = M; a.K = K; a.L = L; a.ldx = ldx; a.ldy = ldy;
  return rq_run<false>({W, (long long)experts * M, K}, {}, {}, a, sorted_rows ? a.rows : tokens, st);
}

int adapter_contract(const int8_t* W, const int64_t* bias, uint64_t delta, int base_shift, int M,
                     int K, const int8_t* A, const int8_t* B, int adapters, int rank,
                     const int32_t* adapter, const uint64_t* X, int ldx, uint64_t* Y, int ldy,
                     int batch, int L, cudaStream_t st) {
  RqArgs a{};
  a.X = X; a.Y = Y; a.bias = bias; a.delta = delta;
  a.which = adapter; a.n_which = adapters;
  a.rows = batch;
  a.M = M; a.K = K; a.L = L; a.ldx = ldx; a.ldy = ldy;
  a.shift = base_shift; a.rank = rank; a.rank16 = (rank + 15) & ~15;
  return rq_run<true>({W, M, K}, {A, (long long)adapters * rank, K}, {B, (long long)adapters * M, rank},
                      a, batch, st);
}

}  // namespace pnb

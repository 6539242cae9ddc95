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

int make_tmap_u8_2d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer,
                    uint64_t pitch_bytes, uint32_t box_inner, uint32_t box_outer);

constexpr int RQ_BM = 128;      // output rows per tile
constexpr int RQ_WORDS = 32;    // output words per tile
constexpr int RQ_BN = 8 * RQ_WORDS;
constexpr int RQ_BK = 128;      // K per stage
constexpr int RQ_KBOX = 32;     // K per X box and MMA step: a ragged K costs at most 31 rows
constexpr int RQ_W_BYTES = RQ_BM * RQ_BK;              // 16 KB
constexpr int RQ_X_BYTES = RQ_BK * RQ_BN;              // 32 KB
constexpr int RQ_A_BYTES = PNB_MAX_RANK * RQ_BK;       // 8 KB
constexpr int RQ_T_BYTES = PNB_MAX_RANK * RQ_BN;       // 16 KB: t as bytes
constexpr int RQ_B_BYTES = RQ_BM * 128;                // 16 KB: B rows, 128-byte pitch
constexpr int RQ_EPI_WARPS = 8;                        // two per TMEM lane quarter
constexpr int RQ_EPI_BYTES = RQ_EPI_WARPS * 32 * 8 * 8;
constexpr uint32_t RQ_WAIT_LIMIT = 1u << 24;

// How X reaches shared memory: rows that start 16-byte aligned (an even pitch) by TMA; other rows
// by 8-byte cp.async from 8 warps.
enum : int { RQ_TMA = 0, RQ_COPY8 = 1 };

template <int MODE, bool ADAPT>
struct RqShape {
  static constexpr int STAGE = RQ_W_BYTES + (ADAPT ? RQ_A_BYTES : 0) + RQ_X_BYTES;
  static constexpr int STAGES = ADAPT || MODE == RQ_COPY8 ? 3 : 4;
  static constexpr int PW = MODE == RQ_TMA ? 1 : 8;  // producer warps
  static constexpr int THREADS = 32 * (PW + 1 + RQ_EPI_WARPS);
  static constexpr int T_AT = STAGES * STAGE;                  // t, then B (adapters only)
  static constexpr int BARS_AT = T_AT + (ADAPT ? RQ_T_BYTES + RQ_B_BYTES : 0);
  static constexpr int SMEM = 1024 + BARS_AT + 256 + RQ_EPI_BYTES;
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
  int m_tiles, n_tiles, k_blocks, w_rows;
};

// Row n's X group (-1: the row is skipped) and its weights (-1: no adapter).
template <bool ADAPT>
__device__ __forceinline__ void rq_row(const RqArgs& a, int n, int& src, int& w) {
  w = __ldg(a.which + n);
  if (w < 0 || w >= a.n_which) w = -1;
  src = n;
  if (!ADAPT) {
    if (w < 0) { src = -1; return; }
    const int c = __ldg(a.row_choice + n);
    if (c < 0 || c >= a.choices)
      src = -1;
    else if (a.top_k > 0)
      src = c / a.top_k;
  }
}

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

template <int MODE, bool ADAPT>
__global__ void __launch_bounds__(RqShape<MODE, ADAPT>::THREADS, 1) request_kernel(
    const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
    const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, RqArgs a) {
  using S = RqShape<MODE, ADAPT>;
  constexpr int STAGES = S::STAGES;
  constexpr int MMA_WARP = S::PW;
  extern __shared__ unsigned char rq_raw[];
  const uint32_t raw = tc::smem_u32(rq_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  auto w_at = [&](int s) { return base + (uint32_t)(s * S::STAGE); };
  auto x_at = [&](int s) { return w_at(s) + RQ_W_BYTES; };
  auto a_at = [&](int s) { return x_at(s) + RQ_X_BYTES; };
  const uint32_t t_at = base + S::T_AT, b_at = t_at + RQ_T_BYTES;
  const uint32_t bars = base + S::BARS_AT;
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (STAGES + s); };
  auto acc_full = [&](int b) { return bars + 8u * (2 * STAGES + b); };
  auto acc_empty = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
  const uint32_t low_full = bars + 8u * (2 * STAGES + 4), t_full = low_full + 8,
                 b_full = low_full + 16, b_empty = low_full + 24;
  const uint32_t holder = low_full + 32;
  volatile int* abort_s = reinterpret_cast<volatile int*>(rq_raw + (holder + 8 - raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(full(s), MODE == RQ_TMA ? 1 : 32 * S::PW + 1);
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
    *abort_s = 0;
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tmW);
    if (MODE == RQ_TMA) tc::prefetch_tmap(&tmX);
    if (ADAPT) {
      tc::prefetch_tmap(&tmA);
      tc::prefetch_tmap(&tmB);
    }
  }
  if (warp == MMA_WARP) tc::tmem_alloc(holder, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(rq_raw + (holder - raw));

  const long long total = (long long)a.rows * a.m_tiles * a.n_tiles;
  // tile -> (row n, 128 output rows mt, 32 words nt), nt fastest
  auto decode = [&](long long t, int& n, int& mt, int& nt) {
    const int per = a.m_tiles * a.n_tiles;
    n = (int)(t / per);
    const int r = (int)(t - (long long)n * per);
    mt = r / a.n_tiles;
    nt = r - mt * a.n_tiles;
  };
  // K rows of block kb, rounded up to whole MMA steps
  auto k_rows = [&](int kb) {
    return min(RQ_BK, ((a.K - kb * RQ_BK) + RQ_KBOX - 1) / RQ_KBOX * RQ_KBOX);
  };
  const uint32_t w_bytes = (uint32_t)(a.w_rows * RQ_BK), a_bytes = (uint32_t)(a.rank16 * RQ_BK);

  if (warp < S::PW) {
    // ---------------- producers -----------------------------------------------------------------
    constexpr int LAG = STAGES - 1;
    int kbg = 0, released = 0, has_n = 0;
    const bool lead = warp == 0 && lane == 0;
    if (MODE != RQ_TMA || lead) {
      for (long long t = blockIdx.x; t < total && !*abort_s; t += gridDim.x) {
        int n, mt, nt, src, w;
        decode(t, n, mt, nt);
        rq_row<ADAPT>(a, n, src, w);
        if (src < 0) continue;
        const bool has = ADAPT && w >= 0;
        const int w_row = (ADAPT ? 0 : w * a.M) + mt * RQ_BM;
        bool ok = true;
        for (int kb = 0; kb < a.k_blocks; ++kb, ++kbg) {
          const int s = kbg % STAGES;
          const uint32_t use = (uint32_t)(kbg / STAGES);
          if (use > 0 && !rq_wait(empty(s), (use - 1) & 1u, abort_s)) { ok = false; break; }
          const int kr = k_rows(kb);
          if (lead) {
            tc::mbar_expect_tx(full(s), w_bytes + (has ? a_bytes : 0u) +
                                            (MODE == RQ_TMA ? (uint32_t)(kr * RQ_BN) : 0u));
            tc::tma_load_2d(w_at(s), &tmW, kb * RQ_BK, w_row, full(s));
            if (has) tc::tma_load_2d(a_at(s), &tmA, kb * RQ_BK, w * a.rank, full(s));
          }
          if (MODE == RQ_TMA) {
            // rows past K belong to the next group (or lie past the tensor and read as zeros)
            // and meet zero weights
            for (int r = 0; r < kr; r += RQ_KBOX) {
              const int row = src * a.K + kb * RQ_BK + r;
              tc::tma_load_2d(x_at(s) + r * 128, &tmX, nt * RQ_BN, row, full(s));
              tc::tma_load_2d(x_at(s) + RQ_BK * 128 + r * 128, &tmX, nt * RQ_BN + 128, row,
                              full(s));
            }
          } else {
            const int col = nt * RQ_WORDS + lane;
            const int box = lane >> 4, ch = (lane & 15) >> 1, half = lane & 1;
            const uint64_t* xp = a.X + ((size_t)src * a.K + kb * RQ_BK) * a.ldx + col;
#pragma unroll 4
            for (int r = warp; r < kr; r += S::PW) {
              const bool in = col < a.L && kb * RQ_BK + r < a.K;
              const uint32_t dst = x_at(s) + box * (RQ_BK * 128) + (r >> 3) * 1024 +
                                   (r & 7) * 128 + ((ch ^ (r & 7)) << 4) + half * 8;
              asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst),
                           "l"(in ? xp + (size_t)r * a.ldx : a.X), "r"(in ? 8u : 0u)
                           : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (kbg + 1 - released > LAG) {
              asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              tc::mbar_arrive(full(released % STAGES));
              ++released;
            }
          }
        }
        if (!ok) break;
        if (has && lead) {
          if (MODE != RQ_TMA) {  // the previous tile must not wait for copies that lag behind
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            for (; released < kbg; ++released) tc::mbar_arrive(full(released % STAGES));
          }
          // after this tile's K blocks: the wait for the previous tile's last MMA is then short
          if (has_n > 0 && !rq_wait(b_empty, (uint32_t)(has_n - 1) & 1u, abort_s)) break;
          tc::mbar_expect_tx(b_full, RQ_B_BYTES);
          tc::tma_load_2d(b_at, &tmB, 0, w * a.M + mt * RQ_BM, b_full);
          ++has_n;
        }
      }
      if (MODE != RQ_TMA) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        for (; released < kbg; ++released) tc::mbar_arrive(full(released % STAGES));
      }
      // no copy may still be landing when the block exits: the last use of each slot completes
      // when its copies have landed (bounded; immediate unless a wait ran out)
      if (lead) {
        for (int k = kbg > STAGES ? kbg - STAGES : 0; k < kbg; ++k)
          (void)tc::mbar_wait(full(k % STAGES), (uint32_t)(k / STAGES) & 1u, RQ_WAIT_LIMIT);
        if (has_n > 0) (void)tc::mbar_wait(b_full, (uint32_t)(has_n - 1) & 1u, RQ_WAIT_LIMIT);
      }
    }
  } else if (warp == MMA_WARP) {
    // ---------------- MMA issue (one lane) -------------------------------------------------------
    if (lane == 0) {
      constexpr uint32_t MAIN = tc::idesc_i8(RQ_BM, RQ_BN, true, false, false, true);
      const uint32_t LOW = tc::idesc_i8(128, a.rank16, false, true, true, false);
      int kbg = 0, tt = 0, has_n = 0;
      for (long long t = blockIdx.x; t < total && !*abort_s; t += gridDim.x) {
        int n, mt, nt, src, w;
        decode(t, n, mt, nt);
        rq_row<ADAPT>(a, n, src, w);
        if (src < 0) continue;
        const bool has = ADAPT && w >= 0;
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
          const int steps = k_rows(kb) / RQ_KBOX;
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
            tc::mma_i8(tmem + 256u, tc::smem_desc_sw128(b_at + 32u * k, 16u, 1024u),
                       tc::smem_desc_sw128(t_at + 4096u * k, PNB_MAX_RANK * 128u, 1024u), MAIN,
                       k != 0 ? 1u : 0u);
          tc::mma_commit(b_empty);
          ++has_n;
        }
        tc::mma_commit(acc_full(buf));
        ++tt;
      }
    }
  } else {
    // ---------------- epilogue -------------------------------------------------------------------
    // Warp w reads TMEM lane quarter w % 4 (32 output rows) and half eh of the tile's words, two
    // chunks of 8 words; limbs become u64 words, staged in shared memory (32 rows x 8 words,
    // XOR-swizzled) and written as 64-byte row segments.
    const int e_w = warp - MMA_WARP - 1;
    const int q = warp & 3, eh = e_w >> 2;
    constexpr int EW = RQ_WORDS / 2;
    uint64_t* stage =
        reinterpret_cast<uint64_t*>(rq_raw + (bars + 256 - raw)) + (size_t)e_w * 32 * 8;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    int tt = 0, has_n = 0;
    for (long long t = blockIdx.x; t < total && !*abort_s; t += gridDim.x) {
      int n, mt, nt, src, w;
      decode(t, n, mt, nt);
      rq_row<ADAPT>(a, n, src, w);
      if (src < 0) continue;
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
          tc::tmem_ld_wait();
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
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc::tc_fence_before();
        tc::mbar_arrive(t_full);
        ++has_n;
      }
      const int buf = ADAPT ? 0 : tt & 1;
      const int turn = ADAPT ? tt : tt >> 1;
      if (!rq_wait(acc_full(buf), (uint32_t)turn & 1u, abort_s)) break;
      tc::tc_fence_after();
      const uint32_t c_tmem = tmem + (uint32_t)(buf * 256) + lanes + (uint32_t)(eh * EW * 8);
#pragma unroll 1
      for (int cp = 0; cp < EW / 8; ++cp) {
        uint64_t y[8];
        uint32_t r0[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tc::tmem_ld_32x32(c_tmem + (uint32_t)(cp * 64 + h * 32), r0);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint64_t v = 0;
#pragma unroll
            for (int b = 0; b < 8; ++b)
              v += (uint64_t)(int64_t)(int32_t)r0[u * 8 + b] << (8 * b);
            y[h * 4 + u] = ADAPT ? v << a.shift : v;
          }
          if (has) {
            tc::tmem_ld_32x32(c_tmem + (uint32_t)(256 + cp * 64 + h * 32), r0);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int b = 0; b < 8; ++b)
                y[h * 4 + u] += (uint64_t)(int64_t)(int32_t)r0[u * 8 + b] << (8 * b);
          }
        }
        if (cp == EW / 8 - 1) {
          tc::tc_fence_before();
          tc::mbar_arrive(acc_empty(buf));
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) stage[lane * 8 + (u ^ (lane & 7))] = y[u];
        __syncwarp();
        // 4 rows per instruction, 8 lanes x 8 bytes = one 64-byte row segment each
        const int wd = lane & 7;
        const int col = nt * RQ_WORDS + eh * EW + cp * 8 + wd;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = 4 * i + (lane >> 3);
          const int row = mt * RQ_BM + q * 32 + rr;
          uint64_t v = stage[rr * 8 + (wd ^ (rr & 7))];
          if (row < a.M && col < a.L) {
            if (col == a.L - 1 && a.bias)
              v += (uint64_t)a.bias[(ADAPT ? (size_t)0 : (size_t)w * a.M) + row] * a.delta;
            a.Y[((size_t)n * a.M + row) * a.ldy + col] = v;
          }
        }
        __syncwarp();
      }
      ++tt;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
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

static int rq_map(CUtensorMap* map, const RqMatrix& m, int box_rows) {
  return make_tmap_u8_2d(map, m.p, (uint64_t)m.pitch(), (uint64_t)m.rows, (uint64_t)m.pitch(), 128,
                         (uint32_t)box_rows);
}

template <int MODE, bool ADAPT>
static int rq_launch(int grid, const CUtensorMap (&tm)[4], const RqArgs& a, cudaStream_t st) {
  using S = RqShape<MODE, ADAPT>;
  static_assert(S::SMEM <= 227 * 1024, "shared memory of one block");
  PNB_CUDA(cudaFuncSetAttribute(request_kernel<MODE, ADAPT>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
  request_kernel<MODE, ADAPT><<<grid, S::THREADS, S::SMEM, st>>>(tm[0], tm[1], tm[2], tm[3], a);
  PNB_CHECK_LAUNCH("request_kernel");
  return PNB_OK;
}

template <bool ADAPT>
static int rq_run(RqMatrix W, RqMatrix A, RqMatrix B, RqArgs a, int x_groups, cudaStream_t st) {
  // TMA coordinates are 32-bit, and a tile reaches up to a stage past its first row
  constexpr long long MOST = 0x7fffffffLL - RQ_BK;
  if ((long long)x_groups * a.K > MOST || W.rows > MOST || A.rows > MOST || B.rows > MOST) {
    set_error("%s: %lld ciphertexts or %lld weight rows exceed a 32-bit index",
              ADAPT ? "adapter_contract" : "expert_contract", (long long)x_groups * a.K,
              std::max(W.rows, std::max(A.rows, B.rows)));
    return PNB_ERR_INVALID;
  }
  a.m_tiles = (a.M + RQ_BM - 1) / RQ_BM;
  a.n_tiles = (a.L + RQ_WORDS - 1) / RQ_WORDS;
  a.k_blocks = (a.K + RQ_BK - 1) / RQ_BK;
  a.w_rows = std::min(RQ_BM, (a.M + 7) & ~7);
  size_t need = W.in_place() ? 0 : W.copy_bytes();
  if (ADAPT) need += (A.in_place() ? 0 : A.copy_bytes()) + (B.in_place() ? 0 : B.copy_bytes());
  int8_t* own = nullptr;
  if (need) PNB_CUDA(cudaMallocAsync((void**)&own, need, st));
  int8_t* ws = own;
  int rc = rq_place(W, ws, st);
  if (ADAPT && !rc) rc = rq_place(A, ws, st);
  if (ADAPT && !rc) rc = rq_place(B, ws, st);
  const bool aligned = a.ldx % 2 == 0 && ((uintptr_t)a.X % 16) == 0;
  CUtensorMap tm[4] = {};
  if (!rc) rc = rq_map(&tm[0], W, a.w_rows);
  if (!rc && aligned)
    rc = make_tmap_u8_2d(&tm[1], a.X, (uint64_t)a.ldx * 8, (uint64_t)x_groups * a.K,
                         (uint64_t)a.ldx * 8, 128, RQ_KBOX);
  if (ADAPT && !rc) rc = rq_map(&tm[2], A, a.rank16);
  if (ADAPT && !rc) rc = rq_map(&tm[3], B, RQ_BM);
  if (!rc) {
    int dev = 0, sms = 148;
    PNB_CUDA(cudaGetDevice(&dev));
    PNB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const int grid = (int)std::min<long long>((long long)a.rows * a.m_tiles * a.n_tiles, sms);
    rc = aligned ? rq_launch<RQ_TMA, ADAPT>(grid, tm, a, st)
                 : rq_launch<RQ_COPY8, ADAPT>(grid, tm, a, st);
  }
  if (own) {
    cudaError_t e = cudaFreeAsync(own, st);
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

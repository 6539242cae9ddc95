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
// One kernel for both, on the tensor cores (calls of few products take plain multiply-adds, below).
// A u64 word is 8 little-endian byte limbs, so the K ciphertexts of a row are a u8 matrix [K][8 ld],
// N-contiguous: kind::i8 reads it as an MN-major operand and the epilogue puts the limb sums together,
//     y = sum_b C[.][8c + b] << 8b  (mod 2^64),  |C| <= 128 * 255 * K < 2^31 for K < 65794.
// A tile is 128 output rows x 32 words (adapters: 16) of one ciphertext row; persistent blocks walk
// groups of tiles that share their X.  Weights are picked per tile by the TMA coordinate, so rows of
// different experts share a launch.
//
// The floor is HBM: X read once and Y written once (256 requests 784->128: 3.83 GB, 586 us at the
// measured copy bandwidth, where the MMAs need 251 us at twice the measured bf16 rate).  What stands
// between is the path from L2 to the SM: a tile reads K x 256 bytes of X, and as many weight rows
// again unless they stay.  So weights stay in shared memory while consecutive tiles of a block use
// the same ones (rows sorted by expert see to that), and where the output has several tiles of 128
// rows, X stays while they take turns (122 rows 130->200: one tile at a time 181 -> 237 us).
// Groups are dealt out to the blocks in turn, so that the blocks work on one ciphertext row at a
// time and its lines are still in L2 for all of them; consecutive runs for each block keep weights
// longer but cost more (45 x 257->384: 263 -> 295 us).
//
// Measured (sustained, SM clock falling to 1.2-1.7 GHz under the power cap; in brackets the best
// launch): 256 x 784->128 of 16 experts 736 us (616) = 5.2 TB/s (6.2); with adapters of rank 16 888 us
// (755) = 4.3 TB/s (5.1); one request 10.4 us a call and 9.4 replayed in a graph, 16.9 and 11.5 with an
// adapter of rank 8.  122 x 130->200 144 us (120), 45 x 257->384 of rank 33 240 us (220).  At an odd pitch
// 256 x 784->128 946 us (788), 122 x 130->200 163-171 us (145), 45 x 257->384 of rank 33 262 us (251).
// Where weights stream (large K times M) every tile reads them again: 32 x 2048->1024 1207 us, 1760
// at an odd pitch, 1726 with adapters of rank 16; 64 x 256->2048 683.  DRAM is busy 73% of a short run of
// 64 x 784->128 (its bytes are the algorithm's), the tensor pipe 34%.
//
// Adapters: the low-rank pair rides on the same pass over X.  While the K loop accumulates
// C = W X it also accumulates the transposed low product  L^T = X^T A^T  (the X tile as the M = 128
// operand, A's rows as N: 46 cycles a step of 32 against 64 for the main product; A as a padded M
// operand would take 64 for any rank).  The epilogue warps add up the limbs of t = A X mod 2^64
// across lanes, write t's bytes to shared memory as the next MN-major operand, and a short MMA makes
// D = B t.  y = (C << s) + D.  X is read once; t never leaves the SM.  C, L^T and D of two tiles
// fill the 512 TMEM columns at 16 words (32 words with one accumulator: 45 x 257->384 263 -> 388 us).
// MMAs that narrow (N = 128) read 8 KB of shared memory in their 64 cycles, and a step of 32 also has 46
// of L^T and about 36 of writing X and A, which makes shared memory busy for half the time of 64 x
// 784->128 (202 us: DRAM 57%, tensor pipe 31%); the rest is waiting, for X or for t.
//
// Rows that start 16-byte aligned (an even pitch) move by TMA straight into the operand layout, and
// results leave by TMA.  Other rows (contiguous [count][kN+1] ciphertexts) are off by one word
// every other row, which no tiled load can shift: they land unshifted in a ring of raw slots, and
// four warps copy them word by word into the operand layout.  (8-byte cp.async into place, without
// the ring and the copy, is slower: 256 x 784->128 760 -> 1024 us at its best.)
#include <algorithm>
#include <atomic>
#include <type_traits>

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
constexpr int RQ_WK = 128;      // K per weight slot
constexpr int RQ_KSTEP = 32;    // K per MMA; a ragged K costs at most 31 rows
constexpr int RQ_W_SLOT = RQ_BM * RQ_WK;               // 16 KB
constexpr int RQ_EPI_WARPS = 8;                        // two per TMEM lane quarter
constexpr int RQ_COPY_WARPS = 4;                       // each copies every fourth raw slot
constexpr int RQ_B_SLOTS = 2;
constexpr int RQ_MAX_W = 13, RQ_MAX_X = 13, RQ_MAX_RAW = 16;  // most slots of each ring
constexpr int RQ_LISTS = 2;                            // lists of groups, each
constexpr int RQ_LIST = 32;                            // one round of a warp long
constexpr int RQ_BARS = 2 * (RQ_MAX_W + RQ_MAX_X + RQ_MAX_RAW + RQ_B_SLOTS + RQ_LISTS) + 7;
// the barriers, two words, the lists' lengths, the lists
constexpr int RQ_LIST_AT = (8 * RQ_BARS + 16 + 4 * RQ_LISTS + 15) / 16 * 16;
constexpr int RQ_BAR_BYTES = (RQ_LIST_AT + 16 * RQ_LISTS * RQ_LIST + 127) / 128 * 128;
constexpr int RQ_SMEM = 227 * 1024;                    // of one block
constexpr uint32_t RQ_WAIT_LIMIT = 1u << 24;

template <bool SHIFTED, bool ADAPT>
struct RqShape {
  static constexpr int WORDS = ADAPT ? 16 : 32;        // words per tile
  static constexpr int BN = 8 * WORDS;                 // limb columns per tile
  static constexpr int BOXES = BN / 128;               // swizzle spans per X row
  static constexpr int XK = ADAPT ? 128 : 64;          // K per X slot
  static constexpr int X_SLOT = XK * BN;               // 16 KB
  static constexpr int RAW_PITCH = BN + 16;            // one word of shift, to 16 bytes
  static constexpr int RAW_ROWS = ADAPT ? 64 : 32;     // rows per raw slot, half of each parity
  static constexpr int RAW_SLOT = RAW_ROWS * RAW_PITCH;
  static constexpr int EW = WORDS / 2;                 // words per epilogue warp
  static constexpr int OUT = 32 * EW * 8;              // its staging: 32 rows
  static constexpr bool MAY_SPLIT = !SHIFTED;          // which may be done in two parts
  static constexpr int COPY = SHIFTED ? RQ_COPY_WARPS : 0;
  static constexpr int MMA_WARP = 2 + COPY;            // warp 0 loads X, warp 1 the weights
  static constexpr int MMA_WARPS = SHIFTED && ADAPT ? 1 : 2;  // two: one per accumulator
  static constexpr int LOW_WARP = MMA_WARP + MMA_WARPS;       // adapters: L^T = X^T A^T and D = B t
  static constexpr int LOW_WARPS = !ADAPT ? 0 : SHIFTED ? 1 : 2;  // (16 warps are all that fit)
  static constexpr int EPI_WARP = LOW_WARP + LOW_WARPS;
  static constexpr int THREADS = 32 * (EPI_WARP + RQ_EPI_WARPS);
};

struct RqMaps {
  CUtensorMap W, A, B, Y;
  CUtensorMap X[2];  // aligned: boxes of one slot's and of 32 rows; shifted: rows 0, 2, .. and 1, 3, ..
};

struct RqArgs {
  uint64_t* Y;
  const int64_t* bias;
  const int32_t* row_choice;  // the choice of each row (experts)
  const int32_t* which;       // expert or adapter of each row
  uint64_t delta;
  int rows, top_k, choices, n_which;  // top_k = 0: row n reads X row group n
  int M, K, L, ldy;
  int shift, rank, rank16;    // adapters
  int b_row;                  // bytes of B's rows in shared memory: one swizzle span, 32 or 64
  int off0, off1;             // words by which rows 0, 2, .. / 1, 3, .. start past 16-byte alignment
  int w_rows;                 // weight rows per load
  int n_tiles, m_tiles, m_group;  // tiles of 128 rows that share one load of X
  int groups;                 // of m_group tiles in one row
  int w_slots, x_slots, raw_slots;
  int out_split;              // results are staged, and leave, in two parts
  int keep_w;                 // the group's weights stay for the next group that uses them
  int x_at, raw_at, a_at, b_at, t_at, out_at, bars_at;  // shared-memory offsets; weights at 0
};

// One group: row n, tiles mg * m_group .. of 128 output rows, tile nt of words.
struct RqGroup {
  int n, mg, nt;
  int src;    // the row's X group
  int w;      // its expert or adapter, -1 when it has no adapter
  bool load;  // its weights are not those of the group before
  bool drop;  // the next group is known to need others
};
// In a list a group is four words: n; src and mg (adapters: mg); w; nt and the two flags.
constexpr int RQ_MG_BITS = 12, RQ_NT_BITS = 30;
constexpr int RQ_LAST = 256;  // in a list's length: no list follows
static_assert(PNB_MAX_CHOICES <= 1 << (32 - RQ_MG_BITS), "a row's token beside its group");

// A block's groups, one grid apart, words fastest.  One warp works them out, a round of 32 at a time,
// without those whose row is skipped; every role reads them from its lists, so that no role has to
// follow the tables, whose loads and branches cost a thread on its own over a thousand cycles a
// tile, more than the MMAs of a short K take.
template <bool ADAPT>
struct RqLister {
  int done = 0;                  // rounds
  int last_w = -2, last_mg = -1;  // of the last group listed
  // The next list: its groups go to `to`; returns its length, with RQ_LAST when it is the last.
  __device__ __forceinline__ int fill(const RqArgs& a, int lane, uint4* to) {
    const long long total = (long long)a.rows * a.groups * a.n_tiles;
    const unsigned per_row = (unsigned)(a.groups * a.n_tiles);
    for (;;) {
      const long long t = blockIdx.x + ((long long)done * 32 + lane) * gridDim.x;
      ++done;
      const bool last = blockIdx.x + (long long)done * 32 * gridDim.x >= total;
      int n = 0, mg = 0, nt = 0, w = -1, src = 0;
      bool used = t < total;
      if (used) {
        // 32-bit divisions wherever the numbers allow
        n = total <= 0xffffffffll ? (int)((unsigned)t / per_row) : (int)(t / per_row);
        const unsigned r = (unsigned)(t - (long long)n * per_row);
        mg = (int)(r / (unsigned)a.n_tiles);
        nt = (int)(r - (unsigned)(mg * a.n_tiles));
        w = __ldg(a.which + n);
        if (w < 0 || w >= a.n_which) w = -1;
        src = n;
        if (!ADAPT) {
          const int c = __ldg(a.row_choice + n);
          used = w >= 0 && c >= 0 && c < a.choices;
          if (a.top_k > 0) src = c / a.top_k;
        }
      }
      const unsigned mask = __ballot_sync(0xffffffffu, used);
      if (mask == 0 && !last) continue;
      const unsigned below = mask & ((1u << lane) - 1u), above = mask & ~(2u * (1u << lane) - 1u);
      const int before = below ? 31 - __clz(below) : lane, after = above ? __ffs(above) - 1 : lane;
      const int w0 = __shfl_sync(0xffffffffu, w, before), mg0 = __shfl_sync(0xffffffffu, mg, before);
      const int w1 = __shfl_sync(0xffffffffu, w, after), mg1 = __shfl_sync(0xffffffffu, mg, after);
      // same weights: the tile rows, and for experts the expert, are the same
      const bool load = !a.keep_w || (below ? mg0 != mg || (!ADAPT && w0 != w)
                                            : last_mg != mg || (!ADAPT && last_w != w));
      const bool drop = !a.keep_w || (above && (mg1 != mg || (!ADAPT && w1 != w)));
      if (used)
        to[__popc(below)] = make_uint4(
            (unsigned)n, ADAPT ? (unsigned)mg : (unsigned)src << RQ_MG_BITS | (unsigned)mg, (unsigned)w,
            (unsigned)nt | (load ? 1u << RQ_NT_BITS : 0u) | (drop ? 2u << RQ_NT_BITS : 0u));
      if (mask) {
        const int end = 31 - __clz(mask);
        last_w = __shfl_sync(0xffffffffu, w, end);
        last_mg = __shfl_sync(0xffffffffu, mg, end);
      }
      return __popc(mask) | (last ? RQ_LAST : 0);
    }
  }
  static __device__ __forceinline__ RqGroup read(const uint4* from) {
    const uint4 e = *from;
    RqGroup g;
    g.n = (int)e.x;
    g.src = ADAPT ? (int)e.x : (int)(e.y >> RQ_MG_BITS);
    g.mg = ADAPT ? (int)e.y : (int)(e.y & ((1u << RQ_MG_BITS) - 1u));
    g.w = (int)e.z;
    g.nt = (int)(e.w & ((1u << RQ_NT_BITS) - 1u));
    g.load = e.w >> RQ_NT_BITS & 1u;
    g.drop = e.w >> RQ_NT_BITS & 2u;
    return g;
  }
};

// A ring of slots: the current one and the parity of its use.
struct RqRing {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int slots) {
    if (++slot == slots) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// Bounded wait that also gives up as soon as another role has flagged an abort.  A completed phase
// is found by the plain test: 145 cycles against a suspending wait's 186, which the thread that
// issues the MMAs pays at every slot.  The rest is out of line: the roles' loops
// share the instruction cache, and a thread on its own runs at the pace of its fetches.
__device__ __noinline__ bool rq_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_s) {
  for (uint32_t it = 0; it < RQ_WAIT_LIMIT; it += 1024) {
    if (tc::mbar_wait(bar, parity, 1024)) return true;
    if (*abort_s) return false;
  }
  *abort_s = 1;
  atomicExch(&g_rq_status, 1);
  return false;
}
__device__ __forceinline__ bool rq_wait(uint32_t bar, uint32_t parity, volatile int* abort_s) {
  return tc::mbar_test(bar, parity & 1u) || rq_wait_slow(bar, parity & 1u, abort_s);
}

// No load may still be landing when the block exits: the last use of each slot completes when it has
// landed (bounded; immediate unless a wait ran out).  `bars` are the ring's full barriers.
__device__ __forceinline__ void rq_drain(uint32_t bars, RqRing ring, bool wrapped, int slots) {
  for (int i = 0; i < slots; ++i)
    if (i < ring.slot)
      (void)tc::mbar_wait(bars + 8u * i, ring.phase, RQ_WAIT_LIMIT);
    else if (wrapped)
      (void)tc::mbar_wait(bars + 8u * i, ring.phase ^ 1u, RQ_WAIT_LIMIT);
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

template <bool SHIFTED, bool ADAPT, bool SPLIT>
__global__ void __launch_bounds__(RqShape<SHIFTED, ADAPT>::THREADS, 1)
    request_kernel(const __grid_constant__ RqMaps tm, const __grid_constant__ RqArgs a) {
  using S = RqShape<SHIFTED, ADAPT>;
  // the swizzles want 1024-byte boundaries; aligning by hand instead would cost 1 KB
  extern __shared__ __align__(1024) unsigned char rq_raw[];
  const uint32_t raw = tc::smem_u32(rq_raw), base = raw;
  if (raw & 1023u) {
    if (threadIdx.x == 0) atomicExch(&g_rq_status, 1);
    return;
  }
  const int a_slot = a.rank16 * RQ_WK;  // A's rows beside one X slot
  const int b_slot = RQ_BM * a.b_row;
  auto w_at = [&](int s) { return base + (uint32_t)(s * RQ_W_SLOT); };
  auto x_at = [&](int s) { return base + (uint32_t)(a.x_at + s * S::X_SLOT); };
  auto raw_at = [&](int s) { return base + (uint32_t)(a.raw_at + s * S::RAW_SLOT); };
  auto a_at = [&](int s) { return base + (uint32_t)(a.a_at + s * a_slot); };
  auto b_at = [&](int s) { return base + (uint32_t)(a.b_at + s * b_slot); };
  const uint32_t t_at = base + (uint32_t)a.t_at;
  const uint32_t bars = base + (uint32_t)a.bars_at;
  constexpr int W0 = 0, X0 = 2 * RQ_MAX_W, R0 = X0 + 2 * RQ_MAX_X, B0 = R0 + 2 * RQ_MAX_RAW,
                L0 = B0 + 2 * RQ_B_SLOTS, C0 = L0 + 2 * RQ_LISTS;
  const uint32_t w_full = bars + 8 * W0, w_empty = w_full + 8 * RQ_MAX_W;
  const uint32_t x_full = bars + 8 * X0, x_empty = x_full + 8 * RQ_MAX_X;
  const uint32_t r_full = bars + 8 * R0, r_empty = r_full + 8 * RQ_MAX_RAW;
  const uint32_t b_full = bars + 8 * B0, b_empty = b_full + 8 * RQ_B_SLOTS;
  const uint32_t list_full = bars + 8 * L0, list_empty = list_full + 8 * RQ_LISTS;
  const uint32_t acc_full = bars + 8 * C0, acc_empty = acc_full + 16;
  const uint32_t low_full = acc_full + 32, t_full = acc_full + 48;
  const uint32_t holder = bars + 8 * RQ_BARS;
  volatile int* abort_s = reinterpret_cast<volatile int*>(rq_raw + (holder + 8 - raw));
  volatile int* list_n = abort_s + 1;
  uint4* lists = reinterpret_cast<uint4*>(rq_raw + (bars - raw) + RQ_LIST_AT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // adapters with one tile to a group: the second warp's answers cost more than its share gains
  // (256 x 784->128 of rank 16: 937 -> 957 us; with four tiles, 64 x 512->512, it is 512 -> 484)
  const int mma_warps = ADAPT && a.m_group == 1 ? 1 : S::MMA_WARPS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.w_slots; ++s) {
      tc::mbar_init(w_full + 8 * s, 1);
      tc::mbar_init(w_empty + 8 * s, mma_warps);
    }
    for (int s = 0; s < a.x_slots; ++s) {
      tc::mbar_init(x_full + 8 * s, SHIFTED ? S::COPY + (ADAPT ? 1 : 0) : 1);
      tc::mbar_init(x_empty + 8 * s, mma_warps + (ADAPT ? 1 : 0));
    }
    for (int s = 0; s < a.raw_slots; ++s) {
      tc::mbar_init(r_full + 8 * s, 1);
      tc::mbar_init(r_empty + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(b_full + 8 * s, 1);
      tc::mbar_init(b_empty + 8 * s, 1);
      tc::mbar_init(acc_full + 8 * s, 1 + S::LOW_WARPS);
      tc::mbar_init(acc_empty + 8 * s, RQ_EPI_WARPS);
      tc::mbar_init(low_full + 8 * s, 1);
      tc::mbar_init(list_full + 8 * s, 1);
      tc::mbar_init(list_empty + 8 * s, S::THREADS / 32);
    }
    tc::mbar_init(t_full, RQ_EPI_WARPS);
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
  // what came before in the stream is done from here on (rq_pad_kernel lets this one start early)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(rq_raw + (holder - raw));

  constexpr uint32_t D_AT = 256;               // adapters: TMEM columns of L^T and D
  const int kb_n = (a.K + RQ_WK - 1) / RQ_WK;  // weight slots of one tile
  const int kx_n = (a.K + S::XK - 1) / S::XK;  // X slots of one tile
  // rows of X slot kx, rounded up to whole MMAs.  Those past K belong to the next group (or lie past
  // the tensor and read as zeros) and meet zero weights.
  auto x_rows = [&](int kx) {
    return min(S::XK, (a.K - kx * S::XK + RQ_KSTEP - 1) / RQ_KSTEP * RQ_KSTEP);
  };
  auto tiles = [&](int mg) { return min(a.m_group, a.m_tiles - mg * a.m_group); };
  // body(group) for every group of the block, until it returns false; a lane on its own, or the first
  // of a warp that goes together, says when a list has been read
  auto each = [&](bool alone, auto&& body) {
    for (int c = 0;; ++c) {
      const int l = c % RQ_LISTS;
      if (!rq_wait(list_full + 8 * l, (uint32_t)(c / RQ_LISTS), abort_s)) return;
      const int n = list_n[l];
      for (int j = 0; j < (n & (RQ_LAST - 1)); ++j)
        if (!body(RqLister<ADAPT>::read(lists + l * RQ_LIST + j))) return;
      if (n & RQ_LAST) return;
      if (!alone) __syncwarp();
      if (lane == 0) tc::mbar_arrive(list_empty + 8 * l);
    }
  };

  if (warp == 0) {
    // ---------------- X loads (one lane) ---------------------------------------------------------
    if (lane == 0) {
      RqRing ring;
      bool wrapped = false;
      const int slots = SHIFTED ? a.raw_slots : a.x_slots;
      each(true, [&](const RqGroup& g) {
        const bool has = ADAPT && g.w >= 0;
        for (int k = 0; k < a.K; k += SHIFTED ? S::RAW_ROWS : S::XK) {
          const int s = ring.slot;
          const uint32_t full = (SHIFTED ? r_full : x_full) + 8 * s;
          if (!rq_wait((SHIFTED ? r_empty : x_empty) + 8 * s, ring.phase ^ 1u, abort_s)) return false;
          const int row = g.src * a.K + k;
          if (SHIFTED) {
            tc::mbar_expect_tx(full, S::RAW_SLOT);  // the rows of either parity, in order
            tc::tma_load_2d(raw_at(s), &tm.X[row & 1], g.nt * S::WORDS, row >> 1, full);
            tc::tma_load_2d(raw_at(s) + S::RAW_SLOT / 2, &tm.X[(row + 1) & 1], g.nt * S::WORDS,
                            (row + 1) >> 1, full);
          } else {
            const int rows = x_rows(k / S::XK);
            const CUtensorMap* map = rows == S::XK ? &tm.X[0] : &tm.X[1];
            const int box = rows == S::XK ? S::XK : RQ_KSTEP;
            tc::mbar_expect_tx(full, (uint32_t)(rows * S::BN + (has ? a_slot : 0)));
            for (int r = 0; r < rows; r += box)
#pragma unroll
              for (int b = 0; b < S::BOXES; ++b)
                tc::tma_load_2d(x_at(s) + (b * S::XK + r) * 128, map, g.nt * S::BN + b * 128, row + r,
                                full);
            if (has) tc::tma_load_2d(a_at(s), &tm.A, k, g.w * a.rank, full);
          }
          ring.advance(slots);
          wrapped |= ring.slot == 0;
        }
        return true;
      });
      rq_drain(SHIFTED ? r_full : x_full, ring, wrapped, slots);
    }
  } else if (warp == 1) {
    // ---------------- the lists (the warp) and weight loads (one lane) ---------------------------
    RqRing br;
    bool b_wrap = false, ok = true;
    int w_slot = 0;
    uint32_t w_par = 0, w_used = 0;  // a bit per slot
    auto load = [&](const RqGroup& g) {
      const bool has = ADAPT && g.w >= 0;
      const int m_n = tiles(g.mg);
      if (a.keep_w) w_slot = 0;
      for (int m = 0; m < m_n; ++m) {
        const int m_row = (g.mg * a.m_group + m) * RQ_BM;
        for (int kb = 0; kb < kb_n && g.load; ++kb) {
          const int s = w_slot;
          if (!rq_wait(w_empty + 8 * s, (w_par >> s) ^ 1u, abort_s)) return false;
          tc::mbar_expect_tx(w_full + 8 * s, (uint32_t)(a.w_rows * RQ_WK));
          tc::tma_load_2d(w_at(s), &tm.W, kb * RQ_WK, (ADAPT ? 0 : g.w * a.M) + m_row,
                          w_full + 8 * s);
          w_par ^= 1u << s;
          w_used |= 1u << s;
          if (++w_slot == a.w_slots) w_slot = 0;
        }
        if (has) {
          const int s = br.slot;
          if (!rq_wait(b_empty + 8 * s, br.phase ^ 1u, abort_s)) return false;
          tc::mbar_expect_tx(b_full + 8 * s, (uint32_t)b_slot);
          tc::tma_load_2d(b_at(s), &tm.B, 0, g.w * a.M + m_row, b_full + 8 * s);
          br.advance(RQ_B_SLOTS);
          b_wrap |= br.slot == 0;
        }
      }
      return true;
    };
    RqLister<ADAPT> lister;
    auto list = [&](int c) {  // list c, once its place has been read by every warp
      const int l = c % RQ_LISTS;
      if (!__all_sync(0xffffffffu,
                      rq_wait(list_empty + 8 * l, (uint32_t)(c / RQ_LISTS) ^ 1u, abort_s)))
        return 0;
      const int n = lister.fill(a, lane, lists + l * RQ_LIST);
      if (lane == 0) list_n[l] = n;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(list_full + 8 * l);
      return n;
    };
    for (int c = 0, n = list(0), next = 0;; ++c, n = next) {
      // the next list is made a few groups into this one, when the other warps have left the last
      const int count = n & (RQ_LAST - 1), early = min(8, count);
      const uint4* from = lists + c % RQ_LISTS * RQ_LIST;
      if (lane == 0)
        for (int j = 0; j < early && ok; ++j) ok = load(RqLister<ADAPT>::read(from + j));
      if (!(n & RQ_LAST)) next = list(c + 1);
      if (lane == 0)
        for (int j = early; j < count && ok; ++j) ok = load(RqLister<ADAPT>::read(from + j));
      if ((n & RQ_LAST) || !__all_sync(0xffffffffu, ok && !*abort_s)) break;
      if (lane == 0) tc::mbar_arrive(list_empty + 8 * (c % RQ_LISTS));
    }
    if (lane == 0) {
      for (int s = 0; s < a.w_slots; ++s)
        if ((w_used >> s) & 1u)
          (void)tc::mbar_wait(w_full + 8 * s, ((w_par >> s) ^ 1u) & 1u, RQ_WAIT_LIMIT);
      if (ADAPT) rq_drain(b_full, br, b_wrap, RQ_B_SLOTS);
    }
  } else if (warp < S::MMA_WARP) {
    // ---------------- raw rows -> operand layout (shifted rows only) -----------------------------
    // Raw slot r is always copied by warp r % 4 (their number is a multiple of 4).  Every warp waits
    // for every X slot's turn and answers it, also where it copies nothing: a parity tells only
    // neighbouring turns apart, so the slot must not be filled and used again before a warp has seen
    // its turn.  (An idle warp answers early, so this costs nothing that shows: 122 x 130->200 163 us
    // either way, 45 x 257->384 of rank 33 262.)
    const int cw = warp - 2;
    constexpr int PER = 32 / S::WORDS;  // rows per pass of a warp
    constexpr int BATCH = 16;           // passes whose words are on their way together
    const int word = lane % S::WORDS, sub = lane / S::WORDS;
    const int box = word >> 4, ch = (word & 15) >> 1, half = word & 1;
    RqRing xr, rr;
    bool x_wrap = false;
    each(false, [&](const RqGroup& g) {
      const int w = g.w;
      const int parity = g.src * a.K & 1;  // of the group's first row (slots hold an even number)
      const int off_e = parity ? a.off1 : a.off0, off_o = parity ? a.off0 : a.off1;
      for (int kx = 0; kx < kx_n; ++kx) {
        if (!rq_wait(x_empty + 8 * xr.slot, xr.phase ^ 1u, abort_s)) return false;
        const uint32_t full = x_full + 8 * xr.slot;
        if (ADAPT && cw == 0 && lane == 0) {  // A's rows beside the slot
          tc::mbar_expect_tx(full, w >= 0 ? (uint32_t)a_slot : 0u);
          if (w >= 0) tc::tma_load_2d(a_at(xr.slot), &tm.A, kx * S::XK, w * a.rank, full);
        }
        const int raws = (x_rows(kx) + S::RAW_ROWS - 1) / S::RAW_ROWS;
        for (int i = 0; i < raws; ++i) {
          if ((rr.slot & 3) == cw) {
            if (!rq_wait(r_full + 8 * rr.slot, rr.phase, abort_s)) return false;
            // row r of the slot: its parity's half, r / 2; one word further where it is shifted
            const unsigned char* from = rq_raw + (raw_at(rr.slot) - raw) + word * 8;
            unsigned char* to = rq_raw + (x_at(xr.slot) - raw) + box * (S::XK * 128) +
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
        if (lane == 0) tc::mbar_arrive(full);  // its words are in place, if it had any
        xr.advance(a.x_slots);
        x_wrap |= xr.slot == 0;
      }
      return true;
    });
    if (ADAPT && cw == 0 && lane == 0) rq_drain(x_full, xr, x_wrap, a.x_slots);
  } else if (warp < S::MMA_WARP + S::MMA_WARPS) {
    // ---------------- main products (one lane of each warp) --------------------------------------
    // Tiles alternate between two warps, each with an accumulator of its own: waiting for a slot,
    // issuing its MMAs and letting it go takes a thread longer than the tensor cores take to run
    // them, the more so between tiles, so one thread's bookkeeping hides behind the other's MMAs
    // (64 x 512->512 350 -> 335 us, 122 x 130->200 154 -> 144).  Either answers for every slot, also
    // those of tiles that are not its own: a parity tells only neighbouring uses apart.  (Adapters
    // at odd pitches have no warp left for it: 16 are all that get 128 registers a thread.)
    if (lane == 0) {
      constexpr uint32_t MAIN = tc::idesc_i8(RQ_BM, S::BN, true, false, false, true);
      constexpr int STEPS = S::XK / RQ_KSTEP;
      constexpr int W_STEPS = RQ_WK / RQ_KSTEP;
      const uint64_t wd = tc::smem_desc_sw128(w_at(0), 16u, 1024u);
      const uint64_t xd = tc::smem_desc_sw128(x_at(0), S::XK * 128u, 1024u);
      const uint32_t w_hi = (uint32_t)(wd >> 32), x_hi = (uint32_t)(xd >> 32);
      const int steps = (a.K + RQ_KSTEP - 1) / RQ_KSTEP;  // MMAs of one tile
      const int x_slots = a.x_slots, w_slots = a.w_slots;
      const bool keep_w = a.keep_w != 0;
      const int me = warp - S::MMA_WARP;
      RqRing x;
      int w_slot = 0;
      uint32_t w_par = 0;
      int tt = 0;  // tiles of this warp
      const bool turns = mma_warps == 2;
      bool mine = me == 0;  // the next tile
      int unreleased = 0;   // weight slots kept for a group that has not come
      // One tile.  Those whose weights are there and stay (kept), whose X nobody else uses (alone), and
      // both, are compiled apart, without the branches that ask.
      using yes = std::true_type;
      using no = std::false_type;
      auto tile = [&](auto kept, auto alone, bool load, bool drop, bool first, bool last) {
        if (kept) load = drop = false;
        if (alone) first = last = true;
        const int buf = turns ? me : tt & 1;
        const uint32_t c_tmem = tmem + (uint32_t)(buf * S::BN);
        if (!rq_wait(acc_empty + 8 * buf, (uint32_t)(turns ? tt : tt >> 1) ^ 1u, abort_s))
          return false;
        ++tt;
        tc::tc_fence_after();  // (operands in shared memory need none: their mbarriers order them)
        uint32_t acc = 0;
        auto slot = [&](uint32_t w_lo, int n, bool whole) {  // n MMAs of one X slot
          if (first && !rq_wait(x_full + 8 * x.slot, x.phase, abort_s)) return false;
          const uint32_t x_lo = (uint32_t)xd + (uint32_t)(x.slot * (S::X_SLOT / 16));
#pragma unroll
          for (int k = 0; k < STEPS; ++k)
            if (whole || k < n)
              tc::mma_i8_lo(c_tmem, w_lo + 2 * k, w_hi, x_lo + 256 * k, x_hi, MAIN, k ? 1u : acc);
          acc = 1;
          if (last) tc::mma_commit(x_empty + 8 * x.slot);
          x.advance(x_slots);
          return true;
        };
        for (int left = steps; left > 0; left -= W_STEPS) {  // one weight slot: 128 of K
          if (load) {
            if (!rq_wait(w_full + 8 * w_slot, w_par >> w_slot, abort_s)) return false;
            w_par ^= 1u << w_slot;
          }
          const uint32_t w_lo = (uint32_t)wd + (uint32_t)(w_slot * (RQ_W_SLOT / 16));
          if (left >= W_STEPS) {
#pragma unroll
            for (int h = 0; h < W_STEPS; h += STEPS)
              if (!slot(w_lo + 2 * h, STEPS, true)) return false;
          } else {
            for (int h = 0; h < left; h += STEPS)
              if (!slot(w_lo + 2 * h, left - h, false)) return false;
          }
          if (drop) tc::mma_commit(w_empty + 8 * w_slot);
          if (++w_slot == w_slots) w_slot = 0;
        }
        tc::mma_commit(acc_full + 8 * buf);
        return true;
      };
      // A tile of the other warp: its weight slots, and (alone) its X slots, in its order.
      auto skip = [&](bool load, bool drop, bool alone) {
        for (int left = steps; left > 0; left -= W_STEPS) {
          if (load) {
            if (!rq_wait(w_full + 8 * w_slot, w_par >> w_slot, abort_s)) return false;
            w_par ^= 1u << w_slot;
          }
          if (drop) {
            if (keep_w)
              tc::mma_commit(w_empty + 8 * w_slot);  // earlier groups' MMAs may still read it
            else
              tc::mbar_arrive(w_empty + 8 * w_slot);
          }
          if (++w_slot == w_slots) w_slot = 0;
          if (!alone) continue;
          for (int h = 0; h < left && h < W_STEPS; h += STEPS) {
            if (!rq_wait(x_full + 8 * x.slot, x.phase, abort_s)) return false;
            tc::mbar_arrive(x_empty + 8 * x.slot);
            x.advance(x_slots);
          }
        }
        return true;
      };
      each(true, [&](const RqGroup& g) {
        if (me >= mma_warps) return true;
        const int m_n = tiles(g.mg);
        if (g.load)
          for (int s = 0; s < unreleased; ++s) tc::mma_commit(w_empty + 8 * s);
        // weights are let go with their last use when the next group is known to need others
        unreleased = g.drop ? 0 : m_n * kb_n;
        if (keep_w) w_slot = 0;
        const bool kept = !g.load && !g.drop;
        const bool own = mine;
        if (turns && (m_n & 1)) mine = !mine;
        if (m_n == 1)
          return !own   ? skip(g.load, g.drop, true)
                 : kept ? tile(yes{}, yes{}, false, false, true, true)
                        : tile(no{}, yes{}, g.load, g.drop, true, true);
        const RqRing x0 = x;
        const int m0 = own ? 0 : 1;
        for (int m = 0; m < m_n; ++m) {
          if (turns && ((m ^ m0) & 1)) {
            if (!skip(g.load, g.drop, false)) return false;
            continue;
          }
          x = x0;
          const bool first = m == m0, last = m + mma_warps >= m_n;
          if (!(kept ? tile(yes{}, no{}, false, false, first, last)
                     : tile(no{}, no{}, g.load, g.drop, first, last)))
            return false;
        }
        return true;
      });
    }
  } else if (ADAPT && warp < S::LOW_WARP + S::LOW_WARPS) {
    // ---------------- low products L^T = X^T A^T and D = B t (one lane of each warp) --------------
    // Two warps, or one that does both and looks for t between its slots: D waits for the epilogue's
    // t, and a thread that waits for it issues no L^T for the next group (256 x 784->128 of rank 16:
    // 943 us with one, 908 with two).
    if (lane == 0) {
      constexpr uint32_t MAIN = tc::idesc_i8(RQ_BM, S::BN, true, false, false, true);
      const bool low = warp == S::LOW_WARP, d = warp == S::LOW_WARP + S::LOW_WARPS - 1;
      const uint32_t LOW = tc::idesc_i8(128, a.rank16, false, true, true, false);
      const uint64_t xd = tc::smem_desc_sw128(x_at(0), S::XK * 128u, 1024u);
      const uint64_t ad = tc::smem_desc_sw128(a_at(0), 16u, 1024u);
      const uint32_t x_hi = (uint32_t)(xd >> 32), a_hi = (uint32_t)(ad >> 32);
      const int steps = (a.K + RQ_KSTEP - 1) / RQ_KSTEP;
      RqRing x, br;
      int tt = 0;
      uint32_t t_par = 0;
      int pending = -1;  // the accumulator whose t and D are still to come
      auto product = [&](int buf) {  // D = B t
        if (!rq_wait(b_full + 8 * br.slot, br.phase, abort_s)) return false;
        tc::tc_fence_after();
        // columns of B past the rank are zero, so t's rows past it do not matter
        for (int k = 0; k < (a.rank + 31) / 32; ++k)
          tc::mma_i8(tmem + D_AT + (uint32_t)(buf * 128),
                     a.b_row == 32 ? tc::smem_desc_sw32(b_at(br.slot), 16u, 256u)
                                   : tc::smem_desc_sw64(b_at(br.slot) + 32u * k, 16u, 512u),
                     tc::smem_desc_sw128(t_at + 4096u * k, 16u, 1024u), MAIN, k != 0 ? 1u : 0u);
        tc::mma_commit(b_empty + 8 * br.slot);
        tc::mma_commit(acc_full + 8 * buf);
        br.advance(RQ_B_SLOTS);
        return true;
      };
      auto finish = [&](bool block) {  // the pending D, once t is there
        if (pending < 0) return true;
        if (block) {
          if (!rq_wait(t_full, t_par, abort_s)) return false;
        } else if (!tc::mbar_test(t_full, t_par & 1u)) {
          return true;
        }
        t_par ^= 1u;
        const int buf = pending;
        pending = -1;
        return product(buf);
      };
      each(true, [&](const RqGroup& g) {
        const bool has = g.w >= 0;
        const int m_n = tiles(g.mg);
        for (int m = 0; m < m_n; ++m, ++tt) {
          // Every tile's turn is waited for and answered, also where nothing is issued: a parity
          // tells only neighbouring turns apart, so no role may get two turns ahead of another.  The
          // warp of D answers when D is there; that of L^T, whose products have a barrier of their
          // own, at once.
          const int buf = tt & 1;
          if (!rq_wait(acc_empty + 8 * buf, (uint32_t)(tt >> 1) ^ 1u, abort_s)) return false;
          tc::tc_fence_after();
          if (!d) tc::mbar_arrive(acc_full + 8 * buf);
          if (m > 0 && !finish(true)) return false;
          if (low && m == 0) {
            const uint32_t l_tmem = tmem + D_AT + (uint32_t)(buf * 128);
            uint32_t acc = 0;
            for (int left = steps; left > 0; left -= S::XK / RQ_KSTEP) {
              if (!rq_wait(x_full + 8 * x.slot, x.phase, abort_s)) return false;
              if (has) {
                const uint32_t x_lo = (uint32_t)xd + (uint32_t)(x.slot * (S::X_SLOT / 16));
                const uint32_t a_lo = (uint32_t)ad + (uint32_t)(x.slot * (a_slot / 16));
#pragma unroll
                for (int k = 0; k < S::XK / RQ_KSTEP; ++k)
                  if (k < left)
                    tc::mma_i8_lo(l_tmem, x_lo + 256 * k, x_hi, a_lo + 2 * k, a_hi, LOW,
                                  k > 0 ? 1u : acc);
                acc = 1;
                tc::mma_commit(x_empty + 8 * x.slot);
              } else {
                tc::mbar_arrive(x_empty + 8 * x.slot);
              }
              x.advance(a.x_slots);
              if (!finish(false)) return false;
            }
            if (!finish(true)) return false;
            if (has) tc::mma_commit(low_full + 8 * buf);
          }
          if (!d) continue;
          if (!has) {
            tc::mbar_arrive(acc_full + 8 * buf);
          } else if (m > 0) {
            if (!product(buf)) return false;
          } else {
            pending = buf;
            if (!low && !finish(true)) return false;
          }
        }
        return true;
      });
      (void)finish(true);
    }
  } else {
    // ---------------- epilogue -------------------------------------------------------------------
    // Warp w reads TMEM lane quarter w % 4 (32 output rows, one per lane) and half eh of the tile's
    // words.  Limb sums become u64 words, staged in shared memory with their 16-byte chunks XORed by
    // the row, and leave as 32 rows x EW words by TMA, or as row segments by plain stores.
    const int e_w = warp - S::EPI_WARP;
    const int q = warp & 3, eh = e_w >> 2;
    // Adapters read two accumulators, so half the words of each at a time: both are then on their way
    // together, and nothing spills (256 x 784->128 of rank 16 892 -> 879 us, 45 x 257->384 267 -> 259;
    // several tiles to a group at an even pitch lose 3%).
    constexpr int EW = S::EW, CW = ADAPT ? 2 : 4, CHUNKS = EW / CW, COLS = 8 * CW;
    auto tmem_ld = [](uint32_t at, uint32_t (&r)[COLS]) {
      if constexpr (COLS == 16)
        tc::tmem_ld_32x32_x16(at, r);
      else
        tc::tmem_ld_32x32_nowait(at, r);
    };
    constexpr int PARTS = SPLIT ? 2 : 1, PITCH = EW * 8 / PARTS;  // staged one after the other
    const uint32_t out_at = base + (uint32_t)(a.out_at + e_w * (S::OUT / PARTS));
    unsigned char* out = rq_raw + (out_at - raw);
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    auto xored = [](int row) {  // its swizzle
      return PITCH == 128 ? row & 7 : PITCH == 64 ? (row >> 1) & 3 : (row >> 2) & 1;
    };
    unsigned char* out_row = out + lane * PITCH;
    const int out_x = xored(lane);
    int tt = 0;
    uint32_t low_par = 0;  // a bit per accumulator
    bool ok = true;
    each(false, [&](const RqGroup& g) {
      const int w = g.w, mg = g.mg, nt = g.nt;
      const bool has = ADAPT && w >= 0;
      const int m_n = tiles(mg);
      for (int m = 0; m < m_n; ++m, ++tt) {
        const int buf = tt & 1;
        const uint32_t d_tmem = tmem + D_AT + (uint32_t)(buf * 128) + lanes;
        const bool low = has && m == 0;
        if (low) {
          // t = A X: lane l of quarter q holds limb l % 8 of word 4q + l/8 for every rank row.  Eight
          // lanes add up 16 rows at a time, halving the rows they keep at each step.
          ok = rq_wait(low_full + 8 * buf, low_par >> buf, abort_s);
          if (!ok) break;
          tc::tc_fence_after();
          const int word = q * 4 + (lane >> 3);
          for (int r0 = 16 * eh; r0 < a.rank16; r0 += 32) {
            uint32_t c[16];
            tc::tmem_ld_32x32_x16(d_tmem + r0, c);
            tc::tmem_ld_wait_for(c);
            uint64_t v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              v[j] = (uint64_t)(int64_t)(int32_t)c[j] << (8 * (lane & 7));
#pragma unroll
            for (int half = 8; half >= 2; half >>= 1) {
              const bool up = (lane & (half >> 1)) != 0;
#pragma unroll
              for (int j = 0; j < half; ++j) {
                const uint64_t give = up ? v[j] : v[j + half];
                v[j] = (up ? v[j + half] : v[j]) + shfl_xor_u64(give, half >> 1);
              }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int r = r0 + 2 * (lane & 7) + j;
              const uint32_t to = t_at + (r >> 3) * 1024 + (r & 7) * 128 +
                                  (((word >> 1) ^ (r & 7)) << 4) + (word & 1) * 8;
              *reinterpret_cast<uint64_t*>(rq_raw + (to - raw)) = v[j];
            }
          }
          tc::fence_async_smem();
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(t_full);
          low_par ^= 1u << buf;
        }
        const uint32_t c_tmem = tmem + (uint32_t)(buf * S::BN) + lanes + (uint32_t)(eh * EW * 8);
        const int row0 = (mg * a.m_group + m) * RQ_BM + q * 32, col0 = nt * S::WORDS + eh * EW;
        ok = rq_wait(acc_full + 8 * buf, (uint32_t)(tt >> 1), abort_s);
        if (!ok) break;
        tc::tc_fence_after();
        if (row0 >= a.M || col0 >= a.L) {  // nothing of this warp's share is kept
          tc::tc_fence_before();
          if (lane == 0) tc::mbar_arrive(acc_empty + 8 * buf);
          continue;
        }
        // the word of this half that is the body, and its bias
        const int body = a.L - 1 - col0;
        uint64_t bias = 0;
        if (a.bias && body < EW && row0 + lane < a.M)
          bias = (uint64_t)__ldg(a.bias + (ADAPT ? (size_t)0 : (size_t)w * a.M) + row0 + lane) *
                 a.delta;
        // CW words at a time, the next ones' columns on their way while these are added up
        uint32_t c[2][COLS], d[2][COLS];
        auto fetch = [&](int i) {
          tmem_ld(c_tmem + (uint32_t)(i * COLS), c[i & 1]);
          if (has) tmem_ld(d_tmem + (uint32_t)(eh * EW * 8 + i * COLS), d[i & 1]);
        };
        fetch(0);
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
          tc::tmem_ld_wait_for(c[i & 1]);
          if (has) tc::tmem_ld_wait_for(d[i & 1]);
          if (i + 1 < CHUNKS) {
            fetch(i + 1);
          } else {
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(acc_empty + 8 * buf);
          }
          uint64_t y[CW];
#pragma unroll
          for (int u = 0; u < CW; ++u) {
            y[u] = add_limbs(0, c[i & 1] + 8 * u);
            if (ADAPT) y[u] <<= a.shift;
          }
          if (has) {
#pragma unroll
            for (int u = 0; u < CW; ++u) y[u] = add_limbs(y[u], d[i & 1] + 8 * u);
          }
          constexpr int STAGED = CHUNKS / PARTS;
          const int c2 = CW / 2 * (i % STAGED);
          if (!SHIFTED && c2 == 0) {  // what was staged before has left
            if (lane == 0) tc::tma_store_wait_read();
            __syncwarp();
          }
#pragma unroll
          for (int u = 0; u < CW; u += 2)
            *reinterpret_cast<ulonglong2*>(out_row + (((c2 + u / 2) ^ out_x) << 4)) =
                make_ulonglong2(y[u], y[u + 1]);
          if ((i + 1) % STAGED != 0) continue;
          const int w0 = (i + 1 - STAGED) * CW;  // the first staged word
          if (body >= w0 && body < (i + 1) * CW) {
            uint64_t* p = reinterpret_cast<uint64_t*>(
                out_row + ((((body - w0) >> 1) ^ out_x) << 4) + (body & 1) * 8);
            *p += bias;
            // tiled stores end on 16-byte boundaries, so the last word of an odd count goes alone
            if (!SHIFTED && (a.L & 1) && row0 + lane < a.M)
              a.Y[((size_t)g.n * a.M + row0 + lane) * a.ldy + a.L - 1] = *p;
          }
          if (!SHIFTED) {
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0 && col0 + w0 < (a.L & ~1))
              tc::tma_store_3d(&tm.Y, col0 + w0, row0, g.n, out_at);
          }
        }
        if (SHIFTED) {
          __syncwarp();
          constexpr int PER = 32 / EW;  // rows per instruction
          const int wd = lane % EW, sub = lane / EW;
          const unsigned char* from = out + sub * PITCH + (wd & 1) * 8;
          const int ch = (wd >> 1) ^ xored(sub);  // (the rows' other bits join below)
          const int left = col0 + wd < a.L ? a.M - row0 - sub : 0;
          uint64_t* y = a.Y + ((size_t)g.n * a.M + row0 + sub) * a.ldy + col0 + wd;
          // Eight rows' words are read before the first is stored: the compiler keeps the order of loads
          // and stores, and one at a time costs their latency each.  122 x 130->200: 179 -> 167 us,
          // adapters 45 x 257->384: 276 -> 262, 256 x 128->10: 177 -> 153; where the epilogue has time
          // (256 x 784->128: 900 -> 930, 64 x 512->512: 537 -> 555) the bursts hold up the copies of X.
          constexpr int BATCH = 8;
#pragma unroll 1
          for (int b = 0; b < 32; b += BATCH * PER, from += BATCH * PER * PITCH) {
            uint64_t v[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j)
              v[j] = *reinterpret_cast<const uint64_t*>(from + j * PER * PITCH +
                                                        ((ch ^ xored(j * PER)) << 4));
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
              if (b + j * PER < left) *y = v[j];
              y += (size_t)PER * a.ldy;
            }
          }
          __syncwarp();
        }
      }
      return ok;
    });
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
  __host__ __device__ int pitch() const { return (cols + 15) & ~15; }
  bool in_place() const { return cols % 16 == 0 && ((uintptr_t)p % 16) == 0; }
  size_t copy_bytes() const { return (size_t)rows * pitch(); }
};

size_t padded_weight_bytes(const int8_t* W, long long rows, int cols) {
  const RqMatrix m{W, rows, cols};
  return m.in_place() ? 0 : m.copy_bytes();
}

struct RqCopy {
  RqMatrix m[3];
  int8_t* to[3];
  size_t first[4];  // the bytes of copy i are first[i] .. first[i + 1]
};

// Up to three matrices in one launch, 16 bytes (of one row) per thread.
__global__ void rq_pad_kernel(const __grid_constant__ RqCopy c) {
  asm volatile("griddepcontrol.launch_dependents;");
  const size_t i = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * 16;
  if (i >= c.first[3]) return;
  const int w = i >= c.first[2] ? 2 : i >= c.first[1] ? 1 : 0;
  const RqMatrix& m = c.m[w];
  const size_t at = i - c.first[w];
  const int pitch = m.pitch();
  const size_t r = at / pitch;
  const int col = (int)(at - r * pitch);
  const int8_t* from = m.p + r * m.cols + col;
  union { int8_t b[16]; uint4 v; } u;
#pragma unroll
  for (int j = 0; j < 16; ++j) u.b[j] = col + j < m.cols ? from[j] : (int8_t)0;
  *reinterpret_cast<uint4*>(c.to[w] + at) = u.v;
}

// Copies the matrices that TMA cannot read in place to ws, and points them there.
static int rq_place(RqMatrix* (&m)[3], int8_t* ws, cudaStream_t st, bool& placed) {
  RqCopy c{};
  for (int i = 0; i < 3; ++i) {
    c.first[i + 1] = c.first[i];
    if (m[i]->rows == 0 || m[i]->in_place()) continue;
    c.m[i] = *m[i];
    c.to[i] = ws + c.first[i];
    c.first[i + 1] += m[i]->copy_bytes();
    m[i]->p = c.to[i];
  }
  const size_t threads = c.first[3] / 16;
  placed = threads != 0;
  if (!placed) return PNB_OK;
  rq_pad_kernel<<<(unsigned)((threads + 127) / 128), 128, 0, st>>>(c);
  PNB_CHECK_LAUNCH("rq_pad_kernel");
  return PNB_OK;
}

// A tiled map of `rank` dimensions (strides of all but the first, in bytes).  No promotion to larger
// L2 reads: rows at an odd pitch would bring their neighbours' lines again (880 -> 790 us for 256 x
// 784->128 without it; even pitches show no difference).
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
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return PNB_OK;
  set_error("cuTensorMapEncodeTiled failed (%d): %llu x %llu, pitch %llu", (int)r,
            (unsigned long long)dims[0], (unsigned long long)dims[1],
            (unsigned long long)strides[0]);
  return PNB_ERR_CUDA;
}

// The swizzle whose span is a box row of these bytes.
static CUtensorMapSwizzle rq_swizzle(int bytes) {
  return bytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
         : bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                       : CU_TENSOR_MAP_SWIZZLE_32B;
}

// Byte matrix [rows][cols] at a pitch, in boxes of box_cols bytes (one swizzle span) x box_rows.
static int rq_map_bytes(CUtensorMap* map, const void* p, uint64_t cols, uint64_t rows,
                        uint64_t pitch, int box_cols, int box_rows) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  return rq_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, 2, dims, strides, box,
                rq_swizzle(box_cols));
}
static int rq_map_weights(CUtensorMap* map, const RqMatrix& m, int box_cols, int box_rows) {
  return rq_map_bytes(map, m.p, (uint64_t)m.pitch(), (uint64_t)m.rows, (uint64_t)m.pitch(), box_cols,
                      box_rows);
}

// How one block's shared memory is shared out.  Weights stay (keep_w) when the slots of a group's
// weights leave X enough; X stays for all tiles of 128 rows (m_group) when it fits beside a ring of
// weights and the batch fills the machine without splitting them.  Beyond that, slots of X in flight
// are what hides memory's latency: with weights kept, 256 x 784->128 takes 848, 713, 664 and 606 us
// (best launches) with 3, 4, 5 and 6 of them, adapters of 640->128 713, 646, 609 and 600.  So where X
// has fewer than six (five), results are staged in two halves, which costs short K something (256 x
// 128->10: 110 -> 119 us) and pays for a slot.  (These rules were weighed at K up to 1024 and M up to
// 512; beyond that the weights stream, and only the times above are known.)
template <bool SHIFTED, bool ADAPT>
static void rq_plan(RqArgs& a, int sms) {
  using S = RqShape<SHIFTED, ADAPT>;
  const int kb = (a.K + RQ_WK - 1) / RQ_WK, kx = (a.K + S::XK - 1) / S::XK;
  const int rank32 = (a.rank + 31) & ~31;
  const int t_bytes = ADAPT ? rank32 * S::BN : 0;
  const int b_bytes = ADAPT ? RQ_B_SLOTS * RQ_BM * a.b_row : 0;
  const int a_slot = ADAPT ? a.rank16 * RQ_WK : 0;  // beside each X slot
  int out_bytes = RQ_EPI_WARPS * S::OUT;
  int room = RQ_SMEM - RQ_BAR_BYTES - t_bytes - b_bytes - out_bytes;
  // what X wants at least before weights may stay: four slots (shifted: three, and 40 KB of raw rows);
  // for adapters, whose weights would come twice as often, one less.  256 rows of 784->128: one slot
  // less costs experts at an odd pitch 928 -> 1065 us by letting the weights stay, and gains rank 64
  // 1359 -> 1147 us, rank 16 at an odd pitch 1423 -> 1333 us.  (Shifted rows are in flight in the raw
  // ring: with four slots of it and more of X, 256 x 784->128 takes 1042 us instead of 760.)
  const int raw_min = SHIFTED ? 40 * 1024 / S::RAW_SLOT : 0;
  const int x_min = 4 - (SHIFTED ? 1 : 0) - (ADAPT ? 1 : 0);
  auto x_bytes = [&](int slots) { return slots * (S::X_SLOT + a_slot) + raw_min * S::RAW_SLOT; };
  const long long columns = (long long)a.rows * a.n_tiles;
  a.m_group = a.m_tiles;
  while (a.m_group > 1 && columns * ((a.m_tiles + a.m_group - 1) / a.m_group) < sms)
    a.m_group = (a.m_group + 1) / 2;
  if (a.m_group > 1 && x_bytes(kx + 1) + 3 * RQ_W_SLOT > room) a.m_group = 1;
  const int x_need = std::min(RQ_MAX_X, a.m_group > 1 ? std::max(x_min, kx + 1) : x_min);
  a.keep_w = (long long)a.m_group * kb <= std::min(RQ_MAX_W, (room - x_bytes(x_need)) / RQ_W_SLOT);
  a.w_slots = a.keep_w ? a.m_group * kb
                       : std::max(3, std::min(4, (room - x_bytes(x_need)) / RQ_W_SLOT));
  room -= a.w_slots * RQ_W_SLOT;
  if (SHIFTED) {
    a.x_slots = x_need;
    a.raw_slots =
        std::min(RQ_MAX_RAW, (room - a.x_slots * (S::X_SLOT + a_slot)) / S::RAW_SLOT & ~3);
  } else {
    a.x_slots = std::min(RQ_MAX_X, room / (S::X_SLOT + a_slot));
    if (S::MAY_SPLIT && a.x_slots < (ADAPT ? 5 : 6)) {
      a.out_split = 1;
      out_bytes /= 2;
      a.x_slots = (room + out_bytes) / (S::X_SLOT + a_slot);
    }
    a.raw_slots = 0;
  }
  a.x_at = a.w_slots * RQ_W_SLOT;
  a.t_at = a.x_at + a.x_slots * S::X_SLOT;
  a.b_at = a.t_at + t_bytes;
  a.a_at = a.b_at + b_bytes;
  a.out_at = a.a_at + a.x_slots * a_slot;
  a.raw_at = a.out_at + out_bytes;
  a.bars_at = a.raw_at + a.raw_slots * S::RAW_SLOT;
}

// ---- few products -------------------------------------------------------------------------------
// A tile of the tensor cores costs its block about 2000 cycles however small K and M are (lists, waits
// and one warp's limb sums), so calls of few products take plain 64-bit multiply-adds instead: one
// thread per word, 16 output rows at a time, weights in shared memory.  Weights are stored as
// w + 128 >= 0, so that a product is one 32 x 32 + 64 and one 32 x 32 + 32 bit multiply-add, and
// sum w x = sum (w + 128) x - 128 sum x.
constexpr int FEW_ROWS = 16;      // per pass, and the largest rank
constexpr int FEW_THREADS = 256;
// Most weights (rows padded to 16) that go this way.  2049-word rows at an even pitch (odd in brackets):
// 256 of experts 10->4 take 110 us (132) on the tensor cores and 54 here with 160 weights, 110 (135)
// and 230 with 1024; 128 with adapters of rank 8 234 us (308) and 57 with 576, 230 (306) and 208 with
// 2304, 230 (304) and 322 with 3584.
template <bool ADAPT> constexpr int few_weights() { return ADAPT ? 2048 : 384; }

struct FewArgs {
  RqArgs a;
  const int8_t *W, *A, *B;
  const uint64_t* X;
  int ldx, per_row, words;  // blocks of a row, and their words
};

__device__ __forceinline__ void few_madd(uint64_t& acc, uint64_t x, uint32_t w) {
  const uint64_t lo = acc + (uint64_t)(uint32_t)x * w;
  acc = lo + ((uint64_t)((uint32_t)(x >> 32) * w) << 32);
}

// acc[u] += sum_k (w[k][u] + 128) x_k;  returns sum_k x_k.  w: rows of `pitch` 32-bit weights.
template <typename Load>
__device__ __forceinline__ uint64_t few_rows(uint64_t (&acc)[FEW_ROWS], const uint32_t* w, int pitch,
                                             int K, Load load) {
  uint64_t sum = 0;
#pragma unroll 4
  for (int k = 0; k < K; ++k) {
    const uint64_t x = load(k);
    sum += x;
    const uint4* wk = reinterpret_cast<const uint4*>(w + k * pitch);
#pragma unroll
    for (int u = 0; u < FEW_ROWS / 4; ++u) {
      const uint4 v = wk[u];
      few_madd(acc[4 * u], x, v.x);
      few_madd(acc[4 * u + 1], x, v.y);
      few_madd(acc[4 * u + 2], x, v.z);
      few_madd(acc[4 * u + 3], x, v.w);
    }
  }
  return sum;
}

template <bool ADAPT>
__global__ void __launch_bounds__(FEW_THREADS) few_kernel(const __grid_constant__ FewArgs f) {
  extern __shared__ __align__(16) uint32_t few_w[];  // [K][M16]; adapters: [K][16] of A, [16][M16] of B
  const RqArgs& a = f.a;
  const int n = (int)(blockIdx.x / (unsigned)f.per_row);
  const int c = (int)(blockIdx.x - (unsigned)n * f.per_row) * f.words + (int)threadIdx.x;
  int w = __ldg(a.which + n), src = n;
  if (w < 0 || w >= a.n_which) w = -1;
  if (!ADAPT) {
    const int choice = __ldg(a.row_choice + n);
    if (w < 0 || choice < 0 || choice >= a.choices) return;
    if (a.top_k > 0) src = choice / a.top_k;
  }
  const bool has = ADAPT && w >= 0;
  const int m16 = (a.M + FEW_ROWS - 1) / FEW_ROWS * FEW_ROWS;
  uint32_t *wa = few_w + a.K * m16, *wb = wa + a.K * FEW_ROWS;
  // weights [rows][cols] transposed to `to` [cols][pitch]; padding is w = 0
  auto stage = [&](uint32_t* to, const int8_t* from, int rows, int cols, int pitch, int lines) {
    for (int i = threadIdx.x; i < lines * pitch; i += FEW_THREADS) {
      const int col = i / pitch, row = i - col * pitch;
      to[i] = 128u + (uint32_t)(row < rows && col < cols ? (int)__ldg(from + (size_t)row * cols + col) : 0);
    }
  };
  stage(few_w, f.W + (ADAPT ? (size_t)0 : (size_t)w * a.M * a.K), a.M, a.K, m16, a.K);
  if (has) {
    stage(wa, f.A + (size_t)w * a.rank * a.K, a.rank, a.K, FEW_ROWS, a.K);
    stage(wb, f.B + (size_t)w * a.M * a.rank, a.M, a.rank, m16, FEW_ROWS);
  }
  __syncthreads();
  if ((int)threadIdx.x >= f.words || c >= a.L) return;
  const uint64_t* x = f.X + (size_t)src * a.K * f.ldx + c;
  auto load = [&](int k) { return __ldg(x + (size_t)k * f.ldx); };
  uint64_t t[FEW_ROWS] = {}, t_sum = 0;
  if (has) {
    const uint64_t sum = few_rows(t, wa, FEW_ROWS, a.K, load);
#pragma unroll
    for (int q = 0; q < FEW_ROWS; ++q) {  // rows past the rank are zero: 128 sum - 128 sum
      t[q] -= 128 * sum;
      t_sum += t[q];
    }
  }
  uint64_t* y = a.Y + (size_t)n * a.M * a.ldy + c;
  for (int j0 = 0; j0 < a.M; j0 += FEW_ROWS) {
    uint64_t acc[FEW_ROWS] = {}, low[FEW_ROWS] = {};
    const uint64_t sum = few_rows(acc, few_w + j0, m16, a.K, load);
    if (has) {
#pragma unroll
      for (int q = 0; q < FEW_ROWS; ++q) {
        const uint4* wq = reinterpret_cast<const uint4*>(wb + q * m16 + j0);
#pragma unroll
        for (int u = 0; u < FEW_ROWS / 4; ++u) {
          const uint4 v = wq[u];
          few_madd(low[4 * u], t[q], v.x);
          few_madd(low[4 * u + 1], t[q], v.y);
          few_madd(low[4 * u + 2], t[q], v.z);
          few_madd(low[4 * u + 3], t[q], v.w);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < FEW_ROWS; ++u) {
      if (j0 + u >= a.M) break;
      uint64_t v = acc[u] - 128 * sum;
      if (ADAPT) v <<= a.shift;
      if (has) v += low[u] - 128 * t_sum;
      if (a.bias && c == a.L - 1)
        v += (uint64_t)__ldg(a.bias + (ADAPT ? (size_t)0 : (size_t)w * a.M) + j0 + u) * a.delta;
      y[(size_t)(j0 + u) * a.ldy] = v;
    }
  }
}

// Launches it when it is the faster one, and says so.
template <bool ADAPT>
static int few_run(const RqArgs& a, const int8_t* W, const int8_t* A, const int8_t* B,
                   const uint64_t* X, int ldx, bool& done, cudaStream_t st) {
  done = false;
  const long long m16 = (a.M + FEW_ROWS - 1) / FEW_ROWS * FEW_ROWS;
  if (ADAPT && a.rank > FEW_ROWS) return PNB_OK;
  const long long weights = a.K * m16 + (ADAPT ? FEW_ROWS * (a.K + m16) : 0);
  FewArgs f{a, W, A, B, X, ldx};
  f.per_row = (a.L + FEW_THREADS - 1) / FEW_THREADS;
  f.words = (a.L + f.per_row - 1) / f.per_row;
  if (weights > few_weights<ADAPT>() || (long long)a.rows * f.per_row > 0x7fffffffLL) return PNB_OK;
  done = true;
  few_kernel<ADAPT><<<(unsigned)(a.rows * f.per_row), FEW_THREADS, (size_t)weights * 4, st>>>(f);
  PNB_CHECK_LAUNCH("few_kernel");
  return PNB_OK;
}

// What the device needs once (its number of SMs read, the kernel's shared-memory limit raised), and
// the plan.
template <bool SHIFTED, bool ADAPT>
static int rq_prepare(RqArgs& a, int& sms) {
  static std::atomic<int> sm_count[64];
  int dev = 0;
  PNB_CUDA(cudaGetDevice(&dev));
  sms = dev < 64 ? sm_count[dev].load(std::memory_order_acquire) : 0;
  if (sms == 0) {
    PNB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    PNB_CUDA(cudaFuncSetAttribute(request_kernel<SHIFTED, ADAPT, false>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, RQ_SMEM));
    if (RqShape<SHIFTED, ADAPT>::MAY_SPLIT)
      PNB_CUDA(cudaFuncSetAttribute(
          request_kernel<SHIFTED, ADAPT, RqShape<SHIFTED, ADAPT>::MAY_SPLIT>,
          cudaFuncAttributeMaxDynamicSharedMemorySize, RQ_SMEM));
    if (dev < 64) sm_count[dev].store(sms, std::memory_order_release);
  }
  rq_plan<SHIFTED, ADAPT>(a, sms);
  if (a.x_slots < 2 || a.w_slots < 1 || (SHIFTED && a.raw_slots < RQ_COPY_WARPS) ||
      a.bars_at + RQ_BAR_BYTES > RQ_SMEM) {
    set_error("%s: no plan for M=%d K=%d rank=%d", ADAPT ? "adapter_contract" : "expert_contract",
              a.M, a.K, a.rank);
    return PNB_ERR_INVALID;
  }
  a.groups = (a.m_tiles + a.m_group - 1) / a.m_group;
  if (a.groups < 1 << RQ_MG_BITS && (long long)a.groups * a.n_tiles < 1 << RQ_NT_BITS) return PNB_OK;
  set_error("%s: %d x %d tiles of one row exceed one launch",
            ADAPT ? "adapter_contract" : "expert_contract", a.groups, a.n_tiles);
  return PNB_ERR_INVALID;
}

// `early`: behind rq_pad_kernel, whose launch and whose run the set-up of this one then hides.
template <bool SHIFTED, bool ADAPT>
static int rq_launch(const RqMaps& tm, const RqArgs& a, int sms, bool early, cudaStream_t st) {
  using S = RqShape<SHIFTED, ADAPT>;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(
      (unsigned)std::min<long long>((long long)a.rows * a.groups * a.n_tiles, sms));
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = (size_t)(a.bars_at + RQ_BAR_BYTES);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  auto kernel = a.out_split ? request_kernel<SHIFTED, ADAPT, S::MAY_SPLIT>
                            : request_kernel<SHIFTED, ADAPT, false>;
  PNB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tm, a));
  return PNB_OK;
}

template <bool ADAPT>
static int rq_run(RqMatrix W, RqMatrix A, RqMatrix B, RqArgs a, const uint64_t* X, int ldx,
                  int x_groups, void* ws, size_t ws_bytes, cudaStream_t st) {
  size_t need = W.in_place() ? 0 : W.copy_bytes();
  if (ADAPT) need += (A.in_place() ? 0 : A.copy_bytes()) + (B.in_place() ? 0 : B.copy_bytes());
  if (need && ws && (ws_bytes < need || ((uintptr_t)ws % 16) != 0)) {
    set_error("%s: workspace of %zu bytes at %p, %zu bytes 16-byte aligned are needed",
              ADAPT ? "adapter_contract" : "expert_contract", ws_bytes, ws, need);
    return PNB_ERR_INVALID;
  }
  using S = RqShape<false, ADAPT>;
  bool done;
  const int few = few_run<ADAPT>(a, W.p, A.p, B.p, X, ldx, done, st);
  if (few || done) return few;
  const long long x_rows = (long long)x_groups * a.K;
  // TMA coordinates are 32-bit, and a tile reaches up to a slot past its first row
  constexpr long long MOST = 0x7fffffffLL - RQ_BM;
  if (x_rows > MOST || W.rows > MOST || A.rows > MOST || B.rows > MOST) {
    set_error("%s: %lld ciphertexts or %lld weight rows exceed a 32-bit index",
              ADAPT ? "adapter_contract" : "expert_contract", x_rows,
              std::max(W.rows, std::max(A.rows, B.rows)));
    return PNB_ERR_INVALID;
  }
  a.n_tiles = (a.L + S::WORDS - 1) / S::WORDS;
  a.m_tiles = (a.M + RQ_BM - 1) / RQ_BM;
  a.w_rows = std::min(RQ_BM, (a.M + 7) & ~7);
  const uintptr_t xw = (uintptr_t)X / 8;
  a.off0 = (int)(xw & 1);
  a.off1 = (int)((xw + (uintptr_t)ldx) & 1);
  const bool shifted = a.off0 || a.off1 || a.ldy % 2 != 0 || ((uintptr_t)a.Y % 16) != 0;
  RqMaps tm{};
  int sms = 0;
  int rc = shifted ? rq_prepare<true, ADAPT>(a, sms) : rq_prepare<false, ADAPT>(a, sms);
  if (rc) return rc;
  if (!shifted) {
    const uint64_t pitch = (uint64_t)ldx * 8;
    rc = rq_map_bytes(&tm.X[0], X, pitch, (uint64_t)x_rows, pitch, 128, S::XK);
    if (!rc) rc = rq_map_bytes(&tm.X[1], X, pitch, (uint64_t)x_rows, pitch, 128, RQ_KSTEP);
    // writes end at word L (rounded down to 16 bytes) of row M of each ciphertext row
    const cuuint64_t dims[3] = {(cuuint64_t)std::max(2, a.L & ~1), (cuuint64_t)a.M,
                                (cuuint64_t)a.rows};
    const cuuint64_t strides[2] = {(cuuint64_t)a.ldy * 8, (cuuint64_t)a.M * a.ldy * 8};
    const int words = a.out_split ? S::EW / 2 : S::EW;
    const cuuint32_t box[3] = {(cuuint32_t)words, 32, 1};
    if (!rc)
      rc = rq_map(&tm.Y, CU_TENSOR_MAP_DATA_TYPE_UINT64, a.Y, 3, dims, strides, box,
                  rq_swizzle(8 * words));
  } else {
    // rows p, p + 2, ..: from the 16-byte boundary at or before row p, at twice the pitch.  A row
    // off by one word has that word's 16 bytes inside its allocation (allocations start aligned).
    for (int p = 0; p < 2 && !rc; ++p) {
      // (a single row has no row 1: both maps are its own, and the second meets zero weights)
      const bool second = p && x_rows > 1;
      const int off = second ? a.off1 : a.off0;
      const cuuint64_t dims[2] = {(cuuint64_t)ldx + off,
                                  (cuuint64_t)std::max<long long>(1, (x_rows + 1 - p) / 2)};
      const cuuint64_t strides[1] = {(cuuint64_t)ldx * 16};
      const cuuint32_t box[2] = {S::WORDS + 2, S::RAW_ROWS / 2};
      rc = rq_map(&tm.X[p], CU_TENSOR_MAP_DATA_TYPE_UINT64, X + (second ? ldx : 0) - off, 2, dims,
                  strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    }
  }
  if (rc) return rc;
  int8_t* own = nullptr;
  if (need && !ws) PNB_CUDA(cudaMallocAsync((void**)&own, need, st));
  RqMatrix* all[3] = {&W, &A, &B};
  bool placed = false;
  rc = rq_place(all, own ? own : (int8_t*)ws, st, placed);
  if (!rc) rc = rq_map_weights(&tm.W, W, 128, a.w_rows);
  if (ADAPT && !rc) rc = rq_map_weights(&tm.A, A, 128, a.rank16);
  if (ADAPT && !rc) rc = rq_map_weights(&tm.B, B, a.b_row, RQ_BM);
  if (!rc)
    rc = shifted ? rq_launch<true, ADAPT>(tm, a, sms, placed, st)
                 : rq_launch<false, ADAPT>(tm, a, sms, placed, st);
  if (own) {
    const cudaError_t e = cudaFreeAsync(own, st);
    if (!rc && e != cudaSuccess) rc = cuda_status(e, "cudaFreeAsync(padded weights)");
  }
  return rc;
}

int expert_contract(const int32_t* row_choice, const int32_t* row_expert, int tokens, int top_k,
                    int experts, bool sorted_rows, const int8_t* W, const int64_t* bias,
                    uint64_t delta, int M, int K, const uint64_t* X, int ldx, uint64_t* Y, int ldy,
                    int L, void* ws, size_t ws_bytes, cudaStream_t st) {
  RqArgs a{};
  a.Y = Y; a.bias = bias; a.delta = delta;
  a.row_choice = row_choice; a.which = row_expert;
  a.rows = a.choices = tokens * top_k;
  a.top_k = sorted_rows ? 0 : top_k;
  a.n_which = experts;
  a.M = M; a.K = K; a.L = L; a.ldy = ldy;
  return rq_run<false>({W, (long long)experts * M, K}, {}, {}, a, X, ldx,
                       sorted_rows ? a.rows : tokens, ws, ws_bytes, st);
}

int adapter_contract(const int8_t* W, const int64_t* bias, uint64_t delta, int base_shift, int M,
                     int K, const int8_t* A, const int8_t* B, int adapters, int rank,
                     const int32_t* adapter, const uint64_t* X, int ldx, uint64_t* Y, int ldy,
                     int batch, int L, void* ws, size_t ws_bytes, cudaStream_t st) {
  RqArgs a{};
  a.Y = Y; a.bias = bias; a.delta = delta;
  a.which = adapter; a.n_which = adapters;
  a.rows = batch;
  a.M = M; a.K = K; a.L = L; a.ldy = ldy;
  a.shift = base_shift; a.rank = rank; a.rank16 = (rank + 15) & ~15;
  a.b_row = rank <= 32 ? 32 : 64;
  return rq_run<true>({W, M, K}, {A, (long long)adapters * rank, K}, {B, (long long)adapters * M, rank},
                      a, X, ldx, batch, ws, ws_bytes, st);
}

}  // namespace pnb

// expert.cu -- rows of ciphertext tokens sorted by expert, moved there and back.
//
// A token is `features` LWE ciphertexts; it chooses top_k experts, in the clear.  Choice
// c = t * top_k + i is used when its expert lies in [0, experts); the used choices, sorted by
// expert with ties in choice order, are the rows.  Three operators, all exact mod 2^64:
//   route     row_choice[r] = c, row_expert[r], choice_row[c] = r (-1 where unused), offsets[e] =
//             the first row of expert e, offsets[experts] = R
//   dispatch  out[choice_row[c]] = w[c] * X[t]
//   combine   out[t] = sum_i w[t][i] * Y[choice_row[t][i]]
// Dispatch is the transpose of combine, so with the same weights each is the other's gradient.
// The reference has no routed layers; these stand beside the Linear contraction
// (runtime/src/ops/linear.rs:52-75) for networks whose weights differ from request to request.
#include <algorithm>

#include <cooperative_groups.h>

#include "pnb_internal.cuh"
#include "pnb_keys.h"

namespace pnb {

namespace cg = cooperative_groups;

// ---- route --------------------------------------------------------------------------------------
// Latency, not traffic: 12 bytes a choice.  A counting sort whose counters are per (warp, expert).
// Warp w of the launch owns one run of consecutive choices, so "warps in order, choices in order
// within a warp" is choice order and the sort is stable without atomics whose order could matter.
// Many choices are shared out over the blocks of one cluster, which read each other's totals: what
// one block spends its time on is the scattered stores, one line after another (8191 x 4 choices of
// 64 experts: 41 us with one block, 12 with a cluster; 8 x 2: 7 us a call, 3 replayed in a graph).
constexpr int RT_MAX_WARPS = 32;
constexpr int RT_CLUSTER = 8;
constexpr int RT_AHEAD = 4;  // loads of a lane on their way together
constexpr int RT_ONE_BLOCK = 32 * RT_MAX_WARPS;  // one choice per thread

__global__ void __launch_bounds__(32 * RT_MAX_WARPS) route_kernel(
    const int32_t* __restrict__ ids, int n, int experts, int32_t* __restrict__ offsets,
    int32_t* __restrict__ row_choice, int32_t* __restrict__ row_expert,
    int32_t* __restrict__ choice_row) {
  extern __shared__ int rt_cnt[];  // [warps][experts], then the block's totals [experts]
  __shared__ int warp_sum[RT_MAX_WARPS];
  __shared__ int carry_s;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = gridDim.x, rank = blockIdx.x;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* totals = rt_cnt + warps * experts;
  for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) rt_cnt[i] = 0;
  if (threadIdx.x == 0) carry_s = 0;
  __syncthreads();
  const int per = ((n + blocks * warps - 1) / (blocks * warps) + 31) & ~31;  // choices per warp
  const int lo = min(n, (rank * warps + warp) * per), hi = min(n, lo + per);
  int* cnt = rt_cnt + warp * experts;
  auto load = [&](int i0, int (&e)[RT_AHEAD]) {  // -1: unused or behind the end
#pragma unroll
    for (int j = 0; j < RT_AHEAD; ++j) {
      const int i = i0 + 32 * j + lane;
      e[j] = i < hi ? __ldg(ids + i) : -1;
    }
#pragma unroll
    for (int j = 0; j < RT_AHEAD; ++j)
      if (e[j] < 0 || e[j] >= experts) e[j] = -1;
  };
  int e[RT_AHEAD];
  for (int i0 = lo; i0 < hi; i0 += 32 * RT_AHEAD) {
    load(i0, e);
#pragma unroll
    for (int j = 0; j < RT_AHEAD; ++j)
      if (e[j] >= 0) atomicAdd(&cnt[e[j]], 1);
  }
  __syncthreads();
  for (int x = threadIdx.x; x < experts; x += blockDim.x) {
    int total = 0;
    for (int w = 0; w < warps; ++w) total += rt_cnt[w * experts + x];
    totals[x] = total;
  }
  if (blocks > 1) cluster.sync(); else __syncthreads();
  // exclusive prefix over (expert, block, warp), blockDim.x experts at a time
  for (int e0 = 0; e0 < experts; e0 += blockDim.x) {
    const int x = e0 + threadIdx.x;
    int total = 0, mine = 0;  // of the expert, and in the blocks before this one
    if (x < experts)
      for (int b = 0; b < blocks; ++b) {
        const int t = blocks > 1 ? *cluster.map_shared_rank(totals + x, b) : totals[x];
        if (b < rank) mine += t;
        total += t;
      }
    int incl = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int before = carry_s, all = 0;
    for (int w = 0; w < warps; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    if (x < experts) {
      int first = before + incl - total;
      if (rank == 0) offsets[x] = first;
      first += mine;
      for (int w = 0; w < warps; ++w) {
        const int c = rt_cnt[w * experts + x];
        rt_cnt[w * experts + x] = first;
        first += c;
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) carry_s += all;
    __syncthreads();
  }
  const int rows = carry_s;
  const int bits = 32 - __clz(experts - 1);
  if (rank == 0 && threadIdx.x == 0) offsets[experts] = rows;
  // places: within 32 choices, the lanes of one expert (one ballot per bit of its number) rank by
  // lane number
  for (int i0 = lo; i0 < hi; i0 += 32 * RT_AHEAD) {
    if (hi - lo > 32 * RT_AHEAD) load(i0, e);  // else they are still here
#pragma unroll
    for (int j = 0; j < RT_AHEAD; ++j) {
      unsigned same = __ballot_sync(0xffffffffu, e[j] >= 0);
      for (int b = 0; b < bits; ++b) {
        const bool set = (e[j] >> b) & 1;
        const unsigned with = __ballot_sync(0xffffffffu, set);
        same &= set ? with : ~with;
      }
      const int place = __popc(same & ((1u << lane) - 1u));
      int at = -1;
      if (e[j] >= 0) at = cnt[e[j]] + place;
      __syncwarp();
      if (e[j] >= 0 && place == 0) cnt[e[j]] += __popc(same);
      __syncwarp();
      const int i = i0 + 32 * j + lane;
      if (i < hi) choice_row[i] = at;
      if (at >= 0) {
        row_choice[at] = i;
        row_expert[at] = e[j];
      }
    }
  }
  for (int r = rows + rank * blockDim.x + threadIdx.x; r < n; r += blocks * blockDim.x) {
    row_choice[r] = -1;
    row_expert[r] = -1;
  }
  if (blocks > 1) cluster.sync();  // the others may still be reading this block's totals
}

int expert_route(const int32_t* ids, int n, int experts, int32_t* offsets, int32_t* row_choice,
                 int32_t* row_expert, int32_t* choice_row, cudaStream_t st) {
  const int blocks = n > RT_ONE_BLOCK ? RT_CLUSTER : 1;
  const int warps = std::max(1, std::min(RT_MAX_WARPS, (n + 32 * blocks - 1) / (32 * blocks)));
  const int smem = (warps + 1) * experts * (int)sizeof(int);
  if (smem > 48 * 1024)
    PNB_CUDA(cudaFuncSetAttribute(route_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (RT_MAX_WARPS + 1) * PNB_MAX_EXPERTS * (int)sizeof(int)));
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)blocks, 1, 1};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  PNB_CUDA(cudaLaunchKernelEx(&cfg, route_kernel, ids, n, experts, offsets, row_choice, row_expert,
                              choice_row));
  return PNB_OK;
}

// ---- dispatch and combine -----------------------------------------------------------------------
// Copies with at most one multiply per word: HBM bounds them.  A block takes a run of one token's
// words, so that dispatch reads a token once however many rows it becomes, and combine writes it
// once.  Rows at even pitches with aligned bases move 16 bytes at a time, others 8.  Runs do not end
// with a ciphertext: 1025 units of 16 bytes would leave every second round of a block to one
// thread.  What is left is to have enough loads on their way: units per thread times the threads
// that fit, four blocks a multiprocessor.  Measured on 96 x 2 tokens of 128 ciphertexts (604 MB, floor
// 92 us): combine, which holds two rows' words beside the sums, 94 us with three units of 16 bytes (106
// with one in eight blocks, 104 with three in three, 129 with three in five, which leave 48
// registers), dispatch 98 us with four (105 with one); at an odd pitch combine 113 us with four of 8
// bytes (162 with one), dispatch 107 us with five (115 with four).
constexpr int MV_THREADS = 256, MV_BLOCKS = 4;
template <int WORDS, bool COMBINE> constexpr int mv_ahead() {
  return (COMBINE ? 3 : 4) + (WORDS == 1 ? 1 : 0);
}

struct MoveArgs {
  const int32_t* choice_row;  // [tokens][top_k]
  const int32_t* weights;     // [tokens][top_k] or null
  const uint64_t* in;
  uint64_t* out;
  int tokens, top_k, features, L, ldi, ldo;
  int per_row;                // units (1 or 2 words) of one ciphertext
  uint32_t magic;             // u / per_row = umulhi(u, magic) >> shift for u < 2^21; 0: per_row = 1
  int shift;
};

template <int WORDS> struct MvUnit;
template <> struct MvUnit<1> { using T = unsigned long long; };
template <> struct MvUnit<2> { using T = ulonglong2; };

__device__ __forceinline__ void mv_madd(unsigned long long& a, unsigned long long v,
                                        unsigned long long w) { a += v * w; }
__device__ __forceinline__ void mv_madd(ulonglong2& a, ulonglong2 v, unsigned long long w) {
  a.x += v.x * w;
  a.y += v.y * w;
}

template <int WORDS, bool COMBINE>
__global__ void __launch_bounds__(MV_THREADS, MV_BLOCKS) move_kernel(const MoveArgs a) {
  constexpr int MV_AHEAD = mv_ahead<WORDS, COMBINE>(), MV_RUN = MV_THREADS * MV_AHEAD;
  using T = typename MvUnit<WORDS>::T;
  const int choices = a.tokens * a.top_k;
  const long long units = (long long)a.features * a.per_row;
  const long long first = (long long)blockIdx.x * MV_RUN;
  for (int t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    const int32_t* row_of = a.choice_row + (size_t)t * a.top_k;
    const int32_t* weight = a.weights ? a.weights + (size_t)t * a.top_k : nullptr;
    const long long f0 = first / a.per_row;
    const int u0 = (int)(first - f0 * a.per_row) + threadIdx.x;
    const int left = (int)min((long long)MV_RUN, units - first);
    size_t in_at[MV_AHEAD], out_at[MV_AHEAD];
    bool live[MV_AHEAD], whole[MV_AHEAD];
#pragma unroll
    for (int j = 0; j < MV_AHEAD; ++j) {
      const int u = u0 + j * MV_THREADS;
      const int f = a.magic ? (int)(__umulhi((uint32_t)u, a.magic) >> a.shift) : u;
      const int c = (u - f * a.per_row) * WORDS;
      live[j] = (int)threadIdx.x + j * MV_THREADS < left;
      whole[j] = c + WORDS <= a.L;  // else the last word of an odd count
      in_at[j] = (size_t)(f0 + f) * a.ldi + c;
      out_at[j] = (size_t)(f0 + f) * a.ldo + c;
    }
    // the row of choice k and its weight; -1 past the last and where unused
    auto row = [&](int k, unsigned long long& w) {
      w = 1;
      if (k >= a.top_k) return -1;
      if (weight) w = (unsigned long long)(long long)__ldg(weight + k);
      const int r = __ldg(row_of + k);
      return r < choices ? r : -1;
    };
    auto load = [&](long long token, T (&v)[MV_AHEAD]) {
#pragma unroll
      for (int j = 0; j < MV_AHEAD; ++j) {
        v[j] = T{};
        if (token >= 0 && live[j])
          v[j] = __ldg(
              reinterpret_cast<const T*>(a.in + (size_t)token * a.features * a.ldi + in_at[j]));
      }
    };
    auto store = [&](long long token, const T (&v)[MV_AHEAD]) {
#pragma unroll
      for (int j = 0; j < MV_AHEAD; ++j) {
        if (token < 0 || !live[j]) continue;
        uint64_t* to = a.out + (size_t)token * a.features * a.ldo + out_at[j];
        if (whole[j])
          __stcs(reinterpret_cast<T*>(to), v[j]);
        else
          *to = *reinterpret_cast<const uint64_t*>(&v[j]);
      }
    };
    if (COMBINE) {
      T sum[MV_AHEAD] = {};
      for (int k = 0; k < a.top_k; k += 2) {  // two rows' loads at a time
        unsigned long long w0, w1;
        const int r0 = row(k, w0), r1 = row(k + 1, w1);
        T v0[MV_AHEAD], v1[MV_AHEAD];
        load(r0, v0);
        load(r1, v1);
#pragma unroll
        for (int j = 0; j < MV_AHEAD; ++j) {
          mv_madd(sum[j], v0[j], w0);
          mv_madd(sum[j], v1[j], w1);
        }
      }
      store(t, sum);
    } else {
      T v[MV_AHEAD];
      load(t, v);
      for (int k = 0; k < a.top_k; ++k) {
        unsigned long long w;
        const int r = row(k, w);
        T p[MV_AHEAD] = {};
#pragma unroll
        for (int j = 0; j < MV_AHEAD; ++j) mv_madd(p[j], v[j], w);
        store(r, p);
      }
    }
  }
}

template <bool COMBINE>
static int move_launch(MoveArgs a, cudaStream_t st) {
  const bool wide = a.ldi % 2 == 0 && a.ldo % 2 == 0 && ((uintptr_t)a.in % 16) == 0 &&
                    ((uintptr_t)a.out % 16) == 0;
  a.per_row = wide ? (a.L + 1) / 2 : a.L;
  // ceil(2^(32 + shift) / per_row) with 2^shift >= per_row / 2: exact for u < 2^21 (at most
  // PNB_MAX_REQUEST_WORDS into a ciphertext, and a run)
  a.shift = 0;
  while ((2 << a.shift) < a.per_row) ++a.shift;
  a.magic = (uint32_t)((((uint64_t)1 << (32 + a.shift)) + a.per_row - 1) / a.per_row);
  const int run = MV_THREADS * (wide ? mv_ahead<2, COMBINE>() : mv_ahead<1, COMBINE>());
  const long long runs = ((long long)a.features * a.per_row + run - 1) / run;
  if (runs > 0x7fffffffLL) {
    set_error("%s: tokens of %d ciphertexts of %d words exceed one launch",
              COMBINE ? "expert_combine" : "expert_dispatch", a.features, a.L);
    return PNB_ERR_INVALID;
  }
  const dim3 grid((unsigned)runs, (unsigned)std::min(65535, a.tokens));
  if (wide)
    move_kernel<2, COMBINE><<<grid, MV_THREADS, 0, st>>>(a);
  else
    move_kernel<1, COMBINE><<<grid, MV_THREADS, 0, st>>>(a);
  PNB_CHECK_LAUNCH("move_kernel");
  return PNB_OK;
}

int expert_dispatch(const int32_t* choice_row, int tokens, int top_k, const int32_t* weights,
                    const uint64_t* X, int features, int ldx, uint64_t* out, int ldo, int L,
                    cudaStream_t st) {
  return move_launch<false>({choice_row, weights, X, out, tokens, top_k, features, L, ldx, ldo}, st);
}

int expert_combine(const int32_t* choice_row, int tokens, int top_k, const int32_t* weights,
                   const uint64_t* Y, int features, int ldy, uint64_t* out, int ldo, int L,
                   cudaStream_t st) {
  return move_launch<true>({choice_row, weights, Y, out, tokens, top_k, features, L, ldy, ldo}, st);
}

}  // namespace pnb

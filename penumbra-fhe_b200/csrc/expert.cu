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

#include "pnb_internal.cuh"
#include "pnb_keys.h"

namespace pnb {

// ---- route --------------------------------------------------------------------------------------
// One block: a counting sort whose counters are per (warp, expert).  Warp w owns one run of
// consecutive choices, so "warps in order, choices in order within a warp" is choice order and the
// sort is stable without atomics whose order could matter.
constexpr int RT_MAX_WARPS = 32;

__global__ void __launch_bounds__(32 * RT_MAX_WARPS) route_kernel(
    const int32_t* __restrict__ ids, int n, int experts, int32_t* __restrict__ offsets,
    int32_t* __restrict__ row_choice, int32_t* __restrict__ row_expert,
    int32_t* __restrict__ choice_row) {
  extern __shared__ int rt_cnt[];  // [warps][experts]
  __shared__ int warp_sum[RT_MAX_WARPS];
  __shared__ int carry_s;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) rt_cnt[i] = 0;
  if (threadIdx.x == 0) carry_s = 0;
  __syncthreads();
  const int per = ((n + warps - 1) / warps + 31) & ~31;  // choices per warp
  const int lo = min(n, warp * per), hi = min(n, lo + per);
  int* cnt = rt_cnt + warp * experts;
  for (int i = lo + lane; i < hi; i += 32) {
    const int e = ids[i];
    if (e >= 0 && e < experts) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  // exclusive prefix over (expert, warp), blockDim.x experts at a time
  for (int e0 = 0; e0 < experts; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int total = 0;
    if (e < experts) {
      for (int w = 0; w < warps; ++w) {
        const int c = rt_cnt[w * experts + e];
        rt_cnt[w * experts + e] = total;
        total += c;
      }
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
    const int first = before + incl - total;
    if (e < experts) {
      offsets[e] = first;
      for (int w = 0; w < warps; ++w) rt_cnt[w * experts + e] += first;
    }
    __syncthreads();
    if (threadIdx.x == 0) carry_s += all;
    __syncthreads();
  }
  const int rows = carry_s;
  if (threadIdx.x == 0) offsets[experts] = rows;
  // places: within 32 choices, the lanes of one expert rank by lane number
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    int e = -1;
    if (i < hi) {
      e = ids[i];
      if (e >= experts || e < 0) e = -1;
    }
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int at = -1;
    if (e >= 0) at = cnt[e] + rank;
    __syncwarp();
    if (e >= 0 && rank == 0) cnt[e] += __popc(same);
    __syncwarp();
    if (i < hi) choice_row[i] = at;
    if (e >= 0) {
      row_choice[at] = i;
      row_expert[at] = e;
    }
  }
  for (int r = rows + threadIdx.x; r < n; r += blockDim.x) {
    row_choice[r] = -1;
    row_expert[r] = -1;
  }
}

int expert_route(const int32_t* ids, int n, int experts, int32_t* offsets, int32_t* row_choice,
                 int32_t* row_expert, int32_t* choice_row, cudaStream_t st) {
  const int warps = std::max(1, std::min(RT_MAX_WARPS, (n + 31) / 32));
  const int smem = warps * experts * (int)sizeof(int);
  PNB_CUDA(cudaFuncSetAttribute(route_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                RT_MAX_WARPS * PNB_MAX_EXPERTS * (int)sizeof(int)));
  route_kernel<<<1, 32 * warps, smem, st>>>(ids, n, experts, offsets, row_choice, row_expert,
                                            choice_row);
  PNB_CHECK_LAUNCH("route_kernel");
  return PNB_OK;
}

// ---- dispatch and combine -----------------------------------------------------------------------
struct MoveArgs {
  const int32_t* choice_row;  // [tokens][top_k]
  const int32_t* weights;     // [tokens][top_k] or null
  const uint64_t* in;
  uint64_t* out;
  int tokens, top_k, features, L, ldi, ldo;
};

__global__ void dispatch_kernel(MoveArgs a) {
  const int t = blockIdx.x;
  const long long words = (long long)a.features * a.L;
  const int choices = a.tokens * a.top_k;
  for (long long i = (long long)blockIdx.y * blockDim.x + threadIdx.x; i < words;
       i += (long long)gridDim.y * blockDim.x) {
    const long long f = i / a.L;
    const int c = (int)(i % a.L);
    const uint64_t v = a.in[((size_t)t * a.features + f) * a.ldi + c];
    for (int k = 0; k < a.top_k; ++k) {
      const int r = a.choice_row[t * a.top_k + k];
      if (r < 0 || r >= choices) continue;
      const uint64_t w = a.weights ? (uint64_t)(int64_t)a.weights[t * a.top_k + k] : 1ull;
      a.out[((size_t)r * a.features + f) * a.ldo + c] = w * v;
    }
  }
}

__global__ void combine_kernel(MoveArgs a) {
  const int t = blockIdx.x;
  const long long words = (long long)a.features * a.L;
  const int choices = a.tokens * a.top_k;
  for (long long i = (long long)blockIdx.y * blockDim.x + threadIdx.x; i < words;
       i += (long long)gridDim.y * blockDim.x) {
    const long long f = i / a.L;
    const int c = (int)(i % a.L);
    uint64_t v = 0;
    for (int k = 0; k < a.top_k; ++k) {
      const int r = a.choice_row[t * a.top_k + k];
      if (r < 0 || r >= choices) continue;
      const uint64_t w = a.weights ? (uint64_t)(int64_t)a.weights[t * a.top_k + k] : 1ull;
      v += w * a.in[((size_t)r * a.features + f) * a.ldi + c];
    }
    a.out[((size_t)t * a.features + f) * a.ldo + c] = v;
  }
}

static int move_launch(bool combine, const MoveArgs& a, cudaStream_t st) {
  const long long words = (long long)a.features * a.L;
  const dim3 grid((unsigned)a.tokens, (unsigned)std::min<long long>((words + 1023) / 1024, 4096));
  if (combine)
    combine_kernel<<<grid, 256, 0, st>>>(a);
  else
    dispatch_kernel<<<grid, 256, 0, st>>>(a);
  PNB_CHECK_LAUNCH(combine ? "combine_kernel" : "dispatch_kernel");
  return PNB_OK;
}

int expert_dispatch(const int32_t* choice_row, int tokens, int top_k, const int32_t* weights,
                    const uint64_t* X, int features, int ldx, uint64_t* out, int ldo, int L,
                    cudaStream_t st) {
  return move_launch(false, {choice_row, weights, X, out, tokens, top_k, features, L, ldx, ldo},
                     st);
}

int expert_combine(const int32_t* choice_row, int tokens, int top_k, const int32_t* weights,
                   const uint64_t* Y, int features, int ldy, uint64_t* out, int ldo, int L,
                   cudaStream_t st) {
  return move_launch(true, {choice_row, weights, Y, out, tokens, top_k, features, L, ldy, ldo},
                     st);
}

}  // namespace pnb

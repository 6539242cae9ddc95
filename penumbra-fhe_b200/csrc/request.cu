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
#include <algorithm>

#include "pnb_internal.cuh"
#include "pnb_keys.h"

namespace pnb {

// One thread per word of RQ_ROWS output rows.
constexpr int RQ_ROWS = 8;

__device__ __forceinline__ void rq_dot(uint64_t (&acc)[RQ_ROWS], const int8_t* W, int rows, int K,
                                       const uint64_t* X, int ldx) {
  for (int k = 0; k < K; ++k) {
    const uint64_t x = X[(size_t)k * ldx];
#pragma unroll
    for (int j = 0; j < RQ_ROWS; ++j)
      if (j < rows) acc[j] += (uint64_t)(int64_t)W[(size_t)j * K + k] * x;
  }
}

// out [n][M][ldo] = 2^shift W[w] X (+ out when add) + bias; w = which[n] (0 when which is null).
__global__ void request_kernel(const int32_t* which, int n_w, const int32_t* row_choice, int top_k,
                               int choices, const int8_t* W, const int64_t* bias, int bias_rows,
                               uint64_t delta, int shift, int add, int M, int K, const uint64_t* X,
                               int ldx, uint64_t* out, int ldo, int L) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  const int j0 = blockIdx.y * RQ_ROWS;
  const int n = blockIdx.z;
  const int w = which ? which[n] : 0;
  if (w < 0 || w >= n_w || c >= L) return;
  long long src = n;
  if (row_choice) {
    const int ch = row_choice[n];
    if (ch < 0 || ch >= choices) return;
    src = ch / top_k;
  }
  uint64_t acc[RQ_ROWS] = {};
  rq_dot(acc, W + ((size_t)w * M + j0) * K, min(RQ_ROWS, M - j0), K, X + (size_t)src * K * ldx + c,
         ldx);
#pragma unroll
  for (int j = 0; j < RQ_ROWS; ++j) {
    if (j0 + j >= M) break;
    uint64_t* o = out + ((size_t)n * M + j0 + j) * ldo + c;
    uint64_t v = acc[j] << shift;
    if (add) v += *o;
    if (bias && c == L - 1) v += (uint64_t)bias[(bias_rows ? (size_t)w * M : 0) + j0 + j] * delta;
    *o = v;
  }
}

int expert_contract(const int32_t* row_choice, const int32_t* row_expert, int tokens, int top_k,
                    int experts, bool sorted_rows, const int8_t* W, const int64_t* bias,
                    uint64_t delta, int M, int K, const uint64_t* X, int ldx, uint64_t* Y, int ldy,
                    int L, cudaStream_t st) {
  const int rows = tokens * top_k;
  for (int z = 0; z < rows; z += 32768) {
    const int n = std::min(rows - z, 32768);
    const dim3 grid((L + 127) / 128, (M + RQ_ROWS - 1) / RQ_ROWS, n);
    request_kernel<<<grid, 128, 0, st>>>(row_expert + z, experts,
                                         sorted_rows ? nullptr : row_choice + z, top_k, rows, W,
                                         bias, 1, delta, 0, 0, M, K,
                                         X + (sorted_rows ? (size_t)z * K * ldx : 0), ldx,
                                         Y + (size_t)z * M * ldy, ldy, L);
    PNB_CHECK_LAUNCH("request_kernel");
  }
  return PNB_OK;
}

int adapter_contract(const int8_t* W, const int64_t* bias, uint64_t delta, int base_shift, int M,
                     int K, const int8_t* A, const int8_t* B, int adapters, int rank,
                     const int32_t* adapter, const uint64_t* X, int ldx, uint64_t* Y, int ldy,
                     int batch, int L, cudaStream_t st) {
  uint64_t* low = nullptr;
  PNB_CUDA(cudaMallocAsync((void**)&low, (size_t)batch * rank * L * 8, st));
  for (int z = 0; z < batch; z += 32768) {
    const int n = std::min(batch - z, 32768);
    const unsigned cols = (L + 127) / 128;
    const uint64_t* Xz = X + (size_t)z * K * ldx;
    uint64_t* lowz = low + (size_t)z * rank * L;
    uint64_t* Yz = Y + (size_t)z * M * ldy;
    request_kernel<<<dim3(cols, (rank + RQ_ROWS - 1) / RQ_ROWS, n), 128, 0, st>>>(
        adapter + z, adapters, nullptr, 1, batch, A, nullptr, 0, 0, 0, 0, rank, K, Xz, ldx, lowz, L,
        L);
    request_kernel<<<dim3(cols, (M + RQ_ROWS - 1) / RQ_ROWS, n), 128, 0, st>>>(
        nullptr, 1, nullptr, 1, batch, W, bias, 0, delta, base_shift, 0, M, K, Xz, ldx, Yz, ldy, L);
    request_kernel<<<dim3(cols, (M + RQ_ROWS - 1) / RQ_ROWS, n), 128, 0, st>>>(
        adapter + z, adapters, nullptr, 1, batch, B, nullptr, 0, 0, 0, 1, M, rank, lowz, L, Yz, ldy,
        L);
  }
  cudaError_t le = cudaGetLastError();
  cudaError_t fe = cudaFreeAsync(low, st);
  if (le != cudaSuccess) return cuda_status(le, "request_kernel");
  if (fe != cudaSuccess) return cuda_status(fe, "cudaFreeAsync(low-rank rows)");
  return PNB_OK;
}

}  // namespace pnb

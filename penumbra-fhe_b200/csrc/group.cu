// group.cu -- contractions with 4-bit weights, a scale and a zero point per group of inputs.
//
//   w[j][i] = s[j][i / g] (q[j][i] - z[j][i / g]),   q and z in 0..15 (z = 8 where none are given)
//   Y[b][j] = sum_i w[j][i] X[b][i] + bias[j] * delta on the body       (transposed: sum over j)
//
// mod 2^64 over LWE ciphertexts.  |w| <= 128 * 15 = 1920.  X comes as rows of u64 words, or as the
// rounded words of a cache (cache.cu), whose limbs below the kept ones are zero.  The reference's
// Linear holds one integer per weight (runtime/src/ops/linear.rs:52-75).
#include <algorithm>

#include "pnb_internal.cuh"
#include "pnb_keys.h"

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

size_t group_workspace_bytes(int n_in, int n_out) {
  return (size_t)2 * n_out * (((size_t)n_in + 15) & ~(size_t)15);
}

static int group_run(const GroupArgs& a, int bits, void* ws, size_t ws_bytes, cudaStream_t st) {
  const size_t need = group_workspace_bytes(a.n_in, a.n_out);
  if (ws && (ws_bytes < need || ((uintptr_t)ws % 16) != 0)) {
    set_error("%s: workspace of %zu bytes at %p, %zu bytes 16-byte aligned are needed",
              a.slots ? "group_contract_cached" : "group_contract", ws_bytes, ws, need);
    return PNB_ERR_INVALID;
  }
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

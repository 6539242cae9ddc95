// cache.cu -- ciphertexts held in fewer bits: rows written into slots of a cache, and read back.
//
//   write:  q = floor((x + 2^(63-n)) / 2^(64-n)) mod 2^n      every word to its nearest multiple of
//   read:   x = q 2^(64-n)                                    2^(64-n), ties upwards
//
// An LWE phase b - <a, s> takes every word's rounding error, at most 2^(63-n) and uniform for uniform
// words: with a binary key of D words the phase moves by a standard deviation of about
// 2^(64-n) sqrt((D / 2 + 1) / 12), 2^(35.2) for n = 32 and D = 2048 against 2^59 between 4-bit messages.
// The reference holds every ciphertext in full (SignedRadixCiphertext, runtime/src/ops/mod.rs:58).
//
// A row of the cache is L little-endian words of n / 8 bytes (n = 16, 24, 32), padded to a multiple of
// 16 bytes: the bytes of a word are the limbs that the tensor-core contraction multiplies, so it
// reads a row as it lies.
#include <algorithm>

#include "pnb_internal.cuh"
#include "pnb_keys.h"

namespace pnb {

constexpr int CH_THREADS = 256;
constexpr int CH_AHEAD = 8;   // words of a thread on their way together
constexpr int CH_RUN = CH_THREADS * CH_AHEAD;
constexpr int CH_TOKENS = 8;  // most tokens of a block

struct CacheArgs {
  const int32_t* slots;  // [tokens]
  const uint64_t* in;    // write: the tokens' rows
  uint64_t* out;         // read: the tokens' rows
  unsigned char* cache;
  int tokens, n_slots, features, L, ld;
  int per_block;         // tokens
  size_t row_bytes;
  int per_row;           // words of a row, rounded up to 4
  uint32_t magic;        // u / per_row = umulhi(u, magic) >> shift for u < 2^21
  int shift;
};

// A block takes the same run of words of a few tokens.  One word per thread and step, so that a warp's
// 64-bit words are 256 consecutive bytes at any pitch.
// Words of three bytes go through registers of four: lane k < 3 of every four holds bytes 4k .. 4k+3 of
// their twelve, which is its own word without its first k bytes and the next lane's first k + 1.
template <int BYTES, bool WRITE>
__global__ void __launch_bounds__(CH_THREADS, 4) cache_kernel(const __grid_constant__ CacheArgs a) {
  constexpr int BITS = 8 * BYTES;
  __shared__ int slot_s[CH_TOKENS];  // of the block's tokens, -1 for those to leave out
  const long long units = (long long)a.features * a.per_row;
  const long long first = (long long)blockIdx.x * CH_RUN;
  const long long f0 = first / a.per_row;
  const int u0 = (int)(first - f0 * a.per_row) + (int)threadIdx.x;
  const int left = (int)min((long long)CH_RUN, units - first) - (int)threadIdx.x;
  const int sub = threadIdx.x & 3;
  size_t word[CH_AHEAD], cell[CH_AHEAD];  // where it is among a token's words, and among its bytes
  bool live[CH_AHEAD];
#pragma unroll
  for (int j = 0; j < CH_AHEAD; ++j) {
    const int u = u0 + j * CH_THREADS;
    const int f = (int)(__umulhi((uint32_t)u, a.magic) >> a.shift);
    const int col = u - f * a.per_row;
    live[j] = j * CH_THREADS < left && col < a.L;
    word[j] = (size_t)(f0 + f) * a.ld + col;
    cell[j] = (size_t)(f0 + f) * a.row_bytes;
    // of four words of three bytes the first three lanes move four bytes each, up to the last word's
    if (BYTES != 3)
      cell[j] += (size_t)col * BYTES;
    else if (sub < 3 && j * CH_THREADS < left && 4 * (col / 4 * 3 + sub) < 3 * a.L)
      cell[j] += 4 * (size_t)(col / 4 * 3 + sub);
    else
      cell[j] = ~(size_t)0;
  }
  for (int t0 = blockIdx.y * a.per_block; t0 < a.tokens; t0 += gridDim.y * a.per_block) {
    const int n = min(a.per_block, a.tokens - t0);
    __syncthreads();
    if ((int)threadIdx.x < n) {
      const int s = __ldg(a.slots + t0 + threadIdx.x);
      slot_s[threadIdx.x] = s >= 0 && s < a.n_slots ? s : -1;
    }
    __syncthreads();
    if (WRITE) {  // of two tokens that name the same slot the later one stays
      unsigned again = 0;
      for (int i = t0 + 1 + (int)threadIdx.x; i < a.tokens; i += CH_THREADS) {
        const int s = __ldg(a.slots + i);
        for (int k = 0; k < n; ++k) again |= t0 + k < i && slot_s[k] == s ? 1u << k : 0u;
      }
      __syncthreads();
      for (int k = 0; k < n; ++k)
        if (again >> k & 1u) slot_s[k] = -1;
      __syncthreads();
    }
    for (int k = 0; k < n; ++k) {
      const int slot = slot_s[k];
      if (slot < 0) continue;
      unsigned char* cells = a.cache + (size_t)slot * a.features * a.row_bytes;
      const size_t x0 = (size_t)(t0 + k) * a.features * a.ld;
      if (WRITE) {
        uint64_t x[CH_AHEAD];
#pragma unroll
        for (int j = 0; j < CH_AHEAD; ++j) x[j] = live[j] ? __ldcs(reinterpret_cast<const unsigned long long*>(a.in + x0 + word[j])) : 0;
#pragma unroll
        for (int j = 0; j < CH_AHEAD; ++j) {
          const uint32_t q = (uint32_t)((x[j] + (1ull << (63 - BITS))) >> (64 - BITS));
          if (BYTES == 4) {
            if (live[j]) *reinterpret_cast<uint32_t*>(cells + cell[j]) = q;
          } else if (BYTES == 2) {
            if (live[j]) *reinterpret_cast<uint16_t*>(cells + cell[j]) = (uint16_t)q;
          } else {
            const uint32_t next = __shfl_down_sync(0xffffffffu, q, 1);
            if (cell[j] != ~(size_t)0)
              *reinterpret_cast<uint32_t*>(cells + cell[j]) = q >> (8 * sub) | next << (24 - 8 * sub);
          }
        }
      } else {
        uint32_t q[CH_AHEAD];
#pragma unroll
        for (int j = 0; j < CH_AHEAD; ++j) {
          if (BYTES == 3)
            q[j] = cell[j] != ~(size_t)0 ? __ldcs(reinterpret_cast<const uint32_t*>(cells + cell[j])) : 0;
          else if (BYTES == 4)
            q[j] = live[j] ? __ldcs(reinterpret_cast<const uint32_t*>(cells + cell[j])) : 0;
          else
            q[j] = live[j] ? __ldcs(reinterpret_cast<const uint16_t*>(cells + cell[j])) : 0;
        }
#pragma unroll
        for (int j = 0; j < CH_AHEAD; ++j) {
          if (BYTES == 3) {  // word k: the last k bytes of the lane before, then its own first 3 - k
            const uint32_t before = __shfl_up_sync(0xffffffffu, q[j], 1);
            q[j] = sub == 0 ? q[j] : before >> (32 - 8 * sub) | q[j] << (8 * sub);
          }
          if (live[j]) __stcs(reinterpret_cast<unsigned long long*>(a.out + x0 + word[j]),
                               (unsigned long long)q[j] << (64 - BITS));
        }
      }
    }
  }
}

size_t cache_row_bytes(int L, int bits) { return ((size_t)L * (bits / 8) + 15) / 16 * 16; }

template <bool WRITE>
static int cache_launch(CacheArgs a, int bits, cudaStream_t st) {
  a.row_bytes = cache_row_bytes(a.L, bits);
  a.per_row = (a.L + 3) & ~3;
  // ceil(2^(32 + shift) / per_row) with 2^shift >= per_row / 2: exact for u < 2^21 (at most
  // PNB_MAX_REQUEST_WORDS into a row, and a run)
  a.shift = 0;
  while ((2 << a.shift) < a.per_row) ++a.shift;
  a.magic = (uint32_t)((((uint64_t)1 << (32 + a.shift)) + a.per_row - 1) / a.per_row);
  const long long runs = ((long long)a.features * a.per_row + CH_RUN - 1) / CH_RUN;
  if (runs > 0x7fffffffLL) {
    set_error("%s: tokens of %d ciphertexts of %d words exceed one launch",
              WRITE ? "cache_write" : "cache_read", a.features, a.L);
    return PNB_ERR_INVALID;
  }
  // several tokens to a block where that leaves every multiprocessor its blocks
  a.per_block = (int)std::max<long long>(1, std::min<long long>(CH_TOKENS, runs * a.tokens / 1184));
  const dim3 grid((unsigned)runs,
                  (unsigned)std::min(65535, (a.tokens + a.per_block - 1) / a.per_block));
  if (bits == 16)
    cache_kernel<2, WRITE><<<grid, CH_THREADS, 0, st>>>(a);
  else if (bits == 24)
    cache_kernel<3, WRITE><<<grid, CH_THREADS, 0, st>>>(a);
  else
    cache_kernel<4, WRITE><<<grid, CH_THREADS, 0, st>>>(a);
  PNB_CHECK_LAUNCH("cache_kernel");
  return PNB_OK;
}

int cache_write(const int32_t* slots, int tokens, const uint64_t* X, int features, int ldx, int L,
                void* cache, int n_slots, int bits, cudaStream_t st) {
  CacheArgs a{};
  a.slots = slots; a.tokens = tokens; a.in = X; a.features = features; a.ld = ldx; a.L = L;
  a.cache = (unsigned char*)cache; a.n_slots = n_slots;
  return cache_launch<true>(a, bits, st);
}

int cache_read(const int32_t* slots, int tokens, const void* cache, int n_slots, int bits,
               int features, uint64_t* out, int ldo, int L, cudaStream_t st) {
  CacheArgs a{};
  a.slots = slots; a.tokens = tokens; a.out = out; a.features = features; a.ld = ldo; a.L = L;
  a.cache = (unsigned char*)cache; a.n_slots = n_slots;
  return cache_launch<false>(a, bits, st);
}

}  // namespace pnb

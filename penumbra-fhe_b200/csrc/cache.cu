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
constexpr int CH_AHEAD = 8;  // words of a thread on their way together
constexpr int CH_RUN = CH_THREADS * CH_AHEAD;

struct CacheArgs {
  const int32_t* slots;  // [tokens]
  const uint64_t* in;    // write: the tokens' rows
  uint64_t* out;         // read: the tokens' rows
  unsigned char* cache;
  int tokens, n_slots, features, L, ld;
  size_t row_bytes;
  int per_row;           // words of a row, rounded up to 4
  uint32_t magic;        // u / per_row = umulhi(u, magic) >> shift for u < 2^21
  int shift;
};

// One word per thread and step, so that a warp's 64-bit words are 256 consecutive bytes at any pitch.
// Words of three bytes go through registers of four: lane k < 3 of every four holds bytes 4k .. 4k+3 of
// their twelve, which is its own word without its first k bytes and the next lane's first k + 1.
template <int BYTES, bool WRITE>
__global__ void __launch_bounds__(CH_THREADS) cache_kernel(const __grid_constant__ CacheArgs a) {
  constexpr int BITS = 8 * BYTES;
  const long long units = (long long)a.features * a.per_row;
  const long long first = (long long)blockIdx.x * CH_RUN;
  const long long f0 = first / a.per_row;
  const int u0 = (int)(first - f0 * a.per_row) + (int)threadIdx.x;
  const int left = (int)min((long long)CH_RUN, units - first) - (int)threadIdx.x;
  const int sub = threadIdx.x & 3;
  size_t row[CH_AHEAD];
  int col[CH_AHEAD];
#pragma unroll
  for (int j = 0; j < CH_AHEAD; ++j) {
    const int u = u0 + j * CH_THREADS;
    const int f = (int)(__umulhi((uint32_t)u, a.magic) >> a.shift);
    row[j] = (size_t)(f0 + f);
    col[j] = j * CH_THREADS < left ? u - f * a.per_row : a.per_row;
  }
  for (int t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    const int slot = __ldg(a.slots + t);
    if (slot < 0 || slot >= a.n_slots) continue;
    const size_t c_row = (size_t)slot * a.features, x_row = (size_t)t * a.features;
    if (WRITE) {
      uint64_t x[CH_AHEAD];
#pragma unroll
      for (int j = 0; j < CH_AHEAD; ++j)
        x[j] = col[j] < a.L ? __ldcs(a.in + (x_row + row[j]) * a.ld + col[j]) : 0;
      // of two tokens that name the same slot the later one stays
      bool later = false;
      for (int i = t + 1 + (int)threadIdx.x; i < a.tokens; i += CH_THREADS)
        later |= __ldg(a.slots + i) == slot;
      if (__syncthreads_or(later)) continue;
#pragma unroll
      for (int j = 0; j < CH_AHEAD; ++j) {
        const uint32_t q = (uint32_t)((x[j] + (1ull << (63 - BITS))) >> (64 - BITS));
        unsigned char* to = a.cache + (c_row + row[j]) * a.row_bytes;
        if (BYTES == 4) {
          if (col[j] < a.L) reinterpret_cast<uint32_t*>(to)[col[j]] = q;
        } else if (BYTES == 2) {
          if (col[j] < a.L) reinterpret_cast<uint16_t*>(to)[col[j]] = (uint16_t)q;
        } else {
          const uint32_t next = __shfl_down_sync(0xffffffffu, q, 1);
          const int at = col[j] / 4 * 3 + sub;  // its four bytes, of the row
          if (sub < 3 && 4 * at < 3 * a.L)
            reinterpret_cast<uint32_t*>(to)[at] = q >> (8 * sub) | next << (24 - 8 * sub);
        }
      }
    } else {
      uint32_t q[CH_AHEAD];
#pragma unroll
      for (int j = 0; j < CH_AHEAD; ++j) {
        const unsigned char* from = a.cache + (c_row + row[j]) * a.row_bytes;
        if (BYTES == 3) {
          const int at = col[j] / 4 * 3 + sub;
          q[j] = sub < 3 && 4 * at < 3 * a.L
                     ? __ldcs(reinterpret_cast<const uint32_t*>(from) + at) : 0;
        } else if (BYTES == 4) {
          q[j] = col[j] < a.L ? __ldcs(reinterpret_cast<const uint32_t*>(from) + col[j]) : 0;
        } else {
          q[j] = col[j] < a.L ? __ldcs(reinterpret_cast<const uint16_t*>(from) + col[j]) : 0;
        }
      }
#pragma unroll
      for (int j = 0; j < CH_AHEAD; ++j) {
        if (BYTES == 3) {  // word k: the last k bytes of the lane before, then its own first 3 - k
          const uint32_t before = __shfl_up_sync(0xffffffffu, q[j], 1);
          q[j] = sub == 0 ? q[j] : before >> (32 - 8 * sub) | q[j] << (8 * sub);
        }
        if (col[j] < a.L)
          a.out[(x_row + row[j]) * a.ld + col[j]] = (uint64_t)q[j] << (64 - BITS);
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
  const dim3 grid((unsigned)runs, (unsigned)std::min(65535, a.tokens));
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

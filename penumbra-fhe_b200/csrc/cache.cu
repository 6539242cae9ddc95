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
// Both move each byte once, which HBM bounds: 512 tokens of 128 ciphertexts of 2049 words, one in twenty
// unused, are written in 24 bits at an odd pitch in 239-250 us (floor 203; the look for later tokens of a
// slot is part of the rest) and read from 32 bits in 242 (floor 234).  That look grows with the square of the
// tokens: one ciphertext each of 4096 tokens takes 25 us (floor 14), of 16384 123 (56), of 65536 1481 (226).
//
// A row of the cache is L little-endian words of n / 8 bytes (n = 16, 24, 32), padded to a multiple of
// 16 bytes: the bytes of a word are the limbs that the tensor-core contraction multiplies, so it
// reads a row as it lies.
#include <algorithm>

#include "pnb_internal.cuh"
#include "pnb_keys.h"

namespace pnb {

constexpr int CH_WARPS = 8, CH_BLOCKS = 5;
constexpr int CH_AHEAD = 4;    // pairs of words of a thread on their way together
// Words of a row that a warp takes at a time: 512 x 128 ciphertexts written in 24 bits 239 us with 256, 249
// with 512, read from 32 bits 262 and 251.
constexpr int CH_PIECE_WRITE = 256, CH_PIECE_READ = 512;
// Most pieces of a block.  Writing, a block looks for later tokens of its slot first, which more pieces
// share (in 24 bits, pieces of 512: 259 us with 8, 249 with 32, 265 with 128); reading, fewer are better
// (from 32 bits: 251, 264, 281).
constexpr int CH_PIECES_WRITE = 32, CH_PIECES_READ = 8;

struct CacheArgs {
  const int32_t* slots;  // [tokens]
  const uint64_t* in;    // write: the tokens' rows
  uint64_t* out;         // read: the tokens' rows
  unsigned char* cache;
  int tokens, n_slots, features, L, ld;
  int row_pieces, block_pieces;
  size_t row_bytes;
};

// A block takes some pieces of one token's rows, a warp one at a time: a piece lies in one row, so nothing
// of its addresses but a constant step changes on the way (with runs that go on from row to row, whose
// lanes each find their own row, the instructions bound these kernels).  Lanes take neighbouring pairs of
// words, 16 aligned bytes at a time: where the row starts off by one word, the words before and of an even
// column, and the lane before or behind has the other half of a pair.  (So the eight bytes before such a row
// are read, inside the 16 that its first word is in, and dropped; they are never written.)
//
// Words of three bytes go in groups of eight: lane k of the group's four has b_k, its pair's six bytes, and
// for k < 3 moves eight of the 24 bytes, s_k = b_k >> 16k | b_(k+1) << (48 - 16k).
template <int BYTES, bool WRITE>
__global__ void __launch_bounds__(32 * CH_WARPS, CH_BLOCKS)
    cache_kernel(const __grid_constant__ CacheArgs a) {
  using word = unsigned long long;
  constexpr int STEP = 64;  // words of a warp's turn
  constexpr int PIECE = WRITE ? CH_PIECE_WRITE : CH_PIECE_READ;
  constexpr int UP = 32 - 8 * BYTES;
  constexpr uint32_t HALF = BYTES == 4 ? 0u : 1u << (31 - 8 * BYTES);  // in the high half of a word
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 3;
  const long long pieces = (long long)a.features * a.row_pieces;
  const long long first = (long long)blockIdx.x * a.block_pieces;
  const int n = (int)min((long long)a.block_pieces, pieces - first);
  for (int t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    const int slot = __ldg(a.slots + t);
    if (WRITE) {  // of two tokens that name the same slot the later one stays
      bool skip = slot < 0 || slot >= a.n_slots;
      for (int i = t + 1 + (int)threadIdx.x; i < a.tokens; i += 32 * CH_WARPS)
        skip |= __ldg(a.slots + i) == slot;
      if (__syncthreads_or(skip)) continue;
    } else if (slot < 0 || slot >= a.n_slots) {
      continue;
    }
#pragma unroll 1
    for (int p = warp; p < n; p += CH_WARPS) {
      const long long f = (first + p) / a.row_pieces;
      const int c0 = (int)(first + p - f * a.row_pieces) * PIECE, c1 = min(a.L, c0 + PIECE);
      word* row = reinterpret_cast<word*>(WRITE ? const_cast<uint64_t*>(a.in) : a.out) +
                  ((size_t)t * a.features + f) * a.ld;
      unsigned char* cell = a.cache + ((size_t)slot * a.features + f) * a.row_bytes;
      const bool off = (uintptr_t)row & 8;  // (the same in all lanes)
      // the bytes of column c's pair, or of the eight that this lane moves of its group
      auto at = [&](int c) { return cell + (BYTES == 3 ? c / 8 * 24 + 8 * sub : c * BYTES); };
      auto moves = [&](int c) { return BYTES == 3 ? sub < 3 && c / 8 * 24 + 8 * sub < 3 * c1 : c < c1; };
      for (int c = c0 + 2 * lane; c - 2 * lane < c1; c += CH_AHEAD * STEP) {
        if (WRITE) {
          ulonglong2 x[CH_AHEAD];
#pragma unroll
          for (int j = 0; j < CH_AHEAD; ++j) {
            const int cj = c + j * STEP;
            x[j] = make_ulonglong2(0, 0);
            if (off) {
              if (cj < c1) x[j] = __ldcs(reinterpret_cast<const ulonglong2*>(row + cj - 1));
            } else if (cj + 1 < c1) {
              x[j] = __ldcs(reinterpret_cast<const ulonglong2*>(row + cj));
            } else if (cj < c1) {
              x[j].x = __ldcs(row + cj);
            }
          }
          if (off) {
            word more[CH_AHEAD];  // where the lane behind has not got it
#pragma unroll
            for (int j = 0; j < CH_AHEAD; ++j) {
              const int cj = c + j * STEP;
              more[j] = (lane == 31 || cj + 2 >= c1) && cj + 1 < c1 ? __ldcs(row + cj + 1) : 0;
            }
#pragma unroll
            for (int j = 0; j < CH_AHEAD; ++j) {
              const word behind = __shfl_down_sync(0xffffffffu, x[j].x, 1);
              x[j] = make_ulonglong2(
                  x[j].y, lane == 31 || c + j * STEP + 2 >= c1 ? more[j] : behind);
            }
          }
#pragma unroll
          for (int j = 0; j < CH_AHEAD; ++j) {
            const int cj = c + j * STEP;
            auto rounded = [](word v) {
              const uint32_t hi = (uint32_t)(v >> 32);
              return BYTES == 4 ? hi + ((uint32_t)v >> 31) : (hi + HALF) >> UP;
            };
            const uint32_t q0 = rounded(x[j].x), q1 = rounded(x[j].y);
            if constexpr (BYTES == 3) {
              const word b = q0 | (word)q1 << 24;
              const word next = __shfl_down_sync(0xffffffffu, b, 1);
              if (moves(cj))
                *reinterpret_cast<word*>(at(cj)) = b >> (16 * sub) | next << (48 - 16 * sub);
            } else if (moves(cj)) {  // (a second word behind the last goes to the row's padding)
              if constexpr (BYTES == 4)
                *reinterpret_cast<uint2*>(at(cj)) = make_uint2(q0, q1);
              else
                *reinterpret_cast<uint32_t*>(at(cj)) = q0 | q1 << 16;
            }
          }
        } else {
          word v[CH_AHEAD];
#pragma unroll
          for (int j = 0; j < CH_AHEAD; ++j) {
            v[j] = 0;
            if (moves(c + j * STEP)) {
              if constexpr (BYTES == 2)
                v[j] = __ldcs(reinterpret_cast<const uint32_t*>(at(c + j * STEP)));
              else
                v[j] = __ldcs(reinterpret_cast<const word*>(at(c + j * STEP)));
            }
          }
#pragma unroll
          for (int j = 0; j < CH_AHEAD; ++j) {
            const int cj = c + j * STEP;
            if constexpr (BYTES == 3) {
              const word before = __shfl_up_sync(0xffffffffu, v[j], 1);
              if (sub) v[j] = before >> (64 - 16 * sub) | v[j] << (16 * sub);
            }
            const uint32_t h0 = (uint32_t)v[j] << UP, h1 = (uint32_t)(v[j] >> (8 * BYTES)) << UP;
            const word y0 = (word)h0 << 32, y1 = (word)h1 << 32;
            if (off) {
              const uint32_t before = __shfl_up_sync(0xffffffffu, h1, 1);
              if (cj < c1) {
                if (lane)
                  __stcs(reinterpret_cast<ulonglong2*>(row + cj - 1),
                         make_ulonglong2((word)before << 32, y0));
                else
                  __stcs(row + cj, y0);
                if ((lane == 31 || cj + 2 >= c1) && cj + 1 < c1) __stcs(row + cj + 1, y1);
              }
            } else if (cj + 1 < c1) {
              __stcs(reinterpret_cast<ulonglong2*>(row + cj), make_ulonglong2(y0, y1));
            } else if (cj < c1) {
              __stcs(row + cj, y0);
            }
          }
        }
      }
    }
  }
}

size_t cache_row_bytes(int L, int bits) { return ((size_t)L * (bits / 8) + 15) / 16 * 16; }

template <bool WRITE>
static int cache_launch(CacheArgs a, int bits, cudaStream_t st) {
  a.row_bytes = cache_row_bytes(a.L, bits);
  constexpr int PIECE = WRITE ? CH_PIECE_WRITE : CH_PIECE_READ;
  a.row_pieces = (a.L + PIECE - 1) / PIECE;
  const long long pieces = (long long)a.features * a.row_pieces;
  // more pieces to a block where that leaves every multiprocessor its blocks
  const long long most = WRITE ? CH_PIECES_WRITE : CH_PIECES_READ;
  a.block_pieces = (int)std::max<long long>(
      CH_WARPS, std::min(most, pieces * a.tokens / (2 * CH_BLOCKS * 148)));
  const long long blocks = (pieces + a.block_pieces - 1) / a.block_pieces;
  if (blocks > 0x7fffffffLL) {
    set_error("%s: tokens of %d ciphertexts of %d words exceed one launch",
              WRITE ? "cache_write" : "cache_read", a.features, a.L);
    return PNB_ERR_INVALID;
  }
  const dim3 grid((unsigned)blocks, (unsigned)std::min(65535, a.tokens));
  if (bits == 16)
    cache_kernel<2, WRITE><<<grid, 32 * CH_WARPS, 0, st>>>(a);
  else if (bits == 24)
    cache_kernel<3, WRITE><<<grid, 32 * CH_WARPS, 0, st>>>(a);
  else
    cache_kernel<4, WRITE><<<grid, 32 * CH_WARPS, 0, st>>>(a);
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

// ---- rows without a place -----------------------------------------------------------------------
// Rows whose index is outside [0, limit) become zero: the others' blocks only look.  Of 512 rows of 2 MB
// none takes 4 us, 26 (54 MB) 29 and all 174, where filling the buffer before every call takes 157.
constexpr int ZS_THREADS = 256;

__global__ void __launch_bounds__(ZS_THREADS)
    zero_skipped_kernel(const int32_t* index, int rows, int limit, unsigned long long* out,
                        size_t words) {
  for (int t = blockIdx.y; t < rows; t += gridDim.y) {
    const int i = __ldg(index + t);
    if (i >= 0 && i < limit) continue;
    unsigned long long* row = out + (size_t)t * words;
    for (size_t c = (size_t)blockIdx.x * ZS_THREADS + threadIdx.x; c < words;
         c += (size_t)gridDim.x * ZS_THREADS)
      row[c] = 0;
  }
}

int zero_skipped(const int32_t* index, int rows, int limit, uint64_t* out, size_t words,
                 cudaStream_t st) {
  // blocks for every multiprocessor, of eight words a thread at least
  const size_t most = std::max(1, 16 * 148 / rows), all = words / (8 * ZS_THREADS) + 1;
  const dim3 grid((unsigned)std::min(most, all), (unsigned)std::min(65535, rows));
  zero_skipped_kernel<<<grid, ZS_THREADS, 0, st>>>(index, rows, limit, (unsigned long long*)out, words);
  PNB_CHECK_LAUNCH("zero_skipped_kernel");
  return PNB_OK;
}

}  // namespace pnb

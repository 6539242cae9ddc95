// tc_tiles.cuh -- what the contractions over limbs share (request.cu, group.cu): rings of shared-memory
// slots, limb sums, tiled tensor maps.
#pragma once
#include <cudaTypedefs.h>

#include "pnb_internal.cuh"
#include "tc_primitives.cuh"

namespace pnb {

PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder();

// A ring of slots: the current one and the parity of its use.
struct TileRing {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int slots) {
    if (++slot == slots) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// No load may still be landing when the block exits: the last use of each slot completes when it has
// landed (bounded; immediate unless a wait ran out).  `bars` are the ring's full barriers.
__device__ __forceinline__ void tile_drain(uint32_t bars, TileRing ring, bool wrapped, int slots,
                                           uint32_t limit) {
  for (int i = 0; i < slots; ++i)
    if (i < ring.slot)
      (void)tc::mbar_wait(bars + 8u * i, ring.phase, limit);
    else if (wrapped)
      (void)tc::mbar_wait(bars + 8u * i, ring.phase ^ 1u, limit);
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

// A tiled map of `rank` dimensions (strides of all but the first, in bytes).  No promotion to larger
// L2 reads: rows at an odd pitch would bring their neighbours' lines again (880 -> 790 us for 256 x
// 784->128 without it; even pitches show no difference).
inline int tile_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int rank,
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
inline CUtensorMapSwizzle tile_swizzle(int bytes) {
  return bytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
         : bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                       : CU_TENSOR_MAP_SWIZZLE_32B;
}

// Byte matrix [rows][cols] at a pitch, in boxes of box_cols bytes (one swizzle span) x box_rows.
inline int tile_map_bytes(CUtensorMap* map, const void* p, uint64_t cols, uint64_t rows,
                        uint64_t pitch, int box_cols, int box_rows) {
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  return tile_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p, 2, dims, strides, box,
                tile_swizzle(box_cols));
}
}  // namespace pnb

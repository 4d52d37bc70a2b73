// Pieces that the forward and the backward of attention over packed documents share.
#pragma once
#include "launch.cuh"
#include "packed.cuh"
#include "tc05.cuh"

#include <math_constants.h>
#include <string.h>

extern "C" void pb_count_launch(int n);

namespace pbv {

using namespace pb;
using pbk::Tile;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kChunkBytes = 128 * 128;  // 128 rows of 64 bf16 columns, 128-byte swizzle

// one MUFU instruction; very negative arguments flush to zero, which is what softmax wants
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 w = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&w);
}

// A warp's wait: every lane waits, all take the same branch.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// Loads a tile of 128 rows (kChunks chunks of 64 columns) for the whole warp.  A tile that reaches beyond its document
// (`valid` < 128 rows) also brings rows of the next one, and an Inf or NaN there would spread: 0 * NaN is NaN in the products
// that contract over these rows.  Such a tile is waited for here (on `aux`, whose phase the caller tracks), its foreign rows
// are cleared, and only then is `full` completed.  Happens once per document and operand.
template <int kChunks>
__device__ __forceinline__ bool load_tile(uint8_t* dst, const CUtensorMap* tm, uint64_t* full, uint64_t* aux,
                                          uint32_t* aux_phase, int col, int row, int valid, int lane,
                                          volatile int* abort_flag) {
  const bool whole = valid >= 128;
  uint64_t* bar = whole ? full : aux;
  if (lane == 0) {
    mbar_expect_tx(bar, kChunks * kChunkBytes);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) tma_load_2d(dst + c * kChunkBytes, tm, bar, col + c * 64, row);
  }
  __syncwarp();
  if (whole) return true;
  const bool ok = warp_wait(aux, *aux_phase, abort_flag);
  *aux_phase ^= 1;
  if (!ok) return false;
  // a row is 128 contiguous bytes of each chunk; the swizzle only permutes inside it
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
    for (int at = valid * 128 + lane * 16; at < kChunkBytes; at += 512)
      *reinterpret_cast<uint4*>(dst + c * kChunkBytes + at) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(full);
  return true;
}

// Zeros in rows [first, stop) x D columns of a padding tile; all threads of the block.
template <int D>
__device__ __forceinline__ void clear_rows(__nv_bfloat16* base, long long stride, long long first, int rows, int col) {
  constexpr int kVec = D / 8;
  for (int i = threadIdx.x; i < rows * kVec; i += blockDim.x)
    *reinterpret_cast<uint4*>(base + (first + i / kVec) * stride + col + (i % kVec) * 8) = make_uint4(0, 0, 0, 0);
}

// Frees TMEM after the last use; a block whose wait ran out first gives its copies in flight time to land.
__device__ __forceinline__ void leave(volatile int* abort_flag, int warp, uint32_t tmem_base) {
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);
  }
  tc_fence_after_sync();
  __syncwarp();
  if (warp == 1) tmem_dealloc<1>(tmem_base, 512);
}

}  // namespace pbv

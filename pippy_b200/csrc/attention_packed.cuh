// Pieces that the forward and the backward of attention over packed documents share.
#pragma once
#include "launch.cuh"
#include "packed.cuh"
#include "tc05.cuh"

#include <math_constants.h>
#include <string.h>

extern "C" void pb_count_launch(int n);
extern "C" int pb_device_sm_count();
extern "C" int pb_get_sm_reserve();

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

template <bool V>
struct Flag {
  static constexpr bool value = V;
};

// Moves registers between the warpgroups of a block: all four warps of a warpgroup call it, and over the block the shares add
// up to no more than what it was launched with (threads x registers each), or the increase would wait for good.
template <int N>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// A warp's wait: every lane waits, all take the same branch.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

// ------------------------------------------------------------------------------------------------ pairs of fp32 values
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// One MUFU instruction each.  (A polynomial on the FMA pipe for a quarter or a half of them, degree 4 in pairs, was slower in
// every kernel here: the softmax warps wait for their own chain of instructions, not for the special-function unit.)
__device__ __forceinline__ f32x2 exp2_pair(f32x2 x) {
  const float2 v = both(x);
  return pair(fast_exp2(v.x), fast_exp2(v.y));
}

// ------------------------------------------------------------------------------------------------ tiles
// Issues the load of a tile of 128 rows (kChunks chunks of 64 columns); one thread.
template <int kChunks>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* tm, uint64_t* bar, int col, int row) {
  mbar_expect_tx(bar, kChunks * kChunkBytes);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) tma_load_2d(dst + c * kChunkBytes, tm, bar, col + c * 64, row);
}

// A tile that reaches beyond its document (`valid` < 128 rows) also brings rows of the next one, and an Inf or NaN there would
// spread: 0 * NaN is NaN in the products that contract over these rows.  So it is loaded against a barrier of its own
// (`raw`), on which a warp waits that clears the foreign rows and only then completes `full`.  A row is 128
// contiguous bytes of each chunk; the swizzle only permutes inside it.
template <int kChunks>
__device__ __forceinline__ void clear_tail(uint8_t* tile, int valid, uint64_t* full, int lane) {
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
    for (int at = valid * 128 + lane * 16; at < kChunkBytes; at += 512)
      *reinterpret_cast<uint4*>(tile + c * kChunkBytes + at) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(full);
}

// The blocks of a launch stay and take the work items i = 0, 1, ... (tile of the table, head; longest first): from a counter,
// which begins at 0, whenever they have loaded what the present item needs; without a counter in turns, every other turn
// in reverse, so that no block gets the longer item of every turn.  The results do not depend on who takes what.  One warp
// of a block calls next().
struct Items {
  int n, turn;
  int* counter;
  __device__ __forceinline__ Items(int count, int* counter_) : n(count), turn(-1), counter(counter_) {}
  // next item of this block, -1 after the last
  __device__ __forceinline__ int next(int lane) {
    ++turn;
    int i;
    if (turn == 0 || counter == nullptr) {
      const long long first = (long long)turn * gridDim.x;
      if (first >= n) return -1;
      i = (int)first + ((turn & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
    } else {
      i = lane == 0 ? (int)gridDim.x + atomicAdd(counter, 1) : 0;
      i = __shfl_sync(0xffffffffu, i, 0);
    }
    return i < n ? i : -1;
  }
};

// Zeros in `rows` rows x D columns of a padding tile, by `threads` threads.
template <int D>
__device__ __forceinline__ void clear_rows(__nv_bfloat16* base, long long stride, long long first, int rows, int col,
                                           int thread, int threads) {
  constexpr int kVec = D / 8;
  for (int i = thread; i < rows * kVec; i += threads)
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

// The loading warp decodes an item (a read of the table, three divisions: 1 000 cycles and more) ahead of the others and hands it
// on through shared memory; they take 100 cycles to get it.
struct ItemRing {
  static constexpr int kDepth = 4, kBytes = kDepth * 48, kBars = 2 * kDepth;
  int4* data;  // [kDepth][3]
  uint64_t *full, *empty;
  int n = 0;
  __device__ __forceinline__ ItemRing(uint8_t* mem, uint64_t* bars)
      : data(reinterpret_cast<int4*>(mem)), full(bars), empty(bars + kDepth) {}
  __device__ __forceinline__ void init(int readers) {
    for (int i = 0; i < kDepth; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], readers);
    }
  }
  __device__ __forceinline__ bool put(int4 a, int4 b, int4 c, int lane, volatile int* abort_flag) {
    const int s = n % kDepth;
    if (!warp_wait(&empty[s], ((n / kDepth) & 1) ^ 1, abort_flag)) return false;
    if (lane == 0) {
      data[s * 3] = a, data[s * 3 + 1] = b, data[s * 3 + 2] = c;
      mbar_arrive(&full[s]);
    }
    ++n;
    return true;
  }
  __device__ __forceinline__ bool get(int4& a, int4& b, int4& c, int lane, volatile int* abort_flag) {
    const int s = n % kDepth;
    if (!warp_wait(&full[s], (n / kDepth) & 1, abort_flag)) return false;
    a = data[s * 3], b = data[s * 3 + 1], c = data[s * 3 + 2];
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
    ++n;
    return true;
  }
};

// Blocks of a launch that stays resident: one per SM that is not reserved for others, no more than there are items.
inline unsigned resident_blocks(long long items) {
  int sms = pb_device_sm_count() - pb_get_sm_reserve();
  if (sms < 1) sms = 1;
  return (unsigned)(items < sms ? items : sms);
}

// Whether a launch takes its items from a counter: not for two turns of them or fewer, which it cannot balance much, and
// clearing it may take a launch of its own.
inline bool takes_from_counter(long long items) { return items > 2LL * resident_blocks(items); }

}  // namespace pbv

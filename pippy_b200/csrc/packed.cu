// Documents of different lengths packed into rows of equal length: the layout (positions and tile tables, from the lengths
// alone, on the device) and rotary embedding by position.
#include "launch.cuh"
#include "packed.cuh"

#include <cuda_bf16.h>
#include <stdint.h>

extern "C" void pb_count_launch(int n);

namespace pbk {

// Tiles are listed longest first: tile `rank` of a document sees rank + 1 tiles of keys (as a tile of keys it is seen by as
// many tiles of queries when counted from the document's end), and a long tile that starts last runs alone at the end.
// Ranks above the last bucket share it; they are all long.  Behind rank 0 come the documents of 128 tokens
// or fewer (the attention forward takes two heads of such a one at a time, its backward has a kernel for them), and then
// the padding.
constexpr int kRanks = 2048;
constexpr int kBuckets = kRanks + 1;  // the last one; padding's is kBuckets
constexpr int kCounters = kBuckets + 1;
constexpr int kPlanThreads = 1024;
constexpr int kChunk = 4096;  // tokens a block writes positions for

struct LayoutArgs {
  const int* lengths;  // [rows, docs]
  int rows, docs, seq;
  int* positions;  // [rows * seq]
  int2* segments;  // [rows * (docs + 1)]: start, length; the last of a row is its padding
  Tile* tiles[2];  // of 128 and of 256 rows
  int max_tiles[2];
  int* counts;  // [table][all, those before the half-filled ones, those before the padding]
  int* err;
};

// A document's length as the layout uses it: inside what its row has left.  One warp walks a row, 32 documents a step.
struct RowWalk {
  long long at = 0;  // rows used so far, as given (may exceed the row)
  __device__ int2 step(int raw, int seq, int lane, bool* bad) {
    const long long len = raw < 0 ? 0 : raw;
    long long upto = len;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long below = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += below;
    }
    const long long first = at + upto - len;
    at += __shfl_sync(0xffffffffu, upto, 31);
    const int start = (int)(first < seq ? first : seq);
    const int kept = (int)(len < seq - start ? len : seq - start);
    if (raw < 0 || kept != len) *bad = true;
    return make_int2(start, kept);
  }
};

__device__ void plan_tiles(const LayoutArgs& a, int* s_hist, int* s_part) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  bool bad = false;
  for (int row = warp; row < a.rows; row += warps) {
    RowWalk walk;
    int2* out = a.segments + (long long)row * (a.docs + 1);
    for (int d0 = 0; d0 < a.docs; d0 += 32) {
      const int raw = d0 + lane < a.docs ? a.lengths[(long long)row * a.docs + d0 + lane] : 0;
      const int2 seg = walk.step(raw, a.seq, lane, &bad);
      if (d0 + lane < a.docs) out[d0 + lane] = make_int2(row * a.seq + seg.x, seg.y);
    }
    const int used = (int)(walk.at < a.seq ? walk.at : a.seq);
    if (lane == 0) out[a.docs] = make_int2(row * a.seq + used, a.seq - used);
  }
  if (bad) atomicExch(a.err, ERR_LAYOUT);
  __syncthreads();
  // Both tables at once: count the tiles of every bucket, sum the counts up, place the tiles.  A thread has a document; the
  // tiles of a long one are shared by its warp.
  const int nseg = a.rows * (a.docs + 1);
  for (int i = tid; i < 2 * kCounters; i += blockDim.x) s_hist[i] = 0;
  __syncthreads();
  for (int sweep = 0; sweep < 2; ++sweep) {
    auto add = [&](int table, int start, int len, int r, bool pad) {
      const bool half = len <= 128;
      const int bucket = pad ? kBuckets : (half ? kRanks : kRanks - 1 - min(r, kRanks - 1));  // high ranks first
      const int at = atomicAdd(&s_hist[table * kCounters + bucket], 1);
      if (sweep == 1 && at < a.max_tiles[table]) a.tiles[table][at] = Tile{start, len, r, pad ? 1 : 0};
    };
    for (int i0 = warp * 32; i0 < nseg; i0 += blockDim.x) {
      const int i = i0 + lane;
      const int2 seg = i < nseg ? a.segments[i] : make_int2(0, 0);
      const bool pad = i % (a.docs + 1) == a.docs, is_long = seg.y > 512;
      if (!is_long) {
        for (int r = 0; r * 128 < seg.y; ++r) add(0, seg.x, seg.y, r, pad);
        for (int r = 0; r * 256 < seg.y; ++r) add(1, seg.x, seg.y, r, pad);
      }
      for (unsigned left = __ballot_sync(0xffffffffu, is_long); left; left &= left - 1) {
        const int from = __ffs(left) - 1;
        const int start = __shfl_sync(0xffffffffu, seg.x, from), len = __shfl_sync(0xffffffffu, seg.y, from);
        const bool its_pad = (i0 + from) % (a.docs + 1) == a.docs;
        for (int r = lane; (long long)r * 128 < len; r += 32) add(0, start, len, r, its_pad);
        for (int r = lane; (long long)r * 256 < len; r += 32) add(1, start, len, r, its_pad);
      }
    }
    __syncthreads();
    if (sweep == 0) {  // counts -> first places: an exclusive sum for each table, by half of the warps, a run of counters a thread
      const int table = warp / (warps / 2), mine = tid - table * (kPlanThreads / 2);
      int* hist = s_hist + table * kCounters;
      const int per = (kCounters + kPlanThreads / 2 - 1) / (kPlanThreads / 2);
      int sum = 0;
      for (int k = 0; k < per; ++k)
        if (mine * per + k < kCounters) sum += hist[mine * per + k];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
      }
      if (lane == 31) s_part[warp] = upto;
      __syncthreads();
      int base = upto - sum;
      for (int k = table * (warps / 2); k < warp; ++k) base += s_part[k];
      for (int k = 0; k < per; ++k) {
        const int i = mine * per + k;
        if (i < kCounters) {
          const int n = hist[i];
          hist[i] = base;
          base += n;
        }
      }
      if (mine == kPlanThreads / 2 - 1) a.counts[table * 4] = min(base, a.max_tiles[table]);
      __syncthreads();
      if (mine == 0) {
        a.counts[table * 4 + 1] = min(hist[kRanks], a.max_tiles[table]);
        a.counts[table * 4 + 2] = min(hist[kBuckets], a.max_tiles[table]);
      }
      __syncthreads();
    }
  }
}

// Block 0 plans the tiles, the others write the positions of kChunk tokens of one row each.  The lengths stay on
// the device, so that nothing waits for the host.  Bound by block 0's chain of phases: 7 us for 333 tokens in one row, 11 for 16
// rows of 2047.
__global__ void __launch_bounds__(kPlanThreads) layout_kernel(LayoutArgs a) {
  __shared__ int s_hist[2 * kCounters];
  __shared__ int s_part[kPlanThreads / 32];
  pb::let_next_start();
  if (blockIdx.x == 0) {
    plan_tiles(a, s_hist, s_part);
    return;
  }
  const int chunks = (a.seq + kChunk - 1) / kChunk;
  const int row = (blockIdx.x - 1) / chunks;
  const int t0 = (blockIdx.x - 1 - row * chunks) * kChunk, t1 = min(t0 + kChunk, a.seq);
  int* out = a.positions + (long long)row * a.seq;
  // every warp walks the row's documents and fills its share of those that meet this block's tokens
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  RowWalk walk;
  bool bad = false;  // reported by block 0
  for (int d0 = 0; d0 < a.docs && walk.at < t1; d0 += 32) {
    const int raw = d0 + lane < a.docs ? a.lengths[(long long)row * a.docs + d0 + lane] : 0;
    const int2 seg = walk.step(raw, a.seq, lane, &bad);
    for (int i = 0; i < 32; ++i) {
      const int start = __shfl_sync(0xffffffffu, seg.x, i), len = __shfl_sync(0xffffffffu, seg.y, i);
      for (int t = max(start, t0) + warp * 32 + lane; t < min(start + len, t1); t += warps * 32) out[t] = t - start;
    }
  }
  const int used = (int)(walk.at < a.seq ? walk.at : a.seq);
  for (int t = max(used, t0) + warp * 32 + lane; t < t1; t += warps * 32) out[t] = -1;
}

// Rotates the first `heads` heads of every row ("rotate-half" pairing: element i with i + D / 2) by the row's position;
// rows at position -1 (padding) are copied.  src and dst may be the same memory: a thread reads the 32 bytes that it
// writes.  A block takes one row at a time, its threads the 16-byte vectors of half heads; rows are stepped by the grid, so
// that no index is divided.  The turned values are rounded to bf16, the type that the products take them in.  Bound by
// bandwidth, one read and one write: 41 us for 8192 tokens of 64 heads of 128 elements, 6.5 TB/s.
__global__ void __launch_bounds__(256) packed_rope_kernel(const __nv_bfloat16* src, long long src_stride,
                                                          __nv_bfloat16* dst, long long dst_stride,
                                                          const float* __restrict__ cs, const float* __restrict__ sn,
                                                          const int* __restrict__ positions, long long T, int heads,
                                                          int half, int table_rows, int* clear, int* err) {
  const int per_head = half / 8, n = heads * per_head;
  pb::after_previous();
  pb::let_next_start();
  if (clear && blockIdx.x == 0 && threadIdx.x == 0) *clear = 0;
  for (long long t = blockIdx.x; t < T; t += gridDim.x) {
    int pos = positions[t];
    if (pos >= table_rows) {
      if (threadIdx.x == 0) atomicExch(err, ERR_INDEX);
      pos = -1;
    }
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int h = i / per_head, v = (i - h * per_head) * 8;
      const long long col = (long long)h * 2 * half + v;
      const uint4 lo = *reinterpret_cast<const uint4*>(src + t * src_stride + col);
      const uint4 hi = *reinterpret_cast<const uint4*>(src + t * src_stride + col + half);
      uint4 ro = lo, rh = hi;
      if (pos >= 0) {
        const float4* cp = reinterpret_cast<const float4*>(cs + (long long)pos * half + v);
        const float4* sp = reinterpret_cast<const float4*>(sn + (long long)pos * half + v);
        const __nv_bfloat162* a = reinterpret_cast<const __nv_bfloat162*>(&lo);
        const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&hi);
        __nv_bfloat162* oa = reinterpret_cast<__nv_bfloat162*>(&ro);
        __nv_bfloat162* ob = reinterpret_cast<__nv_bfloat162*>(&rh);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 c = __ldg(cp + j), s = __ldg(sp + j);
          const float2 a0 = __bfloat1622float2(a[2 * j]), a1 = __bfloat1622float2(a[2 * j + 1]);
          const float2 b0 = __bfloat1622float2(b[2 * j]), b1 = __bfloat1622float2(b[2 * j + 1]);
          oa[2 * j] = __floats2bfloat162_rn(a0.x * c.x - b0.x * s.x, a0.y * c.y - b0.y * s.y);
          oa[2 * j + 1] = __floats2bfloat162_rn(a1.x * c.z - b1.x * s.z, a1.y * c.w - b1.y * s.w);
          ob[2 * j] = __floats2bfloat162_rn(b0.x * c.x + a0.x * s.x, b0.y * c.y + a0.y * s.y);
          ob[2 * j + 1] = __floats2bfloat162_rn(b1.x * c.z + a1.x * s.z, b1.y * c.w + a1.y * s.w);
        }
      }
      *reinterpret_cast<uint4*>(dst + t * dst_stride + col) = ro;
      *reinterpret_cast<uint4*>(dst + t * dst_stride + col + half) = rh;
    }
  }
}

}  // namespace pbk

extern "C" {

// lengths [rows, docs] -> positions [rows * seq] (-1 in padding), segments [rows * (docs + 1)] pairs, tile tables of 128 and
// 256 rows (max128 / max256 entries of 4 ints; the host takes an upper bound), counts [2][4].
int pb_packed_layout(const int* lengths, int rows, int docs, int seq, int* positions, int* segments, int* tiles128,
                     int max128, int* tiles256, int max256, int* counts, int* err_dev, void* stream_) {
  using namespace pbk;
  if (rows < 1 || docs < 0 || seq < 1) return -1;
  const long long blocks = 1 + (long long)rows * ((seq + kChunk - 1) / kChunk);
  // half of the range, so that a token's number plus a block's step is one of 32 bits too
  if ((long long)rows * seq > 0x3fffffffLL || (long long)rows * (docs + 1) > 0x3fffffffLL || blocks > 0x3fffffffLL) return -2;
  LayoutArgs a;
  a.lengths = lengths;
  a.rows = rows, a.docs = docs, a.seq = seq;
  a.positions = positions;
  a.segments = reinterpret_cast<int2*>(segments);
  a.tiles[0] = reinterpret_cast<Tile*>(tiles128), a.tiles[1] = reinterpret_cast<Tile*>(tiles256);
  a.max_tiles[0] = max128, a.max_tiles[1] = max256;
  a.counts = counts;
  a.err = err_dev;
  layout_kernel<<<(unsigned)blocks, kPlanThreads, 0, reinterpret_cast<cudaStream_t>(stream_)>>>(a);
  pb_count_launch(1);
  return (int)cudaGetLastError();
}

// clear: a word that is set to 0 on the way, may be null.
int pb_packed_rope(const void* src, long long src_stride, void* dst, long long dst_stride, const float* cs,
                   const float* sn, const int* positions, long long T, int heads, int D, int table_rows, int* clear,
                   int* err_dev, void* stream_) {
  using namespace pbk;
  if (D % 16 != 0 || src_stride % 8 != 0 || dst_stride % 8 != 0) return -1;
  if ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(cs) |
       reinterpret_cast<uintptr_t>(sn)) & 15)
    return -2;
  if (T == 0) return 0;
  const unsigned grid = (unsigned)(T < 148 * 16 ? T : 148 * 16);
  pb_count_launch(1);
  return (int)pb::launch_chained(packed_rope_kernel, grid, 256, 0, reinterpret_cast<cudaStream_t>(stream_),
                                 reinterpret_cast<const __nv_bfloat16*>(src), src_stride, reinterpret_cast<__nv_bfloat16*>(dst),
                                 dst_stride, cs, sn, positions, T, heads, D / 2, table_rows, clear, err_dev);
}

}  // extern "C"

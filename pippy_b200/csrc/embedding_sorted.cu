// Scaled token (+ position) embedding with positions given per token, and its gradient by sorted tokens.
//
//   out[t] = scale * wte[ids[t]] + wpe[pos[t]]         (no second term where pos[t] = -1)
//   dwte[v] = scale * sum of dout[t] over ids[t] = v,  dwpe[p] = sum of dout[t] over pos[t] = p
//
// The sums are formed in the order of t: the same bits on every run, and a token that fills a third of the batch costs no
// contended atomics.  Three launches: the tokens are sorted (stable radix sort, one cluster per table), tiles of the sorted
// order sum their runs of equal tokens, and runs that cross tiles are folded from the tiles' partial sums.
#include "launch.cuh"
#include "packed.cuh"
#include "tc05.cuh"

#include <cuda_bf16.h>
#include <stdint.h>
#include <string.h>

extern "C" void pb_count_launch(int n);

namespace pbs {

using pbk::ERR_INDEX;

// ------------------------------------------------------------------------------------------------ forward
// One row per threadIdx.y and step, 16-byte vectors along threadIdx.x: no index is divided.  Bound by bandwidth:
// 17 us for 8192 tokens of 4096 columns.
__global__ void __launch_bounds__(256) embed_scaled_kernel(const long long* __restrict__ ids,
                                                           const __nv_bfloat16* __restrict__ wte,
                                                           const __nv_bfloat16* __restrict__ wpe,
                                                           const int* __restrict__ positions, int seq,
                                                           __nv_bfloat16* __restrict__ out, long long T, int vec,
                                                           long long vocab, int n_positions, float scale, int* err) {
  for (long long t = blockIdx.x * (long long)blockDim.y + threadIdx.y; t < T; t += (long long)gridDim.x * blockDim.y) {
    const long long id = ids[t];
    int pos = wpe ? (positions ? positions[t] : (int)(t % seq)) : -1;
    const bool id_ok = id >= 0 && id < vocab;
    if (!id_ok || pos >= n_positions) {
      if (threadIdx.x == 0) atomicExch(err, ERR_INDEX);
      if (pos >= n_positions) pos = -1;
    }
    const uint4* row = reinterpret_cast<const uint4*>(wte) + (id_ok ? id : 0) * vec;
    const uint4* prow = reinterpret_cast<const uint4*>(wpe) + (long long)(pos < 0 ? 0 : pos) * vec;
    uint4* orow = reinterpret_cast<uint4*>(out) + t * vec;
    for (int v = threadIdx.x; v < vec; v += blockDim.x) {
      uint4 a = id_ok ? __ldg(row + v) : make_uint4(0, 0, 0, 0);
      uint4 p = pos >= 0 ? __ldg(prow + v) : make_uint4(0, 0, 0, 0);
      __nv_bfloat162* ab = reinterpret_cast<__nv_bfloat162*>(&a);
      const __nv_bfloat162* pb = reinterpret_cast<const __nv_bfloat162*>(&p);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = __bfloat1622float2(ab[j]), y = __bfloat1622float2(pb[j]);
        ab[j] = __floats2bfloat162_rn(x.x * scale + y.x, x.y * scale + y.y);
      }
      orow[v] = a;
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort
constexpr int kCluster = 8;
constexpr int kSortThreads = 1024;
constexpr int kWarps = kSortThreads / 32;

struct Table {
  const long long* ids;  // keys: 64-bit token ids, else 32-bit positions, else t % seq
  const int* positions;
  int seq;
  int size;      // rows of the table; keys outside [0, size) are sorted last and summed into nothing
  int2* sorted;  // [T] (key, t), by key and then by t
  int2* other;   // [T] the passes' second buffer
  float* partial;      // [2 * tiles, H]: sums of the runs that enter and that leave a tile
  int* crossing;       // tiles in which a run begins that leaves them
  int* n_crossing;     // how many
  void* grad;          // [size, H]: fp32, added to, or bf16, written whole
  float scale;
};
struct SortArgs {
  Table table[2];
  int tables;
  long long T;
  int H;
  int write;  // bf16 gradient, written whole: the blocks that do not sort clear it meanwhile
};

__device__ __forceinline__ uint32_t load_cluster(const uint32_t* local, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(pb::mapa_u32(pb::smem_u32(local), rank)) : "memory");
  return v;
}

// Stable least-significant-digit radix sort of (key, t), 8 bits a pass at most: 2 passes up to 65 535 rows.  A cluster of 8
// blocks holds the counters in shared memory and steps from phase to phase on cluster barriers, 2 per pass, where a
// grid would need launches.  Every warp owns a contiguous run of the block's run, so that ranks follow the order of t.  Bound by
// latency, not by bytes: 13 us for 2048 tokens and two tables, 22 for 32 752.
__device__ void sort_table(const SortArgs& a, const Table& tb, uint32_t* s_hist, uint32_t* s_total, uint32_t* s_base,
                           uint32_t* s_scan) {
  const uint32_t rank = pb::cluster_ctarank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t below = (1u << lane) - 1;
  uint32_t* hist = s_hist + warp * 256;
  const int bits = 32 - __clz(tb.size);  // keys 0..size
  const int passes = (bits + 7) / 8, per = (bits + passes - 1) / passes;
  const uint32_t mask = (1u << per) - 1;
  const long long share = (a.T + kCluster * kWarps - 1) / (kCluster * kWarps);
  const long long per_warp = (share + 31) / 32 * 32;
  const long long begin = ((long long)rank * kWarps + warp) * per_warp;
  const long long end = begin + per_warp < a.T ? begin + per_warp : a.T;
  auto entry = [&](int pass, long long i) -> int2 {
    if (pass > 0) return __ldcg(((passes - pass) & 1 ? tb.other : tb.sorted) + i);
    long long key = tb.ids ? tb.ids[i] : (tb.positions ? (long long)tb.positions[i] : i % tb.seq);
    if (key < 0 || key >= tb.size) key = tb.size;
    return make_int2((int)key, (int)i);
  };
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * per;
    int2* out = (passes - 1 - pass) & 1 ? tb.other : tb.sorted;
    for (int i = lane; i < 256; i += 32) hist[i] = 0;
    __syncwarp();
    for (long long i0 = begin; i0 < end; i0 += 128) {  // four loads in flight
      int2 e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) e[u] = i0 + u * 32 + lane < end ? entry(pass, i0 + u * 32 + lane) : make_int2(0, -1);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t d = e[u].y >= 0 ? ((uint32_t)e[u].x >> shift) & mask : 256u;
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        if (d < 256 && (same & below) == 0) hist[d] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t run = 0;
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t n = s_hist[w * 256 + tid];
        s_hist[w * 256 + tid] = run;
        run += n;
      }
      s_total[tid] = run;
    }
    pb::cluster_sync_all();
    uint32_t all = 0, before = 0, upto = 0;
    if (tid < 256) {
      for (uint32_t c = 0; c < kCluster; ++c) {
        const uint32_t n = load_cluster(s_total + tid, c);
        all += n;
        if (c < rank) before += n;
      }
      upto = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      if (lane == 31) s_scan[warp] = upto;
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t first = upto - all;
      for (int w = 0; w < warp; ++w) first += s_scan[w];
      s_base[tid] = first + before;
    }
    __syncthreads();
    for (long long i0 = begin; i0 < end; i0 += 128) {
      int2 e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) e[u] = i0 + u * 32 + lane < end ? entry(pass, i0 + u * 32 + lane) : make_int2(0, -1);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t d = e[u].y >= 0 ? ((uint32_t)e[u].x >> shift) & mask : 256u;
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        uint32_t at = 0;
        if (d < 256) at = s_base[d] + hist[d] + __popc(same & below);
        __syncwarp();
        if (d < 256 && (same & below) == 0) hist[d] += __popc(same);
        __syncwarp();
        if (d < 256) out[at] = e[u];
      }
    }
    pb::cluster_sync_all();  // the next pass reads what the cluster's other blocks wrote, and reuses the counters
  }
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kSortThreads, 1) embed_sort_kernel(SortArgs a) {
  __shared__ uint32_t s_hist[kWarps * 256];
  __shared__ uint32_t s_total[256], s_base[256], s_scan[8];
  const int cluster = blockIdx.x / kCluster;
  pb::let_next_start();
  if (cluster < a.tables) {
    if (blockIdx.x % kCluster == 0 && threadIdx.x == 0) *(cluster == 0 ? a.table[0] : a.table[1]).n_crossing = 0;
    sort_table(a, cluster == 0 ? a.table[0] : a.table[1], s_hist, s_total, s_base, s_scan);
    return;
  }
  // the other blocks clear; writes alone run at 3.7 TB/s here, with plain stores and with bulk copies alike
  const long long at = (blockIdx.x - a.tables * kCluster) * (long long)blockDim.x + threadIdx.x;
  const long long step = (long long)(gridDim.x - a.tables * kCluster) * blockDim.x;
  for (int k = 0; k < a.tables; ++k) {
    uint4* grad = reinterpret_cast<uint4*>(a.table[k].grad);
    const long long n = (long long)a.table[k].size * a.H / 8;
    for (long long i = at; i < n; i += step) grad[i] = make_uint4(0, 0, 0, 0);
  }
}

// ------------------------------------------------------------------------------------------------ sums of runs
constexpr int kMaxTile = 64;

__device__ __forceinline__ void put_row(const SortArgs& a, const Table& tb, long long key, int col, const float* sum) {
  if (a.write) {
    uint4 w;
    __nv_bfloat162* b = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = __floats2bfloat162_rn(sum[2 * j] * tb.scale, sum[2 * j + 1] * tb.scale);
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(tb.grad) + key * a.H + col) = w;
  } else {
    // An addition that memory makes: the thread need not wait for what is there.  Each element gets one in a launch, so there
    // is no order that could matter.
    float4* g = reinterpret_cast<float4*>(reinterpret_cast<float*>(tb.grad) + key * a.H + col);
    atomicAdd(g, make_float4(sum[0] * tb.scale, sum[1] * tb.scale, sum[2] * tb.scale, sum[3] * tb.scale));
    atomicAdd(g + 1, make_float4(sum[4] * tb.scale, sum[5] * tb.scale, sum[6] * tb.scale, sum[7] * tb.scale));
  }
}

// A block sums one tile of the sorted order for 1024 columns, 8 per thread, with eight rows' loads in flight.  A run inside the
// tile is a finished row of the gradient; one that enters or leaves it becomes a partial sum in fp32.  27 us for 32 752
// tokens of 1024 columns and two tables (39 when a thread waited for the row that it adds to).
__global__ void __launch_bounds__(128) embed_runs_kernel(SortArgs a, const __nv_bfloat16* __restrict__ dout, int tile_rows) {
  const Table& tb = blockIdx.z == 0 ? a.table[0] : a.table[1];
  __shared__ int s_key[kMaxTile + 2], s_tok[kMaxTile];
  const long long t0 = (long long)blockIdx.x * tile_rows;
  const int n = (int)(a.T - t0 < tile_rows ? a.T - t0 : tile_rows);
  pb::after_previous();
  pb::let_next_start();
  for (int i = threadIdx.x; i < n + 2; i += blockDim.x) {  // one neighbour on each side
    const long long t = t0 - 1 + i;
    const int2 e = t >= 0 && t < a.T ? tb.sorted[t] : make_int2(-1, 0);
    s_key[i] = e.x;
    if (i >= 1 && i <= n) s_tok[i - 1] = e.y;
  }
  __syncthreads();
  if (blockIdx.y == 0 && threadIdx.x == 0) {
    // the last key goes on in the next tile, is one of the table's and did not enter this tile
    const int key = s_key[n];
    if (key < tb.size && s_key[n + 1] == key && !(s_key[1] == key && s_key[0] == key))
      tb.crossing[atomicAdd(tb.n_crossing, 1)] = blockIdx.x;
  }
  const int col = (blockIdx.y * 128 + threadIdx.x) * 8;
  if (col >= a.H) return;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  bool entered = s_key[0] == s_key[1];
  for (int r0 = 0; r0 < n; r0 += 8) {
    uint4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = r0 + u < n && s_key[r0 + u + 1] < tb.size
                 ? __ldg(reinterpret_cast<const uint4*>(dout + (long long)s_tok[r0 + u] * a.H + col))
                 : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int r = r0 + u;
      if (r >= n) break;
      const int key = s_key[r + 1];
      if (key >= tb.size) return;  // sorted last: nothing but such keys from here on
      const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&v[u]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(b[j]);
        acc[2 * j] += f.x, acc[2 * j + 1] += f.y;
      }
      const bool last = r + 1 == n;
      const bool goes_on = s_key[r + 2] == key;
      if (last ? true : !goes_on) {
        if (entered || goes_on) {
          float4* p = reinterpret_cast<float4*>(tb.partial + ((long long)blockIdx.x * 2 + (entered ? 0 : 1)) * a.H + col);
          p[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
          p[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        } else {
          put_row(a, tb, key, col, acc);
        }
        entered = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.f;
      }
    }
  }
}

// A run that crosses tiles: the last partial sum of the tile that it begins in and the first ones of the tiles after it, in
// order.  The list's order is not that of the keys, but each run has a row of its own.  A warp takes a run that ends within 32
// tiles; a longer one is left to the block, whose warps look for its end together and take consecutive shares.  10 us for 8192 tokens of 4096 columns;
// 25 where a third of 32 752 tokens is one id.
constexpr int kFoldWarps = 8;

__global__ void __launch_bounds__(32 * kFoldWarps) embed_fold_kernel(SortArgs a, int tile_rows) {
  const Table& tb = blockIdx.z == 0 ? a.table[0] : a.table[1];
  const long long tiles = (a.T + tile_rows - 1) / tile_rows;
  const int lane = threadIdx.x, y = threadIdx.y;
  const int col = (blockIdx.y * 32 + lane) * 8;
  __shared__ float s_acc[kFoldWarps][32][9];
  __shared__ int s_long[kFoldWarps];
  pb::after_previous();
  const int runs = *tb.n_crossing;
  float acc[8];
  auto clear = [&]() {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  };
  auto add = [&](long long t, int which) {
    const float4* p = reinterpret_cast<const float4*>(tb.partial + (t * 2 + which) * a.H + col);
    const float4 lo = p[0], hi = p[1];
    acc[0] += lo.x, acc[1] += lo.y, acc[2] += lo.z, acc[3] += lo.w;
    acc[4] += hi.x, acc[5] += hi.y, acc[6] += hi.z, acc[7] += hi.w;
  };
  for (int r0 = blockIdx.x * kFoldWarps; r0 < runs; r0 += gridDim.x * kFoldWarps) {
    bool is_long = false;
    if (r0 + y < runs) {
      const long long tile = tb.crossing[r0 + y];
      const long long t = tile + 1 + lane;
      const int mine = t < tiles ? tb.sorted[t * tile_rows].x : -1, key = __shfl_sync(0xffffffffu, mine, 0);
      const unsigned same = __ballot_sync(0xffffffffu, mine == key);  // keys are in order: the run's tiles come first
      is_long = same == 0xffffffffu;
      if (!is_long && col < a.H) {
        clear();
        add(tile, 1);
        const int more = __popc(same);
#pragma unroll 8
        for (int k = 1; k <= more; ++k) add(tile + k, 0);
        put_row(a, tb, key, col, acc);
      }
    }
    if (lane == 0) s_long[y] = is_long;
    __syncthreads();
    for (int w = 0; w < kFoldWarps; ++w) {
      if (!s_long[w]) continue;
      const long long tile = tb.crossing[r0 + w];
      const int key = tb.sorted[(tile + 1) * tile_rows].x;
      long long more = 0;  // tiles after this one that the run reaches
      for (int got = 32 * kFoldWarps; got == 32 * kFoldWarps; more += got) {
        const long long t = tile + 1 + more + y * 32 + lane;
        got = __syncthreads_count(t < tiles && tb.sorted[t * tile_rows].x == key);
      }
      clear();
      if (col < a.H) {
        if (y == 0) add(tile, 1);
        const long long share = (more + kFoldWarps - 1) / kFoldWarps;
        const long long first = tile + 1 + y * share, stop = min(first + share, tile + 1 + more);
#pragma unroll 8
        for (long long t = first; t < stop; ++t) add(t, 0);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s_acc[y][lane][j] = acc[j];
      __syncthreads();
      if (y == 0 && col < a.H) {
        for (int k = 1; k < kFoldWarps; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += s_acc[k][lane][j];
        put_row(a, tb, key, col, acc);
      }
      __syncthreads();
    }
    __syncthreads();  // before s_long is written again
  }
}

// Rows of the sorted order per tile.  Larger tiles leave fewer partial sums, smaller ones more blocks.
static int tile_rows_for(long long T, int H) {
  const long long slabs = (H / 8 + 127) / 128;
  for (int rows = kMaxTile; rows > 16; rows /= 2)
    if ((T + rows - 1) / rows * slabs >= 4 * 148) return rows;
  return 16;
}

}  // namespace pbs

extern "C" {

// positions [T] may be null (then t % seq); wpe may be null.  Ids outside the table and positions beyond wpe set the error
// word to 5 and contribute zeros.
int pb_embed_scaled_fwd(const long long* ids, const void* wte, const void* wpe, const int* positions, void* out,
                        long long T, int H, int seq, long long vocab, int n_positions, float scale, int* err_dev,
                        void* stream_) {
  using namespace pbs;
  if (H % 8 != 0 || H < 8) return -1;
  if (wpe && !positions && seq < 1) return -1;
  if ((reinterpret_cast<uintptr_t>(wte) | reinterpret_cast<uintptr_t>(wpe) | reinterpret_cast<uintptr_t>(out)) & 15) return -2;
  if (T == 0) return 0;
  const int vec = H / 8;
  const int tx = vec >= 128 ? 128 : (vec + 31) / 32 * 32, ty = 256 / tx;
  long long blocks = (T + ty - 1) / ty;
  if (blocks > 148 * 64) blocks = 148 * 64;
  embed_scaled_kernel<<<(unsigned)blocks, dim3(tx, ty), 0, reinterpret_cast<cudaStream_t>(stream_)>>>(
      ids, reinterpret_cast<const __nv_bfloat16*>(wte), reinterpret_cast<const __nv_bfloat16*>(wpe), positions, seq,
      reinterpret_cast<__nv_bfloat16*>(out), T, vec, vocab, n_positions, scale, err_dev);
  pb_count_launch(1);
  return (int)cudaGetLastError();
}

// Bytes of scratch that pb_embed_sorted_bwd needs for `tables` (1 or 2) tables.
long long pb_embed_sorted_scratch(long long T, int H, int tables) {
  using namespace pbs;
  const int rows = tile_rows_for(T, H);
  const long long tiles = (T + rows - 1) / rows;
  return tables * (2 * T * (long long)sizeof(int2) + 2 * tiles * H * (long long)sizeof(float) + (tiles + 1) * (long long)sizeof(int) + 32);
}

// dout [T, H] bf16.  gw [vocab, H] and gp [n_positions, H], either null where that gradient is not wanted: fp32 and added to,
// or with `write` bf16 and written whole.  scratch: 16-byte aligned, pb_embed_sorted_scratch bytes, of this call alone.
int pb_embed_sorted_bwd(const long long* ids, const int* positions, const void* dout, void* gw, void* gp, long long T,
                        int H, int seq, int vocab, int n_positions, float scale, int write, void* scratch,
                        void* stream_) {
  using namespace pbs;
  if (H % 8 != 0 || H < 8 || (gw && vocab < 1) || (gp && n_positions < 1) || (gp && !positions && seq < 1)) return -1;
  if (T < 0 || T > 0x7fffffffLL - 1024 || vocab == 0x7fffffff || n_positions == 0x7fffffff) return -2;
  if ((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(gw) | reinterpret_cast<uintptr_t>(gp) |
       reinterpret_cast<uintptr_t>(scratch)) & 15)
    return -3;
  if (!gw && !gp) return 0;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  SortArgs a;
  memset(&a, 0, sizeof(a));
  a.T = T;
  a.H = H;
  a.write = write;
  const int rows = tile_rows_for(T, H);
  const long long tiles = (T + rows - 1) / rows;
  char* at = reinterpret_cast<char*>(scratch);
  for (int k = 0; k < 2; ++k) {
    if (!(k == 0 ? gw : gp)) continue;
    Table& tb = a.table[a.tables++];
    tb.ids = k == 0 ? ids : nullptr;
    tb.positions = positions;
    tb.seq = seq;
    tb.size = k == 0 ? vocab : n_positions;
    tb.grad = k == 0 ? gw : gp;
    tb.scale = k == 0 ? scale : 1.f;
    tb.partial = reinterpret_cast<float*>(at);
    tb.sorted = reinterpret_cast<int2*>(at + 2 * tiles * H * sizeof(float));
    tb.other = tb.sorted + T;
    tb.n_crossing = reinterpret_cast<int*>(tb.other + T);
    tb.crossing = tb.n_crossing + 1;
    at += (2 * tiles * H * sizeof(float) + 2 * T * sizeof(int2) + (tiles + 1) * sizeof(int) + 15) / 16 * 16;
  }
  const int clearing = write ? 128 : 0;
  embed_sort_kernel<<<a.tables * kCluster + clearing, kSortThreads, 0, stream>>>(a);
  pb_count_launch(1);
  if (T == 0) return (int)cudaGetLastError();
  const int slabs = (H / 8 + 127) / 128;
  pb_count_launch(1);
  if (cudaError_t e = pb::launch_chained(embed_runs_kernel, dim3((unsigned)tiles, slabs, a.tables), 128, 0, stream, a,
                                         reinterpret_cast<const __nv_bfloat16*>(dout), rows);
      e != cudaSuccess)
    return (int)e;
  if (tiles > 1) {
    const long long most = (tiles + kFoldWarps - 1) / kFoldWarps < 148 * 2 ? (tiles + kFoldWarps - 1) / kFoldWarps : 148 * 2;
    pb_count_launch(1);
    return (int)pb::launch_chained(embed_fold_kernel, dim3((unsigned)most, (H / 8 + 31) / 32, a.tables), dim3(32, kFoldWarps), 0,
                                   stream, a, rows);
  }
  return (int)cudaGetLastError();
}

}  // extern "C"

// Pieces that the kernels of the packed attention's backward share.
#pragma once
#include "attention_packed.cuh"

namespace pbv {

struct BwdArgs {
  const __nv_bfloat16* o;  // pass 1: delta
  long long o_stride;
  const float* lse;  // [Hq, T] natural log
  float* delta;      // [Hq, T]: written by pass 1, read by pass 2
  __nv_bfloat16* out_a;  // pass 1: dQ; pass 2: dK
  __nv_bfloat16* out_b;  // pass 2: dV
  long long out_stride;
  const float *cs, *sn;  // [table_rows, D / 2], null: no rotation
  int table_rows;
  long long T;
  const Tile* tiles;  // of 128 rows
  const int* counts;  // all tiles, those before the documents of 128 tokens or fewer, those before the padding
  int max_tiles, Hq, Hkv;
  int split;       // pass 2: items that share the query heads of a key head
  float* partial;  // split > 1: [split][dK, dV][T, Hkv * D], neither scaled nor turned back
  float scale, scale_log2;
  int causal;
  int head_group;
  int* counter;  // pass 2: of items, see Items
  int* err;
};

// Mask of a packed pair of bf16 of which the first `n` values stay (all for n >= 2, none for n <= 0).
__device__ __forceinline__ uint32_t keep_below(int n) {
  uint32_t m;
  asm("shr.u32 %0, 0xffffffff, %1;" : "=r"(m) : "r"(max(32 - 16 * n, 0)));  // shifts by 32 and more give 0
  return m;
}

// The 64 columns of a lane at `taddr`, 16 at a time: f(chunk, values) while the next ones are on their way.
template <class F>
__device__ __forceinline__ void by_chunks(uint32_t taddr, F f) {
  uint32_t t[2][16];
  tmem_ld_32x16(taddr, t[0]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tmem_ld_wait();
    if (c < 3) tmem_ld_32x16(taddr + (c + 1) * 16, t[(c + 1) & 1]);
    f(c, t[c & 1]);
  }
}

// Memory of its own that a warp needs for write_rows and write_partial.
constexpr int kStageBytes = 4096;

// A warp's share of the rotation tables for 32 rows, 16 columns at a time: those of its columns [sub * D / 4, + D / 4) of each.
// The first ones are fetched while the products that they are for are still running.  pos: position of the first row; rows:
// how many of the 32 are the document's.
template <int D>
struct Turn {
  float4 cs[4], sn[4];
  const float *c0, *s0;
  int limit;  // of the row numbers u * 8
  __device__ __forceinline__ Turn(const BwdArgs& p, int pos, int rows, int sub, int lane) {
    const int r = lane >> 2;
    const long long at = (long long)(pos + r) * (D / 2) + sub * (D / 4) + (lane & 3) * 4;
    c0 = p.cs + at, s0 = p.sn + at;
    limit = min(rows, p.table_rows - pos) - r;
  }
  __device__ __forceinline__ void fetch(int chunk) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      cs[u] = u * 8 < limit ? __ldg(reinterpret_cast<const float4*>(c0 + u * 8 * (D / 2) + chunk * 16)) : make_float4(1.f, 1.f, 1.f, 1.f);
      sn[u] = u * 8 < limit ? __ldg(reinterpret_cast<const float4*>(s0 + u * 8 * (D / 2) + chunk * 16)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
};

// A lane's D / 2 results, bf16 pairs [half][D / 8] of its row, to global memory through `stage`.
template <int D>
__device__ __forceinline__ void store_rows(const uint32_t (&out)[D / 4], int sub, int rows, uint8_t* stage, int lane,
                                           __nv_bfloat16* dst, long long stride) {
  constexpr int N = D / 4;
  constexpr int kPieces = D / 16;          // 16-byte pieces of a row's results
  constexpr int kRowsPer = 32 / kPieces;  // rows of one access
  auto at = [&](int row, int piece) {
    const int x = kPieces == 8 ? (row & 7) : ((row >> 1) & 3);
    return reinterpret_cast<uint4*>(stage + row * (kPieces * 16) + ((piece ^ x) << 4));
  };
#pragma unroll
  for (int u = 0; u < kPieces; ++u) *at(lane, u) = make_uint4(out[u * 4], out[u * 4 + 1], out[u * 4 + 2], out[u * 4 + 3]);
  __syncwarp();
  const int u = lane % kPieces;
  dst += (lane / kPieces) * stride + (u < kPieces / 2 ? 0 : D / 2) + sub * N + (u % (kPieces / 2)) * 8;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int r = i * kRowsPer + lane / kPieces;
    const uint4 w = *at(r, u);
    if (r < rows) *reinterpret_cast<uint4*>(dst) = w;
    dst += kRowsPer * stride;
  }
  __syncwarp();
}

// 32 rows of an accumulator [128, D] to bf16, by one warp, a row per lane.  The warp's columns are [sub * D / 4, + D / 4) of each
// half, so that a thread holds both elements of every pair that the rotation mixes.  A lane that read and wrote its
// own row in global memory touched 32 lines with every access: 6 000 to 9 000 cycles for a tile of 128 x 128, several times
// what its products take.  So the tables come, and the results leave, through `stage` (kStageBytes of the warp's own), as
// segments of 64 bytes.  `turn` holds its first columns.
template <int D, bool kTurn>
__device__ __forceinline__ void write_rows(uint32_t acc, int sub, float scale, Turn<D>& turn, int rows, uint8_t* stage,
                                           int lane, __nv_bfloat16* dst, long long stride) {
  constexpr int N = D / 4;
  uint32_t out[N];  // [half][N / 2]
  const f32x2 scale2 = pair(scale, scale);
  // 64-byte rows, cosines and then sines; two of them share 128 bytes, hence the shift
  const uint32_t put_at = (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
  const uint32_t get_at = lane * 64, turn_by = (lane >> 1) & 3;
#pragma unroll
  for (int c = 0; c < N / 16; ++c) {
    uint32_t a[16], b[16];
    tmem_ld_32x16(acc + sub * N + c * 16, a);
    tmem_ld_32x16(acc + D / 2 + sub * N + c * 16, b);
    if (kTurn) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // row u * 8 + lane / 4
        *reinterpret_cast<float4*>(stage + put_at + u * 512) = turn.cs[u];
        *reinterpret_cast<float4*>(stage + 2048 + put_at + u * 512) = turn.sn[u];
      }
      __syncwarp();
      if (c + 1 < N / 16) turn.fetch(c + 1);
    }
    tmem_ld_wait();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float4 cs, sn;
      if (kTurn) {
        cs = *reinterpret_cast<const float4*>(stage + get_at + ((u ^ turn_by) << 4));
        sn = *reinterpret_cast<const float4*>(stage + 2048 + get_at + ((u ^ turn_by) << 4));
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int e = u * 4 + k * 2;
        f32x2 f = mul2(pair(__uint_as_float(a[e]), __uint_as_float(a[e + 1])), scale2);
        f32x2 g = mul2(pair(__uint_as_float(b[e]), __uint_as_float(b[e + 1])), scale2);
        if (kTurn) {
          const f32x2 cc = k == 0 ? pair(cs.x, cs.y) : pair(cs.z, cs.w), ss = k == 0 ? pair(sn.x, sn.y) : pair(sn.z, sn.w);
          const f32x2 x = fma2(g, ss, mul2(f, cc));
          g = fma2(mul2(f, pair(-1.f, -1.f)), ss, mul2(g, cc));
          f = x;
        }
        const float2 x = both(f), y = both(g);
        out[c * 8 + u * 2 + k] = pack_bf16(x.x, x.y);
        out[N / 2 + c * 8 + u * 2 + k] = pack_bf16(y.x, y.y);
      }
    }
    __syncwarp();
  }
  store_rows<D>(out, sub, rows, stage, lane, dst, stride);
}

// The same rows in fp32, as they are: a part of dK or dV.  The warp's columns are [sub * D / 4, + D / 4) of each half here too.
template <int D>
__device__ __forceinline__ void write_partial(uint32_t acc, int sub, int rows, uint8_t* stage, int lane, float* dst, long long stride) {
  constexpr int N = D / 4;
  auto at64 = [&](int row, int piece) { return reinterpret_cast<uint4*>(stage + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4)); };
#pragma unroll
  for (int c = 0; c < 2 * (N / 16); ++c) {
    const int col = (c < N / 16 ? 0 : D / 2) + sub * N + (c % (N / 16)) * 16;
    uint32_t a[16];
    tmem_ld_32x16(acc + col, a);
    tmem_ld_wait();
#pragma unroll
    for (int u = 0; u < 4; ++u) *at64(lane, u) = make_uint4(a[u * 4], a[u * 4 + 1], a[u * 4 + 2], a[u * 4 + 3]);
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = u * 8 + (lane >> 2);
      const uint4 w = *at64(r, lane & 3);
      if (r < rows) *reinterpret_cast<uint4*>(dst + r * stride + col + (lane & 3) * 4) = w;
    }
    __syncwarp();
  }
}

// write_rows with the tables of the lane's row in registers, [pair of columns]: for documents that begin at the tile's first row
// they are the same in every item.
template <int D, bool kTurn>
__device__ __forceinline__ void write_rows_held(uint32_t acc, int sub, float scale, const f32x2 (&cs)[D / 8], const f32x2 (&sn)[D / 8],
                                                bool turn, int rows, uint8_t* stage, int lane, __nv_bfloat16* dst,
                                                long long stride) {
  constexpr int N = D / 4;
  uint32_t out[N];
  const f32x2 scale2 = pair(scale, scale);
#pragma unroll
  for (int c = 0; c < N / 16; ++c) {
    uint32_t a[16], b[16];
    tmem_ld_32x16(acc + sub * N + c * 16, a);
    tmem_ld_32x16(acc + D / 2 + sub * N + c * 16, b);
    tmem_ld_wait();
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      f32x2 f = mul2(pair(__uint_as_float(a[u * 2]), __uint_as_float(a[u * 2 + 1])), scale2);
      f32x2 g = mul2(pair(__uint_as_float(b[u * 2]), __uint_as_float(b[u * 2 + 1])), scale2);
      if (kTurn && turn) {
        const f32x2 cc = cs[c * 8 + u], ss = sn[c * 8 + u];
        const f32x2 x = fma2(g, ss, mul2(f, cc));
        g = fma2(mul2(f, pair(-1.f, -1.f)), ss, mul2(g, cc));
        f = x;
      }
      const float2 x = both(f), y = both(g);
      out[c * 8 + u] = pack_bf16(x.x, x.y);
      out[N / 2 + c * 8 + u] = pack_bf16(y.x, y.y);
    }
  }
  store_rows<D>(out, sub, rows, stage, lane, dst, stride);
}

// 16-byte piece `u` of row `row` of a tile: inside the 128 bytes of a chunk it lies at u ^ (row & 7).
__device__ __forceinline__ uint4 piece_of(const uint8_t* tile, int row, int u) {
  return *reinterpret_cast<const uint4*>(tile + (u >> 3) * kChunkBytes + row * 128 + (((u & 7) ^ (row & 7)) << 4));
}

// delta = dO O of a warp's rows to out[row].  D / 8 lanes share a row, so that O is read in whole lines: lane has piece u of
// rows first + k * 32 / (D / 8) in y[k], kCount of them, and dO comes from its tile.
template <int D, int kCount>
__device__ __forceinline__ void row_dots(const uint8_t* tile_do, const uint4 (&y)[kCount], int first, int u, float* out) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  float dot[kCount];
#pragma unroll
  for (int k = 0; k < kCount; ++k) {
    const uint4 x = piece_of(tile_do, first + k * kRows, u);
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
    f32x2 sum = pair(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e)  // a bf16 is the upper half of its fp32
      sum = fma2(pair(__uint_as_float(xs[e] << 16), __uint_as_float(xs[e] & 0xffff0000u)),
                 pair(__uint_as_float(ys[e] << 16), __uint_as_float(ys[e] & 0xffff0000u)), sum);
    const float2 v = both(sum);
    dot[k] = v.x + v.y;
  }
  // the kCount sums of every lane, added over the lanes of a row: each step halves the sums that a lane still carries, and lane
  // u ends with row u % kCount of its group's
#pragma unroll
  for (int o = kLanes / 2; o >= kCount; o >>= 1)
#pragma unroll
    for (int k = 0; k < kCount; ++k) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
#pragma unroll
  for (int o = kCount / 2; o > 0; o >>= 1) {
    const bool upper = u & o;
#pragma unroll
    for (int k = 0; k < o; ++k) {
      const float keep = upper ? dot[k + o] : dot[k], give = upper ? dot[k] : dot[k + o];
      dot[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  if (u < kCount) out[first + u * kRows] = dot[0];
}

// Documents of 128 tokens or fewer, and padding (attention_packed_short.cu).
template <int D, bool kTurn>
int launch_short_bwd(const CUtensorMap& tq, const CUtensorMap& tdo, const CUtensorMap& tk, const CUtensorMap& tv, BwdArgs p,
                     __nv_bfloat16* dq, __nv_bfloat16* dk, __nv_bfloat16* dv, cudaStream_t stream);

}  // namespace pbv

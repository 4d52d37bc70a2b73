// Attention over packed documents, forward, for sm_100a: head size 64 or 128, grouped heads, causal or not.
//
//   o_i = sum_j exp(s q_i k_j - lse_i) v_j over the tokens j of i's document (j <= i if causal)
//
// An item is two tiles of 128 query rows: 256 consecutive rows of one document and head, or, of a document of 128 tokens or
// fewer, two heads.  A tile never mixes documents, and no score of two documents is formed.  Per block of 128 keys and
// tile: S = Q K^T (tcgen05.mma, fp32 in TMEM), softmax with one thread per query row, bf16 P back into TMEM over S,
// O += P V with P as the TMEM operand.  The running maximum is only moved when it grew by more than 2^8 (probabilities
// stay <= 256, the division by the sum makes it exact).  The two tiles alternate on the tensor pipe: one's softmax runs
// under the other's products.  P is rounded to bf16, the type of V; sums and statistics are fp32.
//
// Blocks stay resident and walk a list of items (Items): the next item's operands are loaded, and its first scores formed,
// under the end of the present one.
// Bound by each tile's chain of scores, softmax, P V and the next scores: at D = 128 TMEM holds one score buffer for each of the
// two tiles beside their accumulators.  Measured, D = 128, causal: one row of 16 384 tokens in 4 documents, 8 heads: 239 us,
// 1.06 PFLOP/s of the scores that causal attention needs, 65% of what a large product reaches; 2 x 4096 tokens in 24
// documents, 32 heads: 95 us; 4 x 2999 tokens in 192 documents, 32 heads: 119 us, where an item's start and end are most of it.
// Tried without a gain: a part of the exponentials as polynomials, leaving out the columns that a short document does not have,
// the last P V of one tile behind the next item's first scores.
//
// Warps: 0 loads (TMA), 1 issues MMAs and owns TMEM, 2 clears what reaches beyond a document, 4..7 and 8..11 are the tiles'
// softmax and epilogue.
#include "attention_packed.cuh"

namespace pbv {

struct FwdArgs {
  __nv_bfloat16* o;  // [T, o_stride], head h at column h * D
  long long o_stride;
  float* lse;  // [Hq, T] natural log
  long long T;
  const Tile* tiles;  // of 256 rows
  const int* counts;  // all, those before the documents of 128 tokens or fewer, those before the padding
  int Hq, Hkv;
  float scale_log2;  // softmax scale * log2(e)
  int causal;
  int head_group;
  int* counter;  // of items, see Items
  int* err;
};

constexpr int kFwdThreads = 384;

template <int D>
__global__ void __launch_bounds__(kFwdThreads, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, FwdArgs p) {
  constexpr int NCH = D / 64;
  constexpr int TILE_BYTES = NCH * kChunkBytes;

  // addresses of shared memory are constants, as long as nothing is computed from where it begins
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {  // the launch reserves no slack for re-alignment
    if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sQ = smem;                 // 2 tiles
  uint8_t* sK = sQ + 2 * TILE_BYTES;  // 2 stages
  uint8_t* sV = sK + 2 * TILE_BYTES;  // 2 stages
  uint8_t* sOut = sV + 2 * TILE_BYTES;  // 4 KB for each softmax warp
  uint64_t* bars = reinterpret_cast<uint64_t*>(sOut + 32768);
  uint64_t* q_full = bars;        // [tile]
  uint64_t* q_empty = bars + 2;   // [tile]
  uint64_t* k_full = bars + 4;    // [stage]
  uint64_t* k_empty = bars + 6;   // [stage]
  uint64_t* v_full = bars + 8;    // [stage]
  uint64_t* v_empty = bars + 10;  // [stage]
  uint64_t* v_raw = bars + 12;    // [stage]
  uint64_t* s_full = bars + 14;   // [tile]
  uint64_t* p_ready = bars + 16;  // [tile]
  uint64_t* o_full = bars + 18;   // [tile]: the item's last P V
  ItemRing ring(sOut + 32768 + 256, bars + 20);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20 + ItemRing::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  after_previous();
  let_next_start();
  const int n_all = p.counts[0], n_wide = p.counts[1], n_docs = p.counts[2];
  const int G = p.Hq / p.Hkv, head_pairs = (p.Hq + 1) / 2;

  struct Item {
    int start, len;       // the document
    int row[2], head[2];  // first row and head of the two tiles
    int blocks[2];        // blocks of keys that they see; 0: no such tile
    int pad_rows;         // padding: rows to clear
    bool split;           // two heads with keys of their own (one block each)
  };
  // decoded by the loading warp, taken from the ring by the others; false after the last
  Items items(n_wide * p.Hq + (n_docs - n_wide) * head_pairs + (n_all - n_docs) * p.Hq, p.counter);
  bool ok = true;
  Item w;
  auto decode = [&]() {
    int i = items.next(lane), entry;
    if (i < 0) {
      w.start = -1;
      return;
    }
    bool two_heads = false;
    if (i < n_wide * p.Hq) {
      const TileOrder order = tile_order(i, n_wide, p.Hq, p.head_group);
      entry = order.tile_rank;
      w.head[0] = w.head[1] = order.index;
    } else if ((i -= n_wide * p.Hq) < (n_docs - n_wide) * head_pairs) {
      entry = i / head_pairs;
      w.head[0] = 2 * (i - entry * head_pairs), w.head[1] = w.head[0] + 1;
      entry += n_wide;
      two_heads = true;
    } else {
      i -= (n_docs - n_wide) * head_pairs;
      entry = i / p.Hq;
      w.head[0] = w.head[1] = i - entry * p.Hq;
      entry += n_docs;
    }
    const Tile tile = p.tiles[entry];
    w.start = tile.start, w.len = tile.len;
    w.row[0] = tile.rank * 256, w.row[1] = two_heads ? w.row[0] : w.row[0] + 128;
#pragma unroll
    for (int t = 0; t < 2; ++t)
      w.blocks[t] = tile.pad || w.row[t] >= tile.len || w.head[t] >= p.Hq
                        ? 0 : ((p.causal ? min(tile.len, w.row[t] + 128) : tile.len) + 127) / 128;
    w.split = two_heads && w.blocks[1] > 0 && w.head[0] / G != w.head[1] / G;
    w.pad_rows = tile.pad ? min(256, tile.len - w.row[0]) : 0;
  };
  auto publish_next = [&]() {
    decode();
    ok = ring.put(make_int4(w.start, w.len, w.row[0], w.row[1]), make_int4(w.head[0], w.head[1], w.blocks[0], w.blocks[1]),
                  make_int4(w.split, w.pad_rows, 0, 0), lane, abort_flag);
    return ok && w.start >= 0;
  };
  auto next_item = [&]() {
    int4 a, b, c;
    if (!(ok = ring.get(a, b, c, lane, abort_flag))) return false;
    w.start = a.x, w.len = a.y, w.row[0] = a.z, w.row[1] = a.w;
    w.head[0] = b.x, w.head[1] = b.y, w.blocks[0] = b.z, w.blocks[1] = b.w;
    w.split = c.x, w.pad_rows = c.y;
    return w.start >= 0;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_raw[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_full[i], 1);
    }
    ring.init(10);  // MMA, clearing, softmax
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;  // S/P of tile t: columns [128 t, 128 t + 128); O: [256 + 128 t, + D)

  int used[2] = {0, 0};  // items so far that had the tile
  int n = 0;             // K / V stages so far
  // launched with 168 registers a thread: 88 + 2 x 208 = 3 x 168
  if (warp < 4) {
    give_registers<88>();
    if (warp == 0) {
      while (ok && publish_next()) {
        if (w.blocks[0] == 0) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (w.blocks[t] == 0 || !ok) continue;
          ok = warp_wait(&q_empty[t], (used[t] & 1) ^ 1, abort_flag);
          if (ok && lane == 0) load_tile<NCH>(sQ + t * TILE_BYTES, &tmQ, &q_full[t], w.head[t] * D, w.start + w.row[t]);
          ++used[t];
        }
        const int stages = w.split ? 2 : max(w.blocks[0], w.blocks[1]);
        for (int j = 0; ok && j < stages; ++j, ++n) {
          const int s = n & 1;
          const uint32_t ph = ((n >> 1) & 1) ^ 1;
          const int col = (w.head[w.split ? j : 0] / G) * D, key = w.split ? 0 : j * 128;
          if (!(ok = warp_wait(&k_empty[s], ph, abort_flag))) break;
          // keys beyond the document only make scores that the mask replaces: K needs no clearing, V does
          if (lane == 0) load_tile<NCH>(sK + s * TILE_BYTES, &tmK, &k_full[s], col, w.start + key);
          if (!(ok = warp_wait(&v_empty[s], ph, abort_flag))) break;
          if (lane == 0)
            load_tile<NCH>(sV + s * TILE_BYTES, &tmV, w.len - key < 128 ? &v_raw[s] : &v_full[s], col, w.start + key);
        }
      }
    } else if (warp == 1) {
      // the whole warp walks the loops; one elected lane, the same every time, issues the MMAs and their commits
      const uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0);
      const uint32_t idesc_pv = make_idesc_bf16(128, D, 0, 1);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool got = warp_wait(bar, parity, abort_flag);
        tc_fence_after_sync();
        return got;
      };
      auto issue_s = [&](int t, int stage, bool release, bool last) {
        const uint64_t qd = make_smem_desc(smem_u32(sQ + t * TILE_BYTES), 16, 1024);
        const uint64_t kd = make_smem_desc(smem_u32(sK + stage * TILE_BYTES), 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4;
            umma_ss<1>(tmem_base + t * 128, qd + off, kd + off, idesc_s, kk != 0);
          }
          umma_commit(&s_full[t]);
          if (release) umma_commit(&k_empty[stage]);
          if (last) umma_commit(&q_empty[t]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int t, int stage, bool first, bool release, bool last) {
        const uint64_t vd = make_smem_desc(smem_u32(sV + stage * TILE_BYTES), kChunkBytes, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // A = P: 16 bf16 of K per step = 8 TMEM columns
            umma_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + kk * 8, vd + ((kk * 2048) >> 4), idesc_pv,
                    !(first && kk == 0));
          if (release) umma_commit(&v_empty[stage]);
          if (last) umma_commit(&o_full[t]);
        }
        __syncwarp();
      };
      int done[2] = {0, 0};  // blocks so far, by tile
      while (ok && next_item()) {
        if (w.blocks[0] == 0) continue;
        // stage of block j of a tile, and whether the tile is the last to read it
        auto stage_of = [&](int t, int j) { return n + j + (w.split ? t : 0); };
        auto last_reader = [&](int t, int j) { return w.split || t == 1 || j >= w.blocks[1]; };
        const int nblk = max(w.blocks[0], w.blocks[1]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (w.blocks[t] == 0 || !ok) continue;
          const int s = stage_of(t, 0);
          if (!(ok = wait(&q_full[t], used[t] & 1) && wait(&k_full[s & 1], (s >> 1) & 1))) continue;
          issue_s(t, s & 1, last_reader(t, 0), w.blocks[t] == 1);
          ++used[t];
        }
        for (int j = 0; ok && j < nblk; ++j) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= w.blocks[t] || !ok) continue;
            const int s = stage_of(t, j);
            const bool more = j + 1 < w.blocks[t];
            // what the products need is waited for before P, which comes last
            ok = wait(&v_full[s & 1], (s >> 1) & 1) && (!more || wait(&k_full[(s + 1) & 1], ((s + 1) >> 1) & 1)) &&
                 wait(&p_ready[t], done[t] & 1);
            if (!ok) continue;
            issue_pv(t, s & 1, j == 0, last_reader(t, j), !more);
            if (more) issue_s(t, (s + 1) & 1, last_reader(t, j + 1), j + 2 == w.blocks[t]);
            ++done[t];
          }
        }
        n += w.split ? 2 : nblk;
    }
  } else if (warp == 2) {
    uint32_t phases = 0;  // of the v_raw barriers
    while (ok && next_item()) {
      if (w.blocks[0] == 0) continue;
      const int nblk = max(w.blocks[0], w.blocks[1]), stages = w.split ? 2 : nblk;
      const int valid = w.len - (nblk - 1) * 128;  // only the last block can reach beyond the document
      for (int j = valid < 128 ? (w.split ? 0 : stages - 1) : stages; ok && j < stages; ++j) {
        const int s = (n + j) & 1;
        if (!(ok = warp_wait(&v_raw[s], (phases >> s) & 1, abort_flag))) break;
        phases ^= 1u << s;
        clear_tail<NCH>(sV + s * TILE_BYTES, valid, &v_full[s], lane);
      }
      n += stages;
    }
    }
  } else {
    take_registers<208>();
    // ------------------------------------------------------------ softmax + epilogue, one query row per thread
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem_base + t * 128 + lane_off;
    const uint32_t tO = tmem_base + 256 + t * 128 + lane_off;
    const f32x2 scale2 = pair(p.scale_log2, p.scale_log2);
    int done = 0;  // blocks so far
    int mine = 0;  // items so far
    while (ok && next_item()) {
      if (w.pad_rows > 0) {
        clear_rows<D>(p.o, p.o_stride, (long long)w.start + w.row[0], w.pad_rows, w.head[0] * D, threadIdx.x - 128, 256);
        continue;
      }
      const int nblk = w.blocks[t];
      if (nblk == 0) continue;
      const int first_row = w.row[t], h = w.head[t];
      const int q_idx = first_row + quarter * 32 + lane;
      float m = -CUDART_INF_F;
      f32x2 l2 = pair(0.f, 0.f);
      for (int j = 0; j < nblk; ++j, ++done) {
        if (!(ok = warp_wait(&s_full[t], done & 1, abort_flag))) break;
        tc_fence_after_sync();
        const int k0 = j * 128;
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(tS + c * 32, v[c]);
        tmem_ld_wait();
        if ((p.causal && k0 + 127 > first_row) || k0 + 128 > w.len) {
          // keys this row may see: [k0, limit)
          const int limit = (p.causal ? min(w.len, q_idx + 1) : w.len) - k0;
          // as bits: a test of a bit of a register that every element shares is cheaper than a comparison
          uint32_t seen[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int n = min(max(limit - c * 32, 0), 32);
            seen[c] = n == 32 ? 0xffffffffu : (1u << n) - 1;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((seen[c] >> e) & 1)) v[c][e] = 0xff800000u;  // -inf
        }
        float mx[4];  // four chains: one would be 128 dependent steps
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = __uint_as_float(v[c][0]);
#pragma unroll
          for (int e = 1; e < 32; ++e) mx[c] = fmaxf(mx[c], __uint_as_float(v[c][e]));
        }
        const float m_cand = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2);
        // rescale only when some row of the warp moved its maximum by more than 2^8
        if (__any_sync(0xffffffffu, m_cand > m + 8.f)) {
          const float m_use = (m_cand == -CUDART_INF_F) ? 0.f : m_cand;
          const float alpha = exp2f(m - m_use);  // 0 on the first block (m = -inf)
          if (j > 0) {
#pragma unroll 1  // rare: its code should not push the rest out of the instruction cache
            for (int cc = 0; cc < D / 16; ++cc) {  // 16 columns at a time: v is live
              uint32_t o[16];
              tmem_ld_32x16(tO + cc * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st_32x16(tO + cc * 16, o);
            }
            tmem_st_wait();
          }
          l2 = mul2(l2, pair(alpha, alpha));
          m = m_use;
        }
        const f32x2 minus_m = pair(-m, -m);
        f32x2 sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
        // P over the first 64 columns of S, which is in registers by now
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const f32x2 y = exp2_pair(fma2(pair(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), scale2, minus_m));
            sum[e & 1] = add2(sum[e & 1], y);
            const float2 b = both(y);
            pk[e] = pack_bf16(b.x, b.y);
          }
          tmem_st_32x16(tS + c * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);
        l2 = add2(l2, add2(sum[0], sum[1]));
      }
      if (!ok) break;
      if (!(ok = warp_wait(&o_full[t], mine & 1, abort_flag))) break;
      ++mine;
      tc_fence_after_sync();
      const float2 lb = both(l2);
      const float l = lb.x + lb.y, inv_l = 1.f / l;
      // through memory of the warp's own, 128-byte pieces of 32 rows at a time: whole lines leave (see write_rows in
      // attention_packed_bwd.cuh)
      const int first = first_row + quarter * 32;
      __nv_bfloat16* dst = p.o + ((long long)w.start + first) * p.o_stride + h * D;
      uint8_t* stage = sOut + (warp - 4) * 4096;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        uint32_t o[2][32];
        tmem_ld_32x32(tO + c * 64, o[0]);
        tmem_ld_32x32(tO + c * 64 + 32, o[1]);
        tmem_ld_wait();
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          uint32_t b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            b[e] = pack_bf16(__uint_as_float(o[u >> 2][(u & 3) * 8 + e * 2]) * inv_l,
                             __uint_as_float(o[u >> 2][(u & 3) * 8 + e * 2 + 1]) * inv_l);
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((u ^ (lane & 7)) << 4)) = make_uint4(b[0], b[1], b[2], b[3]);
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = k * 4 + (lane >> 3), u = lane & 7;
          const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 128 + ((u ^ (r & 7)) << 4));
          if (first + r < w.len) *reinterpret_cast<uint4*>(dst + r * p.o_stride + c * 64 + u * 8) = x;
        }
        __syncwarp();
      }
      if (q_idx < w.len) p.lse[(long long)h * p.T + w.start + q_idx] = (m + log2f(l)) * 0.6931471805599453f;
      tc_fence_before_sync();
    }
  }
  if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  leave(abort_flag, warp, tmem_base);
}

template <int D>
static int launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const FwdArgs& p, int max_tiles,
                      cudaStream_t stream) {
  constexpr int SMEM = 6 * (D / 64) * kChunkBytes + 32768 + 256 + ItemRing::kBytes;
  constexpr auto kern = packed_fwd_kernel<D>;
  if (cudaError_t e = pb::allow_smem<kern, SMEM>(); e != cudaSuccess) return (int)e;
  pb_count_launch(1);
  return (int)pb::launch_chained(kern, resident_blocks((long long)max_tiles * p.Hq), kFwdThreads, SMEM, stream, tq, tk, tv, p);
}

}  // namespace pbv

extern "C" {

// q/k/v: bf16 [T, ...], head h at columns [h * D, (h + 1) * D) of the respective pointer, row pitches in elements.
// o: [T, o_stride] bf16, every row written (zeros in padding); lse: [Hq, T] fp32, rows of documents written.  counter: a word of
// this call alone; `cleared` where an earlier launch (pb_packed_rope's) has set it to 0.
// tiles / counts: the layout's table of 256-row tiles (max_tiles entries at most).
int pb_packed_attention_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int* counter, int cleared,
                            const int* tiles, const int* counts, int max_tiles, long long T, int Hq, int Hkv, int D, long long q_stride,
                            long long k_stride, long long v_stride, long long o_stride, float softmax_scale, int causal,
                            int* err_dev, void* stream_) {
  using namespace pbv;
  if (D != 64 && D != 128) return -1;
  if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0) return -2;
  if ((q_stride % 8) || (k_stride % 8) || (v_stride % 8) || (o_stride % 8)) return -3;
  if (reinterpret_cast<uintptr_t>(o) & 15) return -3;
  if (T < 1 || T > 0x3fffffffLL || max_tiles < 1 || (long long)max_tiles * Hq > 0x7fff0000LL) return -4;  // room for Items' last turn
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  CUtensorMap tq, tk, tv;
  if (pb::make_tmap_bf16_2d(&tq, q, (uint64_t)Hq * D, T, (uint64_t)q_stride, 64, 128)) return -10;
  if (pb::make_tmap_bf16_2d(&tk, k, (uint64_t)Hkv * D, T, (uint64_t)k_stride, 64, 128)) return -11;
  if (pb::make_tmap_bf16_2d(&tv, v, (uint64_t)Hkv * D, T, (uint64_t)v_stride, 64, 128)) return -12;
  FwdArgs p;
  memset(&p, 0, sizeof(p));
  p.o = reinterpret_cast<__nv_bfloat16*>(o);
  p.o_stride = o_stride;
  p.lse = lse;
  p.T = T;
  p.tiles = reinterpret_cast<const Tile*>(tiles);
  p.counts = counts;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.scale_log2 = softmax_scale * kLog2e;
  p.causal = causal;
  p.err = err_dev;
  if (takes_from_counter((long long)max_tiles * Hq)) {
    p.counter = counter;
    if (!cleared) {
      if (cudaError_t e = cudaMemsetAsync(counter, 0, sizeof(int), stream); e != cudaSuccess) return (int)e;
    }
  }
  p.head_group = pb::attention_head_group(max_tiles, Hq);
  return D == 128 ? launch_fwd<128>(tq, tk, tv, p, max_tiles, stream)
                  : launch_fwd<64>(tq, tk, tv, p, max_tiles, stream);
}

}  // extern "C"

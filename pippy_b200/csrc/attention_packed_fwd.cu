// Attention over packed documents, forward, for sm_100a: head size 64 or 128, grouped heads, causal or not.
//
//   o_i = sum_j exp(s q_i k_j - lse_i) v_j over the tokens j of i's document (j <= i if causal)
//
// A block owns 256 consecutive rows (two tiles of 128) of one document and one head, taken from the layout's table, so a tile
// never mixes documents and no score of two documents is formed.  Per block of 128 keys and tile: S = Q K^T
// (tcgen05.mma, fp32 in TMEM), softmax with one thread per query row, bf16 P back into TMEM over S, O += P V with P as the
// TMEM operand.  The running maximum is only moved when it grew by more than 2^8 (probabilities stay <= 256, the division by
// the sum makes it exact).  The two tiles alternate on the tensor pipe: one's softmax runs under the other's products.  P is
// rounded to bf16, the type of V; sums and statistics are fp32.
// Warps: 0 loads (TMA), 1 issues MMAs and owns TMEM, 2..5 and 6..9 are the tiles' softmax and epilogue.
#include "attention_packed.cuh"

namespace pbv {

struct FwdArgs {
  __nv_bfloat16* o;  // [T, o_stride], head h at column h * D
  long long o_stride;
  float* lse;  // [Hq, T] natural log
  long long T;
  const Tile* tiles;  // of 256 rows
  const int* count;
  int max_tiles, Hq, Hkv;
  float scale_log2;  // softmax scale * log2(e)
  int causal;
  int head_group;
  int* err;
};

template <int D>
__global__ void __launch_bounds__(320, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, FwdArgs p) {
  constexpr int NCH = D / 64;
  constexpr int TILE_BYTES = NCH * kChunkBytes;

  const TileOrder order = tile_order(blockIdx.x, p.max_tiles, p.Hq, p.head_group);
  if (order.tile_rank >= *p.count) return;
  const Tile tile = p.tiles[order.tile_rank];
  const int h = order.index;
  const int q0 = tile.rank * 256;  // first row of the block inside its document
  if (tile.pad) {
    clear_rows<D>(p.o, p.o_stride, (long long)tile.start + q0, min(256, tile.len - q0), h * D);
    return;
  }
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (smem != smem_raw) {
    if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sQ = smem;                 // 2 tiles
  uint8_t* sK = sQ + 2 * TILE_BYTES;  // 2 stages
  uint8_t* sV = sK + 2 * TILE_BYTES;  // 2 stages
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * TILE_BYTES);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = bars + 3;
  uint64_t* v_full = bars + 5;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 9;    // [tile]
  uint64_t* p_ready = bars + 11;  // [tile]
  uint64_t* o_full = bars + 13;   // [tile], once: the tile's last P V
  uint64_t* aux = bars + 15;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int hkv = h / (p.Hq / p.Hkv);
  // blocks of keys that the two tiles see (the second tile may have no rows)
  auto blocks_of = [&](int first_row) {
    if (first_row >= tile.len) return 0;
    return ((p.causal ? min(tile.len, first_row + 128) : tile.len) + 127) / 128;
  };
  const int n_a = blocks_of(q0), n_b = blocks_of(q0 + 128);
  const int nblk = max(n_a, n_b);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(aux, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;  // S/P of tile t: columns [128 t, 128 t + 128); O: [256 + 128 t, + D)

  if (warp == 0) {
    bool ok = true;
    if (lane == 0) {
      mbar_expect_tx(q_full, (n_b > 0 ? 2 : 1) * TILE_BYTES);
      for (int t = 0; t < (n_b > 0 ? 2 : 1); ++t)
#pragma unroll
        for (int c = 0; c < NCH; ++c)
          tma_load_2d(sQ + t * TILE_BYTES + c * kChunkBytes, &tmQ, q_full, h * D + c * 64, tile.start + q0 + t * 128);
    }
    __syncwarp();
    uint32_t aux_phase = 0;
    for (int j = 0; j < nblk; ++j) {
      const int s = j & 1;
      const uint32_t ph = (j >> 1) & 1;
      if (!(ok = warp_wait(&k_empty[s], ph ^ 1, abort_flag))) break;
      // keys beyond the document only make scores that the mask replaces: K needs no clearing, V does
      load_tile<NCH>(sK + s * TILE_BYTES, &tmK, &k_full[s], aux, &aux_phase, hkv * D, tile.start + j * 128, 128, lane,
                     abort_flag);
      if (!(ok = warp_wait(&v_empty[s], ph ^ 1, abort_flag))) break;
      if (!(ok = load_tile<NCH>(sV + s * TILE_BYTES, &tmV, &v_full[s], aux, &aux_phase, hkv * D, tile.start + j * 128,
                                tile.len - j * 128, lane, abort_flag)))
        break;
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  } else if (warp == 1) {
    // the whole warp walks the loop; one elected lane, the same every time, issues the MMAs and their commits
    const uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0);
    const uint32_t idesc_pv = make_idesc_bf16(128, D, 0, 1);
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool got = warp_wait(bar, parity, abort_flag);
      tc_fence_after_sync();
      return got;
    };
    auto issue_s = [&](int t, int j) {
      const uint64_t qd = make_smem_desc(smem_u32(sQ + t * TILE_BYTES), 16, 1024);
      const uint64_t kd = make_smem_desc(smem_u32(sK + (j & 1) * TILE_BYTES), 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4;
          umma_ss<1>(tmem_base + t * 128, qd + off, kd + off, idesc_s, kk != 0);
        }
        umma_commit(&s_full[t]);
      }
      __syncwarp();
    };
    auto issue_pv = [&](int t, int j, bool last) {
      const uint64_t vd = make_smem_desc(smem_u32(sV + (j & 1) * TILE_BYTES), kChunkBytes, 1024);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)  // A = P: 16 bf16 of K per step = 8 TMEM columns
          umma_ts(tmem_base + 256 + t * 128, tmem_base + t * 128 + kk * 8, vd + ((kk * 2048) >> 4), idesc_pv,
                  (j | kk) != 0);
        if (last) umma_commit(&o_full[t]);
      }
      __syncwarp();
    };
    auto release = [&](uint64_t* bar) {
      if (elect_one()) umma_commit(bar);
      __syncwarp();
    };
    bool ok = wait(q_full, 0) && wait(&k_full[0], 0);
    if (ok) {
      issue_s(0, 0);
      if (n_b > 0) issue_s(1, 0);
      release(&k_empty[0]);
    }
    for (int j = 0; j < nblk && ok; ++j) {
      const bool more = j + 1 < nblk;
      ok = wait(&v_full[j & 1], (j >> 1) & 1) && (!more || wait(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1));
      if (!ok) break;
      if (j < n_a) {
        if (!(ok = wait(&p_ready[0], j & 1))) break;
        issue_pv(0, j, j + 1 == n_a);
      }
      if (j + 1 < n_a) issue_s(0, j + 1);
      if (j < n_b) {
        if (!(ok = wait(&p_ready[1], j & 1))) break;
        issue_pv(1, j, j + 1 == n_b);
      }
      release(&v_empty[j & 1]);
      if (j + 1 < n_b) issue_s(1, j + 1);
      if (more) release(&k_empty[(j + 1) & 1]);
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  } else {
    // ------------------------------------------------------------ softmax + epilogue, one query row per thread
    const int t = (warp - 2) >> 2;
    const int quarter = warp & 3;
    const int first_row = q0 + t * 128;
    const int n_t = t == 0 ? n_a : n_b;
    const int q_idx = first_row + quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem_base + t * 128 + lane_off;
    const uint32_t tO = tmem_base + 256 + t * 128 + lane_off;
    float m = -CUDART_INF_F, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_t; ++j) {
      if (!(ok = warp_wait(&s_full[t], j & 1, abort_flag))) break;
      tc_fence_after_sync();
      const int k0 = j * 128;
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(tS + c * 32, v[c]);
      tmem_ld_wait();
      if ((p.causal && k0 + 127 > first_row) || k0 + 128 > tile.len) {
        // keys this row may see: [k0, limit)
        const int limit = (p.causal ? min(tile.len, q_idx + 1) : tile.len) - k0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e >= limit) v[c][e] = 0xff800000u;  // -inf
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
#pragma unroll
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
        l *= alpha;
        m = m_use;
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x0 = fast_exp2(__uint_as_float(v[c][e * 2]) * p.scale_log2 - m);
          const float x1 = fast_exp2(__uint_as_float(v[c][e * 2 + 1]) * p.scale_log2 - m);
          sum[e & 3] += x0 + x1;
          pk[e] = pack_bf16(x0, x1);
        }
        tmem_st_32x16(tS + c * 16, pk);  // P over the first 64 columns of S, which is in registers by now
      }
      tmem_st_wait();
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t]);
    }
    if (ok && n_t > 0) ok = warp_wait(&o_full[t], 0, abort_flag);
    if (ok && n_t > 0) {
      tc_fence_after_sync();
      const float inv_l = 1.f / l;
      const long long row = (long long)tile.start + q_idx;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32(tO + c * 32, o);
        tmem_ld_wait();
        if (q_idx < tile.len) {
          __nv_bfloat16* dst = p.o + row * p.o_stride + h * D + c * 32;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack_bf16(__uint_as_float(o[u * 8 + e * 2]) * inv_l, __uint_as_float(o[u * 8 + e * 2 + 1]) * inv_l);
            reinterpret_cast<uint4*>(dst)[u] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (q_idx < tile.len) p.lse[(long long)h * p.T + row] = (m + log2f(l)) * 0.6931471805599453f;
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  }
  leave(abort_flag, warp, tmem_base);
}

template <int D>
static int launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const FwdArgs& p,
                      cudaStream_t stream) {
  constexpr int SMEM = 6 * (D / 64) * kChunkBytes + 256;
  constexpr auto kern = packed_fwd_kernel<D>;
  if (cudaError_t e = pb::allow_smem<kern, SMEM>(); e != cudaSuccess) return (int)e;
  kern<<<(unsigned)p.max_tiles * p.Hq, 320, SMEM, stream>>>(tq, tk, tv, p);
  pb_count_launch(1);
  return (int)cudaGetLastError();
}

}  // namespace pbv

extern "C" {

// q/k/v: bf16 [T, ...], head h at columns [h * D, (h + 1) * D) of the respective pointer, row pitches in elements.
// o: [T, o_stride] bf16, every row written (zeros in padding); lse: [Hq, T] fp32, rows of documents written.
// tiles / count: the layout's table of 256-row tiles (max_tiles entries at most).
int pb_packed_attention_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int* tiles,
                            const int* count, int max_tiles, long long T, int Hq, int Hkv, int D, long long q_stride,
                            long long k_stride, long long v_stride, long long o_stride, float softmax_scale, int causal,
                            int* err_dev, void* stream_) {
  using namespace pbv;
  if (D != 64 && D != 128) return -1;
  if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0) return -2;
  if ((q_stride % 8) || (k_stride % 8) || (v_stride % 8) || (o_stride % 8)) return -3;
  if (reinterpret_cast<uintptr_t>(o) & 15) return -3;
  if (T < 1 || T > 0x7fffffffLL || max_tiles < 1 || (long long)max_tiles * Hq > 0x7fffffffLL) return -4;
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
  p.count = count;
  p.max_tiles = max_tiles;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.scale_log2 = softmax_scale * kLog2e;
  p.causal = causal;
  p.err = err_dev;
  p.head_group = pb::attention_head_group(max_tiles, Hq);
  return D == 128 ? launch_fwd<128>(tq, tk, tv, p, stream) : launch_fwd<64>(tq, tk, tv, p, stream);
}

}  // extern "C"

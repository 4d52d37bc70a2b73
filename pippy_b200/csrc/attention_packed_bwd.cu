// Attention over packed documents, backward, for sm_100a: two passes without atomics, the same bits on every run.
//
//   p_ij = exp(s q_i k_j - lse_i), dp_ij = do_i v_j, ds_ij = p_ij (dp_ij - delta_i), delta_i = do_i o_i
//   dq_i = s sum_j ds_ij k_j;  dv_j = sum_i p_ij do_i;  dk_j = s sum_i ds_ij q_i
//
// Pass 1 (dQ): a block keeps 128 query rows of one head (Q and dO as bf16 in TMEM, delta formed on the way) and streams the
// blocks of 128 keys: S = Q K^T, dP = dO V^T, dQ += dS K.
// Pass 2 (dK, dV): a block keeps 128 keys of one key head (K, V in shared memory) and streams the blocks of 128 queries of
// every query head of its group: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q.
// Seven products where a single pass needs five, but that one has to add dQ up across blocks, with atomics whose order
// changes the result, or through 4 bytes an element and block of extra traffic.
//
// TMEM is full (512 columns) in both, with one 128-column buffer for each score tile.  The tensor pipe still never waits
// for a buffer, because the softmax is split into two phases that run under two products each (pass 2 in steady state):
//     tensor pipe   dV(i)  S(i+1)  dK(i)  dP(i+1)  dV(i+1)  S(i+2) ...
//     softmax              dS(i)   P(i+1)          dS(i+1)
// and pass 1 likewise: S(i+1) dQ(i) dP(i+1).  P and dS (bf16) overwrite the score columns that they were computed from and
// are the products' TMEM operand; the streamed tiles serve K-major for the scores and MN-major for the accumulation.
//
// P and dS are rounded to bf16, the type of their products' other operand; scores, accumulators, lse and delta are fp32.
// The rotation of q and k is undone on dQ and dK in the epilogues, before their one rounding.
// Warps: 0 loads, 1 issues MMAs and owns TMEM, 2..17 softmax: four per TMEM lane quarter, 32 of the block's columns each.
#include "attention_packed.cuh"

namespace pbv {

struct BwdArgs {
  const __nv_bfloat16 *q, *dO, *o;  // pass 1 reads its resident rows directly
  long long q_stride, do_stride, o_stride;
  const float* lse;  // [Hq, T] natural log
  float* delta;      // [Hq, T]: written by pass 1, read by pass 2
  __nv_bfloat16* out_a;  // pass 1: dQ; pass 2: dK
  __nv_bfloat16* out_b;  // pass 2: dV
  long long out_stride;
  const float *cs, *sn;  // [table_rows, D / 2], null: no rotation
  int table_rows;
  long long T;
  const Tile* tiles;  // of 128 rows
  const int* count;
  int max_tiles, Hq, Hkv;
  float scale, scale_log2;
  int causal;
  int head_group;
  int* err;
};

constexpr int kBwdThreads = 64 + 512;

__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

// One row of an accumulator [128, D] to bf16: this warp's columns are [sub * D / 8, + D / 8) of each half, so that a thread
// holds both elements of every pair that the rotation mixes.  `pos` < 0: no rotation to undo.
template <int D>
__device__ __forceinline__ void write_row(uint32_t acc, int sub, float scale, const BwdArgs& p, int pos, bool row_ok,
                                          __nv_bfloat16* dst) {
  constexpr int N = D / 8;
  uint32_t a[N], b[N];
  if constexpr (N == 16) {
    tmem_ld_32x16(acc + sub * N, a);
    tmem_ld_32x16(acc + D / 2 + sub * N, b);
  } else {
    tmem_ld_32x8(acc + sub * N, a);
    tmem_ld_32x8(acc + D / 2 + sub * N, b);
  }
  tmem_ld_wait();
  if (!row_ok) return;
  const bool turn = pos >= 0 && pos < p.table_rows;
  const float* cs = p.cs + (turn ? (long long)pos * (D / 2) + sub * N : 0);
  const float* sn = p.sn + (turn ? (long long)pos * (D / 2) + sub * N : 0);
#pragma unroll
  for (int u = 0; u < N / 8; ++u) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (turn) {
        c = __ldg(reinterpret_cast<const float4*>(cs + u * 8 + e));
        s = __ldg(reinterpret_cast<const float4*>(sn + u * 8 + e));
      }
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = __uint_as_float(a[u * 8 + e + i]) * scale, g = __uint_as_float(b[u * 8 + e + i]) * scale;
        x[i] = f * cc[i] + g * ss[i];
        y[i] = g * cc[i] - f * ss[i];
      }
      lo[e / 2] = pack_bf16(x[0], x[1]), lo[e / 2 + 1] = pack_bf16(x[2], x[3]);
      hi[e / 2] = pack_bf16(y[0], y[1]), hi[e / 2 + 1] = pack_bf16(y[2], y[3]);
    }
    *reinterpret_cast<uint4*>(dst + sub * N + u * 8) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    *reinterpret_cast<uint4*>(dst + D / 2 + sub * N + u * 8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  }
}

// ------------------------------------------------------------------------------------------------ pass 1: dQ
constexpr int kStagesK = 3, kStagesV = 2;  // a K tile is read by S and, two products later, by dQ

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, BwdArgs p) {
  constexpr int NCH = D / 64;
  constexpr int TILE_BYTES = NCH * kChunkBytes;

  const TileOrder order = tile_order(blockIdx.x, p.max_tiles, p.Hq, p.head_group);
  if (order.tile_rank >= *p.count) return;
  const Tile tile = p.tiles[order.tile_rank];
  const int h = order.index;
  const int q0 = tile.rank * 128;
  if (tile.pad) {
    clear_rows<D>(p.out_a, p.out_stride, (long long)tile.start + q0, min(128, tile.len - q0), h * D);
    return;
  }
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (smem != smem_raw) {
    if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sV = sK + kStagesK * TILE_BYTES;
  float* s_delta = reinterpret_cast<float*>(sV + kStagesV * TILE_BYTES);  // [2][128]: the two halves of a row
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_delta + 256);
  uint64_t* res_ready = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = k_full + kStagesK;
  uint64_t* v_full = k_empty + kStagesK;
  uint64_t* v_empty = v_full + kStagesV;
  uint64_t* s_full = v_empty + kStagesV;
  uint64_t* s_read = s_full + 1;
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_ready = s_full + 3;
  uint64_t* acc_full = s_full + 4;
  uint64_t* aux = s_full + 5;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 6);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int hkv = h / (p.Hq / p.Hkv);
  const int nblk = ((p.causal ? min(tile.len, q0 + 128) : tile.len) + 127) / 128;

  if (threadIdx.x == 0) {
    mbar_init(res_ready, 16);
    for (int i = 0; i < kStagesK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kStagesV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, 16);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 16);
    mbar_init(acc_full, 1);
    mbar_init(aux, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tQ = tmem_base;          // bf16 pairs, D / 2 columns
  const uint32_t tDO = tmem_base + 64;    // bf16 pairs, D / 2 columns
  const uint32_t tS = tmem_base + 128;    // 128 columns
  const uint32_t tDP = tmem_base + 256;   // 128 columns; dS over them
  const uint32_t tAcc = tmem_base + 384;  // D columns

  if (warp == 0) {
    bool ok = true;
    uint32_t aux_phase = 0;
    for (int j = 0; j < nblk; ++j) {
      const int sk = j % kStagesK, sv = j % kStagesV;
      const int valid = tile.len - j * 128;
      if (!(ok = warp_wait(&k_empty[sk], ((j / kStagesK) & 1) ^ 1, abort_flag))) break;
      if (!(ok = load_tile<NCH>(sK + sk * TILE_BYTES, &tmK, &k_full[sk], aux, &aux_phase, hkv * D, tile.start + j * 128,
                                valid, lane, abort_flag)))
        break;
      if (!(ok = warp_wait(&v_empty[sv], ((j / kStagesV) & 1) ^ 1, abort_flag))) break;
      // dP of a key beyond the document is replaced by the mask: V needs no clearing here
      load_tile<NCH>(sV + sv * TILE_BYTES, &tmV, &v_full[sv], aux, &aux_phase, hkv * D, tile.start + j * 128, 128, lane,
                     abort_flag);
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  } else if (warp == 1) {
    const uint32_t idesc_t = make_idesc_bf16(128, 128, 0, 0);
    const uint32_t idesc_acc = make_idesc_bf16(128, D, 0, 1);
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool got = warp_wait(bar, parity, abort_flag);
      tc_fence_after_sync();
      return got;
    };
    // scores: A = resident bf16 rows in TMEM, B = streamed tile, K-major
    auto issue_scores = [&](uint32_t dst, uint32_t a, const uint8_t* tile_b, uint64_t* full, uint64_t* empty) {
      const uint64_t bd = make_smem_desc(smem_u32(tile_b), 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_ts(dst, a + kk * 8, bd + (((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4), idesc_t, kk != 0);
        umma_commit(full);
        if (empty) umma_commit(empty);
      }
      __syncwarp();
    };
    bool ok = wait(res_ready, 0) && wait(&k_full[0], 0);
    if (ok) {
      issue_scores(tS, tQ, sK, s_full, nullptr);
      ok = wait(&v_full[0], 0);
    }
    if (ok) issue_scores(tDP, tDO, sV, dp_full, &v_empty[0]);
    for (int j = 0; j < nblk && ok; ++j) {
      const bool more = j + 1 < nblk;
      const int next = j + 1;
      if (more) {
        ok = wait(&k_full[next % kStagesK], (next / kStagesK) & 1) && wait(s_read, j & 1);
        if (!ok) break;
        issue_scores(tS, tQ, sK + (next % kStagesK) * TILE_BYTES, s_full, nullptr);
      }
      if (!(ok = wait(ds_ready, j & 1))) break;
      const uint64_t kd = make_smem_desc(smem_u32(sK + (j % kStagesK) * TILE_BYTES), kChunkBytes, 1024);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)  // 16 keys a step: their dS sits in 8 columns at (kk / 2) * 32 + (kk & 1) * 8
          umma_ts(tAcc, tDP + (kk >> 1) * 32 + (kk & 1) * 8, kd + ((kk * 2048) >> 4), idesc_acc, (j | kk) != 0);
        umma_commit(&k_empty[j % kStagesK]);
        if (!more) umma_commit(acc_full);
      }
      __syncwarp();
      if (more) {
        if (!(ok = wait(&v_full[next % kStagesV], (next / kStagesV) & 1))) break;
        issue_scores(tDP, tDO, sV + (next % kStagesV) * TILE_BYTES, dp_full, &v_empty[next % kStagesV]);
      }
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  } else {
    const int sub = (warp - 2) >> 2;  // 0..3: columns [32 sub, 32 sub + 32) of a block
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int q_idx = q0 + r;
    const bool row_ok = q_idx < tile.len;
    const long long row = (long long)tile.start + q_idx;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    bool ok = true;
    {
      // subs 0 and 1 bring the halves of the Q row, 2 and 3 those of the dO row and, with O, their part of delta
      constexpr int W = D / 4;  // 32-bit words of a half row
      const int half = sub & 1;
      const __nv_bfloat16* src = sub < 2 ? p.q + row * p.q_stride : p.dO + row * p.do_stride;
      src += h * D + half * (D / 2);
      const __nv_bfloat16* oth = p.o + row * p.o_stride + h * D + half * (D / 2);
      uint32_t w[W];
      float dot = 0.f;
#pragma unroll
      for (int u = 0; u < W / 4; ++u) {
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (row_ok) {
          x = __ldg(reinterpret_cast<const uint4*>(src) + u);
          if (sub >= 2) y = __ldg(reinterpret_cast<const uint4*>(oth) + u);
        }
        w[u * 4] = x.x, w[u * 4 + 1] = x.y, w[u * 4 + 2] = x.z, w[u * 4 + 3] = x.w;
        const __nv_bfloat162* xb = reinterpret_cast<const __nv_bfloat162*>(&x);
        const __nv_bfloat162* yb = reinterpret_cast<const __nv_bfloat162*>(&y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __bfloat1622float2(xb[e]), g = __bfloat1622float2(yb[e]);
          dot += f.x * g.x + f.y * g.y;
        }
      }
      const uint32_t dst = (sub < 2 ? tQ : tDO) + lane_off + half * W;
      if constexpr (W == 32) tmem_st_32x32(dst, w);
      else tmem_st_32x16(dst, w);
      tmem_st_wait();
      if (sub >= 2) s_delta[half * 128 + r] = dot;
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(res_ready);
    }
    named_bar_or(1, 512, false);
    const float delta = s_delta[r] + s_delta[128 + r];
    float lse2 = 0.f;
    if (row_ok) {
      lse2 = p.lse[(long long)h * p.T + row] * kLog2e;
      if (sub == 0) p.delta[(long long)h * p.T + row] = delta;
    }
    const uint32_t my_s = tS + lane_off + sub * 32, my_dp = tDP + lane_off + sub * 32;
    for (int j = 0; j < nblk; ++j) {
      if (!(ok = warp_wait(s_full, j & 1, abort_flag))) break;
      tc_fence_after_sync();
      uint32_t t[32];
      tmem_ld_32x32(my_s, t);
      tmem_ld_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_read);
      float pr[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) pr[e] = fast_exp2(__uint_as_float(t[e]) * p.scale_log2 - lse2);
      if (j == nblk - 1) {  // the diagonal block (causal) and the one in which the document ends
        const int limit = (p.causal ? min(tile.len, q_idx + 1) : tile.len) - j * 128 - sub * 32;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e >= limit) pr[e] = 0.f;
      }
      if (!(ok = warp_wait(dp_full, j & 1, abort_flag))) break;
      tc_fence_after_sync();
      tmem_ld_32x32(my_dp, t);
      tmem_ld_wait();
      uint32_t pk[16];
      if (j == nblk - 1) {  // 0 * (dP - delta) would let an Inf of a masked column through
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float d = __uint_as_float(t[e]) - delta;
          t[e] = __float_as_uint(pr[e] == 0.f ? 0.f : pr[e] * d);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = pack_bf16(__uint_as_float(t[2 * e]), __uint_as_float(t[2 * e + 1]));
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          pk[e] = pack_bf16(pr[2 * e] * (__uint_as_float(t[2 * e]) - delta), pr[2 * e + 1] * (__uint_as_float(t[2 * e + 1]) - delta));
      }
      tmem_st_32x16(my_dp, pk);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
    }
    if (ok) ok = warp_wait(acc_full, 0, abort_flag);
    if (ok) {
      tc_fence_after_sync();
      write_row<D>(tAcc + lane_off, sub, p.scale, p, p.cs ? q_idx : -1, row_ok, p.out_a + row * p.out_stride + h * D);
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  }
  leave(abort_flag, warp, tmem_base);
}

// ------------------------------------------------------------------------------------------------ pass 2: dK, dV
constexpr int kStagesQ = 3, kStagesDO = 2, kStagesStat = 2;  // a Q tile is read by S and, three products later, by dK

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO, BwdArgs p) {
  constexpr int NCH = D / 64;
  constexpr int TILE_BYTES = NCH * kChunkBytes;

  const TileOrder order = tile_order(blockIdx.x, p.max_tiles, p.Hkv, p.head_group);
  if (order.tile_rank >= *p.count) return;
  const Tile tile = p.tiles[order.tile_rank];
  const int hkv = order.index;
  const int tiles_of_doc = (tile.len + 127) / 128;
  // the table lists tiles by the keys that queries see; the first keys are seen by the most queries
  const int kv_tile = tiles_of_doc - 1 - tile.rank;
  const int k0 = kv_tile * 128;
  if (tile.pad) {
    clear_rows<D>(p.out_a, p.out_stride, (long long)tile.start + k0, min(128, tile.len - k0), hkv * D);
    clear_rows<D>(p.out_b, p.out_stride, (long long)tile.start + k0, min(128, tile.len - k0), hkv * D);
    return;
  }
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (smem != smem_raw) {
    if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE_BYTES;
  uint8_t* sQ = sV + TILE_BYTES;
  uint8_t* sDO = sQ + kStagesQ * TILE_BYTES;
  float* s_stat = reinterpret_cast<float*>(sDO + kStagesDO * TILE_BYTES);  // [stage][lse2, delta][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_stat + kStagesStat * 256);
  uint64_t* res_full = bars;
  uint64_t* q_full = bars + 1;
  uint64_t* q_empty = q_full + kStagesQ;
  uint64_t* do_full = q_empty + kStagesQ;
  uint64_t* do_empty = do_full + kStagesDO;
  uint64_t* stat_full = do_empty + kStagesDO;
  uint64_t* stat_empty = stat_full + kStagesStat;
  uint64_t* s_full = stat_empty + kStagesStat;
  uint64_t* p_ready = s_full + 1;
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_ready = s_full + 3;
  uint64_t* acc_full = s_full + 4;
  uint64_t* aux = s_full + 5;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 6);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = p.Hq / p.Hkv;
  const int blk_start = p.causal ? kv_tile : 0;
  const int per_head = tiles_of_doc - blk_start;
  const int n_it = G * per_head;

  if (threadIdx.x == 0) {
    mbar_init(res_full, 1);
    for (int i = 0; i < kStagesQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < kStagesDO; ++i) {
      mbar_init(&do_full[i], 1);
      mbar_init(&do_empty[i], 1);
    }
    for (int i = 0; i < kStagesStat; ++i) {
      mbar_init(&stat_full[i], 1);
      mbar_init(&stat_empty[i], 16);
    }
    mbar_init(s_full, 1);
    mbar_init(p_ready, 16);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 16);
    mbar_init(acc_full, 1);
    mbar_init(aux, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tS = tmem_base;          // 128 columns; P^T over them
  const uint32_t tDP = tmem_base + 128;   // 128 columns; dS^T over them
  const uint32_t tDV = tmem_base + 256;   // D columns
  const uint32_t tDK = tmem_base + 384;   // D columns

  if (warp == 0) {
    bool ok = true;
    if (lane == 0) {
      // rows beyond the document stay in their own accumulator rows, which are not written
      mbar_expect_tx(res_full, 2 * TILE_BYTES);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        tma_load_2d(sK + c * kChunkBytes, &tmK, res_full, hkv * D + c * 64, tile.start + k0);
        tma_load_2d(sV + c * kChunkBytes, &tmV, res_full, hkv * D + c * 64, tile.start + k0);
      }
    }
    __syncwarp();
    uint32_t aux_phase = 0;
    int g = 0, blk = blk_start;
    for (int it = 0; it < n_it; ++it) {
      const int sq = it % kStagesQ, sd = it % kStagesDO, st = it % kStagesStat;
      const int head = hkv * G + g;
      const int valid = tile.len - blk * 128;
      const int row = tile.start + blk * 128;
      if (!(ok = warp_wait(&q_empty[sq], ((it / kStagesQ) & 1) ^ 1, abort_flag))) break;
      if (!(ok = load_tile<NCH>(sQ + sq * TILE_BYTES, &tmQ, &q_full[sq], aux, &aux_phase, head * D, row, valid, lane,
                                abort_flag)))
        break;
      // a query beyond the document gets lse = inf, so P = exp2(0 - inf) = 0: no mask is needed for the document's end
      if (!(ok = warp_wait(&stat_empty[st], ((it / kStagesStat) & 1) ^ 1, abort_flag))) break;
      const float* lse = p.lse + (long long)head * p.T + row;
      const float* delta = p.delta + (long long)head * p.T + row;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = u * 32 + lane;
        s_stat[st * 256 + i] = i < valid ? lse[i] * kLog2e : CUDART_INF_F;
        s_stat[st * 256 + 128 + i] = i < valid ? delta[i] : 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&stat_full[st]);
      if (!(ok = warp_wait(&do_empty[sd], ((it / kStagesDO) & 1) ^ 1, abort_flag))) break;
      if (!(ok = load_tile<NCH>(sDO + sd * TILE_BYTES, &tmDO, &do_full[sd], aux, &aux_phase, head * D, row, valid, lane,
                                abort_flag)))
        break;
      if (++blk == tiles_of_doc) {
        blk = blk_start;
        ++g;
      }
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  } else if (warp == 1) {
    const uint32_t idesc_t = make_idesc_bf16(128, 128, 0, 0);
    const uint32_t idesc_acc = make_idesc_bf16(128, D, 0, 1);
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool got = warp_wait(bar, parity, abort_flag);
      tc_fence_after_sync();
      return got;
    };
    auto issue_scores = [&](uint32_t dst, const uint8_t* tile_a, const uint8_t* tile_b, uint64_t* full) {
      const uint64_t ad = make_smem_desc(smem_u32(tile_a), 16, 1024);
      const uint64_t bd = make_smem_desc(smem_u32(tile_b), 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4;
          umma_ss<1>(dst, ad + off, bd + off, idesc_t, kk != 0);
        }
        umma_commit(full);
      }
      __syncwarp();
    };
    // accumulation: A = P^T or dS^T (bf16 in TMEM), B = streamed tile, MN-major
    auto issue_acc = [&](uint32_t dst, uint32_t a, const uint8_t* tile_b, int it, uint64_t* empty, uint64_t* last) {
      const uint64_t bd = make_smem_desc(smem_u32(tile_b), kChunkBytes, 1024);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_ts(dst, a + (kk >> 1) * 32 + (kk & 1) * 8, bd + ((kk * 2048) >> 4), idesc_acc, (it | kk) != 0);
        umma_commit(empty);
        if (last) umma_commit(last);
      }
      __syncwarp();
    };
    bool ok = wait(res_full, 0) && wait(&q_full[0], 0);
    if (ok) {
      issue_scores(tS, sK, sQ, s_full);
      ok = wait(&do_full[0], 0);
    }
    if (ok) issue_scores(tDP, sV, sDO, dp_full);
    for (int it = 0; it < n_it && ok; ++it) {
      const bool more = it + 1 < n_it;
      const int next = it + 1;
      if (!(ok = wait(p_ready, it & 1))) break;
      issue_acc(tDV, tS, sDO + (it % kStagesDO) * TILE_BYTES, it, &do_empty[it % kStagesDO], nullptr);
      if (more) {
        if (!(ok = wait(&q_full[next % kStagesQ], (next / kStagesQ) & 1))) break;
        issue_scores(tS, sK, sQ + (next % kStagesQ) * TILE_BYTES, s_full);
      }
      if (!(ok = wait(ds_ready, it & 1))) break;
      issue_acc(tDK, tDP, sQ + (it % kStagesQ) * TILE_BYTES, it, &q_empty[it % kStagesQ], more ? nullptr : acc_full);
      if (more) {
        if (!(ok = wait(&do_full[next % kStagesDO], (next / kStagesDO) & 1))) break;
        issue_scores(tDP, sV, sDO + (next % kStagesDO) * TILE_BYTES, dp_full);
      }
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  } else {
    const int sub = (warp - 2) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // key row of this thread
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t my_s = tS + lane_off + sub * 32, my_dp = tDP + lane_off + sub * 32;
    bool ok = true;
    int blk = blk_start;
    for (int it = 0; it < n_it; ++it) {
      const int st = it % kStagesStat;
      const float* lse2 = s_stat + st * 256 + sub * 32;
      const float* delta = lse2 + 128;
      if (!(ok = warp_wait(&stat_full[st], (it / kStagesStat) & 1, abort_flag))) break;
      if (!(ok = warp_wait(s_full, it & 1, abort_flag))) break;
      tc_fence_after_sync();
      uint32_t t[32];
      tmem_ld_32x32(my_s, t);
      tmem_ld_wait();
      float pr[32];
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 l4 = *reinterpret_cast<const float4*>(lse2 + e);
        pr[e] = fast_exp2(__uint_as_float(t[e]) * p.scale_log2 - l4.x);
        pr[e + 1] = fast_exp2(__uint_as_float(t[e + 1]) * p.scale_log2 - l4.y);
        pr[e + 2] = fast_exp2(__uint_as_float(t[e + 2]) * p.scale_log2 - l4.z);
        pr[e + 3] = fast_exp2(__uint_as_float(t[e + 3]) * p.scale_log2 - l4.w);
      }
      const bool diagonal = p.causal && blk == kv_tile;
      if (diagonal) {  // queries before this key
        const int first = r - sub * 32;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e < first) pr[e] = 0.f;
      }
      uint32_t pk[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) pk[e] = pack_bf16(pr[2 * e], pr[2 * e + 1]);
      tmem_st_32x16(my_s, pk);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
      if (!(ok = warp_wait(dp_full, it & 1, abort_flag))) break;
      tc_fence_after_sync();
      tmem_ld_32x32(my_dp, t);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        const float4 d4 = *reinterpret_cast<const float4*>(delta + e);
        pk[e / 2] = pack_bf16(pr[e] * (__uint_as_float(t[e]) - d4.x), pr[e + 1] * (__uint_as_float(t[e + 1]) - d4.y));
        pk[e / 2 + 1] = pack_bf16(pr[e + 2] * (__uint_as_float(t[e + 2]) - d4.z), pr[e + 3] * (__uint_as_float(t[e + 3]) - d4.w));
      }
      tmem_st_32x16(my_dp, pk);
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(ds_ready);
        mbar_arrive(&stat_empty[st]);
      }
      if (++blk == tiles_of_doc) blk = blk_start;
    }
    if (ok) ok = warp_wait(acc_full, 0, abort_flag);
    if (ok) {
      tc_fence_after_sync();
      const int k_idx = k0 + r;
      const bool row_ok = k_idx < tile.len;
      const long long row = (long long)tile.start + k_idx;
      write_row<D>(tDK + lane_off, sub, p.scale, p, p.cs ? k_idx : -1, row_ok, p.out_a + row * p.out_stride + hkv * D);
      write_row<D>(tDV + lane_off, sub, 1.f, p, -1, row_ok, p.out_b + row * p.out_stride + hkv * D);
    }
    if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  }
  leave(abort_flag, warp, tmem_base);
}

template <int D>
static int launch_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                      BwdArgs p, __nv_bfloat16* dq, __nv_bfloat16* dk, __nv_bfloat16* dv, cudaStream_t stream) {
  constexpr int TILE = (D / 64) * kChunkBytes;
  constexpr int SMEM1 = (kStagesK + kStagesV) * TILE + 1024 + 256;
  constexpr int SMEM2 = (2 + kStagesQ + kStagesDO) * TILE + kStagesStat * 1024 + 256;
  static_assert(SMEM2 <= 232448, "one block's shared memory");
  constexpr auto pass1 = packed_dq_kernel<D>;
  constexpr auto pass2 = packed_dkv_kernel<D>;
  if (cudaError_t e = pb::allow_smem<pass1, SMEM1>(); e != cudaSuccess) return (int)e;
  if (cudaError_t e = pb::allow_smem<pass2, SMEM2>(); e != cudaSuccess) return (int)e;
  p.out_a = dq;
  p.head_group = attention_head_group(p.max_tiles, p.Hq);
  pass1<<<(unsigned)p.max_tiles * p.Hq, kBwdThreads, SMEM1, stream>>>(tk, tv, p);
  pb_count_launch(1);
  p.out_a = dk;
  p.out_b = dv;
  p.head_group = attention_head_group(p.max_tiles, p.Hkv);
  pass2<<<(unsigned)p.max_tiles * p.Hkv, kBwdThreads, SMEM2, stream>>>(tk, tv, tq, tdo, p);
  pb_count_launch(1);
  return (int)cudaGetLastError();
}

}  // namespace pbv

extern "C" {

// Layouts as in pb_packed_attention_fwd; q and k rotated as the forward saw them.  dq/dk/dv: bf16 rows of dqkv_stride, every
// row written (zeros in padding).  cs/sn [table_rows, D / 2] (null: none): dq and dk are turned back by the row's position.
// delta: [Hq, T] fp32 scratch of this call.  tiles: the layout's table of 128-row tiles.
int pb_packed_attention_bwd(const void* dO, const void* q, const void* k, const void* v, const void* o,
                            const float* lse, float* delta, void* dq, void* dk, void* dv, const float* cs,
                            const float* sn, int table_rows, const int* tiles, const int* count, int max_tiles,
                            long long T, int Hq, int Hkv, int D, long long q_stride, long long k_stride,
                            long long v_stride, long long o_stride, long long do_stride, long long dqkv_stride,
                            float softmax_scale, int causal, int* err_dev, void* stream_) {
  using namespace pbv;
  if (D != 64 && D != 128) return -1;
  if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0) return -2;
  if ((q_stride % 8) || (k_stride % 8) || (v_stride % 8) || (o_stride % 8) || (do_stride % 8) || (dqkv_stride % 8)) return -3;
  uintptr_t all = 0;
  for (const void* x : {dO, q, o, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)cs, (const void*)sn})
    all |= reinterpret_cast<uintptr_t>(x);
  if (all & 15) return -3;
  if (T < 1 || T > 0x7fffffffLL || max_tiles < 1 || (long long)max_tiles * Hq > 0x7fffffffLL) return -4;
  CUtensorMap tq, tk, tv, tdo;
  int r = 0;
  r |= pb::make_tmap_bf16_2d(&tq, q, (uint64_t)Hq * D, T, (uint64_t)q_stride, 64, 128);
  r |= pb::make_tmap_bf16_2d(&tk, k, (uint64_t)Hkv * D, T, (uint64_t)k_stride, 64, 128);
  r |= pb::make_tmap_bf16_2d(&tv, v, (uint64_t)Hkv * D, T, (uint64_t)v_stride, 64, 128);
  r |= pb::make_tmap_bf16_2d(&tdo, dO, (uint64_t)Hq * D, T, (uint64_t)do_stride, 64, 128);
  if (r) return -10;
  BwdArgs p;
  memset(&p, 0, sizeof(p));
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.dO = reinterpret_cast<const __nv_bfloat16*>(dO);
  p.o = reinterpret_cast<const __nv_bfloat16*>(o);
  p.q_stride = q_stride, p.do_stride = do_stride, p.o_stride = o_stride;
  p.lse = lse;
  p.delta = delta;
  p.out_stride = dqkv_stride;
  p.cs = cs, p.sn = sn;
  p.table_rows = table_rows;
  p.T = T;
  p.tiles = reinterpret_cast<const Tile*>(tiles);
  p.count = count;
  p.max_tiles = max_tiles;
  p.Hq = Hq, p.Hkv = Hkv;
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * kLog2e;
  p.causal = causal;
  p.err = err_dev;
  auto b = [](void* x) { return reinterpret_cast<__nv_bfloat16*>(x); };
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  return D == 128 ? launch_bwd<128>(tq, tk, tv, tdo, p, b(dq), b(dk), b(dv), stream)
                  : launch_bwd<64>(tq, tk, tv, tdo, p, b(dq), b(dk), b(dv), stream);
}

}  // extern "C"

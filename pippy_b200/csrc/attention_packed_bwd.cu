// Attention over packed documents, backward, for sm_100a: two passes, no result is added to by
// atomics: the same bits on every run.
//
//   p_ij = exp(s q_i k_j - lse_i), dp_ij = do_i v_j, ds_ij = p_ij (dp_ij - delta_i), delta_i = do_i o_i
//   dq_i = s sum_j ds_ij k_j;  dv_j = sum_i p_ij do_i;  dk_j = s sum_i ds_ij q_i
//
// Pass 1 (dQ): an item is 128 query rows of one head (Q and dO as bf16 in TMEM, delta formed on the way); the blocks of 128
// keys are streamed: S = Q K^T, dP = dO V^T, dQ += dS K.
// Pass 2 (dK, dV): an item is 128 keys of one key head (K, V in shared memory); the blocks of 128 queries of every query
// head of its group are streamed: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q.
// Seven products where a single pass needs five, but that one has to add dQ up across blocks, with atomics whose order
// changes the result, or through 4 bytes an element and block of extra traffic.
//
// TMEM is full (512 columns) in both, with one 128-column buffer for each score tile.  The tensor pipe need not wait for a
// buffer all the same, because the softmax is split into two phases that run under two products each (pass 2):
//     tensor pipe   dV(i)  S(i+1)  dK(i)  dP(i+1)  dV(i+1)  S(i+2) ...
//     softmax              dS(i)   P(i+1)          dS(i+1)
// and pass 1 likewise: dQ(i) dP(i+1) S(i+2).  P and dS (bf16) overwrite the score columns that they were computed from and
// are the products' TMEM operand; the streamed tiles serve K-major for the scores and MN-major for the accumulation.
//
// Blocks stay resident and walk a list of items (Items), so that the loads of the next item run under the end of the
// present one: with documents of a few hundred tokens an item is one to three blocks, and its start and end took longer
// than they did.
//
// Measured, D = 128, causal: one row of 16 384 tokens in 4 documents, 8 query and 2 key heads: pass 1 319 us (1.19 PFLOP/s of
// its three products), pass 2 417 us (1.21 of its four) and 17 to add its parts; 2 x 4096 tokens in 24 documents, 32 heads:
// 139 and 165 us.  Pass 1 is bound by the chain of a block through its one buffer for each score tile, pass 2 by the
// shared-memory port besides: both operands of its score products and one of the others come from there.
//
// P and dS are rounded to bf16, the type of their products' other operand; scores, accumulators, lse and delta are fp32.
// The rotation of q and k is undone on dQ and dK in the epilogues, before their one rounding.
#include "attention_packed_bwd.cuh"

namespace pbv {

// ------------------------------------------------------------------------------------------------ pass 1: dQ
constexpr int kStagesK = 3, kStagesV = 2;  // a K tile is read by S and, two products later, by dQ
constexpr int kDqThreads = 512;

// Warps: 0 loads (TMA), 1 issues MMAs and owns TMEM, 2 clears what reaches beyond a document, 4..11 softmax (two per TMEM lane
// quarter, 64 of a block's columns each), 12..15 bring an item's Q and dO from shared memory to TMEM and form delta.
template <int D, bool kTurn>
__global__ void __launch_bounds__(kDqThreads, 1)
packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                 const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, BwdArgs p) {
  constexpr int NCH = D / 64;
  constexpr int TILE_BYTES = NCH * kChunkBytes;

  // addresses of shared memory are constants, as long as nothing is computed from where it begins
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {  // the launch reserves no slack for re-alignment
    if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sQ = smem;  // staging for the next item's resident rows
  uint8_t* sDO = sQ + TILE_BYTES;
  uint8_t* sK = sDO + TILE_BYTES;
  uint8_t* sV = sK + kStagesK * TILE_BYTES;
  float* s_stat = reinterpret_cast<float*>(sV + kStagesV * TILE_BYTES);  // [item & 1][lse2, delta][128]
  float* s_delta = s_stat + 512;                                         // [128] delta of the item that is being brought
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_delta + 128);
  uint64_t* stage_full = bars;       // Q and dO of an item are in shared memory
  uint64_t* stage_empty = bars + 1;  // ... and have been taken to TMEM
  uint64_t* res_ready = bars + 2;    // Q, dO in TMEM; lse and delta in s_stat
  uint64_t* res_empty = bars + 3;    // the item's last scores are complete, and its lse and delta have been read
  uint64_t* k_full = bars + 4;
  uint64_t* k_empty = k_full + kStagesK;
  uint64_t* k_raw = k_empty + kStagesK;
  uint64_t* v_full = k_raw + kStagesK;
  uint64_t* v_empty = v_full + kStagesV;
  uint64_t* s_full = v_empty + kStagesV;
  uint64_t* s_read = s_full + 1;
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_ready = s_full + 3;
  uint64_t* acc_full = s_full + 4;
  uint8_t* sStage = reinterpret_cast<uint8_t*>(bars) + 256 + ItemRing::kBytes;  // D = 64 only
  ItemRing ring(reinterpret_cast<uint8_t*>(bars) + 256, s_full + 5);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 5 + ItemRing::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  let_next_start();
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.counter) *p.counter = 0;  // pass 2's
  const int count = p.counts[1];  // longer documents only: see attention_packed_short.cu
  const int G = p.Hq / p.Hkv;
  // an item: a tile of queries of head h and the blocks of keys that it sees
  Items items(count * p.Hq, nullptr);
  bool ok = true;
  Tile tile;
  int h = 0, nblk = 0;
  auto publish_next = [&]() {  // by the loading warp; false after the last
    const int i = items.next(lane);
    tile.start = -1;
    if (i >= 0) {
      const TileOrder order = tile_order(i, count, p.Hq, p.head_group);
      tile = p.tiles[order.tile_rank];
      h = order.index;
      nblk = ((p.causal ? min(tile.len, tile.rank * 128 + 128) : tile.len) + 127) / 128;
    }
    ok = ring.put(make_int4(tile.start, tile.len, tile.rank, h), make_int4(nblk, 0, 0, 0), make_int4(0, 0, 0, 0), lane, abort_flag);
    return ok && tile.start >= 0;
  };
  auto next_item = [&]() {  // by the others
    int4 a, b, c;
    if (!(ok = ring.get(a, b, c, lane, abort_flag))) return false;
    tile.start = a.x, tile.len = a.y, tile.rank = a.z, h = a.w, nblk = b.x;
    return tile.start >= 0;
  };

  if (threadIdx.x == 0) {
    mbar_init(stage_full, 1);
    mbar_init(stage_empty, 4);
    mbar_init(res_ready, 4);
    mbar_init(res_empty, 9);
    for (int i = 0; i < kStagesK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&k_raw[i], 1);
    }
    for (int i = 0; i < kStagesV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 8);
    }
    mbar_init(s_full, 1);
    mbar_init(s_read, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 8);
    mbar_init(acc_full, 1);
    ring.init(14);  // MMA, clearing, softmax, Q and dO
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

  int it = 0;  // items so far
  int n = 0;   // blocks so far
  // launched with 128 registers a thread: 64 + 2 x 168 + 112 = 4 x 128
  if (warp < 4) {
    give_registers<64>();
    if (warp == 0) {
      while (ok && publish_next()) {
        const int hkv = h / G;
        if (!(ok = warp_wait(stage_empty, (it & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          mbar_expect_tx(stage_full, 2 * TILE_BYTES);
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            tma_load_2d(sQ + c * kChunkBytes, &tmQ, stage_full, h * D + c * 64, tile.start + tile.rank * 128);
            tma_load_2d(sDO + c * kChunkBytes, &tmDO, stage_full, h * D + c * 64, tile.start + tile.rank * 128);
          }
        }
        for (int j = 0; j < nblk; ++j, ++n) {
          const int sk = n % kStagesK, sv = n % kStagesV;
          if (!(ok = warp_wait(&k_empty[sk], ((n / kStagesK) & 1) ^ 1, abort_flag))) break;
          if (lane == 0)
            load_tile<NCH>(sK + sk * TILE_BYTES, &tmK, tile.len - j * 128 < 128 ? &k_raw[sk] : &k_full[sk], hkv * D,
                           tile.start + j * 128);
          if (!(ok = warp_wait(&v_empty[sv], ((n / kStagesV) & 1) ^ 1, abort_flag))) break;
          // dP of a key beyond the document is replaced by the mask: V needs no clearing here
          if (lane == 0) load_tile<NCH>(sV + sv * TILE_BYTES, &tmV, &v_full[sv], hkv * D, tile.start + j * 128);
        }
        ++it;
      }
    } else if (warp == 1) {
      // the whole warp walks the loops; one elected lane, the same every time, issues the MMAs and their commits
      const uint32_t idesc_t = make_idesc_bf16(128, 128, 0, 0);
      const uint32_t idesc_acc = make_idesc_bf16(128, D, 0, 1);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool got = warp_wait(bar, parity, abort_flag);
        tc_fence_after_sync();
        return got;
      };
      // scores: A = resident bf16 rows in TMEM, B = streamed tile, K-major
      auto issue_scores = [&](uint32_t dst, uint32_t a, const uint8_t* tile_b, uint64_t* full, uint64_t* last) {
        const uint64_t bd = make_smem_desc(smem_u32(tile_b), 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_ts(dst, a + kk * 8, bd + (((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4), idesc_t, kk != 0);
          umma_commit(full);
          if (last) umma_commit(last);
        }
        __syncwarp();
      };
      while (ok && next_item()) {
        if (!(ok = wait(res_ready, it & 1) && wait(&k_full[n % kStagesK], (n / kStagesK) & 1))) break;
        issue_scores(tS, tQ, sK + (n % kStagesK) * TILE_BYTES, s_full, nullptr);
        if (!(ok = wait(&v_full[n % kStagesV], (n / kStagesV) & 1))) break;
        issue_scores(tDP, tDO, sV + (n % kStagesV) * TILE_BYTES, dp_full, nblk == 1 ? res_empty : nullptr);
        for (int j = 0; j < nblk; ++j, ++n) {
          const bool more = j + 1 < nblk;
          const int m = n + 1;
          if (more) {
            if (!(ok = wait(&k_full[m % kStagesK], (m / kStagesK) & 1) && wait(s_read, n & 1))) break;
            issue_scores(tS, tQ, sK + (m % kStagesK) * TILE_BYTES, s_full, nullptr);
            // what the next scores need is waited for while there is nothing to issue anyway
            if (!(ok = wait(&v_full[m % kStagesV], (m / kStagesV) & 1))) break;
          }
          if (!(ok = wait(ds_ready, n & 1))) break;
          const uint64_t kd = make_smem_desc(smem_u32(sK + (n % kStagesK) * TILE_BYTES), kChunkBytes, 1024);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)  // 16 keys a step: their dS sits in 8 columns at (kk / 4) * 64 + (kk % 4) * 8
              umma_ts(tAcc, tDP + (kk >> 2) * 64 + (kk & 3) * 8, kd + ((kk * 2048) >> 4), idesc_acc, (j | kk) != 0);
            umma_commit(&k_empty[n % kStagesK]);
            if (!more) umma_commit(acc_full);
          }
          __syncwarp();
          if (more)
            issue_scores(tDP, tDO, sV + (m % kStagesV) * TILE_BYTES, dp_full, j + 2 == nblk ? res_empty : nullptr);
        }
        ++it;
    }
  } else if (warp == 2) {
    uint32_t phases = 0;  // of the k_raw barriers
    while (ok && next_item()) {
      n += nblk;
      const int valid = tile.len - (nblk - 1) * 128;  // only an item's last block can reach beyond its document
      if (valid >= 128) continue;
      const int sk = (n - 1) % kStagesK;
      if (!(ok = warp_wait(&k_raw[sk], (phases >> sk) & 1, abort_flag))) break;
      phases ^= 1u << sk;
      clear_tail<NCH>(sK + sk * TILE_BYTES, valid, &k_full[sk], lane);
    }
    }
  } else if (warp >= 12) {
    give_registers<112>();
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    while (ok && next_item()) {
      const bool row_ok = tile.rank * 128 + r < tile.len;
      const long long row = (long long)tile.start + tile.rank * 128 + r;
      const float lse2 = row_ok ? p.lse[(long long)h * p.T + row] * kLog2e : 0.f;
      // delta = dO O: D / 8 lanes to a row, so that O is read in whole lines, all of them on their way before dO is waited for
      constexpr int kLanes = D / 8, kRows = 32 / kLanes;
      const int u = lane % kLanes, first = quarter * 32 + lane / kLanes;
      uint4 y[kLanes];
#pragma unroll
      for (int k = 0; k < kLanes; ++k)
        y[k] = tile.rank * 128 + first + k * kRows < tile.len
                   ? __ldg(reinterpret_cast<const uint4*>(p.o + ((long long)tile.start + tile.rank * 128 + first + k * kRows) * p.o_stride + h * D) + u)
                   : make_uint4(0, 0, 0, 0);
      if (!(ok = warp_wait(stage_full, it & 1, abort_flag))) break;
      row_dots<D, kLanes>(sDO, y, first, u, s_delta);
      __syncwarp();
      const float delta = s_delta[r];
      __syncwarp();
      if (row_ok) p.delta[(long long)h * p.T + row] = delta;
      if (!(ok = warp_wait(res_empty, (it & 1) ^ 1, abort_flag))) break;
      tc_fence_after_sync();
      // (the softmax takes part in res_empty: without it this warp could be two items ahead of it, and res_ready two phases)
      s_stat[(it & 1) * 256 + r] = lse2;
      s_stat[(it & 1) * 256 + 128 + r] = row_ok ? delta : 0.f;
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          uint32_t w[32];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const uint4 x = piece_of(which == 0 ? sQ : sDO, r, c * 8 + u);
            w[u * 4] = x.x, w[u * 4 + 1] = x.y, w[u * 4 + 2] = x.z, w[u * 4 + 3] = x.w;
          }
          tmem_st_32x32((which == 0 ? tQ : tDO) + lane_off + c * 32, w);
        }
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(stage_empty);
        mbar_arrive(res_ready);
      }
      ++it;
    }
  } else {
    take_registers<168>();
    const int sub = (warp - 4) >> 2;  // 0, 1: columns [64 sub, 64 sub + 64) of a block
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t my_s = tS + lane_off + sub * 64, my_dp = tDP + lane_off + sub * 64;
    while (ok && next_item()) {
      const int q0 = tile.rank * 128, q_idx = q0 + r;
      if (!(ok = warp_wait(res_ready, it & 1, abort_flag))) break;
      const float lse2 = s_stat[(it & 1) * 256 + r], delta = s_stat[(it & 1) * 256 + 128 + r];
      __syncwarp();
      if (lane == 0) mbar_arrive(res_empty);
      const f32x2 scale2 = pair(p.scale_log2, p.scale_log2), minus_lse = pair(-lse2, -lse2), minus_delta = pair(-delta, -delta);
      for (int j = 0; j < nblk; ++j, ++n) {
        if (!(ok = warp_wait(s_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        f32x2 pr[32];
        {
          uint32_t t[2][32];
          tmem_ld_32x32(my_s, t[0]);
          tmem_ld_32x32(my_s + 32, t[1]);
          tmem_ld_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_read);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            pr[e] = exp2_pair(fma2(pair(__uint_as_float(t[e >> 4][(e & 15) * 2]), __uint_as_float(t[e >> 4][(e & 15) * 2 + 1])), scale2, minus_lse));
        }
        if (!(ok = warp_wait(dp_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        // dP was the only reader of this V tile; the last one's memory serves the epilogue first
        if (lane == 0 && j + 1 < nblk) mbar_arrive(&v_empty[n % kStagesV]);
        // the diagonal block (causal) and the one in which the document ends are masked, in the packed result: what a masked
        // score gave, Inf or NaN, is gone with it
        const int limit = j < nblk - 1 ? 64 : (p.causal ? min(tile.len, q_idx + 1) : tile.len) - j * 128 - sub * 64;
        const bool masked = j == nblk - 1;
        by_chunks(my_dp, [&](int c, const uint32_t(&x)[16]) {
          uint32_t pk[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 d = both(mul2(pr[c * 8 + e], add2(pair(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), minus_delta)));
            pk[e] = pack_bf16(d.x, d.y);
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[e] &= keep_below(limit - 2 * (c * 8 + e));
          }
          tmem_st_32x8(my_dp + c * 8, pk);
        });
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
      }
      if (!ok) break;
      const int first = q0 + quarter * 32;
      const int sv = (n - 1) % kStagesV;
      Turn<D> turn(p, first, tile.len - first, sub, lane);
      if (kTurn) turn.fetch(0);
      if (!(ok = warp_wait(acc_full, it & 1, abort_flag))) break;
      tc_fence_after_sync();
      uint8_t* stage = (D == 128 ? sV + sv * TILE_BYTES : sStage) + (warp - 4) * kStageBytes;
      __nv_bfloat16* dst = p.out_a + ((long long)tile.start + first) * p.out_stride + h * D;
      write_rows<D, kTurn>(tAcc + lane_off, sub, p.scale, turn, tile.len - first, stage, lane, dst, p.out_stride);
      tc_fence_before_sync();
      fence_proxy_async_smem();  // the tile's next content comes by TMA
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_empty[sv]);
      ++it;
    }
  }
  if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  // its memory and that of the launch before are apart; what follows may need both
  if (threadIdx.x == 0) after_previous();
  leave(abort_flag, warp, tmem_base);
}

// ------------------------------------------------------------------------------------------------ pass 2: dK, dV
constexpr int kStagesQ = 3, kStagesDO = 2, kStagesStat = 2;  // a Q tile is read by S and, three products later, by dK
constexpr int kDkvThreads = 384;

// Warps: 0 loads (TMA), 1 issues MMAs and owns TMEM, 2 brings lse and delta of a block's queries, 3 clears what reaches beyond
// a document, 4..11 softmax (two per TMEM lane quarter, 64 of a block's columns each).
template <int D, bool kTurn>
__global__ void __launch_bounds__(kDkvThreads, 1)
packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                  const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, BwdArgs p) {
  constexpr int NCH = D / 64;
  constexpr int TILE_BYTES = NCH * kChunkBytes;

  // addresses of shared memory are constants, as long as nothing is computed from where it begins
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {  // the launch reserves no slack for re-alignment
    if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE_BYTES;
  uint8_t* sQ = sV + TILE_BYTES;
  uint8_t* sDO = sQ + kStagesQ * TILE_BYTES;
  float* s_stat = reinterpret_cast<float*>(sDO + kStagesDO * TILE_BYTES);  // [stage][-lse2, -delta][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_stat + kStagesStat * 256);
  uint64_t* k_full = bars;
  uint64_t* k_empty = bars + 1;
  uint64_t* v_full = bars + 2;
  uint64_t* v_empty = bars + 3;
  uint64_t* q_full = bars + 4;
  uint64_t* q_empty = q_full + kStagesQ;
  uint64_t* q_raw = q_empty + kStagesQ;
  uint64_t* do_full = q_raw + kStagesQ;
  uint64_t* do_empty = do_full + kStagesDO;
  uint64_t* do_raw = do_empty + kStagesDO;
  uint64_t* stat_full = do_raw + kStagesDO;
  uint64_t* stat_empty = stat_full + kStagesStat;
  uint64_t* s_full = stat_empty + kStagesStat;
  uint64_t* p_ready = s_full + 1;
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_ready = s_full + 3;
  uint64_t* acc_full = s_full + 4;
  uint8_t* sStage = reinterpret_cast<uint8_t*>(bars) + 320 + ItemRing::kBytes;  // D = 64 only
  ItemRing ring(reinterpret_cast<uint8_t*>(bars) + 320, s_full + 5);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_full + 5 + ItemRing::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  after_previous();
  let_next_start();
  const int count = p.counts[1];  // longer documents only: see attention_packed_short.cu
  const int G = p.Hq / p.Hkv / p.split;  // query heads of an item
  // an item: rows [k0, k0 + 128) of a document as keys, blocks [first, tiles) of queries of G heads.  The table lists tiles by
  // the keys that queries see; the first keys are seen by the most queries.
  struct Item {
    int start, len, hkv, part, kv_tile, first, tiles, blocks;
  };
  Items items(count * p.Hkv * p.split, p.counter);
  bool ok = true;
  Item w;
  auto decode = [&](int i) {
    const TileOrder order = tile_order(i, count, p.Hkv * p.split, p.head_group);
    const Tile tile = p.tiles[order.tile_rank];
    w.start = tile.start, w.len = tile.len, w.hkv = order.index / p.split;
    w.part = order.index - w.hkv * p.split;
    w.tiles = (tile.len + 127) / 128;
    w.kv_tile = w.tiles - 1 - tile.rank;
    w.first = p.causal ? w.kv_tile : 0;
    w.blocks = G * (w.tiles - w.first);
  };
  auto publish_next = [&]() {  // by the loading warp; false after the last
    const int i = items.next(lane);
    w.start = -1;
    if (i >= 0) decode(i);
    ok = ring.put(make_int4(w.start, w.len, w.hkv, w.kv_tile), make_int4(w.first, w.tiles, w.blocks, w.part), make_int4(0, 0, 0, 0), lane, abort_flag);
    return ok && w.start >= 0;
  };
  auto next_item = [&]() {  // by the others
    int4 a, b, c;
    if (!(ok = ring.get(a, b, c, lane, abort_flag))) return false;
    w.start = a.x, w.len = a.y, w.hkv = a.z, w.kv_tile = a.w;
    w.first = b.x, w.tiles = b.y, w.blocks = b.z, w.part = b.w;
    return w.start >= 0;
  };

  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    mbar_init(v_full, 1);
    mbar_init(v_empty, 8);
    for (int i = 0; i < kStagesQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&q_raw[i], 1);
    }
    for (int i = 0; i < kStagesDO; ++i) {
      mbar_init(&do_full[i], 1);
      mbar_init(&do_empty[i], 1);
      mbar_init(&do_raw[i], 1);
    }
    for (int i = 0; i < kStagesStat; ++i) {
      mbar_init(&stat_full[i], 1);
      mbar_init(&stat_empty[i], 8);
    }
    mbar_init(s_full, 1);
    mbar_init(p_ready, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, 8);
    mbar_init(acc_full, 1);
    ring.init(11);  // MMA, lse and delta, clearing, softmax
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

  int it = 0;  // items so far
  int n = 0;   // blocks so far
  // launched with 168 registers a thread: 72 + 2 x 216 = 3 x 168
  if (warp < 4) {
    give_registers<72>();
    if (warp == 0) {
      while (ok && publish_next()) {
        // rows beyond the document stay in their own accumulator rows, which are not written
        if (!(ok = warp_wait(k_empty, (it & 1) ^ 1, abort_flag))) break;
        if (lane == 0) load_tile<NCH>(sK, &tmK, k_full, w.hkv * D, w.start + w.kv_tile * 128);
        int head = (w.hkv * p.split + w.part) * G, blk = w.first;
        for (int b = 0; b < w.blocks; ++b, ++n) {
          const int sq = n % kStagesQ, sd = n % kStagesDO;
          const bool tail = w.len - blk * 128 < 128;
          if (!(ok = warp_wait(&q_empty[sq], ((n / kStagesQ) & 1) ^ 1, abort_flag))) break;
          if (lane == 0) load_tile<NCH>(sQ + sq * TILE_BYTES, &tmQ, tail ? &q_raw[sq] : &q_full[sq], head * D, w.start + blk * 128);
          if (b == 0) {
            if (!(ok = warp_wait(v_empty, (it & 1) ^ 1, abort_flag))) break;
            if (lane == 0) load_tile<NCH>(sV, &tmV, v_full, w.hkv * D, w.start + w.kv_tile * 128);
          }
          if (!(ok = warp_wait(&do_empty[sd], ((n / kStagesDO) & 1) ^ 1, abort_flag))) break;
          if (lane == 0) load_tile<NCH>(sDO + sd * TILE_BYTES, &tmDO, tail ? &do_raw[sd] : &do_full[sd], head * D, w.start + blk * 128);
          if (++blk == w.tiles) blk = w.first, ++head;
        }
        ++it;
      }
    } else if (warp == 1) {
      const uint32_t idesc_t = make_idesc_bf16(128, 128, 0, 0);
      const uint32_t idesc_acc = make_idesc_bf16(128, D, 0, 1);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool got = warp_wait(bar, parity, abort_flag);
        tc_fence_after_sync();
        return got;
      };
      auto issue_scores = [&](uint32_t dst, const uint8_t* tile_a, const uint8_t* tile_b, uint64_t* full, uint64_t* last) {
        const uint64_t ad = make_smem_desc(smem_u32(tile_a), 16, 1024);
        const uint64_t bd = make_smem_desc(smem_u32(tile_b), 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4;
            umma_ss<1>(dst, ad + off, bd + off, idesc_t, kk != 0);
          }
          umma_commit(full);
          if (last) umma_commit(last);
        }
        __syncwarp();
      };
      // accumulation: A = P^T or dS^T (bf16 in TMEM: 16 queries in 8 columns), B = streamed tile, MN-major
      auto issue_acc = [&](uint32_t dst, uint32_t a, const uint8_t* tile_b, int b, uint64_t* empty, uint64_t* last) {
        const uint64_t bd = make_smem_desc(smem_u32(tile_b), kChunkBytes, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ts(dst, a + (kk >> 2) * 64 + (kk & 3) * 8, bd + ((kk * 2048) >> 4), idesc_acc, (b | kk) != 0);
          umma_commit(empty);
          if (last) umma_commit(last);
        }
        __syncwarp();
      };
      while (ok && next_item()) {
        const int blocks = w.blocks;
        if (!(ok = wait(k_full, it & 1) && wait(&q_full[n % kStagesQ], (n / kStagesQ) & 1))) break;
        issue_scores(tS, sK, sQ + (n % kStagesQ) * TILE_BYTES, s_full, blocks == 1 ? k_empty : nullptr);
        if (!(ok = wait(v_full, it & 1) && wait(&do_full[n % kStagesDO], (n / kStagesDO) & 1))) break;
        issue_scores(tDP, sV, sDO + (n % kStagesDO) * TILE_BYTES, dp_full, nullptr);
        for (int b = 0; b < blocks; ++b, ++n) {
          const bool more = b + 1 < blocks;
          const int m = n + 1;
          // what the next scores need is waited for while there is nothing to issue anyway
          if (more && !(ok = wait(&q_full[m % kStagesQ], (m / kStagesQ) & 1))) break;
          if (!(ok = wait(p_ready, n & 1))) break;
          issue_acc(tDV, tS, sDO + (n % kStagesDO) * TILE_BYTES, b, &do_empty[n % kStagesDO], nullptr);
          if (more) {
            issue_scores(tS, sK, sQ + (m % kStagesQ) * TILE_BYTES, s_full, b + 2 == blocks ? k_empty : nullptr);
            if (!(ok = wait(&do_full[m % kStagesDO], (m / kStagesDO) & 1))) break;
          }
          if (!(ok = wait(ds_ready, n & 1))) break;
          issue_acc(tDK, tDP, sQ + (n % kStagesQ) * TILE_BYTES, b, &q_empty[n % kStagesQ], more ? nullptr : acc_full);
          if (more) issue_scores(tDP, sV, sDO + (m % kStagesDO) * TILE_BYTES, dp_full, nullptr);
        }
        ++it;
    }
  } else if (warp == 2) {
    // lse and delta of a block's queries, negative as the softmax adds them; fetched one block ahead of their buffer.  A query
    // beyond the document gets lse = inf, so P = 2^-inf = 0: no mask at a document's end.
    float next[8];
    auto fetch = [&](const Item& w, int head, int blk) {
      const int row = w.start + blk * 128;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int x = u * 32 + lane;
        const bool in = blk * 128 + x < w.len;
        next[u] = in ? -kLog2e * p.lse[(long long)head * p.T + row + x] : -CUDART_INF_F;
        next[4 + u] = in ? -p.delta[(long long)head * p.T + row + x] : 0.f;
      }
    };
    while (ok && next_item()) {
      int head = (w.hkv * p.split + w.part) * G, blk = w.first;
      fetch(w, head, blk);
      for (int b = 0; b < w.blocks; ++b, ++n) {
        const int st = n % kStagesStat;
        if (!(ok = warp_wait(&stat_empty[st], ((n / kStagesStat) & 1) ^ 1, abort_flag))) break;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          s_stat[st * 256 + u * 32 + lane] = next[u];
          s_stat[st * 256 + 128 + u * 32 + lane] = next[4 + u];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&stat_full[st]);
        if (++blk == w.tiles) blk = w.first, ++head;
        if (b + 1 < w.blocks) fetch(w, head, blk);
      }
    }
  } else {
    uint32_t q_phases = 0, do_phases = 0;  // of the raw barriers
    while (ok && next_item()) {
      const int per_head = w.tiles - w.first, valid = w.len - (w.tiles - 1) * 128;
      if (valid >= 128) {
        n += w.blocks;
        continue;
      }
      for (int g = 0; g < G; ++g) {  // the last block of each head
        n += per_head;
        const int sq = (n - 1) % kStagesQ, sd = (n - 1) % kStagesDO;
        if (!(ok = warp_wait(&q_raw[sq], (q_phases >> sq) & 1, abort_flag))) break;
        q_phases ^= 1u << sq;
        clear_tail<NCH>(sQ + sq * TILE_BYTES, valid, &q_full[sq], lane);
        if (!(ok = warp_wait(&do_raw[sd], (do_phases >> sd) & 1, abort_flag))) break;
        do_phases ^= 1u << sd;
        clear_tail<NCH>(sDO + sd * TILE_BYTES, valid, &do_full[sd], lane);
      }
    }
    }
  } else {
    take_registers<216>();
    const int sub = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // key row of this thread
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t my_s = tS + lane_off + sub * 64, my_dp = tDP + lane_off + sub * 64;
    const f32x2 scale2 = pair(p.scale_log2, p.scale_log2);
    while (ok && next_item()) {
      const int k0 = w.kv_tile * 128;
      int blk = w.first;
      for (int b = 0; b < w.blocks; ++b, ++n) {
        const int st = n % kStagesStat;
        const f32x2* minus_lse = reinterpret_cast<const f32x2*>(s_stat + st * 256 + sub * 64);
        const f32x2* minus_delta = minus_lse + 64;
        if (!(ok = warp_wait(&stat_full[st], (n / kStagesStat) & 1, abort_flag))) break;
        // what shared memory gives is asked for ahead of the scores: while the products read their operands there at its full
        // rate, a load takes its time
        f32x2 pr[32];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const ulonglong2 l = *reinterpret_cast<const ulonglong2*>(minus_lse + e);
          pr[e] = l.x, pr[e + 1] = l.y;
        }
        if (!(ok = warp_wait(s_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        by_chunks(my_s, [&](int c, const uint32_t(&x)[16]) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            pr[c * 8 + e] = exp2_pair(fma2(pair(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), scale2, pr[c * 8 + e]));
        });
        // queries before this key are masked, in the packed results
        const bool masked = p.causal && blk == w.kv_tile;
        const int first = r - sub * 64;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 v = both(pr[c * 16 + e]);
            pk[e] = pack_bf16(v.x, v.y);
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[e] &= ~keep_below(first - 2 * (c * 16 + e));
          }
          tmem_st_32x16(my_s + c * 16, pk);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        f32x2 dl[32];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const ulonglong2 d = *reinterpret_cast<const ulonglong2*>(minus_delta + e);
          dl[e] = d.x, dl[e + 1] = d.y;
        }
        if (!(ok = warp_wait(dp_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        by_chunks(my_dp, [&](int c, const uint32_t(&x)[16]) {
          uint32_t pk[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 v = both(mul2(pr[c * 8 + e], add2(pair(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), dl[c * 8 + e])));
            pk[e] = pack_bf16(v.x, v.y);
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[e] &= ~keep_below(first - 2 * (c * 8 + e));
          }
          tmem_st_32x8(my_dp + c * 8, pk);
        });
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(ds_ready);
          mbar_arrive(&stat_empty[st]);
        }
        if (++blk == w.tiles) blk = w.first;
      }
      if (!ok) break;
      const int first = k0 + quarter * 32;
      Turn<D> turn(p, first, w.len - first, sub, lane);
      if (kTurn && p.split == 1) turn.fetch(0);
      if (!(ok = warp_wait(acc_full, it & 1, abort_flag))) break;
      tc_fence_after_sync();
      const long long at = ((long long)w.start + first) * p.out_stride + w.hkv * D;
      uint8_t* stage = (D == 128 ? sV : sStage) + (warp - 4) * kStageBytes;  // V has been read; its next tile is loaded after this
      if (p.split > 1) {
        const long long pitch = (long long)p.Hkv * D, size = p.T * pitch;
        float* dk = p.partial + w.part * 2 * size + ((long long)w.start + first) * pitch + w.hkv * D;
        write_partial<D>(tDK + lane_off, sub, w.len - first, stage, lane, dk, pitch);
        write_partial<D>(tDV + lane_off, sub, w.len - first, stage, lane, dk + size, pitch);
      } else {
        write_rows<D, kTurn>(tDK + lane_off, sub, p.scale, turn, w.len - first, stage, lane, p.out_a + at, p.out_stride);
        write_rows<D, false>(tDV + lane_off, sub, 1.f, turn, w.len - first, stage, lane, p.out_b + at, p.out_stride);
      }
      tc_fence_before_sync();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(v_empty);
      ++it;
    }
  }
  if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  leave(abort_flag, warp, tmem_base);
}

// Adds the parts of dK and dV up, in their order; scale and rotation as in write_rows, zeros in padding.  Bound by bandwidth.  A
// thread has 4 columns of both halves of a row.
template <int D>
__global__ void __launch_bounds__(256) packed_dkv_sum_kernel(BwdArgs p, const int* __restrict__ positions) {
  constexpr int kPer = D / 8;
  const int width = p.Hkv * D, per_row = p.Hkv * kPer;
  const long long size = p.T * width;
  after_previous();
  for (long long t = blockIdx.x * (long long)blockDim.y + threadIdx.y; t < p.T; t += (long long)gridDim.x * blockDim.y) {
    const int pos = positions[t];
    for (int i = threadIdx.x; i < per_row; i += blockDim.x) {
      const int h = i / kPer, c = (i - h * kPer) * 4, col = h * D + c;
      float4 sum[4];  // dK low, dK high, dV low, dV high
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (pos >= 0) {
        for (int part = 0; part < p.split; ++part)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 x = *reinterpret_cast<const float4*>(p.partial + (part * 2 + k / 2) * size + t * width + col + (k & 1) * (D / 2));
            sum[k].x += x.x, sum[k].y += x.y, sum[k].z += x.z, sum[k].w += x.w;
          }
#pragma unroll
        for (int k = 0; k < 2; ++k) sum[k].x *= p.scale, sum[k].y *= p.scale, sum[k].z *= p.scale, sum[k].w *= p.scale;
        if (p.cs && pos < p.table_rows) {
          const float4 cc = __ldg(reinterpret_cast<const float4*>(p.cs + (long long)pos * (D / 2) + c));
          const float4 ss = __ldg(reinterpret_cast<const float4*>(p.sn + (long long)pos * (D / 2) + c));
          const float4 f = sum[0], g = sum[1];
          sum[0] = make_float4(f.x * cc.x + g.x * ss.x, f.y * cc.y + g.y * ss.y, f.z * cc.z + g.z * ss.z, f.w * cc.w + g.w * ss.w);
          sum[1] = make_float4(g.x * cc.x - f.x * ss.x, g.y * cc.y - f.y * ss.y, g.z * cc.z - f.z * ss.z, g.w * cc.w - f.w * ss.w);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        __nv_bfloat16* dst = (k < 2 ? p.out_a : p.out_b) + t * p.out_stride + col + (k & 1) * (D / 2);
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(sum[k].x, sum[k].y), pack_bf16(sum[k].z, sum[k].w));
      }
    }
  }
}

// Items that share the query heads of a key head in pass 2.  An item there is G query heads of a tile of keys, so with few
// key heads there are few items, and the longest alone can take longer than the average SM: one row of 16 384
// tokens with 8 query heads on 2 key heads took 660 us unsplit, 333 blocks of 128 x 128 in the longest item against 214 on
// the average SM, and 435 + 17 to add the parts split in two.  The parts cost 16 bytes per split, token and column of K, so the split stops
// at three items for each of 148 SMs.
static int split_for(int max_tiles, int Hq, int Hkv) {
  const int G = Hq / Hkv;
  for (int s = 1; s < G; ++s)
    if (G % s == 0 && (long long)max_tiles * Hkv * s >= 3 * 148) return s;
  return G;
}

template <int D, bool kTurn>
static int launch_bwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo,
                      BwdArgs p, __nv_bfloat16* dq, __nv_bfloat16* dk, __nv_bfloat16* dv, const int* positions, cudaStream_t stream) {
  constexpr int TILE = (D / 64) * kChunkBytes;
  constexpr int STAGE = D == 128 ? 0 : 8 * kStageBytes;  // a V tile of D = 128 has room for it
  constexpr int SMEM1 = (2 + kStagesK + kStagesV) * TILE + 2560 + 256 + ItemRing::kBytes + STAGE;
  constexpr int SMEM2 = (2 + kStagesQ + kStagesDO) * TILE + kStagesStat * 1024 + 320 + ItemRing::kBytes + STAGE;
  static_assert(SMEM1 <= 232448 && SMEM2 <= 232448, "one block's shared memory");
  constexpr auto pass1 = packed_dq_kernel<D, kTurn>;
  constexpr auto pass2 = packed_dkv_kernel<D, kTurn>;
  if (cudaError_t e = pb::allow_smem<pass1, SMEM1>(); e != cudaSuccess) return (int)e;
  if (cudaError_t e = pb::allow_smem<pass2, SMEM2>(); e != cudaSuccess) return (int)e;
  // The short documents first: their launch needs nothing from the others, and so the blocks of pass 1 take the places that its
  // last blocks leave.
  if (int rc = launch_short_bwd<D, kTurn>(tq, tdo, tk, tv, p, dq, dk, dv, stream)) return rc;
  p.out_a = dq;
  p.head_group = attention_head_group(p.max_tiles, p.Hq);
  pb_count_launch(2);
  if (cudaError_t e = launch_chained(pass1, resident_blocks((long long)p.max_tiles * p.Hq), kDqThreads, SMEM1, stream, tq, tdo, tk, tv, p);
      e != cudaSuccess)
    return (int)e;
  p.out_a = dk;
  p.out_b = dv;
  p.head_group = attention_head_group(p.max_tiles, p.Hkv * p.split);
  if (cudaError_t e = launch_chained(pass2, resident_blocks((long long)p.max_tiles * p.Hkv * p.split), kDkvThreads, SMEM2, stream, tq, tdo,
                                     tk, tv, p);
      e != cudaSuccess)
    return (int)e;
  if (p.split > 1) {
    const int x = p.Hkv * D / 8 < 256 ? (p.Hkv * D / 8 + 31) / 32 * 32 : 256, y = 256 / x;
    const long long blocks = (p.T + y - 1) / y;
    pb_count_launch(1);
    return (int)launch_chained(packed_dkv_sum_kernel<D>, (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), dim3(x, y), 0, stream, p,
                               positions);
  }
  return 0;
}

}  // namespace pbv

extern "C" {

// Layouts as in pb_packed_attention_fwd; q and k rotated as the forward saw them.  dq/dk/dv: bf16 rows of dqkv_stride, every
// row written (zeros in padding).  cs/sn [table_rows, D / 2] (null: none): dq and dk are turned back by the row's position.
// scratch: pb_packed_attention_bwd_scratch bytes, 16-byte aligned, of this call alone.  tiles / counts: the layout's table of
// 128-row tiles; positions: the layout's.
long long pb_packed_attention_bwd_scratch(long long T, int Hq, int Hkv, int D, int max_tiles) {
  const int split = pbv::split_for(max_tiles, Hq, Hkv);
  return 16 + (T * Hq * 4 + 15) / 16 * 16 + (split > 1 ? split * 2 * T * Hkv * D * 4 : 0);
}

int pb_packed_attention_bwd(const void* dO, const void* q, const void* k, const void* v, const void* o,
                            const float* lse, void* scratch, void* dq, void* dk, void* dv, const float* cs,
                            const float* sn, int table_rows, const int* tiles, const int* counts, int max_tiles,
                            const int* positions, long long T, int Hq, int Hkv, int D, long long q_stride, long long k_stride,
                            long long v_stride, long long o_stride, long long do_stride, long long dqkv_stride,
                            float softmax_scale, int causal, int* err_dev, void* stream_) {
  using namespace pbv;
  if (D != 64 && D != 128) return -1;
  if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0) return -2;
  if ((q_stride % 8) || (k_stride % 8) || (v_stride % 8) || (o_stride % 8) || (do_stride % 8) || (dqkv_stride % 8)) return -3;
  uintptr_t all = 0;
  for (const void* x : {o, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)cs, (const void*)sn, (const void*)scratch})
    all |= reinterpret_cast<uintptr_t>(x);
  if (all & 15) return -3;
  if (T < 1 || T > 0x3fffffffLL || max_tiles < 1 || (long long)max_tiles * Hq > 0x7fff0000LL) return -4;  // room for Items' last turn
  CUtensorMap tq, tk, tv, tdo;
  int r = 0;
  r |= pb::make_tmap_bf16_2d(&tq, q, (uint64_t)Hq * D, T, (uint64_t)q_stride, 64, 128);
  r |= pb::make_tmap_bf16_2d(&tk, k, (uint64_t)Hkv * D, T, (uint64_t)k_stride, 64, 128);
  r |= pb::make_tmap_bf16_2d(&tv, v, (uint64_t)Hkv * D, T, (uint64_t)v_stride, 64, 128);
  r |= pb::make_tmap_bf16_2d(&tdo, dO, (uint64_t)Hq * D, T, (uint64_t)do_stride, 64, 128);
  if (r) return -10;
  BwdArgs p;
  memset(&p, 0, sizeof(p));
  p.o = reinterpret_cast<const __nv_bfloat16*>(o);
  p.o_stride = o_stride;
  p.lse = lse;
  p.delta = reinterpret_cast<float*>(scratch) + 4;
  p.split = split_for(max_tiles, Hq, Hkv);
  // pass 1 has tiles of about one length in every turn: its items in turns were within 3% of evenly spread in every case here
  p.counter = takes_from_counter((long long)max_tiles * Hkv * p.split) ? reinterpret_cast<int*>(scratch) : nullptr;
  p.partial = reinterpret_cast<float*>(reinterpret_cast<char*>(scratch) + 16 + (T * Hq * 4 + 15) / 16 * 16);
  p.out_stride = dqkv_stride;
  p.cs = cs, p.sn = sn;
  p.table_rows = table_rows;
  p.T = T;
  p.tiles = reinterpret_cast<const Tile*>(tiles);
  p.counts = counts;
  p.max_tiles = max_tiles;
  p.Hq = Hq, p.Hkv = Hkv;
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * kLog2e;
  p.causal = causal;
  p.err = err_dev;
  auto b = [](void* x) { return reinterpret_cast<__nv_bfloat16*>(x); };
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const auto launch = D == 128 ? (cs ? launch_bwd<128, true> : launch_bwd<128, false>) : (cs ? launch_bwd<64, true> : launch_bwd<64, false>);
  return launch(tq, tk, tv, tdo, p, b(dq), b(dk), b(dv), positions, stream);
}

}  // extern "C"

// Attention over packed documents, backward, for documents of 128 tokens or fewer (sm_100a).
//
// Such a document is one tile, so nothing has to be added up across tiles and one pass gives dQ, dK and dV: five products
// instead of seven, one set of exponentials, and each operand is read once (see attention_packed_bwd.cu for the formulas and
// for longer documents).  An item is a document and a key head; K and V stay in shared memory while its query heads
// pass:
//     S = Q K^T, dP = dO V^T                 fp32 in TMEM, a query row per lane
//     P, dS -> shared memory                 bf16 [query][key], which serves as three operands
//     dV += P^T dO, dK += dS^T Q             P and dS read key-major
//     dQ = dS K                              dS read query-major; over dP's columns in TMEM
// The chain of one head is serial; what overlaps it are the next head's loads and its S, and the O rows for its delta.  The
// products run over the document's tokens, rounded up to 16, and not over the tile.
// Roundings as in the longer documents' kernels.
// Warps: 0 loads (TMA), 1 issues MMAs and owns TMEM, 2 clears what reaches beyond the document, 4..11 softmax and
// epilogue (two per TMEM lane quarter, 64 keys each), 12..15 form delta.
#include "attention_packed_bwd.cuh"

namespace pbv {

constexpr int kShortThreads = 512;

template <int D, bool kTurn>
__global__ void __launch_bounds__(kShortThreads, 1)
packed_short_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
                        const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, BwdArgs p,
                        __nv_bfloat16* dq, __nv_bfloat16* dk, __nv_bfloat16* dv) {
  constexpr int NCH = D / 64;
  constexpr int TILE_BYTES = NCH * kChunkBytes;
  constexpr int PAIR_BYTES = 2 * kChunkBytes;  // [128 queries][128 keys]

  // addresses of shared memory are constants, as long as nothing is computed from where it begins
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023) {  // the launch reserves no slack for re-alignment
    if (threadIdx.x == 0) atomicExch(p.err, ERR_BAD_ARG);
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE_BYTES;
  uint8_t* sQ = sV + TILE_BYTES;  // 2 stages
  uint8_t* sDO = sQ + 2 * TILE_BYTES;
  uint8_t* sP = sDO + TILE_BYTES;  // and, when its product is done, the epilogue's memory
  uint8_t* sDS = sP + PAIR_BYTES;
  float* s_stat = reinterpret_cast<float*>(sDS + PAIR_BYTES);  // [step & 1][lse2, delta][128]
  float* s_delta = s_stat + 512;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_delta + 128);
  uint64_t* k_full = bars;
  uint64_t* k_raw = bars + 1;
  uint64_t* v_full = bars + 2;
  uint64_t* kv_empty = bars + 3;
  uint64_t* q_full = bars + 4;   // [2]
  uint64_t* q_raw = bars + 6;    // [2]
  uint64_t* q_empty = bars + 8;  // [2]
  uint64_t* do_full = bars + 10;
  uint64_t* do_raw = bars + 11;
  uint64_t* do_empty = bars + 12;
  uint64_t* stat_full = bars + 13;   // [2]
  uint64_t* stat_empty = bars + 15;  // [2]
  uint64_t* s_full = bars + 17;
  uint64_t* p_ready = bars + 18;
  uint64_t* dp_full = bars + 19;
  uint64_t* ds_ready = bars + 20;
  uint64_t* done = bars + 21;      // all products of a step
  uint64_t* epi_done = bars + 22;  // its results have left TMEM and sP
  ItemRing ring(reinterpret_cast<uint8_t*>(bars) + 320, bars + 23);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23 + ItemRing::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = p.Hq / p.Hkv / p.split;  // query heads of an item
  const int first_entry = p.counts[1], n_all = p.counts[0] - first_entry;
  const int heads = p.Hkv * p.split;

  // an item: a document (or a tile of padding), a key head, and `part` of its query heads
  Items items(n_all * heads);
  bool ok = true;
  int start = 0, len = 0, rank = 0, hkv = 0, part = 0, pad = 0;
  auto publish_next = [&]() {  // by the loading warp; false after the last
    const int i = items.next();
    start = -1;
    if (i >= 0) {
      const int entry = i / heads, index = i - entry * heads;
      const Tile tile = p.tiles[first_entry + entry];
      start = tile.start, len = tile.len, rank = tile.rank, pad = tile.pad;
      hkv = index / p.split, part = index - hkv * p.split;
    }
    ok = ring.put(make_int4(start, len, rank, pad), make_int4(hkv, part, 0, 0), make_int4(0, 0, 0, 0), lane, abort_flag);
    return ok && start >= 0;
  };
  auto next_item = [&]() {  // by the others
    int4 a, b, c;
    if (!(ok = ring.get(a, b, c, lane, abort_flag))) return false;
    start = a.x, len = a.y, rank = a.z, pad = a.w, hkv = b.x, part = b.y;
    return start >= 0;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 23; ++i) {
      int arrivals = 1;
      if (&bars[i] == do_empty) arrivals = 5;                                                    // products, delta
      if (&bars[i] == stat_full || &bars[i] == stat_full + 1) arrivals = 4;                      // delta's warps
      if (&bars[i] == stat_empty || &bars[i] == stat_empty + 1 || &bars[i] == p_ready || &bars[i] == ds_ready ||
          &bars[i] == epi_done)
        arrivals = 8;  // softmax
      mbar_init(&bars[i], arrivals);
    }
    ring.init(14);  // MMA, clearing, softmax, delta
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<1>(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tS = tmem_base;         // 128 columns
  const uint32_t tDP = tmem_base + 128;  // 128 columns; dQ over them
  const uint32_t tDV = tmem_base + 256;  // D columns
  const uint32_t tDK = tmem_base + 384;  // D columns

  int it = 0;  // documents so far
  int n = 0;   // steps (a query head of a document) so far
  // launched with 128 registers a thread: 64 + 2 x 168 + 112 = 4 x 128
  if (warp < 4) {
    give_registers<64>();
    if (warp == 0) {
      while (ok && publish_next()) {
        if (pad) continue;
        const bool tail = len & 15;
        if (!(ok = warp_wait(kv_empty, (it & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          load_tile<NCH>(sK, &tmK, tail ? k_raw : k_full, hkv * D, start);
          load_tile<NCH>(sV, &tmV, v_full, hkv * D, start);
        }
        for (int g = 0; g < G; ++g, ++n) {
          const int s = n & 1, col = ((hkv * p.split + part) * G + g) * D;
          if (!(ok = warp_wait(&q_empty[s], ((n >> 1) & 1) ^ 1, abort_flag))) break;
          if (lane == 0) load_tile<NCH>(sQ + s * TILE_BYTES, &tmQ, tail ? &q_raw[s] : &q_full[s], col, start);
          if (!(ok = warp_wait(do_empty, (n & 1) ^ 1, abort_flag))) break;
          if (lane == 0) load_tile<NCH>(sDO, &tmDO, tail ? do_raw : do_full, col, start);
        }
        ++it;
      }
    } else if (warp == 1) {
      const uint32_t idesc_dkv = make_idesc_bf16(128, D, 1, 1), idesc_dq = make_idesc_bf16(128, D, 0, 1);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool got = warp_wait(bar, parity, abort_flag);
        tc_fence_after_sync();
        return got;
      };
      auto issue_scores = [&](uint32_t dst, const uint8_t* tile_a, const uint8_t* tile_b, uint32_t idesc, uint64_t* full) {
        const uint64_t ad = make_smem_desc(smem_u32(tile_a), 16, 1024);
        const uint64_t bd = make_smem_desc(smem_u32(tile_b), 16, 1024);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = ((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4;
            umma_ss<1>(dst, ad + off, bd + off, idesc, kk != 0);
          }
          umma_commit(full);
        }
        __syncwarp();
      };
      while (ok && next_item()) {
        if (pad) continue;
        const int n16 = (len + 15) & ~15, steps = n16 >> 4;
        const uint32_t idesc_s = make_idesc_bf16(128, n16, 0, 0);
        if (!(ok = wait(k_full, it & 1) && wait(v_full, it & 1))) break;
        for (int g = 0; g < G; ++g, ++n) {
          const uint8_t* q = sQ + (n & 1) * TILE_BYTES;
          if (!(ok = wait(&q_full[n & 1], (n >> 1) & 1))) break;
          issue_scores(tS, q, sK, idesc_s, s_full);
          if (!(ok = wait(do_full, n & 1) && (n == 0 || wait(epi_done, (n - 1) & 1)))) break;
          issue_scores(tDP, sDO, sV, idesc_s, dp_full);
          // sixteen queries a step; P, dS, dO and Q are rows of 128 bytes per query
          const uint64_t pd = make_smem_desc(smem_u32(sP), kChunkBytes, 1024), dsd = make_smem_desc(smem_u32(sDS), kChunkBytes, 1024);
          const uint64_t dod = make_smem_desc(smem_u32(sDO), kChunkBytes, 1024), qd = make_smem_desc(smem_u32(q), kChunkBytes, 1024);
          if (!(ok = wait(p_ready, n & 1))) break;
          if (elect_one())
            for (int kk = 0; kk < steps; ++kk) umma_ss<1>(tDV, pd + kk * 128, dod + kk * 128, idesc_dkv, (g | kk) != 0);
          __syncwarp();
          if (!(ok = wait(ds_ready, n & 1))) break;
          // sixteen keys a step of dQ; dS read query-major
          const uint64_t dsq = make_smem_desc(smem_u32(sDS), 16, 1024), kd = make_smem_desc(smem_u32(sK), kChunkBytes, 1024);
          if (elect_one()) {
            for (int kk = 0; kk < steps; ++kk) umma_ss<1>(tDK, dsd + kk * 128, qd + kk * 128, idesc_dkv, (g | kk) != 0);
            for (int kk = 0; kk < steps; ++kk)
              umma_ss<1>(tDP, dsq + (((kk >> 2) * kChunkBytes + (kk & 3) * 32) >> 4), kd + kk * 128, idesc_dq, kk != 0);
            umma_commit(&q_empty[n & 1]);
            umma_commit(do_empty);
            if (g + 1 == G) umma_commit(kv_empty);
            umma_commit(done);
          }
          __syncwarp();
        }
        ++it;
      }
    } else if (warp == 2) {
      // rows from the document's end to the next multiple of 16 take part in the products: zeros there (load_tile's comment)
      uint32_t phases = 0;  // of k_raw, q_raw[0], q_raw[1], do_raw
      auto clear = [&](uint8_t* tile, uint64_t* raw, int bit, uint64_t* full) {
        if (!warp_wait(raw, (phases >> bit) & 1, abort_flag)) return false;
        phases ^= 1u << bit;
        const int bytes = (((len + 15) & ~15) - len) * 128;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
          for (int at = lane * 16; at < bytes; at += 512)
            *reinterpret_cast<uint4*>(tile + c * kChunkBytes + len * 128 + at) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
        return true;
      };
      while (ok && next_item()) {
        if (pad) continue;
        if ((len & 15) == 0) {
          n += G;
          continue;
        }
        if (!(ok = clear(sK, k_raw, 0, k_full))) break;
        for (int g = 0; ok && g < G; ++g, ++n)
          ok = clear(sQ + (n & 1) * TILE_BYTES, &q_raw[n & 1], 1 + (n & 1), &q_full[n & 1]) && clear(sDO, do_raw, 3, do_full);
      }
    }
  } else if (warp >= 12) {
    give_registers<112>();
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // lanes to a row of O
    const int u = lane % kLanes, first = quarter * 32 + lane / kLanes;
    while (ok && next_item()) {
      if (pad) continue;
      for (int g = 0; g < G; ++g, ++n) {
        const int h = (hkv * p.split + part) * G + g;
        uint4 y[kLanes];
#pragma unroll
        for (int k = 0; k < kLanes; ++k)
          y[k] = first + k * kRows < len ? __ldg(reinterpret_cast<const uint4*>(p.o + ((long long)start + first + k * kRows) * p.o_stride + h * D) + u)
                                         : make_uint4(0, 0, 0, 0);
        const float lse2 = r < len ? p.lse[(long long)h * p.T + start + r] * kLog2e : 0.f;
        if (!(ok = warp_wait(do_full, n & 1, abort_flag) && warp_wait(&stat_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag))) break;
        row_dots<D>(sDO, y, first, u, s_delta);
        __syncwarp();
        s_stat[(n & 1) * 256 + r] = lse2;
        s_stat[(n & 1) * 256 + 128 + r] = r < len ? s_delta[r] : 0.f;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&stat_full[n & 1]);
          mbar_arrive(do_empty);
        }
      }
    }
  } else {
    take_registers<168>();
    const int sub = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // query row of this thread, and its key row in the epilogue of dK and dV
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t my_s = tS + lane_off + sub * 64, my_dp = tDP + lane_off + sub * 64;
    const f32x2 scale2 = pair(p.scale_log2, p.scale_log2);
    uint8_t* stage = sP + (warp - 4) * kStageBytes;
    while (ok && next_item()) {
      const int head0 = (hkv * p.split + part) * G;
      if (pad) {
        const int first = rank * 128, rows = min(128, len - first);
        for (int g = 0; g < G; ++g)
          clear_rows<D>(dq, p.out_stride, (long long)start + first, rows, (head0 + g) * D, threadIdx.x - 128, 256);
        if (p.split == 1) {  // whoever adds the parts up clears theirs
          clear_rows<D>(dk, p.out_stride, (long long)start + first, rows, hkv * D, threadIdx.x - 128, 256);
          clear_rows<D>(dv, p.out_stride, (long long)start + first, rows, hkv * D, threadIdx.x - 128, 256);
        }
        continue;
      }
      const int n16 = (len + 15) & ~15;
      const bool active = quarter * 32 < n16 && sub * 64 < n16;  // this warp has scores that a product reads
      const int limit = r < len ? (p.causal ? min(len, r + 1) : len) - sub * 64 : 0;
      const int first = quarter * 32, rows = len - first;
      const long long row = (long long)start + first;
      for (int g = 0; g < G; ++g, ++n) {
        if (!(ok = warp_wait(&stat_full[n & 1], (n >> 1) & 1, abort_flag))) break;
        const float lse2 = s_stat[(n & 1) * 256 + r], delta = s_stat[(n & 1) * 256 + 128 + r];
        __syncwarp();
        if (lane == 0) mbar_arrive(&stat_empty[n & 1]);
        const f32x2 minus_lse = pair(-lse2, -lse2), minus_delta = pair(-delta, -delta);
        if (!(ok = warp_wait(s_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        f32x2 pr[32];
        if (active) {
          uint32_t t[2][32];
          tmem_ld_32x32(my_s, t[0]);
          tmem_ld_32x32(my_s + 32, t[1]);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            pr[e] = exp2_pair(fma2(pair(__uint_as_float(t[e >> 4][(e & 15) * 2]), __uint_as_float(t[e >> 4][(e & 15) * 2 + 1])), scale2, minus_lse),
                              (e & 7) < kPolyPairs);
        }
        // the memory of P served the last step's epilogue, of other warps too
        if (n > 0 && !(ok = warp_wait(epi_done, (n - 1) & 1, abort_flag))) break;
        // 16-byte piece u of a query's 64 keys lies at u ^ (query & 7), as TMA would have put it
        auto put = [&](uint8_t* tile, const uint32_t* pk, int piece) {
          *reinterpret_cast<uint4*>(tile + sub * kChunkBytes + r * 128 + ((piece ^ (r & 7)) << 4)) =
              make_uint4(pk[0], pk[1], pk[2], pk[3]);
        };
        if (active) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t pk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = both(pr[c * 4 + e]);
              pk[e] = pack_bf16(v.x, v.y) & keep_below(limit - 2 * (c * 4 + e));
            }
            put(sP, pk, c);
          }
        }
        tc_fence_before_sync();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        if (!(ok = warp_wait(dp_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        if (active)
          by_chunks(my_dp, [&](int c, const uint32_t(&x)[16]) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t pk[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int v = half * 4 + e;
                const float2 d = both(mul2(pr[c * 8 + v], add2(pair(__uint_as_float(x[2 * v]), __uint_as_float(x[2 * v + 1])), minus_delta)));
                pk[e] = pack_bf16(d.x, d.y) & keep_below(limit - 2 * (c * 8 + v));
              }
              put(sDS, pk, c * 2 + half);
            }
          });
        tc_fence_before_sync();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
        // dQ, and after the last head dK and dV: one copy of the code for the three
        const int outputs = g + 1 < G ? 1 : (p.split > 1 ? 1 : 3);
#pragma unroll 1
        for (int which = 0; which < outputs; ++which) {
          Turn<D> turn(p, first, which < 2 ? rows : 0, sub, lane);  // dV is not turned
          if (kTurn) turn.fetch(0);
          if (which == 0) {
            if (!(ok = warp_wait(done, n & 1, abort_flag))) break;
            tc_fence_after_sync();
          }
          __nv_bfloat16* base = which == 0 ? dq : (which == 1 ? dk : dv);
          if (rows > 0)
            write_rows<D, kTurn>((which == 0 ? tDP : (which == 1 ? tDK : tDV)) + lane_off, sub, which < 2 ? p.scale : 1.f, turn, rows,
                                 stage, lane, base + row * p.out_stride + (which == 0 ? head0 + g : hkv) * D, p.out_stride);
        }
        if (!ok) break;
        if (g + 1 == G && p.split > 1 && rows > 0) {
          const long long pitch = (long long)p.Hkv * D, size = p.T * pitch;
          float* at = p.partial + part * 2 * size + row * pitch + hkv * D;
          write_partial<D>(tDK + lane_off, sub, rows, stage, lane, at, pitch);
          write_partial<D>(tDV + lane_off, sub, rows, stage, lane, at + size, pitch);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(epi_done);
      }
    }
  }
  if (!ok && lane == 0) atomicExch(p.err, ERR_WAIT_TIMEOUT);
  leave(abort_flag, warp, tmem_base);
}

template <int D, bool kTurn>
int launch_short_bwd(const CUtensorMap& tq, const CUtensorMap& tdo, const CUtensorMap& tk, const CUtensorMap& tv, BwdArgs p,
                     __nv_bfloat16* dq, __nv_bfloat16* dk, __nv_bfloat16* dv, cudaStream_t stream) {
  constexpr int SMEM = 5 * (D / 64) * kChunkBytes + 4 * kChunkBytes + 2560 + 320 + ItemRing::kBytes;
  static_assert(SMEM <= 232448, "one block's shared memory");
  constexpr auto kern = packed_short_bwd_kernel<D, kTurn>;
  if (cudaError_t e = pb::allow_smem<kern, SMEM>(); e != cudaSuccess) return (int)e;
  kern<<<resident_blocks((long long)p.max_tiles * p.Hkv * p.split), kShortThreads, SMEM, stream>>>(tq, tdo, tk, tv, p, dq, dk, dv);
  pb_count_launch(1);
  return (int)cudaGetLastError();
}
#define PB_SHORT(D, TURN)                                                                                               \
  template int launch_short_bwd<D, TURN>(const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, \
                                         BwdArgs, __nv_bfloat16*, __nv_bfloat16*, __nv_bfloat16*, cudaStream_t)
PB_SHORT(64, false);
PB_SHORT(64, true);
PB_SHORT(128, false);
PB_SHORT(128, true);
#undef PB_SHORT

}  // namespace pbv

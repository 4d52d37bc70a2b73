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
// The chain of one head is serial; what overlaps it are the next head's loads and its S.  The
// products run over the document's tokens, rounded up to 16, and not over the tile.
// Measured: 190 documents of 59 tokens on average, 32 query and 8 key heads of 128: 208 us, 5.3 us per head of a document and
// SM.  Bound by that chain: five products of 500 cycles or fewer, two exchanges through shared memory, and the epilogue.
// Roundings as in the longer documents' kernels.
// Warps: 0 loads (TMA), 1 issues MMAs and owns TMEM, 2 clears what reaches beyond the document, 4..11 softmax, delta and
// epilogue (two per TMEM lane quarter, 64 keys each).
#include "attention_packed_bwd.cuh"

namespace pbv {

constexpr int kShortThreads = 384;

__device__ __forceinline__ int up16(int n) { return (n + 15) & ~15; }

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
  float* s_delta = reinterpret_cast<float*>(sDS + PAIR_BYTES);  // [step & 1][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_delta + 256);
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
  uint64_t* delta_ready = bars + 13;
  uint64_t* s_full = bars + 14;
  uint64_t* p_ready = bars + 15;
  uint64_t* dp_full = bars + 16;
  uint64_t* ds_ready = bars + 17;
  uint64_t* done = bars + 18;      // all products of a step
  uint64_t* epi_done = bars + 19;  // its results have left TMEM and sP
  constexpr int kBars = 20;
  ItemRing ring(reinterpret_cast<uint8_t*>(bars) + 320, bars + kBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars + ItemRing::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int G = p.Hq / p.Hkv / p.split;  // query heads of an item
  let_next_start();
  const int first_entry = p.counts[1], n_all = p.counts[0] - first_entry;
  const int heads = p.Hkv * p.split;

  // an item: a document (or a tile of padding), a key head, and `part` of its query heads
  Items items(n_all * heads, nullptr);
  bool ok = true;
  int start = 0, len = 0, rank = 0, hkv = 0, part = 0, pad = 0;
  auto publish_next = [&]() {  // by the loading warp; false after the last
    const int i = items.next(lane);
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
    for (int i = 0; i < kBars; ++i) {
      const uint64_t* bar = &bars[i];
      mbar_init(&bars[i], bar == delta_ready || bar == p_ready || bar == ds_ready || bar == epi_done ? 8 : 1);  // 8: softmax
    }
    ring.init(10);  // MMA, clearing, softmax
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
  // launched with 168 registers a thread: 72 + 2 x 216 = 3 x 168
  if (warp < 4) {
    give_registers<72>();
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
        const int n16 = up16(len), steps = n16 >> 4;
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
        const int bytes = (up16(len) - len) * 128;
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
  } else {
    take_registers<216>();
    const int sub = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // query row of this thread, and its key row in the epilogue of dK and dV
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t my_s = tS + lane_off + sub * 64, my_dp = tDP + lane_off + sub * 64;
    const f32x2 scale2 = pair(p.scale_log2, p.scale_log2);
    uint8_t* stage = sP + (warp - 4) * kStageBytes;
    // the tables of row r: every document begins at row 0 of its tile
    f32x2 cs[D / 8], sn[D / 8];
    if (kTurn) {
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        float4 c = make_float4(1.f, 1.f, 1.f, 1.f), t = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < p.table_rows) {
          c = __ldg(reinterpret_cast<const float4*>(p.cs + r * (D / 2) + sub * (D / 4)) + u);
          t = __ldg(reinterpret_cast<const float4*>(p.sn + r * (D / 2) + sub * (D / 4)) + u);
        }
        cs[u * 2] = pair(c.x, c.y), cs[u * 2 + 1] = pair(c.z, c.w);
        sn[u * 2] = pair(t.x, t.y), sn[u * 2 + 1] = pair(t.z, t.w);
      }
    }
    // delta of 16 rows is this warp's: D / 8 lanes to a row
    constexpr int kLanes = D / 8, kRows = 32 / kLanes, kCount = 16 / kRows;
    const int piece_u = lane % kLanes, dot_first = (warp - 4) * 16 + lane / kLanes;
    // O and lse of a step are fetched under the epilogue of the step before, whose item may be another
    uint4 y[kCount];
    float lse2 = 0.f;
    auto fetch = [&](int h) {
#pragma unroll
      for (int k = 0; k < kCount; ++k)
        y[k] = dot_first + k * kRows < len
                   ? __ldg(reinterpret_cast<const uint4*>(p.o + ((long long)start + dot_first + k * kRows) * p.o_stride + h * D) + piece_u)
                   : make_uint4(0, 0, 0, 0);
      lse2 = r < len ? p.lse[(long long)h * p.T + start + r] * kLog2e : 0.f;
    };
    auto next_document = [&]() {  // clears the padding that comes on the way
      while (next_item()) {
        const int head0 = (hkv * p.split + part) * G;
        if (!pad) {
          fetch(head0);
          return true;
        }
        const int first = rank * 128, rows = min(128, len - first);
        for (int g = 0; g < G; ++g)
          clear_rows<D>(dq, p.out_stride, (long long)start + first, rows, (head0 + g) * D, threadIdx.x - 128, 256);
        if (p.split == 1) {  // whoever adds the parts up clears theirs
          clear_rows<D>(dk, p.out_stride, (long long)start + first, rows, hkv * D, threadIdx.x - 128, 256);
          clear_rows<D>(dv, p.out_stride, (long long)start + first, rows, hkv * D, threadIdx.x - 128, 256);
        }
      }
      return false;
    };
    bool more = next_document();
    while (ok && more) {
      const int head0 = (hkv * p.split + part) * G, hkv0 = hkv, part0 = part;
      const int n16 = up16(len);
      // which of its scores a product reads, and which of these are not masked
      const bool active = quarter * 32 < n16 && sub * 64 < n16;
      const bool zeros = p.causal && sub * 64 > quarter * 32 + 31;
      const bool row_ok = r < len;
      const int limit = row_ok ? (p.causal ? min(len, r + 1) : len) - sub * 64 : 0;
      const bool masked = __any_sync(0xffffffffu, limit < 64);
      const int first = quarter * 32, rows = len - first;
      const long long row = (long long)start + first;
      for (int g = 0; g < G; ++g, ++n) {
        const int h = head0 + g;
        const f32x2 minus_lse = pair(-lse2, -lse2);
        if (!(ok = warp_wait(s_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        // the memory of P served the last step's epilogue, of other warps too
        if (n > 0 && !(ok = warp_wait(epi_done, (n - 1) & 1, abort_flag))) break;
        // 16-byte piece u of a query's 64 keys lies at u ^ (query & 7), as TMA would have put it
        auto put = [&](uint8_t* tile, const uint32_t* pk, int piece) {
          *reinterpret_cast<uint4*>(tile + sub * kChunkBytes + r * 128 + ((piece ^ (r & 7)) << 4)) =
              make_uint4(pk[0], pk[1], pk[2], pk[3]);
        };
        auto probability = [&](const uint32_t(&x)[16], int e) {
          return exp2_pair(fma2(pair(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), scale2, minus_lse));
        };
        auto put_chunk = [&](uint8_t* tile, uint32_t(&pk)[8], int c) {
          if (masked) {
#pragma unroll
            for (int e = 0; e < 8; ++e) pk[e] &= keep_below(limit - 2 * (c * 8 + e));
          }
          put(tile, pk, c * 2);
          put(tile, pk + 4, c * 2 + 1);
        };
        if (active && zeros) {
          const uint32_t none[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            put(sP, none, c);
            put(sDS, none, c);
          }
        } else if (active) {
          by_chunks(my_s, [&](int c, const uint32_t(&x)[16]) {
            uint32_t pk[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 v = both(probability(x, e));
              pk[e] = pack_bf16(v.x, v.y);
            }
            put_chunk(sP, pk, c);
          });
        }
        tc_fence_before_sync();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        // delta, while dP is formed
        if (!(ok = warp_wait(do_full, n & 1, abort_flag))) break;
        row_dots<D, kCount>(sDO, y, dot_first, piece_u, s_delta + (n & 1) * 128);
        __syncwarp();
        if (lane == 0) mbar_arrive(delta_ready);
        if (!(ok = warp_wait(delta_ready, n & 1, abort_flag) && warp_wait(dp_full, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        if (active && !zeros) {
          const float delta = row_ok ? s_delta[(n & 1) * 128 + r] : 0.f;
          const f32x2 minus_delta = pair(-delta, -delta);
          // P once more, from S, which is still there: kept, it would take the registers of the tables
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t x[16], d[16], pk[8];
            tmem_ld_32x16(my_s + c * 16, x);
            tmem_ld_32x16(my_dp + c * 16, d);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 v = both(mul2(probability(x, e), add2(pair(__uint_as_float(d[2 * e]), __uint_as_float(d[2 * e + 1])), minus_delta)));
              pk[e] = pack_bf16(v.x, v.y);
            }
            put_chunk(sDS, pk, c);
          }
        }
        tc_fence_before_sync();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
        if (g + 1 < G) fetch(h + 1);
        else more = next_document();
        if (!ok) break;
        if (!(ok = warp_wait(done, n & 1, abort_flag))) break;
        tc_fence_after_sync();
        if (rows > 0) {
          // dQ, and after the last head dK and dV: one copy of the code for the three
          const int outputs = g + 1 < G || p.split > 1 ? 1 : 3;
#pragma unroll 1
          for (int which = 0; which < outputs; ++which) {
            __nv_bfloat16* base = which == 0 ? dq : (which == 1 ? dk : dv);
            write_rows_held<D, kTurn>((which == 0 ? tDP : (which == 1 ? tDK : tDV)) + lane_off, sub, which < 2 ? p.scale : 1.f, cs, sn,
                                      which < 2, rows, stage, lane, base + row * p.out_stride + (which == 0 ? h : hkv0) * D, p.out_stride);
          }
          if (g + 1 == G && p.split > 1) {
            const long long pitch = (long long)p.Hkv * D, size = p.T * pitch;
            float* at = p.partial + part0 * 2 * size + row * pitch + hkv0 * D;
            write_partial<D>(tDK + lane_off, sub, rows, stage, lane, at, pitch);
            write_partial<D>(tDV + lane_off, sub, rows, stage, lane, at + size, pitch);
          }
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
  constexpr int SMEM = 5 * (D / 64) * kChunkBytes + 4 * kChunkBytes + 1024 + 320 + ItemRing::kBytes;
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

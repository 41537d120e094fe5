// Attention over the paged cache for chunks of many query rows per kv head (prompts): bound by
// the tensor core and the exponentials.
//
// A persistent CTA per SM walks the items of its share: two tiles of 128 query rows (row = token
// * G + g, so the heads of a group share every key they read) against a run of key blocks.
//   warps 0-3, 4-7   softmax of tile 0 and of tile 1, a query row per thread
//   warps 8-11       output: O out of TMEM, normalised, written
//   warp 12          TMA: queries, and K and V blocks through a ring of 32 KB stages
//   warps 13, 14     issue tcgen05.mma, one warp per tile
//   warp 15          V blocks that not all rows see all of: rows that no row sees (whose pages hold
//                    whatever they do) are cleared, values that are not finite are taken out of those
//                    that only some see (weight 0 times either must be 0)
// A key block is worked on in two halves of 64 keys, each with its own S [128 x 64] in TMEM (its
// weights P, in bf16, take the place of its first 32 columns).  While the softmax is on one half,
// the tensor core adds P V of the other and writes the other's next S = Q K^T, so that the softmax
// warps, which set the pace, find their next scores ready.  S of both tiles' halves and both O
// fill the 512 columns of TMEM.
//
// The softmax's reference need not be the running maximum: any value that no weight outgrows by
// more than 2^8, and that is no larger than the true maximum, gives the same quotient O / l with
// the same relative rounding, and takes no more than 8 of the 128 powers of two that O has for
// the values.  So a row takes the maximum of the first half block that it sees a
// key of, and later halves only check their largest score against it; where a row outgrows it, the
// reference moves and O is rescaled.
//
// Measured (32 / 8 heads of 128, 4096 tokens over 16384 cached keys, 0.96 TFLOP): 885 us, 1.09
// PFLOP/s, 66% of a cuBLAS burst and 80% of what cuBLAS sustains under the same 1000 W cap (this
// kernel runs there at 1.59 of 1.965 GHz).  Without the softmax's work the same loads and products
// take 639 us.  A whole block at a time, with the running maximum of every block, took 1316 us; a
// separate issuing warp per tile, elected so that the compiler knows it is one thread, was worth a
// quarter of that (a commit holds its thread until the tensor core has run what came before it).
// Windowed ragged chunks (40 / 8 heads, window 1000, 5600 tokens): 214 us.
// The waits that keep parities unmistakable are in the issuing warps, whose products hide them: in
// the softmax warps one more wait a half cost the first case 932 to 949 us.
#include "paged_tc.cuh"

namespace sf {

constexpr int kChunkThreads = 512;
constexpr int kOddItems = 16;          // more than the items between the V warp and the output

// Of every 8 pairs of weights, this many take the polynomial instead of the special-function unit
// (none 921 us, one 888, two 891, three 921 for the case above: an exponential costs the FMA pipe
// nearly what it costs the other unit).
constexpr int kPolyPairs = 1;

// the larger of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// the largest of 64, NaN if one is
__device__ __forceinline__ float max64(const float* v) {
  float m[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    m[c] = max3(v[c * 16], v[c * 16 + 1], v[c * 16 + 2]);
#pragma unroll
    for (int j = 3; j < 15; j += 2) m[c] = max3(m[c], v[c * 16 + j], v[c * 16 + j + 1]);
  }
  return max3(max3(m[0], m[1], v[15]), max3(m[2], m[3], v[31]), max3(v[47], v[63], v[63]));
}
// How far a row may outgrow its reference (see the head of the file).  (2^60 made O overflow for
// values above 2^67 and was no faster.)
constexpr float kGrowthLog2 = 8.f;

// 2^x of a pair on the FMA and integer pipes: x = i + r with |r| <= 1/2, 2^r by the polynomial of
// degree 4 with p(0) = 1 that is minimax in relative error on that interval (2.8e-6, found by
// linear programming), i added to the exponent.  x <= -127 gives 0.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  const uint64_t t = pair(fmaxf(a, -127.f), fmaxf(b, -127.f));
  const uint64_t magic = pair(12582912.f, 12582912.f);   // 1.5 * 2^23: the sum's low bits are i
  const uint64_t z = add2(t, magic);
  const uint64_t i = add2(z, pair(-12582912.f, -12582912.f));
  const uint64_t r = fma2(i, pair(-1.f, -1.f), t);
  uint64_t y = pair(0.009582576341927052f, 0.009582576341927052f);
  y = fma2(y, r, pair(0.05590682849287987f, 0.05590682849287987f));
  y = fma2(y, r, pair(0.24024106562137604f, 0.24024106562137604f));
  y = fma2(y, r, pair(0.6931241154670715f, 0.6931241154670715f));
  y = fma2(y, r, pair(1.f, 1.f));
  float za, zb, ya, yb;
  unpair(z, za, zb);
  unpair(y, ya, yb);
  return pair(__int_as_float(__float_as_int(ya) + (__float_as_int(za) << 23)),
              __int_as_float(__float_as_int(yb) + (__float_as_int(zb) << 23)));
}

template <int HD>
struct ChunkSmem {
  static constexpr int kTile = HD / 64 * kPagedBox;      // 128 rows
  static constexpr int kStages = HD == 128 ? 5 : 8;
  static constexpr int q = 0;                            // [2][kTile]
  static constexpr int ring = q + 2 * kTile;             // [kStages][kTile]
  static constexpr int ml = ring + kStages * kTile;      // [2 tiles][m (log2 units), l][128]
  static constexpr int bars = ml + 2 * 2 * 128 * 4;
  static constexpr int bytes = bars + (3 * kStages + 26) * 8 + kOddItems * 4 + 8;
};

template <int HD>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_attention_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                 const __grid_constant__ CUtensorMap tmV, PagedAttnParams p) {
  typedef ChunkSmem<HD> L;
  constexpr int KCH = HD / 64, NS = L::kStages;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::bars);
  // [x % kOddItems] x, where the V of the CTA's x-th item (with blocks) lost values
  volatile uint32_t* odd_items = reinterpret_cast<volatile uint32_t*>(bars + 3 * NS + 26);
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 3 * NS + 26 + kOddItems / 2);
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(&tmem_slot + 1);
  if (smem_u32(sm) & 1023) {                             // the swizzled tiles need it; all threads see it
    flag_error(p.err, SF_DEV_ERR_TMEM);
    return;
  }
  uint64_t* full = bars;                                 // [NS]
  uint64_t* empty = bars + NS;                           // [NS]
  uint64_t* fit = bars + 2 * NS;                         // [NS] looked at by the V warp
  uint64_t* q_full = bars + 3 * NS;                      // [2] and so on: one per tile
  uint64_t* q_empty = q_full + 2;
  uint64_t* o_done = q_full + 4;
  uint64_t* o_free = q_full + 6;
  uint64_t* ml_full = q_full + 8;
  uint64_t* ml_free = q_full + 10;
  uint64_t* drain = q_full + 12;
  uint64_t* s_full = q_full + 14;                        // [2 tiles][2 halves]
  uint64_t* p_full = q_full + 18;
  uint64_t* pv_done = q_full + 22;

  pdl_trigger();                                         // the join of cut tiles may line up
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2);                           // both tiles
      mbar_init(&fit[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&s_full[2 * t + h], 1);
        mbar_init(&p_full[2 * t + h], 4);
        mbar_init(&pv_done[2 * t + h], 1);
      }
      mbar_init(&o_done[t], 1);
      mbar_init(&drain[t], 1);
      mbar_init(&o_free[t], 4);
      mbar_init(&ml_full[t], 4);
      mbar_init(&ml_free[t], 4);
    }
    for (int x = 0; x < kOddItems; ++x) odd_items[x] = ~0u;
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 13) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  float* ml = reinterpret_cast<float*>(sm + L::ml);      // [2 tiles][2][128]

  const int first = p.first[blockIdx.x], last = p.first[blockIdx.x + 1];
  const int tq = p.tile_tokens;                          // tokens of one tile
  if (warp >= 12) {
    if (warp == 12) {
      // -------------------------------------------------------------- TMA
      uint32_t u = 0;                                    // ring units issued (K and V blocks)
      uint32_t qn[2] = {0, 0};                           // query tiles issued
      bool ok = true;
      for (int it = first; ok && it < last; ++it) {
        const PagedItem w = p.items[it];
        if (w.i0 == w.i1) continue;
        const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
        const PagedRange range = mask.range(w.tok0, w.tok0 + w.ntok);
        const int tiles = w.ntok > tq ? 2 : 1;
        auto load_q = [&](int t) {
          ok = __all_sync(0xffffffffu, wait_or_abort(&q_empty[t], (qn[t] & 1) ^ 1, p.err, &abort_flag));
          if (!ok) return;
          if (lane == 0) mbar_arrive_expect_tx(&q_full[t], KCH * tq * p.G * 128);
          __syncwarp();
          if (lane < KCH)
            tma_load_3d(sm + L::q + t * L::kTile + lane * kPagedBox, &tmQ, &q_full[t], lane * 64, w.kvh * p.G,
                        w.q0 + w.tok0 + t * tq);
          ++qn[t];
        };
        KeyPages pages(p.pool, w, range, w.block(w.i0), KCH, lane, p.err);
        for (int i = w.i0; ok && i < w.i1; ++i) {
          const KeyPages now = pages;
          if (i + 1 < w.i1) pages = KeyPages(p.pool, w, range, w.block(i + 1), KCH, lane, p.err);
          for (int kv = 0; ok && kv < 2; ++kv, ++u) {
            // the first block's order: tile 0's queries, K, tile 1's queries, V
            if (i == w.i0 && kv < tiles) load_q(kv);
            if (!ok) break;
            const int s = u % NS;
            ok = __all_sync(0xffffffffu, wait_or_abort(&empty[s], ((u / NS) & 1) ^ 1, p.err, &abort_flag));
            if (!ok) break;
            load_key_block(sm + L::ring + s * L::kTile, kv ? &tmV : &tmK, &full[s], now, w.kvh, lane);
          }
        }
      }
      if (!ok && lane == 0) {                            // no load may be in flight at exit
        abort_flag = 1;
        for (uint32_t x = u > NS ? u - NS : 0; x < u; ++x) mbar_wait(&full[x % NS], (x / NS) & 1, p.err);
        for (int t = 0; t < 2; ++t)
          if (qn[t] > 0) mbar_wait(&q_full[t], (qn[t] - 1) & 1, p.err);
      }
    } else if (warp <= 14 && elect_one()) {
      // -------------------------------------------------------------- MMA
      // One warp per tile: a commit holds its thread until the tensor core has run what was
      // issued before it, and the other tile's products must be in the queue by then.
      const int t = warp - 13;
      const uint32_t id_s = idesc_bf16(128, kPagedKB / 2);
      const uint32_t id_pv = idesc_bf16(128, HD, 0, 1);
      const uint32_t ring_lo = smem_u32(sm + L::ring) >> 4;
      const uint32_t q_lo = ((smem_u32(sm + L::q) + t * L::kTile) >> 4) | (1u << 16);
      const uint32_t tS = tmem + t * 128, tO = tmem + 256 + t * 128;
      // parities of this tile's next block (bit 0), item (bit 1) and query tile (bit 2)
      uint32_t par = 0;
      // ring stage and parity of the stream's next K block; of the V block whose P V is due, with
      // whether it begins and ends its item
      uint32_t stage = 0, phase = 0;
      uint32_t due_stage = NS, due_phase = 0;            // NS: none is due
      bool due_begin = false, due_end = false, ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_or_abort(bar, parity & 1, p.err, &abort_flag); };
      auto advance = [&]() {
        phase ^= stage + 1 == NS;
        stage = stage + 1 == NS ? 0 : stage + 1;
      };
      // O += P V of half h of the block that is due
      auto issue_pv = [&](int h) -> bool {
        if (h == 0) {
          if (due_begin) {
            if (!wait(&o_free[t], (par >> 1) ^ 1)) return false;
            par ^= 2;
          }
          if (!wait(&full[due_stage], due_phase) || !wait(&fit[due_stage], due_phase)) return false;
        }
        if (!wait(&p_full[2 * t + h], par)) return false;
        tc_fence_after();
        const uint32_t v_lo = (ring_lo + due_stage * (L::kTile >> 4) + h * 512) | ((kPagedBox >> 4) << 16);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_f16_ts(tO, tS + h * 64 + kk * 8, desc(v_lo + kk * 128), id_pv, (!due_begin || h > 0 || kk > 0) ? 1u : 0u);
        return true;
      };
      // Ahead of what half h commits: the last P V of the other half that was committed must be seen
      // to be done, so that a softmax warp that has this half's scores finds its barrier at most one
      // phase behind.  (That P V came before the products just issued, which hide the wait.)
      auto settle = [&](int h) -> bool {
        return wait(&pv_done[2 * t + (h ^ 1)], h == 1 && due_stage != NS ? par : par ^ 1);
      };
      // after an item's last block O is done; the stage of V is free
      auto commit_pv = [&](int h) {
        umma_commit(&pv_done[2 * t + h]);
        if (h == 0) return;
        umma_commit(&empty[due_stage]);
        if (due_end) umma_commit(&o_done[t]);
        par ^= 1;
      };
#pragma unroll 1
      for (int it = first; ok && it < last; ++it) {
        const int i0 = p.items[it].i0, i1 = p.items[it].i1;
        if (i0 == i1) continue;
        const bool active = t == 0 || p.items[it].ntok > tq;
        if (active) {
          ok = wait(&q_full[t], par >> 2);
          par ^= 4;
        }
#pragma unroll 1
        for (int left = i1 - i0; ok && left > 0; --left) {
          ok = wait(&full[stage], phase);
#pragma unroll 1
          for (int h = 0; ok && h < 2; ++h) {
            if (due_stage != NS) ok = issue_pv(h);
            if (!ok) break;
            if (active) {
              tc_fence_after();
              const uint32_t k_lo = (ring_lo + stage * (L::kTile >> 4) + h * 512) | (1u << 16);
#pragma unroll
              for (int kk = 0; kk < HD / 16; ++kk)
                umma_f16(tS + h * 64, desc(q_lo + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2),
                         desc(k_lo + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2), id_s, kk > 0 ? 1u : 0u);
            }
            ok = settle(h);
            if (!ok) break;
            if (active) {
              umma_commit(&s_full[2 * t + h]);
              if (h == 1) {
                umma_commit(&empty[stage]);
                if (left == 1) umma_commit(&q_empty[t]);
              }
            } else if (h == 1) {
              mbar_arrive(&empty[stage]);
            }
            if (due_stage != NS) commit_pv(h);
          }
          if (!ok) break;
          advance();
          if (active) {
            due_stage = stage;
            due_phase = phase;
            due_begin = left == i1 - i0;
            due_end = left == 1;
          } else {
            due_stage = NS;
            ok = wait(&full[stage], phase) && wait(&fit[stage], phase);
            mbar_arrive(&empty[stage]);
          }
          advance();
        }
      }
      for (int h = 0; ok && due_stage != NS && h < 2; ++h) {
        ok = issue_pv(h);
        if (ok) commit_pv(h);
      }
      if (!ok) abort_flag = 1;
      umma_commit(&drain[t]);
      mbar_wait(&drain[t], 0, p.err);
    } else if (warp == 15) {
      // -------------------------------------------------------------- V
      uint32_t u = 0;                                    // ring units (every one is waited for, so that
                                                         // no parity is mistaken)
      uint32_t nth = 0;                                  // items with blocks
      bool ok = true;
      for (int it = first; ok && it < last; ++it) {
        const PagedItem w = p.items[it];
        if (w.i0 == w.i1) continue;
        ++nth;
        const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
        const PagedRange range = mask.range(w.tok0, w.tok0 + w.ntok);
        const int hi_min = mask.hi(w.tok0), lo_max = mask.lo(w.tok0 + w.ntok - 1);
        for (int i = w.i0; ok && i < w.i1; ++i) {
          const int k0 = w.block(i) * kPagedKB;
          for (int kv = 0; kv < 2; ++kv, ++u) {
            const int s = u % NS;
            ok = __all_sync(0xffffffffu, wait_or_abort(&full[s], (u / NS) & 1, p.err, &abort_flag));
            if (!ok) break;
            if (kv == 1 && (k0 + kPagedKB > hi_min || (k0 < lo_max && k0 + kPagedKB > range.sinks))) {
              bool odd = false;
              // four rows at a time, 16 bytes a lane
#pragma unroll 2
              for (int r = lane / 8; r < kPagedKB; r += 4) {
                const int j = k0 + r;
                const bool seen = range.has(j);
                if (seen && j < hi_min && (j >= lo_max || j < range.sinks)) continue;
                uint4* at = reinterpret_cast<uint4*>(sm + L::ring + s * L::kTile + r * 128) + lane % 8;
#pragma unroll
                for (int c = 0; c < KCH; ++c) {
                  uint4 d = make_uint4(0, 0, 0, 0);
                  bool write = !seen;
                  if (seen) {
                    d = at[c * (kPagedBox / 16)];
                    write = drop_odd(d);
                    odd |= write;
                  }
                  if (write) at[c * (kPagedBox / 16)] = d;
                }
              }
              if (__any_sync(0xffffffffu, odd) && lane == 0) odd_items[nth % kOddItems] = nth;
              fence_async_shared();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&fit[s]);
          }
        }
      }
      if (!ok) abort_flag = 1;
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- output
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    uint32_t on[2] = {0, 0}, nth = 0;
    bool ok = true;
    for (int it = first; ok && it < last; ++it) {
      const PagedItem w = p.items[it];
      const bool any = w.i1 > w.i0;
      nth += any;
      for (int t = 0; ok && t < (w.ntok > tq ? 2 : 1); ++t) {
        const int rows = (min(w.ntok, (t + 1) * tq) - t * tq) * p.G;
        float m = -INFINITY, l = 0.f;
        if (any) {
          ok = __all_sync(0xffffffffu, wait_or_abort(&ml_full[t], on[t] & 1, p.err, &abort_flag) &&
                                           wait_or_abort(&o_done[t], on[t] & 1, p.err, &abort_flag));
          if (!ok) break;
          ++on[t];
          tc_fence_after();
          m = ml[t * 256 + r];
          l = ml[t * 256 + 128 + r];
          __syncwarp();
          if (lane == 0) mbar_arrive(&ml_free[t]);
        }
        const int64_t tok = w.q0 + w.tok0 + t * tq + r / p.G;
        const int64_t row = tok * p.H + w.kvh * p.G + r % p.G;
        const int64_t prow = static_cast<int64_t>(w.slot) * p.rows + t * 128 + r;
        const float f = w.slot >= 0 ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int c = 0; c < HD; c += 8) {
          float o[8];
          __syncwarp();
          if (any) {
            tmem_ld8(tmem + 256 + t * 128 + lane_off + c, o);
            tmem_wait<8>(o);
          }
          if (any && c + 8 == HD) {                      // O is read: the next item may begin
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[t]);
          }
          if (r < rows) {
            if (!any || f == 0.f) {
#pragma unroll
              for (int j = 0; j < 8; ++j) o[j] = 0.f;
            }
            if (w.slot >= 0) {
              float4* dst = reinterpret_cast<float4*>(p.part_O + prow * HD + c);
              dst[0] = make_float4(o[0], o[1], o[2], o[3]);
              dst[1] = make_float4(o[4], o[5], o[6], o[7]);
            } else {
              *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row * HD + c) =
                  make_uint4(pack_bf16(o[0] * f, o[1] * f), pack_bf16(o[2] * f, o[3] * f),
                             pack_bf16(o[4] * f, o[5] * f), pack_bf16(o[6] * f, o[7] * f));
            }
          }
        }
        if (r < rows) {
          if (w.slot >= 0) {
            p.part_ml[2 * prow] = m;
            p.part_ml[2 * prow + 1] = l;
          } else {
            p.lse[row] = m * 0.6931471805599453f + logf(l);
          }
        }
        if (any && odd_items[nth % kOddItems] == nth) {  // values that decide their columns
          const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
          __syncwarp();                                  // the rows are read back
          float sum[HD / 32];
          for (int x = 0, seen = -1; x < 32 && quarter * 32 + x < rows; ++x) {
            const int rx = quarter * 32 + x, tx = w.tok0 + t * tq + rx / p.G;
            if (tx != seen)
              paged_odd_values<__nv_bfloat16, HD>(p, w, tx, true, mask.hi(w.tok0), mask.lo(w.tok0 + w.ntok - 1), kPagedKB, lane, ~0u, sum);
            seen = tx;
            paged_put_odd<__nv_bfloat16, HD>(
                sum, true, static_cast<__nv_bfloat16*>(p.out) + (static_cast<int64_t>(w.q0 + tx) * p.H + w.kvh * p.G + rx % p.G) * HD,
                w.slot >= 0 ? p.part_O + (static_cast<int64_t>(w.slot) * p.rows + t * 128 + rx) * HD : nullptr, lane);
          }
        }
      }
    }
    if (!ok) abort_flag = 1;
  } else {
    // ---------------------------------------------------------------- softmax
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    const float sl2 = p.scale * 1.4426950408889634f;     // scores in log2 units
    uint32_t n = 0, items = 0;                           // this tile's blocks, items
    bool ok = true;
    for (int it = first; ok && it < last; ++it) {
      const PagedItem w = p.items[it];
      if (w.i0 == w.i1 || (t == 1 && w.ntok <= tq)) continue;
      const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
      const PagedRange range = mask.range(w.tok0, w.tok0 + w.ntok);
      const int t0 = w.tok0 + t * tq, t1 = min(w.tok0 + w.ntok, t0 + tq);
      const int tok = min(t0 + r / p.G, t1 - 1);
      const bool valid = r < (t1 - t0) * p.G;
      const int hi = mask.hi(tok), lo = mask.lo(tok);
      const int hi_min = mask.hi(t0), lo_max = mask.lo(t1 - 1);
      float m = -INFINITY, l = 0.f;
      for (int i = w.i0; i < w.i1; ++i, ++n) {
        const int k0 = w.block(i) * kPagedKB;
        const bool edge = k0 + kPagedKB > hi_min || (k0 < lo_max && k0 + kPagedKB > range.sinks);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          ok = __all_sync(0xffffffffu, ok && wait_or_abort(&s_full[2 * t + half], n & 1, p.err, &abort_flag));
          if (!ok) break;
          tc_fence_after();
          const uint32_t tH = tS + half * 64;
          float v[64];
          tmem_ld32(tH, v);
          tmem_ld32(tH + 32, v + 32);
          tmem_wait<64>(v);
          if (edge) {
            const int c0 = k0 + half * 64, h = hi - c0, b = lo - c0, f = range.sinks - c0;
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (!(j < h && (j >= b || j < f))) v[j] = -INFINITY;
          }
          const float mx = max64(v) * sl2;
          if (!__all_sync(0xffffffffu, !valid || mx <= m + kGrowthLog2)) {
            const bool grew = valid && !(mx <= m + kGrowthLog2);
            const float alpha = grew ? ex2(m - mx) : 1.f;
            if (grew) m = mx;
            l *= alpha;
            if (valid && !(mx < INFINITY)) l = NAN;      // an infinite or NaN score in the row
            if (i > w.i0 || half > 0) {
              // the P V of the half before, the last to add to O, must be done: phase n of the first
              // half's barrier, n - 1 of the second's.  The parity means no other: the phase before was
              // over when these scores were committed (settle), the one after needs this row's P.
              wait_or_abort(&pv_done[2 * t + (half ^ 1)], (n & 1) ^ half ^ 1, p.err, &abort_flag);
              __syncwarp();
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD; c += 16) {
                float o[16];
                tmem_ld16(tO + c, o);
                tmem_wait<16>(o);
                uint32_t e[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) e[j] = __float_as_uint(o[j] * alpha);
                tmem_st16(tO + c, e);
              }
            }
          }
          const float ref = m == -INFINITY ? 0.f : m;
          const uint64_t scale2 = pair(sl2, sl2), ref2 = pair(-ref, -ref);
          uint64_t sum = pair(l, 0.f);
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t e[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint64_t y = fma2(pair(v[c + 2 * j], v[c + 2 * j + 1]), scale2, ref2);
              float e0, e1;
              if ((j & 7) < kPolyPairs) {
                unpair(exp2_pair(y), e0, e1);
              } else {
                unpair(y, e0, e1);
                e0 = ex2(e0);
                e1 = ex2(e1);
              }
              sum = add2(sum, pair(e0, e1));
              e[j] = pack_bf16(e0, e1);
            }
            tmem_st16(tH + c / 2, e);
          }
          float l_even, l_odd;
          unpair(sum, l_even, l_odd);
          l = l_even + l_odd;
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[2 * t + half]);
        }
        if (!ok) break;
      }
      ok = __all_sync(0xffffffffu, ok && wait_or_abort(&ml_free[t], (items & 1) ^ 1, p.err, &abort_flag));
      if (!ok) break;
      ++items;
      ml[t * 256 + r] = m;
      ml[t * 256 + 128 + r] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ml_full[t]);
    }
    if (!ok) abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 13) tmem_dealloc(tmem, 512);
}

template <int HD>
static cudaError_t attention_chunk(const PagedAttnParams& p, cudaStream_t st) {
  CUtensorMap tq, tk, tv;
  if (!query_tmap(&tq, p.q, p.q_tok, p.q_head, p.T, p.H, HD, p.G, p.tile_tokens) ||
      !pool_tmap(&tk, p.pool.k, p.pool, p.Hkv, HD) || !pool_tmap(&tv, p.pool.v, p.pool, p.Hkv, HD))
    return cudaErrorInvalidValue;
  cudaError_t e = allow_smem(paged_attention_chunk_kernel<HD>, ChunkSmem<HD>::bytes);
  if (e != cudaSuccess) return e;
  paged_attention_chunk_kernel<HD><<<p.workers, kChunkThreads, ChunkSmem<HD>::bytes, st>>>(tq, tk, tv, p);
  return launched();
}

cudaError_t launch_paged_attention_chunk(const PagedAttnParams& p, cudaStream_t st) {
  if (p.workers == 0) return cudaSuccess;
  return p.hd == 128 ? attention_chunk<128>(p, st) : attention_chunk<64>(p, st);
}

}  // namespace sf

// Attention over the paged cache for chunks of many query rows per kv head (prompts): bound by
// the tensor core and the exponentials.
//
// A persistent CTA per SM walks the items of its share: two tiles of 128 query rows (row = token
// * G + g, so the heads of a group share every key they read) against a run of key blocks.
//   warps 0-3, 4-7   softmax of tile 0 and of tile 1, a query row per thread
//   warps 8-11       output: O out of TMEM, normalised, written
//   warp 12          TMA: queries, and K and V blocks through a ring of 32 KB stages
//   warp 13          issues tcgen05.mma
// While one tile's softmax runs, the tensor core works on the other tile: P V of the last block,
// then S = Q K^T of the next.  S [128 x 128] fp32 and P (bf16, over S's first 64 columns) of
// both tiles and both O fill the 512 columns of TMEM.  A tile's S of block j + 1 is issued after
// its P V of block j, and its commit covers both: a softmax thread that sees S may change O, so
// the (rare) rescaling needs no wait of its own.
//
// The rescaling waits until a row's maximum has grown by 2^8 (see paged_attention_tokens.cu).
#include "paged_tc.cuh"

namespace sf {

constexpr int kChunkThreads = 512;

template <int HD>
struct ChunkSmem {
  static constexpr int kTile = HD / 64 * kPagedBox;      // 128 rows
  static constexpr int kStages = HD == 128 ? 5 : 8;
  static constexpr int q = 0;                            // [2][kTile]
  static constexpr int ring = q + 2 * kTile;             // [kStages][kTile]
  static constexpr int ml = ring + kStages * kTile;      // [2 tiles][m (log2 units), l][128]
  static constexpr int bars = ml + 2 * 2 * 128 * 4;
  static constexpr int bytes = bars + (2 * kStages + 17) * 8 + 8;
};

template <int HD>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_attention_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                 const __grid_constant__ CUtensorMap tmV, PagedAttnParams p) {
  typedef ChunkSmem<HD> L;
  constexpr int KCH = HD / 64, NS = L::kStages;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint32_t& tmem_slot = *reinterpret_cast<uint32_t*>(bars + 2 * NS + 17);
  volatile int& abort_flag = *reinterpret_cast<volatile int*>(&tmem_slot + 1);
  if (smem_u32(sm) & 1023) {                             // the swizzled tiles need it; all threads see it
    flag_error(p.err, SF_DEV_ERR_TMEM);
    return;
  }
  uint64_t* full = bars;                                 // [NS]
  uint64_t* empty = bars + NS;                           // [NS]
  uint64_t* q_full = bars + 2 * NS;                      // [2] and so on: one per tile
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_full + 4;
  uint64_t* p_full = q_full + 6;
  uint64_t* o_done = q_full + 8;
  uint64_t* o_free = q_full + 10;
  uint64_t* ml_full = q_full + 12;
  uint64_t* ml_free = q_full + 14;
  uint64_t* drain = q_full + 16;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
      mbar_init(&o_free[t], 4);
      mbar_init(&ml_full[t], 4);
      mbar_init(&ml_free[t], 4);
    }
    mbar_init(drain, 1);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
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
          ok = __all_sync(0xffffffffu, !abort_flag && mbar_wait(&q_empty[t], (qn[t] & 1) ^ 1, p.err));
          if (!ok) return;
          if (lane == 0) mbar_arrive_expect_tx(&q_full[t], KCH * tq * p.G * 128);
          __syncwarp();
          if (lane < KCH)
            tma_load_3d(sm + L::q + t * L::kTile + lane * kPagedBox, &tmQ, &q_full[t], lane * 64, w.kvh * p.G,
                        w.q0 + w.tok0 + t * tq);
          ++qn[t];
        };
        for (int i = w.i0; ok && i < w.i1; ++i)
          for (int kv = 0; ok && kv < 2; ++kv, ++u) {
            // the first block's order: tile 0's queries, K, tile 1's queries, V
            if (i == w.i0 && kv < tiles) load_q(kv);
            if (!ok) break;
            const int s = u % NS;
            ok = __all_sync(0xffffffffu, !abort_flag && mbar_wait(&empty[s], ((u / NS) & 1) ^ 1, p.err));
            if (!ok) break;
            load_key_block<HD>(sm + L::ring + s * L::kTile, kv ? &tmV : &tmK, &full[s], p.pool, w, range, w.block(i),
                               lane, p.err);
          }
      }
      if (!ok && lane == 0) {                            // no load may be in flight at exit
        abort_flag = 1;
        for (uint32_t x = u > NS ? u - NS : 0; x < u; ++x) mbar_wait(&full[x % NS], (x / NS) & 1, p.err);
        for (int t = 0; t < 2; ++t)
          if (qn[t] > 0) mbar_wait(&q_full[t], (qn[t] - 1) & 1, p.err);
      }
    } else if (warp == 13 && lane == 0) {
      // -------------------------------------------------------------- MMA
      const uint32_t id_s = idesc_bf16(128, kPagedKB);
      const uint32_t id_pv = idesc_bf16(128, HD, 0, 1);
      uint32_t n = 0;                                    // block of the stream whose P V comes next
      uint32_t sn[2] = {0, 0}, on[2] = {0, 0};           // blocks, items of each tile
      uint32_t qn[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return !abort_flag && mbar_wait(bar, parity, p.err); };
      // S of tile t for block x of the stream (the i-th of an item's [i0, i1))
      auto issue_s = [&](int t, uint32_t x, bool begin, bool end) -> bool {
        const uint32_t u = 2 * x;
        if (begin && !wait(&q_full[t], qn[t]++ & 1)) return false;
        if (!wait(&full[u % NS], (u / NS) & 1)) return false;
        tc_fence_after();
        const uint32_t q_s = smem_u32(sm + L::q + t * L::kTile);
        const uint32_t k_s = smem_u32(sm + L::ring + (u % NS) * L::kTile);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          umma_f16(tmem + t * 128, sdesc_kmajor_sw128(q_s + (kk >> 2) * kPagedBox + (kk & 3) * 32),
                   sdesc_kmajor_sw128(k_s + (kk >> 2) * kPagedBox + (kk & 3) * 32), id_s, kk > 0 ? 1u : 0u);
        umma_commit(&s_full[t]);
        if (end) umma_commit(&q_empty[t]);
        return true;
      };
      int it = first;
      while (it < last && p.items[it].i0 == p.items[it].i1) ++it;
      if (it < last) {
        int i0 = p.items[it].i0, i1 = p.items[it].i1, tiles = p.items[it].ntok > tq ? 2 : 1, i = i0;
        for (int t = 0; ok && t < tiles; ++t) ok = issue_s(t, 0, true, i0 + 1 == i1);
        if (ok) umma_commit(&empty[0]);
        while (ok) {
          // what follows block i: the next one of the item, or the first of the next item
          const bool begin = i == i0, end = i + 1 == i1;
          int nit = it, ni0 = i0, ni1 = i1, ntiles = tiles;
          if (end) {
            ++nit;
            while (nit < last && p.items[nit].i0 == p.items[nit].i1) ++nit;
            if (nit < last) {
              ni0 = p.items[nit].i0;
              ni1 = p.items[nit].i1;
              ntiles = p.items[nit].ntok > tq ? 2 : 1;
            }
          }
          const bool more = nit < last;
          const int ni = end ? ni0 : i + 1;
          const uint32_t u = 2 * n + 1;
          for (int t = 0; ok && t < 2; ++t) {
            if (t < tiles) {
              if (begin) ok = wait(&o_free[t], (on[t]++ & 1) ^ 1);
              ok = ok && wait(&p_full[t], sn[t]++ & 1) && wait(&full[u % NS], (u / NS) & 1);
              if (!ok) break;
              tc_fence_after();
              const uint32_t v_s = smem_u32(sm + L::ring + (u % NS) * L::kTile);
#pragma unroll
              for (int kk = 0; kk < kPagedKB / 16; ++kk)
                umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8,
                            sdesc_mnmajor_sw128(v_s + kk * 2048, kPagedBox), id_pv, (!begin || kk > 0) ? 1u : 0u);
              if (end) umma_commit(&o_done[t]);
              if (t + 1 == tiles) umma_commit(&empty[u % NS]);
            }
            if (more && t < ntiles) {
              ok = issue_s(t, n + 1, end, ni + 1 == ni1);
              if (ok && t + 1 == ntiles) umma_commit(&empty[(2 * n + 2) % NS]);
            }
          }
          if (!more) break;
          ++n;
          it = nit;
          i0 = ni0;
          i1 = ni1;
          i = ni;
          tiles = ntiles;
        }
      }
      if (!ok) abort_flag = 1;
      umma_commit(drain);
      mbar_wait(drain, 0, p.err);
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- output
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    const int quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    uint32_t on[2] = {0, 0};
    bool ok = true;
    for (int it = first; ok && it < last; ++it) {
      const PagedItem w = p.items[it];
      const bool any = w.i1 > w.i0;
      for (int t = 0; ok && t < (w.ntok > tq ? 2 : 1); ++t) {
        const int rows = (min(w.ntok, (t + 1) * tq) - t * tq) * p.G;
        float m = -INFINITY, l = 0.f;
        if (any) {
          ok = __all_sync(0xffffffffu, !abort_flag && mbar_wait(&ml_full[t], on[t] & 1, p.err) &&
                                           mbar_wait(&o_done[t], on[t] & 1, p.err));
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
        for (int c = 0; c < HD; c += 32) {
          float o[32];
          __syncwarp();
          if (any) {
            tmem_ld32(tmem + 256 + t * 128 + lane_off + c, o);
            tmem_ld_wait();
          }
          if (any && c + 32 == HD) {                     // O is read: the next item may begin
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[t]);
          }
          if (r < rows) {
            if (!any || f == 0.f) {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0.f;
            }
            if (w.slot >= 0) {
              float4* dst = reinterpret_cast<float4*>(p.part_O + prow * HD + c);
#pragma unroll
              for (int j = 0; j < 8; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            } else {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row * HD + c);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                dst[j] = make_uint4(pack_bf16(o[8 * j] * f, o[8 * j + 1] * f), pack_bf16(o[8 * j + 2] * f, o[8 * j + 3] * f),
                                    pack_bf16(o[8 * j + 4] * f, o[8 * j + 5] * f), pack_bf16(o[8 * j + 6] * f, o[8 * j + 7] * f));
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
      }
    }
    if (!ok) abort_flag = 1;
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    const float sl2 = p.scale * 1.4426950408889634f;     // scores in log2 units
    uint32_t n = 0, items = 0;                           // this tile's blocks and items
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
        ok = __all_sync(0xffffffffu, !abort_flag && mbar_wait(&s_full[t], n & 1, p.err));
        if (!ok) break;
        tc_fence_after();
        float v[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32(tS + c, v + c);
        tmem_ld_wait();
        if (k0 + kPagedKB > hi_min || (k0 < lo_max && k0 + kPagedKB > range.sinks)) {
          const int h = hi - k0, b = lo - k0, f = range.sinks - k0;
#pragma unroll
          for (int j = 0; j < 128; ++j)
            if (!(j < h && (j >= b || j < f))) v[j] = -INFINITY;
        }
        float mx = fmaxf(v[0], v[1]);
#pragma unroll
        for (int j = 2; j < 128; j += 2) mx = fmaxf(mx, fmaxf(v[j], v[j + 1]));
        mx *= sl2;
        // the keys of this block that no row sees hold whatever their pages do: weight 0 times
        // that must be 0 (thread r of tile 0, whose blocks are all of the stream's, clears row r
        // of V; tile 1's P V comes later)
        if (t == 0 && (k0 < range.lo || k0 + kPagedKB > range.hi) && !range.has(k0 + r)) {
          const uint32_t u = 2 * n + 1;
          ok = mbar_wait(&full[u % NS], (u / NS) & 1, p.err);
          unsigned char* row = sm + L::ring + (u % NS) * L::kTile + r * 128;
#pragma unroll
          for (int c = 0; c < KCH; ++c)
#pragma unroll
            for (int y = 0; y < 8; ++y) *reinterpret_cast<uint4*>(row + c * kPagedBox + y * 16) = make_uint4(0, 0, 0, 0);
          fence_async_shared();
        }
        const bool grew = valid && mx > m + 8.f;                  // also the first finite maximum of a row
        if (__any_sync(0xffffffffu, grew)) {
          const float alpha = grew ? ex2(m - mx) : 1.f;
          if (grew) m = mx;
          l *= alpha;
          if (i > w.i0) {
#pragma unroll 1
            for (int c = 0; c < HD; c += 16) {
              float o[16];
              tmem_ld16(tO + c, o);
              tmem_ld_wait();
              uint32_t b[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) b[j] = __float_as_uint(o[j] * alpha);
              tmem_st16(tO + c, b);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          uint32_t b[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float e0 = ex2(fmaf(v[c + j], sl2, -ref)), e1 = ex2(fmaf(v[c + j + 1], sl2, -ref));
            l0 += e0;
            l1 += e1;
            b[j / 2] = pack_bf16(e0, e1);
          }
          tmem_st16(tS + c / 2, b);
        }
        l += l0 + l1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      ok = __all_sync(0xffffffffu, ok && !abort_flag && mbar_wait(&ml_free[t], (items & 1) ^ 1, p.err));
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
  cudaError_t e = cudaFuncSetAttribute(paged_attention_chunk_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       ChunkSmem<HD>::bytes);
  if (e != cudaSuccess) return e;
  paged_attention_chunk_kernel<HD><<<p.workers, kChunkThreads, ChunkSmem<HD>::bytes, st>>>(tq, tk, tv, p);
  return launched();
}

cudaError_t launch_paged_attention_chunk(const PagedAttnParams& p, cudaStream_t st) {
  if (p.workers == 0) return cudaSuccess;
  return p.hd == 128 ? attention_chunk<128>(p, st) : attention_chunk<64>(p, st);
}

}  // namespace sf

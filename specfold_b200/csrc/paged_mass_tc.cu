// Weight accumulation over the paged cache on the tensor core (bf16): every cached key's
// sum over query rows of exp(s - lse).
//
// The scores are computed transposed, S^T = K Q^T with the 128 keys of a block as the rows of the
// MMA, so that a key is a TMEM lane: a thread adds up its own key's weights over the columns (the
// query rows), tile after tile, in registers.  A weight is therefore summed in one place, in one
// order, and added once (atomically: another sequence may hold the same page).  lse is a per-column
// constant: the exponent is one fma.
// A CTA works on two key blocks at a time, so that a query tile, which streams from L2, feeds two
// products.  A pair whose tiles were cut between CTAs leaves its sums for the merge.
//   warps 4-11, 12-19 exponentials and sums of the first and of the second block, two threads per
//                     key: rows 0-63 and 64-127 of a tile.  Two warps on each scheduler for either
//                     block hide each other's waits for TMEM and for the special-function unit: with
//                     one thread per key the largest case took 292 us, with two a fifth less
//   warp 0            TMA: key blocks and query tiles, through rings of their own
//   warp 1            tcgen05.mma, two S^T buffers of 128 columns for each block (all of TMEM)
//   warp 2            lse of the tile's rows into shared memory
// Bound: for chunks by the special-function unit, one exponential per (row, key): 1024 cycles for
// a 128 x 128 tile against 512 of products; for single tokens by the bytes of the keys.
//
// Measured: 28 / 4 heads, 4051 tokens over 5300 and 8192 keys, 0.167 TFLOP, 6.5e8 exponentials: 249
// us, 1.6 times what the special-function units need; 32 tokens over 1000 to 8192 keys of 8 heads,
// 235 MB: 55 us (4.3 TB/s).  A polynomial for some of the exponentials did not help (289 to 328 us
// where none took 292, before there were two threads per key).
#include "paged_tc.cuh"

namespace sf {

constexpr int kMassThreads = 640;

template <int HD>
struct MassSmem {
  static constexpr int kTile = HD / 64 * kPagedBox;      // 128 rows
  static constexpr int kKeys = 4, kQueries = 2;          // stages of keys, of queries
  static constexpr int kRows = 4;                        // stages of lse
  static constexpr int k = 0;                            // [kKeys][kTile]
  static constexpr int q = k + kKeys * kTile;            // [kQueries][kTile]
  static constexpr int lse = q + kQueries * kTile;        // [kRows][128] floats
  static constexpr int half = lse + kRows * 512;         // [2 blocks][2][128] sums of rows 64-127
  static constexpr int odd = half + 4 * 512;             // [kRows] stages with a NaN lse
  static constexpr int bars = odd + kRows * 4;
  static constexpr int bytes = bars + 256 + 1024;        // + alignment of the base
};

// The tiles of an item that meet block kb (0 or 1 of the pair): those with tokens [f, l) that see
// a key of it.
struct MassBlock {
  int kb, f, l;
  __device__ __forceinline__ MassBlock(const PagedMask& mask, int kb_, int kv_len) : kb(kb_), f(0), l(0) {
    if (kb * kPagedKB < kv_len) mask.tokens(kb, &f, &l);
  }
  __device__ __forceinline__ bool meets(int t, int t_end) const { return t < l && t_end > f; }
};

template <int HD>
__global__ void __launch_bounds__(kMassThreads, 1)
    paged_mass_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      PagedMassParams p) {
  typedef MassSmem<HD> L;
  constexpr int KCH = HD / 64, NK = L::kKeys, NQ = L::kQueries, NR = L::kRows;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                       ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* k_full = bars;                               // [NK]
  uint64_t* k_empty = bars + NK;                         // [NK]
  uint64_t* q_full = bars + 2 * NK;                      // [NQ]
  uint64_t* q_empty = q_full + NQ;                       // [NQ]
  uint64_t* r_full = q_empty + NQ;                       // [NR]
  uint64_t* r_empty = r_full + NR;                       // [NR]
  uint64_t* s_full = r_empty + NR;                       // [2 blocks][2 buffers]
  uint64_t* s_empty = s_full + 4;
  uint64_t* drain = s_empty + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    for (int s = 0; s < NK; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < NQ; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < NR; ++s) {
      mbar_init(&r_full[s], 1);
      mbar_init(&r_empty[s], 16);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_empty[s], 8);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  // rows of a query tile past its G * tokens are never loaded: their scores must be finite
  for (int i = threadIdx.x; i < NQ * L::kTile / 16; i += kMassThreads)
    reinterpret_cast<uint4*>(sm + L::q)[i] = make_uint4(0, 0, 0, 0);
  fence_async_shared();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int first = p.first[blockIdx.x], last = p.first[blockIdx.x + 1];
  const int tq = 128 / p.G;                              // tokens of a query tile
  uint32_t kn = 0, qn = 0;                               // key blocks, query tiles so far
  bool ok = true;
  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    // one item ahead: its record, and the pages of its two blocks
    struct Pair {
      KeyPages a, b;
      bool has_a, has_b;
    };
    auto pages = [&](const PagedMassItem& m) {
      const PagedMask mask{p.block, p.window, p.sinks, m.q_len, m.kv_len};
      PagedItem w{};
      w.seq = m.seq;
      const bool second = (m.kb0 + 1) * kPagedKB < m.kv_len;
      const PagedRange ra = mask.block_range(m.kb0), rb = second ? mask.block_range(m.kb0 + 1) : PagedRange{0, 0, 0};
      return Pair{KeyPages(p.pool, w, ra, m.kb0, KCH, lane, p.err), KeyPages(p.pool, w, rb, m.kb0 + 1, KCH, lane, p.err),
                  ra.hi > 0, rb.hi > 0};
    };
    auto load_keys = [&](const KeyPages& k, int kvh) {
      const uint32_t s = kn % NK;
      ok = __all_sync(0xffffffffu, wait_or_abort(&k_empty[s], ((kn / NK) & 1) ^ 1, p.err, abort_flag));
      if (!ok) return;
      load_key_block(sm + L::k + s * L::kTile, &tmK, &k_full[s], k, kvh, lane);
      ++kn;
    };
    PagedMassItem m = p.items[first < last ? first : 0];
    Pair now = pages(m);
    for (int it = first; ok && it < last; ++it) {
      const PagedMassItem next = p.items[it + 1 < last ? it + 1 : it];
      if (now.has_a) load_keys(now.a, m.kvh);
      if (ok && now.has_b) load_keys(now.b, m.kvh);
      for (int x = m.i0; ok && x < m.i1; ++x) {
        const uint32_t s = qn % NQ;
        ok = __all_sync(0xffffffffu, wait_or_abort(&q_empty[s], ((qn / NQ) & 1) ^ 1, p.err, abort_flag));
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&q_full[s], KCH * tq * p.G * 128);
        __syncwarp();
        if (lane < KCH)
          tma_load_3d(sm + L::q + s * L::kTile + lane * kPagedBox, &tmQ, &q_full[s], lane * 64, m.kvh * p.G,
                      m.q0 + m.t0 + x * tq);
        ++qn;
      }
      m = next;
      now = pages(m);
    }
    if (!ok && lane == 0) {                              // no load may be in flight at exit
      *abort_flag = 1;
      for (uint32_t x = kn > NK ? kn - NK : 0; x < kn; ++x) mbar_wait(&k_full[x % NK], (x / NK) & 1, p.err);
      for (uint32_t x = qn > NQ ? qn - NQ : 0; x < qn; ++x) mbar_wait(&q_full[x % NQ], (x / NQ) & 1, p.err);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (elect_one()) {
      uint32_t bn[2] = {0, 0};                           // scores of each block so far
      for (int it = first; ok && it < last; ++it) {
        const PagedMassItem m = p.items[it];
        const PagedMask mask{p.block, p.window, p.sinks, m.q_len, m.kv_len};
        const MassBlock blk[2] = {MassBlock(mask, m.kb0, m.kv_len), MassBlock(mask, m.kb0 + 1, m.kv_len)};
        uint32_t k_lo[2];
        uint32_t ks[2];
#pragma unroll
        for (int y = 0; ok && y < 2; ++y) {
          if (blk[y].f >= blk[y].l) continue;
          ks[y] = kn % NK;
          ok = wait_or_abort(&k_full[ks[y]], (kn / NK) & 1, p.err, abort_flag);
          k_lo[y] = ((smem_u32(sm + L::k) + ks[y] * L::kTile) >> 4) | (1u << 16);
          ++kn;
        }
        for (int x = m.i0; ok && x < m.i1; ++x, ++qn) {
          const uint32_t s = qn % NQ;
          const int t = m.t0 + x * tq, t_end = min(t + tq, m.t1);
          const int cols = ((t_end - t) * p.G + 15) / 16 * 16;
          const uint32_t id = idesc_bf16(128, 16) + (static_cast<uint32_t>(cols / 8 - 2) << 17);
          const uint32_t q_lo = ((smem_u32(sm + L::q) + s * L::kTile) >> 4) | (1u << 16);
          ok = wait_or_abort(&q_full[s], (qn / NQ) & 1, p.err, abort_flag);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            if (!ok || !blk[y].meets(t, t_end)) continue;
            const uint32_t b = 2 * y + (bn[y] & 1);
            ok = wait_or_abort(&s_empty[b], ((bn[y] >> 1) & 1) ^ 1, p.err, abort_flag);
            if (!ok) continue;
            ++bn[y];
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              umma_f16(tmem + b * 128, desc(k_lo[y] + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2),
                       desc(q_lo + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2), id, kk > 0 ? 1u : 0u);
            umma_commit(&s_full[b]);
          }
          if (!ok) break;
          umma_commit(&q_empty[s]);
        }
        if (!ok) break;
#pragma unroll
        for (int y = 0; y < 2; ++y)
          if (blk[y].f < blk[y].l) umma_commit(&k_empty[ks[y]]);
      }
      if (!ok) *abort_flag = 1;
      umma_commit(drain);
      mbar_wait(drain, 0, p.err);
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- lse of the rows
    float* s_lse = reinterpret_cast<float*>(sm + L::lse);
    int* s_odd = reinterpret_cast<int*>(sm + L::odd);
    int tok[4], head[4];                                 // of this lane's four rows
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      tok[j] = (lane + 32 * j) / p.G;
      head[j] = (lane + 32 * j) % p.G;
    }
    for (int it = first; ok && it < last; ++it) {
      const PagedMassItem m = p.items[it];
      for (int x = m.i0; x < m.i1; ++x, ++qn) {
        const uint32_t s = qn % NR;
        const int t = m.t0 + x * tq, n = min(tq, m.t1 - t);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {                    // ahead of the wait: the loads take their time
          v[j] = INFINITY;                               // a column that is no row: weight 0
          if (tok[j] < n)
            v[j] = p.lse[static_cast<int64_t>(m.q0 + t + tok[j]) * p.H + m.kvh * p.G + head[j]] * 1.4426950408889634f;
          if (v[j] == -INFINITY) v[j] = INFINITY;        // a row that saw nothing gives nothing
        }
        const bool odd = __any_sync(0xffffffffu, isnan(v[0]) || isnan(v[1]) || isnan(v[2]) || isnan(v[3]));
        ok = __all_sync(0xffffffffu, wait_or_abort(&r_empty[s], ((qn / NR) & 1) ^ 1, p.err, abort_flag));
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) s_lse[s * 128 + lane + 32 * j] = -v[j];
        if (lane == 0) s_odd[s] = odd;
        __syncwarp();
        if (lane == 0) mbar_arrive(&r_full[s]);
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- exponentials and sums
    const int y = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t tS = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + y * 256;
    const float* s_lse = reinterpret_cast<const float*>(sm + L::lse);
    const int* s_odd = reinterpret_cast<const int*>(sm + L::odd);
    const float sl2 = p.scale * 1.4426950408889634f;
    const uint64_t scale2 = pair(sl2, sl2);
    uint32_t bn = 0;                                     // this block's scores so far
    // One item ahead: which key is this thread's, the tokens that see it, and where its sum goes
    // (the page id is on its way while the item before is worked on).
    struct Ahead {
      PagedMassItem m;
      int f, l, id;                                      // tokens [f, l) see the key; its page
    };
    auto begin = [&](int it) {
      Ahead a;
      a.m = p.items[it];
      const int key = (a.m.kb0 + y) * kPagedKB + r;
      a.f = a.l = a.id = 0;
      if (key < a.m.kv_len) {
        const PagedMask mask{p.block, p.window, p.sinks, a.m.q_len, a.m.kv_len};
        mask.key_tokens(key, &a.f, &a.l);
        if (a.f < a.l && a.m.slot < 0) a.id = p.pool.table[a.m.seq * p.pool.table_stride + (key >> p.pool.page_shift)];
      }
      return a;
    };
    auto target = [&](const Ahead& a) -> float* {
      if (a.f >= a.l) return nullptr;
      if (a.m.slot >= 0) return p.part + static_cast<int64_t>(a.m.slot) * kMassBlocks * kPagedKB + y * kPagedKB + r;
      const int key = (a.m.kb0 + y) * kPagedKB + r;
      int id = a.id;
      if (id < 0 || id >= p.pool.num_pages) {            // flagged, and nothing is written
        flag_error(p.err, SF_DEV_ERR_INDEX);
        return nullptr;
      }
      return p.pool.mass + ((static_cast<int64_t>(id) * p.Hkv + a.m.kvh) << p.pool.page_shift) +
             (key & ((1 << p.pool.page_shift) - 1));
    };
    Ahead cur = begin(first < last ? first : 0);
    float* dst = target(cur);
    float* s_half = reinterpret_cast<float*>(sm + L::half) + y * 256;
    for (int it = first; it < last; ++it) {              // (to the end whatever fails: the halves meet)
      const PagedMassItem& m = cur.m;
      const Ahead next = begin(it + 1 < last ? it + 1 : it);
      const PagedMask mask{p.block, p.window, p.sinks, m.q_len, m.kv_len};
      const MassBlock blk(mask, m.kb0 + y, m.kv_len);
      uint64_t sum0 = pair(0.f, 0.f), sum1 = sum0;
      for (int x = m.i0; x < m.i1; ++x, ++qn) {
        const uint32_t s = qn % NR, b = bn & 1;
        const int t = m.t0 + x * tq, t_end = min(t + tq, m.t1);
        const int rows = (t_end - t) * p.G;
        const bool mine = blk.meets(t, t_end);
        ok = __all_sync(0xffffffffu, ok && (!mine || wait_or_abort(&s_full[2 * y + b], (bn >> 1) & 1, p.err, abort_flag)) &&
                                         wait_or_abort(&r_full[s], (qn / NR) & 1, p.err, abort_flag));
        if (!ok) break;
        if (mine && half * 64 >= rows) ++bn;
        else if (mine) {
          tc_fence_after();
          // columns [c_lo, c_hi) are rows that see this thread's key
          const int c_lo = max(cur.f - t, 0) * p.G, c_hi = max(min(cur.l, t_end) - t, 0) * p.G;
          // the weights of columns [c, c + 32); what is no row of the tile is outside [c_lo, c_hi)
          auto add = [&](float* v, int c) {
            const float4* lse4 = reinterpret_cast<const float4*>(s_lse + s * 128 + c);
            if (__any_sync(0xffffffffu, c < c_lo || c + 32 > c_hi)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j < c_lo || c + j >= c_hi) v[j] = -INFINITY;
            }
#pragma unroll
            for (int g = 0; g < 32; g += 8) {
              if (c + g >= rows) break;
#pragma unroll
              for (int j = g; j < g + 8; j += 4) {
                const float4 e = lse4[j / 4];
                float a0, a1, a2, a3;
                unpair(fma2(pair(v[j], v[j + 1]), scale2, pair(e.x, e.y)), a0, a1);
                unpair(fma2(pair(v[j + 2], v[j + 3]), scale2, pair(e.z, e.w)), a2, a3);
                sum0 = add2(sum0, pair(ex2(a0), ex2(a1)));
                sum1 = add2(sum1, pair(ex2(a2), ex2(a3)));
              }
            }
          };
          const uint32_t tB = tS + b * 128;
          const int c_end = min(rows, half * 64 + 64);
          if (s_odd[s]) {                                // -inf + NaN is NaN: only the columns themselves
#pragma unroll 1
            for (int c = half * 64; c < c_end; c += 8) {
              float v[8];
              tmem_ld8(tB + c, v);
              tmem_wait<8>(v);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (c + j >= c_lo && c + j < c_hi) sum0 = add2(sum0, pair(ex2(fmaf(v[j], sl2, s_lse[s * 128 + c + j])), 0.f));
            }
          } else {
#pragma unroll 1
            for (int c = half * 64; c < c_end; c += 32) {
              float v[32];
              tmem_ld32(tB + c, v);
              tmem_wait<32>(v);
              add(v, c);
            }
          }
          tc_fence_before();
          ++bn;
        }
        __syncwarp();
        if (lane == 0) {
          if (mine) mbar_arrive(&s_empty[2 * y + b]);
          mbar_arrive(&r_empty[s]);
        }
      }
      float* next_dst = target(next);
      float a0, a1;
      unpair(add2(sum0, sum1), a0, a1);
      float* other = s_half + (it - first & 1) * 128 + r;  // two by turns: read while the next is written
      if (half == 1) *other = a0 + a1;
      asm volatile("bar.sync %0, 256;" ::"r"(1 + y) : "memory");
      if (half == 0 && dst != nullptr && ok) {
        const float sum = a0 + a1 + *other;
        if (m.slot < 0) atomicAdd(dst, sum);
        else *dst = sum;
      }
      cur = next;
      dst = next_dst;
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

template <int HD>
static cudaError_t mass_tc(const PagedMassParams& p, cudaStream_t st) {
  CUtensorMap tq, tk;
  if (!query_tmap(&tq, p.q, p.q_tok, p.q_head, p.T, p.H, HD, p.G, 128 / p.G) ||
      !pool_tmap(&tk, p.pool.k, p.pool, p.Hkv, HD))
    return cudaErrorInvalidValue;
  cudaError_t e = allow_smem(paged_mass_kernel<HD>, MassSmem<HD>::bytes);
  if (e != cudaSuccess) return e;
  paged_mass_kernel<HD><<<p.workers, kMassThreads, MassSmem<HD>::bytes, st>>>(tq, tk, p);
  return launched();
}

cudaError_t launch_paged_mass_tc(const PagedMassParams& p, cudaStream_t st) {
  if (p.workers == 0) return cudaSuccess;
  return p.hd == 128 ? mass_tc<128>(p, st) : mass_tc<64>(p, st);
}

}  // namespace sf

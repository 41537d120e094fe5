// Attention over the paged cache when a sequence brings few query rows per kv head (at most 128:
// single tokens, small blocks): bound by the bytes of the keys and values.
//
// A persistent CTA per SM walks the items of its share.  Keys and values stream through a ring
// of TMA stages (one key block of 128 rows of K or of V each, a box per page), the products run
// on tcgen05 with M = 128 query rows:
//     S = Q K^T        accumulator in TMEM, double-buffered, one block ahead of the softmax
//     softmax          4 warps, a query row per thread, running (m, l)
//     O += P V         P (bf16) from TMEM, V as the MN-major operand, O in TMEM
// A token's G query heads fill only G of the 128 rows.  The products cost the same whatever
// they hold, and at 2 x 512 cycles a block they hide behind its 64 KB (2800 cycles at the HBM
// rate); the softmax would not, with all of a row's 128 exponentials in one thread.  So with at
// most 32 (64) rows they are loaded 4 (2) times, copy c takes the keys [c, c + 1) * 128 / REP of
// every block, its weights elsewhere stay zero, and each copy accumulates its own (m, l, O);
// they are joined once per item.
//
// The rescaling of O waits until a row's maximum has grown by 2^8: until then the weights are
// merely up to 2^8 instead of 1, relative to the same reference in l and O, and lose nothing.
//
// Measured (32 / 8 heads of 128): 64 single tokens over 1100 to 16384 keys, 1.52 GB, in 297 us (5.1
// TB/s, 79% of a plain copy's rate); 32 tokens that see a window of 4096 and 4 first keys, 244 MB,
// in 60 us.  In the steady state a CTA takes 2200 cycles a block; the rest is the first loads'
// latency (page id, keys, 5000 cycles) and each item's output.  One token over 777 keys: 11 us on
// the device, the latency of the chain item, page id, keys, softmax, output, join.
#include "paged_tc.cuh"

namespace sf {

constexpr int kTokThreads = 192;       // TMA warp, MMA warp, 4 softmax warps
constexpr int kRedLd = 33;             // row of the join buffer

template <int HD>
struct TokSmem {
  static constexpr int kTile = HD / 64 * kPagedBox;      // 128 rows
  static constexpr int kStages = HD == 128 ? 4 : 8;
  static constexpr int q = 0;                            // [2][kTile]
  static constexpr int ring = q + 2 * kTile;             // [kStages][kTile]
  static constexpr int red = ring + kStages * kTile;     // [128][kRedLd] floats
  static constexpr int ml = red + 128 * kRedLd * 4;      // [2][128] floats
  static constexpr int bars = ml + 2 * 128 * 4;
  static constexpr int bytes = bars + 256 + 1024;        // + alignment of the base
};

__device__ __forceinline__ bool vote128(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x))
      : "memory");
  return r != 0;
}

template <int HD, int REP>
__global__ void __launch_bounds__(kTokThreads, 1)
    paged_attention_tokens_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                                  const __grid_constant__ CUtensorMap tmV, PagedAttnParams p) {
  typedef TokSmem<HD> L;
  constexpr int KCH = HD / 64, NS = L::kStages;
  constexpr int RC = 128 / REP;                          // rows of a copy
  constexpr int NC = 128 / REP;                          // keys of a block that a copy takes
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                       ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* full = bars;                                 // [NS]
  uint64_t* empty = bars + NS;                           // [NS]
  uint64_t* q_full = bars + 2 * NS;                      // [2]
  uint64_t* q_empty = q_full + 2;                        // [2]
  uint64_t* s_full = q_full + 4;                         // [2]
  uint64_t* p_full = q_full + 6;
  uint64_t* pv_done = q_full + 7;
  uint64_t* o_free = q_full + 8;
  uint64_t* drain = q_full + 9;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 10);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  pdl_trigger();                                         // the join of cut tiles may line up
  // (on its way while the barriers are set up)
  const PagedItem head = p.heads[blockIdx.x];
  const int first = p.first[blockIdx.x], last = p.first[blockIdx.x + 1];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
    }
    mbar_init(p_full, 4);
    mbar_init(pv_done, 1);
    mbar_init(o_free, 4);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tO = tmem + 256, tP = tmem + 384;       // S buffers at columns 0 and 128

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    uint32_t u = 0;                                      // ring units issued (K and V blocks)
    int qn = 0;                                          // query tiles issued
    bool ok = true;
    for (int it = first; ok && it < last; ++it) {
      const PagedItem w = it == first ? head : p.items[it];
      if (w.i0 == w.i1) continue;
      const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
      const PagedRange range = mask.range(w.tok0, w.tok0 + w.ntok);
      const int qb = qn & 1;
      ok = __all_sync(0xffffffffu, wait_or_abort(&q_empty[qb], ((qn >> 1) & 1) ^ 1, p.err, abort_flag));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&q_full[qb], REP * KCH * (RC / p.G) * p.G * 128);
      __syncwarp();
      if (lane < REP * KCH)
        tma_load_3d(sm + L::q + qb * L::kTile + (lane % KCH) * kPagedBox + (lane / KCH) * RC * 128, &tmQ,
                    &q_full[qb], (lane % KCH) * 64, w.kvh * p.G, w.q0 + w.tok0);
      ++qn;
      KeyPages pages(p.pool, w, range, w.block(w.i0), KCH, lane, p.err);
      for (int i = w.i0; ok && i < w.i1; ++i) {
        const KeyPages now = pages;
        if (i + 1 < w.i1) pages = KeyPages(p.pool, w, range, w.block(i + 1), KCH, lane, p.err);
        for (int kv = 0; kv < 2; ++kv, ++u) {
          const int s = u % NS;
          ok = __all_sync(0xffffffffu, wait_or_abort(&empty[s], ((u / NS) & 1) ^ 1, p.err, abort_flag));
          if (!ok) break;
          load_key_block(sm + L::ring + s * L::kTile, kv ? &tmV : &tmK, &full[s], now, w.kvh, lane);
        }
      }
    }
    if (!ok) {                                           // no load may be in flight at exit
      if (lane == 0) {
        *abort_flag = 1;
        for (uint32_t x = u > NS ? u - NS : 0; x < u; ++x) mbar_wait(&full[x % NS], (x / NS) & 1, p.err);
        for (int x = qn > 2 ? qn - 2 : 0; x < qn; ++x) mbar_wait(&q_full[x & 1], (x >> 1) & 1, p.err);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (elect_one()) {
      const uint32_t id_s = idesc_bf16(128, kPagedKB);
      const uint32_t id_pv = idesc_bf16(128, HD, 0, 1);
      uint32_t n = 0;                                    // key blocks whose S was issued
      int qn = 0, items = 0;                             // query tiles, items whose O was begun
      bool ok = true;
      // O += P V of block x (its place in the stream of blocks)
      auto issue_pv = [&](uint32_t x, bool begin) -> bool {
        if (begin) {
          if (!wait_or_abort(o_free, (items & 1) ^ 1, p.err, abort_flag)) return false;
          ++items;
        }
        const uint32_t u = 2 * x + 1;
        if (!wait_or_abort(&full[u % NS], (u / NS) & 1, p.err, abort_flag) ||
            !wait_or_abort(p_full, x & 1, p.err, abort_flag))
          return false;
        tc_fence_after();
        const uint32_t v_lo = ((smem_u32(sm + L::ring) + (u % NS) * L::kTile) >> 4) | ((kPagedBox >> 4) << 16);
#pragma unroll
        for (int kk = 0; kk < kPagedKB / 16; ++kk)
          umma_f16_ts(tO, tP + kk * 8, desc(v_lo + kk * 128), id_pv, (!begin || kk > 0) ? 1u : 0u);
        umma_commit(pv_done);
        umma_commit(&empty[u % NS]);
        return true;
      };
      bool begin = false, waiting = false;               // the block before: begins an item; P V due
      for (int it = first; ok && it < last; ++it) {
        const int i0 = it == first ? head.i0 : p.items[it].i0, i1 = it == first ? head.i1 : p.items[it].i1;
        if (i0 == i1) continue;
        const int qb = qn & 1;
        ok = wait_or_abort(&q_full[qb], (qn >> 1) & 1, p.err, abort_flag);
        const uint32_t q_lo = ((smem_u32(sm + L::q) + qb * L::kTile) >> 4) | (1u << 16);
        for (int i = i0; ok && i < i1; ++i) {
          const uint32_t u = 2 * n;
          // S buffer n & 1 was read by the softmax of block n - 2 before it handed over its P,
          // which the P V of that block, issued before, has waited for
          ok = wait_or_abort(&full[u % NS], (u / NS) & 1, p.err, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t k_lo = ((smem_u32(sm + L::ring) + (u % NS) * L::kTile) >> 4) | (1u << 16);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            umma_f16(tmem + (n & 1) * 128, desc(q_lo + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2),
                     desc(k_lo + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2), id_s, kk > 0 ? 1u : 0u);
          umma_commit(&s_full[n & 1]);
          umma_commit(&empty[u % NS]);
          if (i + 1 == i1) umma_commit(&q_empty[qb]);
          if (waiting) ok = issue_pv(n - 1, begin);
          begin = i == i0;
          waiting = true;
          ++n;
        }
        ++qn;
      }
      if (ok && waiting) ok = issue_pv(n - 1, begin);
      if (!ok) *abort_flag = 1;
      umma_commit(drain);
      mbar_wait(drain, 0, p.err);
    }
  } else {
    // ---------------------------------------------------------------- softmax and output
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;                   // this thread's row of the MMA tile
    const int copy = r / RC, rr = r % RC;                // copy of the rows, row of the tile
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const float sl2 = p.scale * 1.4426950408889634f;     // scores in log2 units
    float* red = reinterpret_cast<float*>(sm + L::red);
    float* s_m = reinterpret_cast<float*>(sm + L::ml);
    float* s_l = s_m + 128;
    if (REP > 1) {
      const uint32_t zero[16] = {};
#pragma unroll
      for (int c = 0; c < 64; c += 16) tmem_st16(tP + lane_off + c, zero);
      tmem_st_wait();
    }
    uint32_t n = 0;                                      // key blocks done
    bool ok = true;
    for (int it = first; it < last; ++it) {
      const PagedItem w = it == first ? head : p.items[it];
      const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
      const PagedRange range = mask.range(w.tok0, w.tok0 + w.ntok);
      const int rows = w.ntok * p.G;
      const bool valid = rr < rows;
      const bool busy = (quarter * 32) % RC < rows;      // any row of this warp
      const int tok = w.tok0 + (valid ? rr / p.G : 0);
      const int hi = mask.hi(tok), lo = mask.lo(tok);
      const int hi_min = mask.hi(w.tok0), lo_max = mask.lo(w.tok0 + w.ntok - 1);
      float m = -INFINITY, l = 0.f;
      bool finite = true;                                // what this thread saw of V and of the output
      for (int i = w.i0; i < w.i1; ++i, ++n) {
        const int k0 = w.block(i) * kPagedKB;
        const bool edge = k0 + kPagedKB > hi_min || (k0 < lo_max && k0 + kPagedKB > range.sinks);
        ok = __all_sync(0xffffffffu, ok && wait_or_abort(&s_full[n & 1], (n >> 1) & 1, p.err, abort_flag));
        if (!ok) break;
        tc_fence_after();
        float v[NC];
        float mx = -INFINITY;
        if (busy) {
#pragma unroll
          for (int c = 0; c < NC; c += 32) tmem_ld32(tmem + (n & 1) * 128 + lane_off + copy * NC + c, v + c);
          tmem_wait<NC>(v);
          if (edge) {
            const int h = hi - k0 - copy * NC, b = lo - k0 - copy * NC, f = range.sinks - k0 - copy * NC;
#pragma unroll
            for (int j = 0; j < NC; ++j)
              if (!(j < h && (j >= b || j < f))) v[j] = -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < NC; ++j) mx = fmaxf(mx, v[j]);
          mx *= sl2;
        }
        // The keys of this block that no row sees hold whatever their pages do, and those that only
        // some see may hold values that are not finite: weight 0 times either must be 0 (thread r
        // clears row r of V, or takes such values out of it).
        const int key = k0 + r;
        const bool seen = range.has(key);
        if (edge && !(seen && key < hi_min && (key >= lo_max || key < range.sinks))) {
          const uint32_t u = 2 * n + 1;
          ok = mbar_wait(&full[u % NS], (u / NS) & 1, p.err);
          uint4* row = reinterpret_cast<uint4*>(sm + L::ring + (u % NS) * L::kTile + r * 128);
#pragma unroll
          for (int c = 0; c < KCH; ++c)
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              uint4 d = make_uint4(0, 0, 0, 0);
              uint4* at = row + c * (kPagedBox / 16) + ((x + r) & 7);   // (the rows' banks apart)
              bool write = !seen;
              if (seen) {
                d = *at;
                write = drop_odd(d);
                finite &= !write;
              }
              if (write) *at = d;
            }
          fence_async_shared();
        }
        // the P V before reads P and adds to O
        ok = __all_sync(0xffffffffu, ok && (n == 0 || mbar_wait(pv_done, (n - 1) & 1, p.err)));
        if (!ok) break;
        tc_fence_after();
        if (busy) {
          const bool grew = valid && mx > m + 8.f;       // also the first finite maximum of a row
          if (__any_sync(0xffffffffu, grew)) {
            const float alpha = grew ? ex2(m - mx) : 1.f;
            if (grew) m = mx;
            l *= alpha;
            if (i > w.i0) {
#pragma unroll
              for (int c = 0; c < HD; c += 32) {
                float o[32];
                tmem_ld32(tO + lane_off + c, o);
                tmem_wait<32>(o);
                uint32_t b[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) b[j] = __float_as_uint(o[j] * alpha);
                tmem_st16(tO + lane_off + c, b);
                tmem_st16(tO + lane_off + c + 16, b + 16);
              }
            }
          }
          const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int c = 0; c < NC; c += 32) {
            uint32_t b[16];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float e0 = ex2(fmaf(v[c + j], sl2, -ref)), e1 = ex2(fmaf(v[c + j + 1], sl2, -ref));
              l += e0 + e1;
              b[j / 2] = pack_bf16(e0, e1);
            }
            tmem_st16(tP + lane_off + (copy * NC + c) / 2, b);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      const bool any = w.i1 > w.i0;
      if (ok && any) ok = mbar_wait(pv_done, (n - 1) & 1, p.err);
      ok = vote128(ok);
      if (!ok) break;
      tc_fence_after();
      float f = 1.f, L_row = l, M_row = m;               // join of the copies
      if (REP > 1) {
        s_m[r] = m;
        s_l[r] = l;
        vote128(true);
#pragma unroll
        for (int c = 0; c < REP; ++c) M_row = fmaxf(M_row, s_m[c * RC + rr]);
        const float ref = M_row == -INFINITY ? 0.f : M_row;
        L_row = 0.f;
#pragma unroll
        for (int c = 0; c < REP; ++c) L_row = fmaf(s_l[c * RC + rr], ex2(s_m[c * RC + rr] - ref), L_row);
        f = ex2(m - ref);
      }
      const int64_t slot_row = static_cast<int64_t>(w.slot) * p.rows;
      if (w.slot < 0) f *= L_row == 0.f ? 0.f : 1.f / L_row;
      // Through shared memory, so that a warp writes rows and the copies meet: all columns at once
      // where the rows are few, else 32 at a time.
      const int turn = REP * rows * (HD + 1) <= 128 * kRedLd ? HD : 32, ld = turn + 1;
      float* mine = red + (copy * rows + rr) * ld;
#pragma unroll 1
      for (int c0 = 0; c0 < HD; c0 += turn) {
#pragma unroll 1
        for (int c = c0; c < c0 + turn; c += 32) {
          float o[32];
          if (any && busy) {
            tmem_ld32(tO + lane_off + c, o);
            tmem_wait<32>(o);
          }
          if (valid)
#pragma unroll
            for (int j = 0; j < 32; ++j) mine[c - c0 + j] = any && f != 0.f ? o[j] * f : 0.f;
          __syncwarp();
        }
        if (c0 + turn == HD) {                           // O is read: the next item may begin
          tc_fence_before();
          __syncwarp();
          if (any && lane == 0) mbar_arrive(o_free);
        }
        vote128(true);
        // 32 columns of a row per warp and turn, the copies added in their order
        for (int x = quarter; x < rows * (turn / 32); x += 4) {
          const int row = x / (turn / 32), c = x % (turn / 32) * 32 + lane;
          float sum = red[row * ld + c];
#pragma unroll
          for (int y = 1; y < REP; ++y) sum += red[(y * rows + row) * ld + c];
          finite &= fabsf(sum) < INFINITY;
          if (w.slot < 0) {
            const int64_t t = w.q0 + w.tok0 + row / p.G;
            static_cast<__nv_bfloat16*>(p.out)[(t * p.H + w.kvh * p.G + row % p.G) * HD + c0 + c] =
                __float2bfloat16_rn(sum);
          } else {
            p.part_O[(slot_row + row) * HD + c0 + c] = sum;
          }
        }
        finite = vote128(finite);
      }
      if (valid && copy == 0) {
        if (w.slot < 0) {
          const int64_t t = w.q0 + w.tok0 + rr / p.G;
          p.lse[t * p.H + w.kvh * p.G + rr % p.G] = M_row * 0.6931471805599453f + logf(L_row);
        } else {
          p.part_ml[2 * (slot_row + rr)] = M_row;
          p.part_ml[2 * (slot_row + rr) + 1] = L_row;
        }
      }
      // Values that decide their columns.  (Of a row's copies only one has the weight of such a value,
      // the others 0: infinity became NaN, so the sum takes the output's place, unless the scores were NaN.)
      if (!finite) {
        vote128(true);                                   // lse is read back
        float sum[HD / 32];
        for (int tok = quarter; tok < w.ntok; tok += 4) {
          const int64_t row0 = static_cast<int64_t>(w.q0 + w.tok0 + tok) * p.H + w.kvh * p.G;
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + row0 * HD;
          float* part = w.slot >= 0 ? p.part_O + (slot_row + tok * p.G) * HD : nullptr;
          unsigned need = w.ntok == 1 ? 0u : ~0u;        // one token: nothing was left out of V
          for (int g = 0; w.ntok == 1 && g < p.G; ++g)
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) {
              const int at = g * HD + lane * (HD / 32) + e;
              need |= static_cast<unsigned>(!(fabsf(part != nullptr ? part[at] : __bfloat162float(out[at])) < INFINITY)) << e;
            }
          paged_odd_values<__nv_bfloat16, HD>(p, w, w.tok0 + tok, REP == 1, hi_min, lo_max, kPagedKB, lane, need, sum);
          for (int g = 0; g < p.G; ++g)
            if (part != nullptr || !isnan(p.lse[row0 + g]))
              paged_put_odd<__nv_bfloat16, HD>(sum, REP == 1, out + g * HD, part != nullptr ? part + g * HD : nullptr, lane);
        }
      }
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

template <int HD, int REP>
static cudaError_t attention_tokens(const PagedAttnParams& p, cudaStream_t st) {
  CUtensorMap tq, tk, tv;
  if (!query_tmap(&tq, p.q, p.q_tok, p.q_head, p.T, p.H, HD, p.G, 128 / REP / p.G) ||
      !pool_tmap(&tk, p.pool.k, p.pool, p.Hkv, HD) || !pool_tmap(&tv, p.pool.v, p.pool, p.Hkv, HD))
    return cudaErrorInvalidValue;
  cudaError_t e = allow_smem(paged_attention_tokens_kernel<HD, REP>, TokSmem<HD>::bytes);
  if (e != cudaSuccess) return e;
  paged_attention_tokens_kernel<HD, REP><<<p.workers, kTokThreads, TokSmem<HD>::bytes, st>>>(tq, tk, tv, p);
  return launched();
}

// copies: how often the rows of the list's largest tile fit the 128 (4, 2 or 1)
cudaError_t launch_paged_attention_tokens(const PagedAttnParams& p, int copies, cudaStream_t st) {
  if (p.workers == 0) return cudaSuccess;
  if (p.hd == 128)
    return copies == 4 ? attention_tokens<128, 4>(p, st) : copies == 2 ? attention_tokens<128, 2>(p, st) : attention_tokens<128, 1>(p, st);
  return copies == 4 ? attention_tokens<64, 4>(p, st) : copies == 2 ? attention_tokens<64, 2>(p, st) : attention_tokens<64, 1>(p, st);
}

}  // namespace sf

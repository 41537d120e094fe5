// Weight accumulation over the paged cache on the tensor core (bf16): every cached key's
// sum over query rows of exp(s - lse).
//
// The scores are computed transposed, S^T = K Q^T with the 128 keys of a block as the rows of the
// MMA, so that a key is a TMEM lane: a thread adds up its own key's weights over the columns (the
// query rows), tile after tile, in registers.  A weight is therefore summed in one place, in one
// order, and written once; no atomics.  lse is a per-column constant: the exponent is one fma.
//   warps 4-7, 8-11   exponentials and sums of columns 0-63 and 64-127 of every tile
//   warp 0            TMA: key blocks and query tiles, through rings of their own
//   warp 1            tcgen05.mma into four S^T buffers of 128 columns (all of TMEM)
//   warp 2            lse and the mask's bounds of the query tile's rows into shared memory
// Bound: for chunks by the special-function unit, one exponential per (row, key): 1024 cycles for
// a 128 x 128 tile against 512 of products; for single tokens by the bytes of the keys.
#include "paged_tc.cuh"

namespace sf {

constexpr int kMassThreads = 384;

template <int HD>
struct MassSmem {
  static constexpr int kTile = HD / 64 * kPagedBox;      // 128 rows
  static constexpr int kStages = 3;                      // of keys, of queries
  static constexpr int k = 0;                            // [kStages][kTile]
  static constexpr int q = k + kStages * kTile;          // [kStages][kTile]
  static constexpr int lse = q + kStages * kTile;        // [kStages][128] floats
  static constexpr int hi = lse + kStages * 512;         // [kStages][128] ints
  static constexpr int lo = hi + kStages * 512;
  static constexpr int part = lo + kStages * 512;        // [2][128] floats
  static constexpr int bars = part + 2 * 512;
  static constexpr int bytes = bars + 256 + 1024;        // + alignment of the base
};

template <int HD>
__global__ void __launch_bounds__(kMassThreads, 1)
    paged_mass_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      PagedMassParams p) {
  typedef MassSmem<HD> L;
  constexpr int KCH = HD / 64, NS = L::kStages;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                       ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t* k_full = bars;                               // [NS]
  uint64_t* k_empty = bars + NS;                         // [NS]
  uint64_t* q_full = bars + 2 * NS;                      // [NS]
  uint64_t* q_empty = bars + 3 * NS;                     // [NS]
  uint64_t* s_full = bars + 4 * NS;                      // [4]
  uint64_t* s_empty = s_full + 4;                        // [4]
  uint64_t* drain = s_full + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&q_full[s], 2);                          // the tile, the rows' bounds
      mbar_init(&q_empty[s], 9);                         // the products, the sums' warps
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
  for (int i = threadIdx.x; i < NS * L::kTile / 16; i += kMassThreads)
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
    for (int it = first; ok && it < last; ++it) {
      const PagedMassItem m = p.items[it];
      const PagedMask mask{p.block, p.window, p.sinks, m.q_len, m.kv_len};
      PagedItem w{};
      w.seq = m.seq;
      w.kvh = m.kvh;
      for (int kb = m.kb0; ok && kb < m.kb1; ++kb) {
        int t0, t1;
        mask.tokens(kb, &t0, &t1);
        if (t0 >= t1) continue;
        const uint32_t s = kn % NS;
        ok = __all_sync(0xffffffffu, wait_or_abort(&k_empty[s], ((kn / NS) & 1) ^ 1, p.err, abort_flag));
        if (!ok) break;
        load_key_block<HD>(sm + L::k + s * L::kTile, &tmK, &k_full[s], p.pool, w, mask.range(t0, t1), kb, lane, p.err);
        ++kn;
        for (int t = t0; t < t1; t += tq) {
          const uint32_t x = qn % NS;
          ok = __all_sync(0xffffffffu, wait_or_abort(&q_empty[x], ((qn / NS) & 1) ^ 1, p.err, abort_flag));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&q_full[x], KCH * tq * p.G * 128);
          __syncwarp();
          if (lane < KCH)
            tma_load_3d(sm + L::q + x * L::kTile + lane * kPagedBox, &tmQ, &q_full[x], lane * 64, m.kvh * p.G, m.q0 + t);
          ++qn;
        }
      }
    }
    if (!ok && lane == 0) {                              // no load may be in flight at exit
      *abort_flag = 1;
      for (uint32_t x = kn > NS ? kn - NS : 0; x < kn; ++x) mbar_wait(&k_full[x % NS], (x / NS) & 1, p.err);
      for (uint32_t x = qn > NS ? qn - NS : 0; x < qn; ++x) mbar_wait(&q_full[x % NS], (x / NS) & 1, p.err);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (elect_one()) {
      for (int it = first; ok && it < last; ++it) {
        const PagedMassItem m = p.items[it];
        const PagedMask mask{p.block, p.window, p.sinks, m.q_len, m.kv_len};
        for (int kb = m.kb0; ok && kb < m.kb1; ++kb) {
          int t0, t1;
          mask.tokens(kb, &t0, &t1);
          if (t0 >= t1) continue;
          const uint32_t s = kn % NS;
          ok = wait_or_abort(&k_full[s], (kn / NS) & 1, p.err, abort_flag);
          const uint32_t k_lo = ((smem_u32(sm + L::k) + s * L::kTile) >> 4) | (1u << 16);
          for (int t = t0; ok && t < t1; t += tq) {
            const uint32_t x = qn % NS, b = qn & 3;
            ok = wait_or_abort(&q_full[x], (qn / NS) & 1, p.err, abort_flag) &&
                 wait_or_abort(&s_empty[b], ((qn >> 2) & 1) ^ 1, p.err, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const int cols = (min(tq, t1 - t) * p.G + 15) / 16 * 16;
            const uint32_t id = idesc_bf16(128, 16) + (static_cast<uint32_t>(cols / 8 - 2) << 17);
            const uint32_t q_lo = ((smem_u32(sm + L::q) + x * L::kTile) >> 4) | (1u << 16);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              umma_f16(tmem + b * 128, desc(k_lo + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2),
                       desc(q_lo + (kk >> 2) * (kPagedBox >> 4) + (kk & 3) * 2), id, kk > 0 ? 1u : 0u);
            umma_commit(&s_full[b]);
            umma_commit(&q_empty[x]);
            if (t + tq >= t1) umma_commit(&k_empty[s]);
            ++qn;
          }
          ++kn;
        }
      }
      if (!ok) *abort_flag = 1;
      umma_commit(drain);
      mbar_wait(drain, 0, p.err);
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- lse and bounds of the rows
    float* s_lse = reinterpret_cast<float*>(sm + L::lse);
    int* s_hi = reinterpret_cast<int*>(sm + L::hi);
    int* s_lo = reinterpret_cast<int*>(sm + L::lo);
    for (int it = first; ok && it < last; ++it) {
      const PagedMassItem m = p.items[it];
      const PagedMask mask{p.block, p.window, p.sinks, m.q_len, m.kv_len};
      for (int kb = m.kb0; ok && kb < m.kb1; ++kb) {
        int t0, t1;
        mask.tokens(kb, &t0, &t1);
        for (int t = t0; ok && t < t1; t += tq, ++qn) {
          const uint32_t x = qn % NS;
          const int rows = min(tq, t1 - t) * p.G;
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {                  // ahead of the wait: the loads take their time
            const int c = lane + 32 * j;
            v[j] = INFINITY;                             // a column that is no row: weight 0
            if (c < rows)
              v[j] = p.lse[static_cast<int64_t>(m.q0 + t + c / p.G) * p.H + m.kvh * p.G + c % p.G] * 1.4426950408889634f;
          }
          ok = __all_sync(0xffffffffu, wait_or_abort(&q_empty[x], ((qn / NS) & 1) ^ 1, p.err, abort_flag));
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = lane + 32 * j, i = t + min(c, rows - 1) / p.G;
            s_lse[x * 128 + c] = -v[j];
            s_hi[x * 128 + c] = mask.hi(i);
            s_lo[x * 128 + c] = mask.lo(i);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[x]);
        }
      }
    }
    if (!ok) *abort_flag = 1;
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- exponentials and sums
    const int half = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t tS = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * 64;
    const float* s_lse = reinterpret_cast<const float*>(sm + L::lse);
    const int* s_hi = reinterpret_cast<const int*>(sm + L::hi);
    const int* s_lo = reinterpret_cast<const int*>(sm + L::lo);
    float* part = reinterpret_cast<float*>(sm + L::part);
    const float sl2 = p.scale * 1.4426950408889634f;
    const uint64_t scale2 = pair(sl2, sl2);
    for (int it = first; it < last; ++it) {
      const PagedMassItem m = p.items[it];
      const PagedMask mask{p.block, p.window, p.sinks, m.q_len, m.kv_len};
      for (int kb = m.kb0; kb < m.kb1; ++kb) {
        int t0, t1;
        mask.tokens(kb, &t0, &t1);
        if (t0 >= t1) continue;
        const PagedRange range = mask.range(t0, t1);
        const int k0 = kb * kPagedKB, key = k0 + r;
        float* dst = nullptr;                            // this key's weight, read while the tiles run
        float old = 0.f;
        if (half == 0 && range.has(key)) {
          const int page = paged_page(p.pool, m.seq, key >> p.pool.page_shift, p.err);
          dst = p.pool.mass + ((static_cast<int64_t>(page) * p.Hkv + m.kvh) << p.pool.page_shift) +
                (key & ((1 << p.pool.page_shift) - 1));
          old = *dst;
        }
        uint64_t sum = pair(0.f, 0.f);
        for (int t = t0; t < t1; t += tq, ++qn) {
          const uint32_t x = qn % NS, b = qn & 3;
          const int rows = min(tq, t1 - t) * p.G;
          // (a warp whose wait failed goes on: the halves meet at the block's end)
          ok = __all_sync(0xffffffffu, ok && wait_or_abort(&s_full[b], (qn >> 2) & 1, p.err, abort_flag) &&
                                           wait_or_abort(&q_full[x], (qn / NS) & 1, p.err, abort_flag));
          if (ok && half * 64 < rows) {
            tc_fence_after();
            const int tl = min(t + tq, t1) - 1;
            const bool edge = k0 + kPagedKB > mask.hi(t) || (k0 < mask.lo(tl) && k0 + kPagedKB > range.sinks);
#pragma unroll 1
            for (int c = half * 64; c < min(rows, half * 64 + 64); c += 32) {
              float v[32];
              tmem_ld32(tS + b * 128 + (c & 32), v);
              tmem_ld_wait();
              const float4* lse4 = reinterpret_cast<const float4*>(s_lse + x * 128 + c);
              if (c + 32 > rows) {                       // columns that are no rows may hold anything
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (c + j >= rows) v[j] = 0.f;         // (their -lse is -inf)
              }
              if (edge) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                  const int h = s_hi[x * 128 + c + j], l = s_lo[x * 128 + c + j];
                  if (!(key < h && (key >= l || key < range.sinks))) v[j] = -INFINITY;
                }
              }
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 e = lse4[j / 4];
                float a0, a1, a2, a3;
                unpair(fma2(pair(v[j], v[j + 1]), scale2, pair(e.x, e.y)), a0, a1);
                unpair(fma2(pair(v[j + 2], v[j + 3]), scale2, pair(e.z, e.w)), a2, a3);
                a0 = ex2(a0);
                a1 = ex2(a1);
                a2 = ex2(a2);
                a3 = ex2(a3);
                sum = add2(sum, add2(pair(a0, a1), pair(a2, a3)));
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&s_empty[b]);
            mbar_arrive(&q_empty[x]);
          }
        }
        float even, odd;
        unpair(sum, even, odd);
        // the halves' sums (two buffers: the next block's may come while this one is read)
        if (half == 1) part[(kn & 1) * 128 + r] = even + odd;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (dst != nullptr && ok) *dst = old + (even + odd + part[(kn & 1) * 128 + r]);
        ++kn;
      }
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
  cudaError_t e = cudaFuncSetAttribute(paged_mass_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       MassSmem<HD>::bytes);
  if (e != cudaSuccess) return e;
  paged_mass_kernel<HD><<<p.workers, kMassThreads, MassSmem<HD>::bytes, st>>>(tq, tk, p);
  return launched();
}

cudaError_t launch_paged_mass_tc(const PagedMassParams& p, cudaStream_t st) {
  if (p.workers == 0) return cudaSuccess;
  return p.hd == 128 ? mass_tc<128>(p, st) : mass_tc<64>(p, st);
}

}  // namespace sf

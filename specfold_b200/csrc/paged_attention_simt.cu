// Attention over the paged cache and its weight accumulation on the FP32 pipe: the fp32 path
// (the tensor core's tf32 products would round the inputs to 11 bits).
//
// One CTA walks the items of its share.  A tile of R = 16 * RM query rows (row = token * G + g)
// meets 64 keys at a time: S = Q K^T from shared memory with an RM x 4 register tile per
// thread, the running maximum and sum of the softmax per row, P back through shared memory, and
// O += P V with an RM x hd/16 register tile.  K and V share one buffer so that two CTAs fit an
// SM and one's loads run under the other's products.
//
// Products are taken two at a time (fma.rn.f32x2): half the issue slots for the same FMA rate.
// Scores add up even and odd dims apart; for P V each weight is stored twice, side by side.
//
// Measured (12 / 2 heads of 128, 704 tokens over 800 to 2100 keys, block-causal): 264 us, 23
// TFLOP/s of the 70 the FMA pipes could do; single products took 4% longer, and 2% go to the look at
// values that only some rows see.  The FMA pipes are 48% busy, the shared-memory pipe 62%: loads are
// waited for with two CTAs of 8 warps on an SM, and there is no room for a second buffer.
#include "paged_tc.cuh"

namespace sf {

constexpr int kSimtThreads = 256;
constexpr int kSimtKeys = kPagedKeysF32;

// keys [k0, k0 + 64) of a sequence into shared memory [64][HD + 4]; keys outside `range`, which
// no row of the tile sees, are zero: their slots may never have been written (0 * NaN is NaN),
// their pages may be gone
template <int HD>
__device__ __forceinline__ void simt_load_keys(float* dst, const void* pages, const PagedPool& pool,
                                               int seq, int kvh, int k0, PagedRange range, int* err) {
  constexpr int VPR = HD / 4;
  for (int i = threadIdx.x; i < kSimtKeys * VPR; i += kSimtThreads) {
    const int r = i / VPR, e = (i % VPR) * 4;
    const int key = k0 + r;
    float* d = dst + r * (HD + 4);
    if (range.has(key)) {
      const int page = paged_page(pool, seq, key >> pool.page_shift, err);
      const float* src = static_cast<const float*>(pages) + page * pool.page_stride + kvh * pool.head_stride +
                         (key & ((1 << pool.page_shift) - 1)) * pool.row_stride;
      *reinterpret_cast<float4*>(d + e) = *reinterpret_cast<const float4*>(src + e);
    } else {
      *reinterpret_cast<float4*>(d + e) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
}

// Takes values that are not finite out of the keys that not all rows see (not in [all_lo, all_hi), and
// no sink), each thread out of what it loaded; whether there were any.
template <int HD>
__device__ __forceinline__ bool simt_drop_odd(float* dst, int k0, int sinks, int all_lo, int all_hi) {
  constexpr int VPR = HD / 4;
  bool odd = false;
#pragma unroll 1
  for (int i = threadIdx.x; i < kSimtKeys * VPR; i += kSimtThreads) {
    const int r = i / VPR, key = k0 + r;
    if (key < all_hi && (key >= all_lo || key < sinks)) continue;
    float* x = dst + r * (HD + 4) + (i % VPR) * 4;
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (!(fabsf(x[y]) < INFINITY)) {
        x[y] = 0.f;
        odd = true;
      }
  }
  return odd;
}

template <int HD, int RM>
__device__ __forceinline__ void simt_load_q(float* sQ, const void* q, int64_t q_tok, int64_t q_head,
                                            int row0, int kvh, int G, int rows) {
  constexpr int VPR = HD / 4;
  for (int i = threadIdx.x; i < 16 * RM * VPR; i += kSimtThreads) {
    const int r = i / VPR, e = (i % VPR) * 4;
    float* d = sQ + r * (HD + 4);
    if (r < rows) {
      const float* src = static_cast<const float*>(q) + (row0 + r / G) * q_tok + (kvh * G + r % G) * q_head;
      *reinterpret_cast<float4*>(d + e) = *reinterpret_cast<const float4*>(src + e);
    } else {
      *reinterpret_cast<float4*>(d + e) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
}

// s[a][c] = q row (ty + 16 a) . key (tx + 16 c)
template <int HD, int RM>
__device__ __forceinline__ void simt_scores(const float* sQ, const float* sK, float (&s)[RM][4]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  uint64_t s2[RM][4];
#pragma unroll
  for (int a = 0; a < RM; ++a)
#pragma unroll
    for (int c = 0; c < 4; ++c) s2[a][c] = 0;
#pragma unroll 4
  for (int d = 0; d < HD; d += 4) {
    ulonglong2 kf[4], qf[RM];
#pragma unroll
    for (int c = 0; c < 4; ++c) kf[c] = *reinterpret_cast<const ulonglong2*>(sK + (tx + 16 * c) * (HD + 4) + d);
#pragma unroll
    for (int a = 0; a < RM; ++a) qf[a] = *reinterpret_cast<const ulonglong2*>(sQ + (ty + 16 * a) * (HD + 4) + d);
#pragma unroll
    for (int a = 0; a < RM; ++a)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s2[a][c] = fma2(qf[a].x, kf[c].x, s2[a][c]);
        s2[a][c] = fma2(qf[a].y, kf[c].y, s2[a][c]);
      }
  }
#pragma unroll
  for (int a = 0; a < RM; ++a)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float even, odd;
      unpair(s2[a][c], even, odd);
      s[a][c] = even + odd;
    }
}

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The values that were left out of an item decide their columns.  (A call: registers are short above.)
template <int HD>
__device__ __noinline__ void simt_put_odd(const PagedAttnParams& p, int item, int all_lo, int all_hi) {
  const PagedItem w = p.items[item];
  const int lane = threadIdx.x & 31;
  float sum[HD / 32];
  for (int tok = threadIdx.x >> 5; tok < w.ntok; tok += kSimtThreads / 32) {
    paged_odd_values<float, HD>(p, w, w.tok0 + tok, true, all_hi, all_lo, kSimtKeys, lane, ~0u, sum);
    for (int g = 0; g < p.G; ++g) {
      const int64_t row = static_cast<int64_t>(w.q0 + w.tok0 + tok) * p.H + w.kvh * p.G + g;
      paged_put_odd<float, HD>(sum, true, static_cast<float*>(p.out) + row * HD,
                               w.slot >= 0 ? p.part_O + (static_cast<int64_t>(w.slot) * p.rows + tok * p.G + g) * HD : nullptr, lane);
    }
  }
}

template <int HD, int RM>
__global__ void __launch_bounds__(kSimtThreads, 2) paged_attention_simt_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int R = 16 * RM, LD = HD + 4, LP = 2 * kSimtKeys + 4;
  constexpr int DV = HD / 64;                           // float4 groups of O per thread
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;                                       // [R][LD]
  float* sKV = sQ + R * LD;                             // [64][LD]
  float* sP = sKV + kSimtKeys * LD;                     // [R][LP], every weight twice
  __shared__ int s_all[3];                              // all rows see keys [0], [1); values were left out
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float sl2 = p.scale * 1.4426950408889634f;
  const int last = p.first[blockIdx.x + 1];
  for (int it = p.first[blockIdx.x]; it < last; ++it) {
    const PagedItem w = p.items[it];
    const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
    const int rows = w.ntok * p.G;
    float m[RM], l[RM];
    uint64_t o[RM][DV][2];
    int hi[RM], lo[RM];
#pragma unroll
    for (int a = 0; a < RM; ++a) {
      m[a] = -INFINITY;
      l[a] = 0.f;
#pragma unroll
      for (int d = 0; d < DV; ++d) o[a][d][0] = o[a][d][1] = 0;
      const int r = ty + 16 * a;
      const int i = w.tok0 + r / p.G;
      hi[a] = r < rows ? mask.hi(i) : 0;
      lo[a] = r < rows ? mask.lo(i) : 0;
    }
    const PagedRange range = mask.range(w.tok0, w.tok0 + w.ntok);
    __syncthreads();                                    // the previous item's reads are done
    if (threadIdx.x == 0) {
      s_all[0] = mask.lo(w.tok0 + w.ntok - 1);
      s_all[1] = mask.hi(w.tok0);
      s_all[2] = 0;
    }
    simt_load_q<HD, RM>(sQ, p.q, p.q_tok, p.q_head, w.q0 + w.tok0, w.kvh, p.G, rows);
    for (int i = w.i0; i < w.i1; ++i) {
      const int k0 = w.block(i) * kSimtKeys;
      __syncthreads();
      simt_load_keys<HD>(sKV, p.pool.k, p.pool, w.seq, w.kvh, k0, range, p.err);
      __syncthreads();
      float s[RM][4];
      simt_scores<HD, RM>(sQ, sKV, s);
#pragma unroll
      for (int a = 0; a < RM; ++a) {
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int j = k0 + tx + 16 * c;
          const bool see = j < hi[a] && (j >= lo[a] || j < p.sinks);
          s[a][c] = see ? s[a][c] * sl2 : -INFINITY;
          mx = fmaxf(mx, s[a][c]);
        }
        const float mn = fmaxf(m[a], half_warp_max(mx));
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2f(m[a] - ref);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float e = exp2f(s[a][c] - ref);
          sum += e;
          *reinterpret_cast<float2*>(sP + (ty + 16 * a) * LP + 2 * (tx + 16 * c)) = make_float2(e, e);
        }
        l[a] = l[a] * alpha + half_warp_sum(sum);
        m[a] = mn;
        const uint64_t alpha2 = pair(alpha, alpha);
#pragma unroll
        for (int d = 0; d < DV; ++d) {
          o[a][d][0] = fma2(o[a][d][0], alpha2, 0);
          o[a][d][1] = fma2(o[a][d][1], alpha2, 0);
        }
      }
      __syncthreads();                                  // K read, P written
      simt_load_keys<HD>(sKV, p.pool.v, p.pool, w.seq, w.kvh, k0, range, p.err);
      if ((k0 + kSimtKeys > s_all[1] || k0 < s_all[0]) && simt_drop_odd<HD>(sKV, k0, p.window > 0 ? p.sinks : 0, s_all[0], s_all[1]))
        s_all[2] = 1;
      __syncthreads();
      // a row of P is written and read by the same half-warp's 16 threads
#pragma unroll 4
      for (int j = 0; j < kSimtKeys; j += 2) {
        ulonglong2 pf[RM];
#pragma unroll
        for (int a = 0; a < RM; ++a) pf[a] = *reinterpret_cast<const ulonglong2*>(sP + (ty + 16 * a) * LP + 2 * j);
#pragma unroll
        for (int d = 0; d < DV; ++d) {
          const ulonglong2 v0 = *reinterpret_cast<const ulonglong2*>(sKV + j * LD + d * 64 + tx * 4);
          const ulonglong2 v1 = *reinterpret_cast<const ulonglong2*>(sKV + (j + 1) * LD + d * 64 + tx * 4);
#pragma unroll
          for (int a = 0; a < RM; ++a) {
            o[a][d][0] = fma2(pf[a].x, v0.x, o[a][d][0]);
            o[a][d][1] = fma2(pf[a].x, v0.y, o[a][d][1]);
            o[a][d][0] = fma2(pf[a].y, v1.x, o[a][d][0]);
            o[a][d][1] = fma2(pf[a].y, v1.y, o[a][d][1]);
          }
        }
      }
    }
#pragma unroll
    for (int a = 0; a < RM; ++a) {
      const int r = ty + 16 * a;
      if (r >= rows) continue;
      if (w.slot >= 0) {
        const int64_t pr = static_cast<int64_t>(w.slot) * p.rows + r;
#pragma unroll
        for (int d = 0; d < DV; ++d)
          *reinterpret_cast<ulonglong2*>(p.part_O + pr * HD + d * 64 + tx * 4) = make_ulonglong2(o[a][d][0], o[a][d][1]);
        if (tx == 0) {
          p.part_ml[2 * pr] = m[a];
          p.part_ml[2 * pr + 1] = l[a];
        }
      } else {
        const int64_t t = w.q0 + w.tok0 + r / p.G;
        const int h = w.kvh * p.G + r % p.G;
        const float inv = l[a] == 0.f ? 0.f : 1.f / l[a];   // a NaN sum stays one
        float* dst = static_cast<float*>(p.out) + (t * p.H + h) * HD;
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float e0, e1;
            unpair(o[a][d][x], e0, e1);
            dst[d * 64 + tx * 4 + 2 * x] = e0 * inv;
            dst[d * 64 + tx * 4 + 2 * x + 1] = e1 * inv;
          }
        if (tx == 0) p.lse[t * p.H + h] = m[a] * 0.6931471805599453f + logf(l[a]);
      }
    }
    __syncthreads();
    if (s_all[2]) simt_put_odd<HD>(p, it, s_all[0], s_all[1]);
  }
}

// Joins the pieces of the tiles that were cut: one warp per row, pieces in order.
template <typename T, int HD>
__global__ void __launch_bounds__(256) paged_merge_kernel(PagedAttnParams p) {
  const PagedMerge w = p.merges[blockIdx.y];
  pdl_wait();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= w.ntok * p.G) return;
  const int t = r / p.G, half = t / p.tile_tokens;
  const int pr = half * 128 + (t - half * p.tile_tokens) * p.G + r % p.G;
  paged_join_row<T, HD>(p, w, r, pr, lane);
}

cudaError_t launch_paged_merge(int dtype, const PagedAttnParams& p, cudaStream_t st) {
  if (p.n_merges == 0) return cudaSuccess;
  const dim3 grid((p.rows + 7) / 8, p.n_merges);
  // lines up behind the pieces' kernel (which lets it) and waits for its end on the device
  auto go = [&](auto* kernel) {
    const cudaError_t e = launch_attr(kernel, grid, dim3(256), 0, st, false, true, p);
    return e == cudaSuccess ? launched() : e;
  };
  if (dtype == BF16)
    return p.hd == 128 ? go(paged_merge_kernel<__nv_bfloat16, 128>) : go(paged_merge_kernel<__nv_bfloat16, 64>);
  return p.hd == 128 ? go(paged_merge_kernel<float, 128>) : go(paged_merge_kernel<float, 64>);
}

template <int HD, int RM>
static cudaError_t attention_simt(const PagedAttnParams& p, cudaStream_t st) {
  constexpr int R = 16 * RM;
  constexpr int smem = (R * (HD + 4) + kSimtKeys * (HD + 4) + R * (2 * kSimtKeys + 4)) * 4;
  cudaError_t e = allow_smem(paged_attention_simt_kernel<HD, RM>, smem);
  if (e != cudaSuccess) return e;
  paged_attention_simt_kernel<HD, RM><<<p.workers, kSimtThreads, smem, st>>>(p);
  return launched();
}

cudaError_t launch_paged_attention_simt(const PagedAttnParams& p, cudaStream_t st) {
  if (p.workers == 0) return cudaSuccess;
  const bool wide = p.rows == 64;
  if (p.hd == 128) return wide ? attention_simt<128, 4>(p, st) : attention_simt<128, 1>(p, st);
  return wide ? attention_simt<64, 4>(p, st) : attention_simt<64, 1>(p, st);
}

// ------------------------------------------------------------------ weight accumulation
// A key's accumulated weight; a page outside the pool is flagged, and nothing is written.  Atomic:
// sequences that share the page add to it at the same time.
__device__ __forceinline__ void add_mass(const PagedMassParams& p, int seq, int kvh, int key, float sum) {
  const int page = p.pool.table[seq * p.pool.table_stride + (key >> p.pool.page_shift)];
  if (page < 0 || page >= p.pool.num_pages) {
    flag_error(p.err, SF_DEV_ERR_INDEX);
    return;
  }
  atomicAdd(&p.pool.mass[((static_cast<int64_t>(page) * p.Hkv + kvh) << p.pool.page_shift) +
                         (key & ((1 << p.pool.page_shift) - 1))], sum);
}

// A key's weight over all rows that see it: sum of exp(s - lse).  A CTA owns a key block and
// walks the query rows, so each weight is summed in one place, in one order, and added once.
template <int HD, int RM>
__global__ void __launch_bounds__(kSimtThreads, 2) paged_mass_simt_kernel(PagedMassParams p) {
  constexpr int R = 16 * RM, LD = HD + 4;
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;                                       // [R][LD]
  float* sK = sQ + R * LD;                              // [64][LD]
  float* sR = sK + kSimtKeys * LD;                      // [16][64]
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float sl2 = p.scale * 1.4426950408889634f;
  const int last = p.first[blockIdx.x + 1];
  const int tile = R / p.G;
  for (int it = p.first[blockIdx.x]; it < last; ++it) {
    const PagedMassItem w = p.items[it];
    const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
    for (int kb = w.kb0; kb < w.kb0 + kMassBlocks && kb * kPagedKB < w.kv_len; ++kb) {
      const PagedRange range = mask.block_range(kb);
      for (int sub = 0; sub < kPagedKB / kSimtKeys; ++sub) {
        const int k0 = kb * kPagedKB + sub * kSimtKeys;
        if (k0 >= range.hi) break;
        __syncthreads();
        simt_load_keys<HD>(sK, p.pool.k, p.pool, w.seq, w.kvh, k0, range, p.err);
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int x = w.i0; x < w.i1; ++x) {
          const int t = w.t0 + x * tile;
          const int rows = min(tile, w.t1 - t) * p.G;
          __syncthreads();
          simt_load_q<HD, RM>(sQ, p.q, p.q_tok, p.q_head, w.q0 + t, w.kvh, p.G, rows);
          __syncthreads();
          float s[RM][4];
          simt_scores<HD, RM>(sQ, sK, s);
#pragma unroll
          for (int a = 0; a < RM; ++a) {
            const int r = ty + 16 * a;
            if (r >= rows) continue;
            const int i = t + r / p.G;
            const float lse = p.lse[static_cast<int64_t>(w.q0 + i) * p.H + w.kvh * p.G + r % p.G] * 1.4426950408889634f;
            if (lse == -INFINITY) continue;               // a row that saw nothing gives nothing
            const int hi = mask.hi(i), lo = mask.lo(i);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int j = k0 + tx + 16 * c;
              if (j < hi && (j >= lo || j < p.sinks)) acc[c] += exp2f(fmaf(s[a][c], sl2, -lse));
            }
          }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) sR[ty * kSimtKeys + tx + 16 * c] = acc[c];
        __syncthreads();
        if (threadIdx.x < kSimtKeys && range.has(k0 + threadIdx.x)) {
          float sum = 0.f;
          for (int y = 0; y < 16; ++y) sum += sR[y * kSimtKeys + threadIdx.x];
          const int j = k0 + threadIdx.x;
          if (w.slot >= 0)
            p.part[static_cast<int64_t>(w.slot) * kMassBlocks * kPagedKB + j - w.kb0 * kPagedKB] = sum;
          else
            add_mass(p, w.seq, w.kvh, j, sum);
        }
      }
    }
  }
}

// Adds the pieces of the pairs of key blocks that were cut, in order.
__global__ void __launch_bounds__(kMassBlocks * kPagedKB) paged_mass_merge_kernel(PagedMassParams p) {
  const PagedMassMerge w = p.merges[blockIdx.x];
  const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
  const int key = w.kb0 * kPagedKB + threadIdx.x;
  if (key >= w.kv_len) return;
  int f, l;
  mask.key_tokens(key, &f, &l);
  if (f >= l) return;                                   // no token sees it
  float sum = 0.f;
  for (int i = 0; i < w.n; ++i) sum += p.part[static_cast<int64_t>(w.slot0 + i) * kMassBlocks * kPagedKB + threadIdx.x];
  add_mass(p, w.seq, w.kvh, key, sum);
}

cudaError_t launch_paged_mass_merge(const PagedMassParams& p, cudaStream_t st) {
  if (p.n_merges == 0) return cudaSuccess;
  paged_mass_merge_kernel<<<p.n_merges, kMassBlocks * kPagedKB, 0, st>>>(p);
  return launched();
}

template <int HD, int RM>
static cudaError_t mass_simt(const PagedMassParams& p, cudaStream_t st) {
  constexpr int R = 16 * RM;
  constexpr int smem = (R * (HD + 4) + kSimtKeys * (HD + 4) + 16 * kSimtKeys) * 4;
  cudaError_t e = allow_smem(paged_mass_simt_kernel<HD, RM>, smem);
  if (e != cudaSuccess) return e;
  paged_mass_simt_kernel<HD, RM><<<p.workers, kSimtThreads, smem, st>>>(p);
  return launched();
}

cudaError_t launch_paged_mass_simt(const PagedMassParams& p, cudaStream_t st) {
  if (p.workers == 0) return cudaSuccess;
  return p.hd == 128 ? mass_simt<128, 4>(p, st) : mass_simt<64, 4>(p, st);
}

}  // namespace sf

// Paged prefix cache: the append of new rows and the eviction by accumulated weight.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace sf {

// element offset of a position's row in the pool
__device__ __forceinline__ int64_t pool_row(const PagedPool& p, int page, int kvh, int pos) {
  return page * p.page_stride + kvh * p.head_stride + (pos & ((1 << p.page_shift) - 1)) * p.row_stride;
}
__device__ __forceinline__ int64_t mass_at(const PagedPool& p, int page, int Hkv, int kvh, int pos) {
  return ((static_cast<int64_t>(page) * Hkv + kvh) << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
}

// ------------------------------------------------------------------ append
// One thread per 16-byte vector of a new row (key vectors, then value vectors): a row is read
// once, coalesced, from wherever the projection left it, while {sequence, position} and then the
// page are looked up, and written once.  (Several vectors a thread were slower: 36 to 43 us
// against 29 for 14000 rows of 8 heads.)  VPR: vectors of a row, a constant, so that the row is found
// with shifts: 20 us for those rows when they are in L2, 27 (4.4 TB/s) when they are not.
template <typename T, int VPR>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedAppendParams p) {
  constexpr int V = Elt<T>::kVec;
  const unsigned row = blockIdx.x * (256 / (2 * VPR)) + threadIdx.x / (2 * VPR);
  const unsigned t = row / p.Hkv, h = row % p.Hkv;
  if (t >= static_cast<unsigned>(p.T)) return;
  const int e = threadIdx.x % VPR * V;
  const bool value = threadIdx.x / VPR & 1;
  const int2 at = reinterpret_cast<const int2*>(p.tokens)[t];
  const T* src = static_cast<const T*>(value ? p.v_new : p.k_new) + t * p.new_tok + h * p.new_head + e;
  const uint4 d = __ldcs(reinterpret_cast<const uint4*>(src));
  const int id = p.pool.table[at.x * p.pool.table_stride + (at.y >> p.pool.page_shift)];
  if (id < 0 || id >= p.pool.num_pages) {               // nowhere to write: flagged, left out
    flag_error(p.err, SF_DEV_ERR_INDEX);
    return;
  }
  T* dst = static_cast<T*>(const_cast<void*>(value ? p.pool.v : p.pool.k)) + pool_row(p.pool, id, h, at.y) + e;
  *reinterpret_cast<uint4*>(dst) = d;
  if (!value && e == 0 && p.pool.mass != nullptr) p.pool.mass[mass_at(p.pool, id, p.Hkv, h, at.y)] = 0.f;
}

template <typename T, int VPR>
static cudaError_t append_rows(const PagedAppendParams& p, cudaStream_t st) {
  const int64_t threads = static_cast<int64_t>(p.T) * p.Hkv * 2 * VPR;   // T * Hkv < 2^31
  paged_append_kernel<T, VPR><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, st>>>(p);
  return launched();
}

cudaError_t launch_paged_append(int dtype, const PagedAppendParams& p, cudaStream_t st) {
  if (p.T == 0) return cudaSuccess;
  if (dtype == BF16) return p.hd == 128 ? append_rows<__nv_bfloat16, 16>(p, st) : append_rows<__nv_bfloat16, 8>(p, st);
  return p.hd == 128 ? append_rows<float, 32>(p, st) : append_rows<float, 16>(p, st);
}

// ------------------------------------------------------------------ eviction
// Which keys stay.  Of n cached keys the first `sinks` and the last `recent` stay; of the rest
// the m = keep - sinks - recent largest weights, equal ones by position.  A radix select over
// the weights' order-preserving bits (11, 11 and 10 of them) finds the m-th largest value and
// how many of its equals are taken; a count over the positions then places every survivor.
//
// Measured: 8200 keys of 4 heads of 24 sequences, 16 us; 32768 keys of 8 heads, 19 us (the weights
// are 3 and 1 MB: it is the latency of three passes, each a count, a cluster barrier and a scan).
// One CTA per head that read the weights again in every pass took 55 us for the longer.
//
// A cluster of 1 to 8 CTAs works on one (sequence, kv head), a contiguous range of positions
// each: the weights are read once and stay in registers (kSelKeys a thread; what is beyond is
// read again), every pass adds up the CTAs' histograms through distributed shared memory.
constexpr int kSelThreads = 1024;
constexpr int kSelKeys = 8;

// bits that order like the weights: zeros of either sign are equal, a NaN of either is above all
__device__ __forceinline__ uint32_t order_bits(float f) {
  if (isnan(f)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.f);           // -0 + 0 = 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// inclusive sum over the block
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    uint32_t w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  return v + (warp > 0 ? s_warp[warp - 1] : 0);
}

// {cached keys, keys that stay} of a sequence; what the host's bounds do not cover is flagged and
// cut to them (a budget too small for sinks + recent: everything up to it stays)
__device__ __forceinline__ void evict_lens(const PagedEvictParams& p, int b, int* n, int* keep) {
  const int a = p.lens[2 * b], k = p.lens[2 * b + 1];
  *n = min(max(a, 0), p.max_len);
  *keep = min(max(k, 0), p.max_keep);
  if (*n > *keep && *keep < p.sinks + p.recent) *n = *keep;
  if ((*n != a || *keep != k) && threadIdx.x == 0) flag_error(p.err, SF_DEV_ERR_INDEX);
}

__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(PagedEvictParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ uint32_t hist[2][2048];                     // of this pass and the next: two by turns
  __shared__ uint32_t s_warp[32];
  __shared__ uint32_t s_above[kSelKeys][32], s_equal[kSelKeys][32];
  __shared__ uint32_t s_total[2];                        // of this CTA: above, equal
  __shared__ uint32_t s_bin, s_before;
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int n, keep;
  evict_lens(p, b, &n, &keep);
  int32_t* out = p.kept + (static_cast<int64_t>(b) * p.Hkv + h) * p.kept_stride;
  const int tid = rank * kSelThreads + threadIdx.x, all = C * kSelThreads;
  pdl_trigger();                                         // the move may line up
  for (int i = min(n, keep) + tid; i < p.kept_stride; i += all) out[i] = -1;
  if (n <= keep) {                                       // (the whole cluster)
    for (int i = tid; i < n; i += all) out[i] = i;
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;            // the middle
  const int want = keep - p.sinks - p.recent;
  for (int i = tid; i < p.sinks; i += all) out[i] = i;
  for (int i = tid; i < p.recent; i += all) out[keep - p.recent + i] = hi + i;
  if (want == 0) return;
  // this CTA's positions [begin, end), kSelThreads side by side
  const int span = (hi - lo + C - 1) / C;
  const int begin = min(hi, lo + rank * span), end = min(hi, begin + span);
  const int turns = (span + kSelThreads - 1) / kSelThreads;
  auto read = [&](int i) {
    const int page = paged_page(p.pool, b, i >> p.pool.page_shift, p.err);
    return order_bits(p.pool.mass[mass_at(p.pool, page, p.Hkv, h, i)]);
  };
  uint32_t held[kSelKeys];
#pragma unroll
  for (int j = 0; j < kSelKeys; ++j) {
    const int i = begin + j * kSelThreads + threadIdx.x;
    held[j] = i < end ? read(i) : 0;
  }
  for (int i = threadIdx.x; i < 2 * 2048; i += kSelThreads) hist[0][i] = 0;
  __syncthreads();
  // the want-th largest: its bits from the top, `left` of the keys that share them still wanted
  uint32_t prefix = 0, mask = 0, left = want;
  const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    uint32_t* mine = hist[pass & 1];
    const uint32_t field = (1u << bits[pass]) - 1;
    // (counting equal bins of a warp together first was slower: 21 us for the selection, 16 without)
    auto count = [&](uint32_t k, bool live) {
      if (live && (k & mask) == prefix) atomicAdd(&mine[(k >> shifts[pass]) & field], 1u);
    };
#pragma unroll
    for (int j = 0; j < kSelKeys; ++j)
      if (j < turns) count(held[j], begin + j * kSelThreads + threadIdx.x < end);
    for (int j = kSelKeys; j < turns; ++j) {
      const int i = begin + j * kSelThreads + threadIdx.x;
      count(i < end ? read(i) : 0, i < end);
    }
    cluster.sync();                                      // every CTA's counts are there
    // thread t owns bins 2047 - 2t and 2046 - 2t: a scan from the largest bin down
    uint32_t c0 = 0, c1 = 0;
    for (int c = 0; c < C; ++c) {
      const uint2 x = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(mine, c) + 2046 - 2 * threadIdx.x);
      c0 += x.y;
      c1 += x.x;
    }
    const uint32_t before = block_scan(c0 + c1, s_warp) - c0 - c1;
    if (before < left && before + c0 >= left) {
      s_bin = 2047 - 2 * threadIdx.x;
      s_before = before;
    } else if (before + c0 < left && before + c0 + c1 >= left) {
      s_bin = 2046 - 2 * threadIdx.x;
      s_before = before + c0;
    }
    if (pass == 0) {                                     // the buffer of pass 2
      cluster.sync();                                    // (nobody reads it any more)
      for (int i = threadIdx.x; i < 2048; i += kSelThreads) mine[i] = 0;
    }
    __syncthreads();
    prefix |= s_bin << shifts[pass];
    mask |= field << shifts[pass];
    left -= s_before;
    __syncthreads();
  }
  // Positions in order: larger than the threshold, or one of the first `left` equal to it.  Counts
  // per warp and turn, their sums over what comes before, then each survivor's place.
  uint32_t above = 0, equal = 0;                         // in the turns before
#pragma unroll 1
  for (int j0 = 0; j0 < turns; j0 += kSelKeys) {
    const int m = min(kSelKeys, turns - j0);
    if (j0 > 0)
#pragma unroll
      for (int j = 0; j < kSelKeys; ++j) {
        const int i = begin + (j0 + j) * kSelThreads + threadIdx.x;
        held[j] = i < end ? read(i) : 0;
      }
    unsigned gt[kSelKeys], eq[kSelKeys];
#pragma unroll
    for (int j = 0; j < kSelKeys; ++j) {
      const bool live = begin + (j0 + j) * kSelThreads + static_cast<int>(threadIdx.x) < end;
      gt[j] = __ballot_sync(0xffffffffu, live && held[j] > prefix);
      eq[j] = __ballot_sync(0xffffffffu, live && held[j] == prefix);
      if (lane == 0) {
        s_above[j][warp] = __popc(gt[j]);
        s_equal[j][warp] = __popc(eq[j]);
      }
    }
    __syncthreads();
    if (warp == 0) {                                     // sums over (turn, warp) in order
      uint32_t run_a = above, run_e = equal;
      for (int j = 0; j < m; ++j) {
        const uint32_t a = s_above[j][lane], e = s_equal[j][lane];
        uint32_t ia = a, ie = e;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t ua = __shfl_up_sync(0xffffffffu, ia, o), ue = __shfl_up_sync(0xffffffffu, ie, o);
          if (lane >= o) {
            ia += ua;
            ie += ue;
          }
        }
        s_above[j][lane] = run_a + ia - a;
        s_equal[j][lane] = run_e + ie - e;
        run_a += __shfl_sync(0xffffffffu, ia, 31);
        run_e += __shfl_sync(0xffffffffu, ie, 31);
      }
      if (lane == 0) {
        s_total[0] = run_a;
        s_total[1] = run_e;
      }
    }
    __syncthreads();
    above = s_total[0];
    equal = s_total[1];
    // (the CTAs before this one: their totals are known once all have counted, which takes their
    // last turn; what exceeds the registers is counted first and placed in a second walk)
    if (turns > kSelKeys) continue;
    cluster.sync();
    uint32_t base_a = 0, base_e = 0;
    for (int c = 0; c < rank; ++c) {
      const uint32_t* t = cluster.map_shared_rank(s_total, c);
      base_a += t[0];
      base_e += t[1];
    }
#pragma unroll
    for (int j = 0; j < kSelKeys; ++j) {
      const unsigned below = (1u << lane) - 1;
      const uint32_t g = base_a + s_above[j][warp] + __popc(gt[j] & below);
      const uint32_t q = base_e + s_equal[j][warp] + __popc(eq[j] & below);
      if ((gt[j] >> lane & 1) || ((eq[j] >> lane & 1) && q < left))
        out[p.sinks + g + min(q, left)] = begin + j * kSelThreads + threadIdx.x;
    }
  }
  if (turns > kSelKeys) {
    cluster.sync();
    uint32_t base_a = 0, base_e = 0;
    for (int c = 0; c < rank; ++c) {
      const uint32_t* t = cluster.map_shared_rank(s_total, c);
      base_a += t[0];
      base_e += t[1];
    }
#pragma unroll 1
    for (int j = 0; j < turns; ++j) {
      const int i = begin + j * kSelThreads + threadIdx.x;
      const uint32_t k = i < end ? read(i) : 0;
      const bool g = i < end && k > prefix, e = i < end && k == prefix;
      const uint32_t ia = block_scan(g, s_warp);
      const uint32_t ta = s_warp[31];
      __syncthreads();
      const uint32_t ie = block_scan(e, s_warp);
      const uint32_t te = s_warp[31];
      __syncthreads();
      const uint32_t q = base_e + ie - e;
      if (g || (e && q < left)) out[p.sinks + base_a + ia - g + min(q, left)] = i;
      base_a += ta;
      base_e += te;
    }
  }
  cluster.sync();                                        // shared memory is read until here
}

// The survivors' rows to their new pages.  A CTA takes kMoveKeys of one (sequence, kv head): first
// a thread per key finds both rows (survivor, page, destination page: three loads one after the
// other, paid once for 32 KB of bf16) and moves its weight, then all threads copy 16-byte vectors, a
// key's key and value rows side by side, kMoveVecs of them in flight.  Measured: 2048 keys of 4 heads
// of 24 sequences, 198 MB read and written, in 35 us (5.6 TB/s).
constexpr int kMoveKeys = 64;
constexpr int kMoveVecs = 4;

template <typename T, int vpr>                          // vectors of a row
__global__ void __launch_bounds__(256) paged_move_kernel(PagedEvictParams p) {
  constexpr int V = Elt<T>::kVec;
  constexpr int vpk = 2 * vpr;                          // vectors of a key
  __shared__ int64_t s_src[kMoveKeys], s_dst[kMoveKeys];
  const int bh = blockIdx.y, b = bh / p.Hkv, h = bh % p.Hkv;
  int n, keep;
  evict_lens(p, b, &n, &keep);
  const int stay = min(n, keep);
  const int base = blockIdx.x * kMoveKeys, keys = min(kMoveKeys, stay - base);
  if (keys <= 0) return;
  pdl_wait();
  if (static_cast<int>(threadIdx.x) < keys) {
    const int i = base + threadIdx.x, pos = p.kept[static_cast<int64_t>(bh) * p.kept_stride + i];
    const int page = paged_page(p.pool, b, pos >> p.pool.page_shift, p.err);
    const int id = p.dst[b * p.dst_stride + (i >> p.pool.page_shift)];
    s_src[threadIdx.x] = pool_row(p.pool, page, h, pos);
    if (id < 0 || id >= p.pool.num_pages) {             // flagged, left out
      flag_error(p.err, SF_DEV_ERR_INDEX);
      s_dst[threadIdx.x] = -1;
    } else {
      s_dst[threadIdx.x] = pool_row(p.pool, id, h, i);
      p.pool.mass[mass_at(p.pool, id, p.Hkv, h, i)] = p.pool.mass[mass_at(p.pool, page, p.Hkv, h, pos)];
    }
  }
  __syncthreads();
  T* const k = static_cast<T*>(const_cast<void*>(p.pool.k));
  T* const v = static_cast<T*>(const_cast<void*>(p.pool.v));
  for (int x0 = threadIdx.x; x0 < keys * vpk; x0 += 256 * kMoveVecs) {
    uint4 d[kMoveVecs];
#pragma unroll
    for (int y = 0; y < kMoveVecs; ++y) {
      const int x = x0 + y * 256;
      if (x < keys * vpk) d[y] = __ldcs(reinterpret_cast<const uint4*>(((x / vpr) & 1 ? v : k) + s_src[x / vpk] + x % vpr * V));
    }
#pragma unroll
    for (int y = 0; y < kMoveVecs; ++y) {
      const int x = x0 + y * 256;
      if (x < keys * vpk && s_dst[x / vpk] >= 0)
        *reinterpret_cast<uint4*>(((x / vpr) & 1 ? v : k) + s_dst[x / vpk] + x % vpr * V) = d[y];
    }
  }
}

cudaError_t launch_paged_evict(int dtype, const PagedEvictParams& p, cudaStream_t st) {
  if (p.B == 0) return cudaSuccess;
  // CTAs of a cluster: at most 2 keys a thread, as long as all clusters run side by side (a CTA
  // fills an SM: for 96 heads of 8200 keys the selection took 4 us more with two CTAs each than with one)
  const int stay = p.max_len < p.max_keep ? p.max_len : p.max_keep;
  int C = 1;
  while (C < 8 && p.max_len > C * 2 * kSelThreads && 2 * C * p.B * p.Hkv <= p.sms) C *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(C, p.Hkv, p.B);
  cfg.blockDim = dim3(kSelThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, paged_select_kernel, p);
  if (e == cudaSuccess) e = launched();
  if (e != cudaSuccess || stay == 0) return e;
  const dim3 grid((stay + kMoveKeys - 1) / kMoveKeys, p.B * p.Hkv);
  auto move = [&](auto* kernel) { return launch_attr(kernel, grid, dim3(256), 0, st, false, true, p); };
  if (dtype == BF16) e = p.hd == 128 ? move(paged_move_kernel<__nv_bfloat16, 16>) : move(paged_move_kernel<__nv_bfloat16, 8>);
  else e = p.hd == 128 ? move(paged_move_kernel<float, 32>) : move(paged_move_kernel<float, 16>);
  return e == cudaSuccess ? launched() : e;
}

}  // namespace sf

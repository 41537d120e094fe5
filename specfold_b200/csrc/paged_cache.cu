// Paged prefix cache: the append of new rows and the eviction by accumulated weight.
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
// once, coalesced, from wherever the projection left it and written once.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedAppendParams p) {
  constexpr int V = Elt<T>::kVec;
  const int vpr = p.hd / V;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t rows = static_cast<int64_t>(p.T) * p.Hkv;
  const int e = static_cast<int>(i % vpr) * V;
  const bool value = (i / vpr) & 1;
  const int64_t row = i / (2 * vpr);
  if (row >= rows) return;
  const int t = static_cast<int>(row / p.Hkv), h = static_cast<int>(row % p.Hkv);
  const int2 at = reinterpret_cast<const int2*>(p.tokens)[t];
  const int id = p.pool.table[at.x * p.pool.table_stride + (at.y >> p.pool.page_shift)];
  if (id < 0 || id >= p.pool.num_pages) {               // nowhere to write: flagged, left out
    flag_error(p.err, SF_DEV_ERR_INDEX);
    return;
  }
  const T* src = static_cast<const T*>(value ? p.v_new : p.k_new) + t * p.new_tok + h * p.new_head + e;
  T* dst = static_cast<T*>(const_cast<void*>(value ? p.pool.v : p.pool.k)) + pool_row(p.pool, id, h, at.y) + e;
  *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  if (!value && e == 0 && p.pool.mass != nullptr)
    p.pool.mass[mass_at(p.pool, id, p.Hkv, h, at.y)] = 0.f;
}

cudaError_t launch_paged_append(int dtype, const PagedAppendParams& p, cudaStream_t st) {
  if (p.T == 0) return cudaSuccess;
  const int vpr = p.hd / (dtype == BF16 ? 8 : 4);
  const int64_t n = static_cast<int64_t>(p.T) * p.Hkv * 2 * vpr;
  const int64_t blocks = (n + 255) / 256;
  if (dtype == BF16)
    paged_append_kernel<__nv_bfloat16><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p);
  else
    paged_append_kernel<float><<<static_cast<unsigned>(blocks), 256, 0, st>>>(p);
  return launched();
}

// ------------------------------------------------------------------ eviction
// Which keys stay.  Of n cached keys the first `sinks` and the last `recent` stay; of the rest
// the m = keep - sinks - recent largest weights, equal ones by position.  A radix select over
// the weights' order-preserving bits (11, 11 and 10 of them) finds the m-th largest value and
// how many of its equals are taken; one scan over the positions then writes the list in order.
// One CTA per (sequence, kv head).
constexpr int kSelThreads = 1024;

__device__ __forceinline__ uint32_t order_bits(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// inclusive sum over the block of a 64-bit pair of counts
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    uint64_t w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  return v + (warp > 0 ? s_warp[warp - 1] : 0);
}

__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(PagedEvictParams p) {
  __shared__ uint32_t hist[2048];
  __shared__ uint64_t s_warp[32];
  __shared__ uint32_t s_bin, s_above;
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = p.lens[2 * b], keep = p.lens[2 * b + 1];
  int32_t* out = p.kept + (static_cast<int64_t>(b) * p.Hkv + h) * p.kept_stride;
  for (int i = min(n, keep) + threadIdx.x; i < p.kept_stride; i += kSelThreads) out[i] = -1;
  if (n <= keep) {
    for (int i = threadIdx.x; i < n; i += kSelThreads) out[i] = i;
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;            // the middle
  const int want = keep - p.sinks - p.recent;
  auto key_of = [&](int pos) {
    const int page = paged_page(p.pool, b, pos >> p.pool.page_shift, p.err);
    return order_bits(p.pool.mass[mass_at(p.pool, page, p.Hkv, h, pos)]);
  };
  // the want-th largest: its bits from the top, `left` of the keys that share them still wanted
  uint32_t prefix = 0, mask = 0;
  int left = want;
  const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = threadIdx.x; i < 2048; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t field = (1u << bits[pass]) - 1;
      for (int i = lo + threadIdx.x; i < hi; i += kSelThreads) {
        const uint32_t k = key_of(i);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shifts[pass]) & field], 1u);
      }
      __syncthreads();
      // thread t owns bins 2047 - 2t and 2046 - 2t: a scan from the largest bin down
      const uint32_t c0 = hist[2047 - 2 * threadIdx.x], c1 = hist[2046 - 2 * threadIdx.x];
      const uint64_t inc = block_scan(c0 + c1, s_warp);
      const uint32_t before = static_cast<uint32_t>(inc) - c0 - c1;
      const uint32_t l = static_cast<uint32_t>(left);
      if (before < l && before + c0 >= l) {
        s_bin = 2047 - 2 * threadIdx.x;
        s_above = before;
      } else if (before + c0 < l && before + c0 + c1 >= l) {
        s_bin = 2046 - 2 * threadIdx.x;
        s_above = before + c0;
      }
      __syncthreads();
      prefix |= s_bin << shifts[pass];
      mask |= field << shifts[pass];
      left -= static_cast<int>(s_above);
      __syncthreads();
    }
  }
  for (int i = threadIdx.x; i < p.sinks; i += kSelThreads) out[i] = i;
  for (int i = threadIdx.x; i < p.recent; i += kSelThreads) out[keep - p.recent + i] = hi + i;
  if (want == 0) return;
  // positions in order: larger than the threshold, or one of the first `left` equal to it
  uint32_t above = 0, equal = 0;
  for (int i0 = lo; i0 < hi; i0 += kSelThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t k = i < hi ? key_of(i) : 0;
    const bool gt = i < hi && k > prefix, eq = i < hi && k == prefix;
    const uint64_t inc = block_scan((static_cast<uint64_t>(gt) << 32) | eq, s_warp);
    const uint32_t g = above + static_cast<uint32_t>(inc >> 32) - gt;
    const uint32_t q = equal + static_cast<uint32_t>(inc) - eq;
    if (gt || (eq && q < static_cast<uint32_t>(left)))
      out[p.sinks + g + min(q, static_cast<uint32_t>(left))] = i;
    const uint64_t all = s_warp[31];
    above += static_cast<uint32_t>(all >> 32);
    equal += static_cast<uint32_t>(all);
    __syncthreads();
  }
}

// The survivors' rows to their new pages: a thread per 16-byte vector, kCopyRows keys in
// flight each (key and value vectors of one key side by side, so a warp moves whole rows).
constexpr int kCopyRows = 4;

template <typename T>
__global__ void __launch_bounds__(256) paged_move_kernel(PagedEvictParams p) {
  constexpr int V = Elt<T>::kVec;
  const int vpr = p.hd / V, per = 256 / (2 * vpr);      // keys side by side in the CTA
  const int bh = blockIdx.y, b = bh / p.Hkv, h = bh % p.Hkv;
  const int stay = min(p.lens[2 * b], p.lens[2 * b + 1]);
  const int x = threadIdx.x % (2 * vpr), k0 = threadIdx.x / (2 * vpr);
  const bool value = x >= vpr;
  const int e = (x % vpr) * V;
  const int32_t* kept = p.kept + static_cast<int64_t>(bh) * p.kept_stride;
  const int base = blockIdx.x * per * kCopyRows + k0;
  if (base >= stay) return;
  T* pages = static_cast<T*>(const_cast<void*>(value ? p.pool.v : p.pool.k));
  uint4 d[kCopyRows];
  float a[kCopyRows];
#pragma unroll
  for (int r = 0; r < kCopyRows; ++r) {
    const int i = base + r * per;
    if (i >= stay) continue;
    const int pos = kept[i];
    const int page = paged_page(p.pool, b, pos >> p.pool.page_shift, p.err);
    d[r] = *reinterpret_cast<const uint4*>(pages + pool_row(p.pool, page, h, pos) + e);
    if (x == 0) a[r] = p.pool.mass[mass_at(p.pool, page, p.Hkv, h, pos)];
  }
#pragma unroll
  for (int r = 0; r < kCopyRows; ++r) {
    const int i = base + r * per;
    if (i >= stay) continue;
    const int id = p.dst[b * p.dst_stride + (i >> p.pool.page_shift)];
    if (id < 0 || id >= p.pool.num_pages) {
      flag_error(p.err, SF_DEV_ERR_INDEX);
      continue;
    }
    *reinterpret_cast<uint4*>(pages + pool_row(p.pool, id, h, i) + e) = d[r];
    if (x == 0) p.pool.mass[mass_at(p.pool, id, p.Hkv, h, i)] = a[r];
  }
}

cudaError_t launch_paged_evict(int dtype, const PagedEvictParams& p, cudaStream_t st) {
  if (p.B == 0) return cudaSuccess;
  paged_select_kernel<<<dim3(p.Hkv, p.B), kSelThreads, 0, st>>>(p);
  cudaError_t e = launched();
  if (e != cudaSuccess) return e;
  const int stay = p.max_len < p.max_keep ? p.max_len : p.max_keep;
  if (stay == 0) return cudaSuccess;
  const int per = 256 / (2 * (p.hd / (dtype == BF16 ? 8 : 4))) * kCopyRows;
  const dim3 grid((stay + per - 1) / per, p.B * p.Hkv);
  if (dtype == BF16)
    paged_move_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  else
    paged_move_kernel<float><<<grid, 256, 0, st>>>(p);
  return launched();
}

}  // namespace sf

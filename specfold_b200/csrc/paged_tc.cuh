// What the tensor-core kernels of the paged cache share: tensor maps of the pools and the
// queries, the load of a key block by pages, and the device side of a bounded unwind.
#pragma once

#include <cudaTypedefs.h>

#include <mutex>

#include "paged.cuh"

namespace sf {

// TMA load of one box of a 3-D / 4-D tensor map (coordinates in elements of each dimension)
__device__ __forceinline__ void tma_load_3d(void* dst, const void* map, uint64_t* bar, int c0, int c1,
                                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, uint64_t* bar, int c0, int c1,
                                            int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// 32 lanes x 32 bits, 32 consecutive columns per thread
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// 8 consecutive columns per thread
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
// Waits for this thread's TMEM loads; the N values of v count as written here, so that no use of
// them can be scheduled before the wait.
template <int N>
__device__ __forceinline__ void tmem_wait(float* v) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < N; i += 8)
    asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]),
                 "+f"(v[i + 6]), "+f"(v[i + 7]));
}
__device__ __forceinline__ void fence_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
// 2^x by the hardware's approximation (2 units in the last place, below what any use here rounds
// to); -inf gives 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// fp32 pairs: one instruction for two
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t d, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// shared-memory matrix descriptors of sf_common.cuh, in the two words an issue loop steps
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t desc(uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(kDescHi));
  return d;
}

// Bounded wait that also ends when another role of the CTA gave up (sets *abort itself when the
// time is up).  A phase that is complete costs one try.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, int* err, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (true) {
    if (*abort) return false;
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (globaltimer() - t0 > kWaitNs) {
      flag_error(err, SF_DEV_ERR_TIMEOUT);
      *abort = 1;
      return false;
    }
  }
}

// Values that are not finite become 0; whether there were any.  (An exponent of ones is carried into
// the bit above it.)
__device__ __forceinline__ bool drop_odd(uint32_t& x) {
  const uint32_t t = ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  if (t != 0) x &= ~((t & 0x8000u ? 0xffffu : 0u) | (t & 0x80000000u ? 0xffff0000u : 0u));
  return t != 0;
}
__device__ __forceinline__ bool drop_odd(uint4& d) {
  return static_cast<int>(drop_odd(d.x)) | static_cast<int>(drop_odd(d.y)) | static_cast<int>(drop_odd(d.z)) |
         static_cast<int>(drop_odd(d.w));
}

constexpr int kPagedBox = 128 * 128;   // 128 rows of 64 bf16, 128-byte swizzled

// What a lane of the loading warp fetches of a key block: box lane / chunks (a page, or half of a
// large one), 64 columns lane % chunks.  Pages that no row of the tile sees are not read.
struct KeyPages {
  int page, row, at, rows;                               // page < 0: nothing; first row; place; rows of a box
  __device__ __forceinline__ KeyPages(const PagedPool& pool, const PagedItem& w, const PagedRange& range, int kb,
                                      int chunks, int lane, int* err) {
    const int ps = 1 << pool.page_shift;
    rows = ps < 128 ? ps : 128;
    const int x = lane / chunks, k0 = kb * kPagedKB + x * rows;
    at = x * rows;
    row = k0 & (ps - 1);
    page = -1;
    if (x < 128 / rows && range.meets(k0, k0 + rows)) page = paged_page(pool, w.seq, k0 >> pool.page_shift, err);
    at |= (lane % chunks) << 16;
  }
};
// One warp loads the 128 rows of a key block: [hd / 64][128 rows][64], 128-byte swizzle.  Completes
// on `bar` (one arrival with the bytes).
__device__ __forceinline__ void load_key_block(unsigned char* dst, const void* map, uint64_t* bar, const KeyPages& k,
                                               int kvh, int lane) {
  const bool mine = k.page >= 0;
  const unsigned n = __popc(__ballot_sync(0xffffffffu, mine));
  if (lane == 0) mbar_arrive_expect_tx(bar, n * k.rows * 128);
  __syncwarp();
  const int c = k.at >> 16, x = k.at & 0xffff;
  if (mine) tma_load_4d(dst + c * kPagedBox + x * 128, map, bar, c * 64, k.row, kvh, k.page);
}

// ------------------------------------------------------------------ host side
inline PFN_cuTensorMapEncodeTiled_v12000 paged_encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}
inline bool paged_tmap(CUtensorMap* m, const void* ptr, int rank, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box) {
  auto fn = paged_encode_fn();
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(ptr), dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// a pool [num_pages][Hkv][page_size][hd]: boxes of 64 columns and a page (at most 128 rows of it)
inline bool pool_tmap(CUtensorMap* m, const void* pages, const PagedPool& p, int Hkv, int hd) {
  const cuuint64_t ps = 1ull << p.page_shift;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(hd), ps, static_cast<cuuint64_t>(Hkv),
                              static_cast<cuuint64_t>(p.num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p.row_stride) * 2, static_cast<cuuint64_t>(p.head_stride) * 2,
                                 static_cast<cuuint64_t>(p.page_stride) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(ps < 128 ? ps : 128), 1, 1};
  return paged_tmap(m, pages, 4, dims, strides, box);
}
// query rows [T][H][hd]: boxes of 64 columns, the G heads of a group and `tokens` tokens, which
// land as rows token * G + g
inline bool query_tmap(CUtensorMap* m, const void* q, int64_t tok, int64_t head, int T, int H, int hd, int G,
                       int tokens) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(T)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head) * 2, static_cast<cuuint64_t>(tok) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(tokens)};
  return paged_tmap(m, q, 3, dims, strides, box);
}

}  // namespace sf

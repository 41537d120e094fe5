// Paged prefix cache: what its kernels, the plan builder and the C entries share.
//
// A pool of pages [num_pages][Hkv][page_size][hd] holds the keys (and another the values, a
// third the fp32 accumulated attention weight of every key) of many sequences; a table
// [B][width] of page ids maps a sequence's positions to pages.  A step runs the q_b new tokens
// of every sequence against its n_b cached ones (the new ones included).  Token i of a chunk
// sits at position p = n - q + i and sees key j when
//     j < hi(i)  and  (j > p - window  or  j < sinks)
//     hi(i) = min(n, n - q + (i / block + 1) * block), or n when block = 0
// (window = 0: no lower bound).  block = 1 is the causal mask, block = N the block-causal one.
//
// The lengths are known on the host, so the split of the work over the SMs is made there once
// per step, for all layers (paged_plan.cu): an item is a run of key blocks of one (sequence,
// kv head, tile of query rows), and every CTA gets a contiguous share of the items of equal
// cost.  A tile whose run was cut writes fp32 partials (O, m, l) that a merge joins in the
// order of the pieces, so results do not depend on timing.
#pragma once

#include <mutex>
#include <utility>
#include <vector>

#include "../../include/specfold_b200.h"
#include "sf_kernels.cuh"

namespace sf {

constexpr int kPagedKB = 128;         // keys of one block: the unit the plan counts in ...
constexpr int kPagedKeysF32 = 64;     // ... and that of the fp32 attention
constexpr int kPagedMaxGroup = 16;    // query heads per kv head

// A run [i0, i1) of the key blocks that a tile of query rows sees.  The blocks a tile sees
// are the sink blocks 0 .. sink_blks - 1, then lo_blk, lo_blk + 1, ...
struct alignas(16) PagedItem {
  int32_t seq, kvh, tok0, ntok;       // the tile: tokens [tok0, tok0 + ntok) of the chunk
  int32_t i0, i1, slot, sink_blks;    // slot < 0: writes the output itself
  int32_t lo_blk, q0, q_len, kv_len;  // q0: the chunk's first row in q / out
  __host__ __device__ int block(int i) const { return i < sink_blks ? i : i - sink_blks + lo_blk; }
};
// A tile whose run was cut into n pieces, in slots [slot0, slot0 + n)
struct alignas(16) PagedMerge {
  int32_t kvh, tok0, ntok, slot0;
  int32_t n, q0, pad0, pad1;
};
// Weight accumulation: two key blocks of one (sequence, kv head) against tiles [i0, i1) of the
// tokens from t0 on (t0: the first that sees either block, t1: behind the last)
constexpr int kMassBlocks = 2;
struct alignas(16) PagedMassItem {
  int32_t seq, kvh, kb0, t0;
  int32_t t1, i0, i1, slot;           // slot < 0: adds to the weights itself
  int32_t q0, q_len, kv_len, pad;
};
struct alignas(16) PagedMassMerge {
  int32_t seq, kvh, kb0, slot0;
  int32_t n, q_len, kv_len, pad;
};

// The keys that some token of a range sees: [lo, hi) and [0, sinks)
struct PagedRange {
  int lo, hi, sinks;
  __host__ __device__ bool has(int key) const { return key < hi && (key >= lo || key < sinks); }
  // any key of [a, b)
  __host__ __device__ bool meets(int a, int b) const { return a < hi && (b > lo || a < sinks); }
};

struct PagedMask {
  int block, window, sinks, q_len, kv_len;
  __host__ __device__ int pos(int i) const { return kv_len - q_len + i; }
  // keys [0, hi) at most
  __host__ __device__ int hi(int i) const {
    if (block == 0) return kv_len;
    const int64_t h = static_cast<int64_t>(kv_len) - q_len + (static_cast<int64_t>(i / block) + 1) * block;
    return h < kv_len ? static_cast<int>(h) : kv_len;
  }
  // keys [lo, hi) and [0, sinks)
  __host__ __device__ int lo(int i) const {
    if (window == 0) return 0;
    const int l = pos(i) - window + 1;
    return l > 0 ? l : 0;
  }
  // the tokens that see one key, 0 <= key < kv_len: [first, last), empty when last <= first
  __host__ __device__ void key_tokens(int key, int* first, int* last) const {
    const int64_t off = static_cast<int64_t>(key) - (kv_len - q_len);   // its place in the chunk
    int f = 0, l = q_len;
    if (block > 0 && off >= 0) f = static_cast<int>(off / block * block);
    if (window > 0 && key >= sinks && off + window < l) l = off + window > 0 ? static_cast<int>(off + window) : 0;
    *first = f;
    *last = l;
  }
  // keys that some token sees in block kb
  __host__ __device__ PagedRange block_range(int kb) const {
    int f, l;
    tokens(kb, &f, &l);
    return f < l ? range(f, l) : PagedRange{0, 0, 0};
  }
  // the tokens that see a key of any block of a pair
  __host__ __device__ void pair_tokens(int kb0, int* first, int* last) const {
    *first = q_len;
    *last = 0;
    for (int kb = kb0; kb < kb0 + kMassBlocks && kb * kPagedKB < kv_len; ++kb) {
      int f, l;
      tokens(kb, &f, &l);
      if (f >= l) continue;
      if (f < *first) *first = f;
      if (l > *last) *last = l;
    }
  }
  __host__ __device__ PagedRange range(int t0, int t1) const { return {lo(t0), hi(t1 - 1), window > 0 ? sinks : 0}; }
  // the tokens of the chunk that see any key of block kb: [first, last)
  __host__ __device__ void tokens(int kb, int* first, int* last) const {
    const int k0 = kb * kPagedKB;
    const int k1 = k0 + kPagedKB < kv_len ? k0 + kPagedKB : kv_len;   // exclusive
    int f = 0, l = q_len;
    if (block > 0) {
      // hi(i) > k0  <=>  i / block + 1 > (k0 - base) / block
      const int base = kv_len - q_len;
      if (k0 >= base) f = (k0 - base) / block * block;
    }
    if (window > 0 && k0 >= sinks) {
      // lo(i) < k1  <=>  i < k1 + window - 1 - base
      const int64_t e = static_cast<int64_t>(k1) + window - 1 - (kv_len - q_len);
      if (e < l) l = e > 0 ? static_cast<int>(e) : 0;
    }
    *first = f < q_len ? f : q_len;
    *last = l > *first ? l : *first;
  }
};

struct PagedPool {
  const void* k;
  const void* v;
  int64_t page_stride, head_stride, row_stride;   // elements, k and v alike
  float* mass;                                     // [num_pages][Hkv][page_size], contiguous
  int num_pages, page_shift;
  const int32_t* table;
  int64_t table_stride;
  int table_width;
};

struct PagedAttnParams {
  const void* q;
  int64_t q_tok, q_head;            // strides, elements
  PagedPool pool;
  void* out;                        // [T, H, hd] contiguous
  float* lse;                       // [T, H]
  const PagedItem* items;
  const PagedItem* heads;           // [workers] a copy of every CTA's first item
  const int32_t* first;             // [workers + 1] its index
  int workers;
  const PagedMerge* merges;
  int n_merges;
  float* part_O;                    // [slots][rows][hd]
  float* part_ml;                   // [slots][rows][2]
  int rows, tile_tokens;            // rows of a slot; tokens of 128 (64) rows
  int H, Hkv, G, hd, T;
  int block, window, sinks;
  float scale;
  int* err;
};

struct PagedMassParams {
  const void* q;
  int64_t q_tok, q_head;
  PagedPool pool;
  const float* lse;                 // [T, H]
  const PagedMassItem* items;
  const int32_t* first;
  int workers;
  const PagedMassMerge* merges;
  int n_merges;
  float* part;                      // [slots][2 * 128] sums of the pieces
  int H, Hkv, G, hd, T;
  int block, window, sinks;
  float scale;
  int* err;
};

// Raises a kernel's dynamic shared memory limit, once per kernel and device.
template <typename F>
inline cudaError_t allow_smem(F* kernel, int bytes) {
  static std::mutex mu;
  static std::vector<std::pair<const void*, uint64_t>> seen;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const void* key = reinterpret_cast<const void*>(kernel);
  std::lock_guard<std::mutex> lock(mu);
  for (auto& x : seen)
    if (x.first == key) {
      if (dev < 64 && (x.second >> dev & 1)) return cudaSuccess;
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e == cudaSuccess && dev < 64) x.second |= uint64_t{1} << dev;
      return e;
    }
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) seen.push_back({key, uint64_t{1} << dev});
  return e;
}

// page id of position pos; an id outside the pool is flagged and read as page 0
__device__ __forceinline__ int paged_page(const PagedPool& p, int seq, int idx, int* err) {
  const int id = p.table[seq * p.table_stride + idx];
  if (id < 0 || id >= p.num_pages) {
    flag_error(err, SF_DEV_ERR_INDEX);
    return 0;
  }
  return id;
}

// One warp joins the pieces of row r (row pr of the slots) of a cut tile, in their order.  Lane x
// fetches the state of piece x; the first pieces' values are on their way meanwhile.
template <typename T, int HD>
__device__ __forceinline__ void paged_join_row(const PagedAttnParams& p, const PagedMerge& w, int r, int pr, int lane) {
  constexpr int E = HD / 32, AHEAD = 8;
  const int64_t at0 = static_cast<int64_t>(w.slot0) * p.rows + pr;
  float2 v[AHEAD][E / 2];
  auto fetch = [&](int i, int j) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e)
      v[j][e] = i < w.n ? reinterpret_cast<const float2*>(p.part_O + (at0 + static_cast<int64_t>(i) * p.rows) * HD + lane * E)[e]
                        : make_float2(0.f, 0.f);
  };
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) fetch(j, j);
  float m = -INFINITY;
  for (int i = lane; i < w.n; i += 32) m = fmaxf(m, p.part_ml[2 * (at0 + static_cast<int64_t>(i) * p.rows)]);
  m = warp_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int i0 = 0; i0 < w.n; i0 += 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (i0 + lane < w.n) ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (at0 + static_cast<int64_t>(i0 + lane) * p.rows));
    const float f_lane = exp2f(ml.x - ref);
    const int n = min(32, w.n - i0);
    for (int j0 = 0; j0 < n; j0 += AHEAD) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float f = __shfl_sync(0xffffffffu, f_lane, (j0 + j) & 31), lj = __shfl_sync(0xffffffffu, ml.y, (j0 + j) & 31);
        if (j0 + j < n) {
          l = fmaf(lj, f, l);
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            o[2 * e] = fmaf(v[j][e].x, f, o[2 * e]);
            o[2 * e + 1] = fmaf(v[j][e].y, f, o[2 * e + 1]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) fetch(i0 + j0 + AHEAD + j, j);
    }
  }
  const int64_t row = static_cast<int64_t>(w.q0 + w.tok0 + r / p.G) * p.H + w.kvh * p.G + r % p.G;
  const float inv = l == 0.f ? 0.f : 1.f / l;           // a NaN sum stays one
  T* dst = static_cast<T*>(p.out) + row * HD + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = Elt<T>::from_f(o[e] * inv);
  if (lane == 0) p.lse[row] = m * 0.6931471805599453f + logf(l);
}

// Keys that only some rows of a tile see have weight 0 in the others, and 0 times an infinite or NaN
// value is NaN.  Such values are taken out of the tile in shared memory (only keys of that kind are
// looked at) and decide their columns here, at the output of the rows that see them: one warp adds up
// the values that are not finite of the keys that a token sees.  `some`: of those that not all rows of
// the item see (beyond hi_min, or before lo_max and no sink), else of all.  keys: of a block; need:
// which of the lane's columns are asked for.
template <typename T, int HD>
__device__ __forceinline__ void paged_odd_values(const PagedAttnParams& p, const PagedItem& w, int tok, bool some,
                                                 int hi_min, int lo_max, int keys, int lane, unsigned need,
                                                 float (&sum)[HD / 32]) {
  constexpr int E = HD / 32, AHEAD = 8;
  const PagedMask mask{p.block, p.window, p.sinks, w.q_len, w.kv_len};
  const int hi = mask.hi(tok), lo = mask.lo(tok), sinks = p.window > 0 ? p.sinks : 0;
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = 0.f;
#pragma unroll 1
  for (int i = w.i0; i < w.i1; ++i) {
    const int k0 = w.block(i) * keys;
    if (some && k0 + keys <= hi_min && (k0 >= lo_max || k0 + keys <= sinks)) continue;
#pragma unroll 1
    for (int j0 = k0; j0 < k0 + keys; j0 += AHEAD) {       // (in one page)
      bool take[AHEAD], any = false;
#pragma unroll
      for (int y = 0; y < AHEAD; ++y) {
        const int j = j0 + y;
        take[y] = j < hi && (j >= lo || j < sinks) && !(some && j < hi_min && (j >= lo_max || j < sinks));
        any |= take[y];
      }
      if (!any) continue;
      const T* row = static_cast<const T*>(p.pool.v) +
                     paged_page(p.pool, w.seq, j0 >> p.pool.page_shift, p.err) * p.pool.page_stride + w.kvh * p.pool.head_stride +
                     (j0 & ((1 << p.pool.page_shift) - 1)) * p.pool.row_stride + lane * E;
      float v[AHEAD][E];
#pragma unroll
      for (int y = 0; y < AHEAD; ++y)
#pragma unroll
        for (int e = 0; e < E; ++e) v[y][e] = take[y] ? Elt<T>::to_f(row[y * p.pool.row_stride + e]) : 0.f;
      bool open = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int y = 0; y < AHEAD; ++y)
          if (!(fabsf(v[y][e]) < INFINITY)) sum[e] += v[y][e];
        open |= (need >> e & 1) && !isnan(sum[e]);
      }
      if (!__any_sync(0xffffffffu, open)) return;          // (NaN stays NaN)
    }
  }
}
// ... into an output row (or its partial, where given): added, or in its place
template <typename T, int HD>
__device__ __forceinline__ void paged_put_odd(const float (&sum)[HD / 32], bool add, T* out, float* part, int lane) {
#pragma unroll
  for (int e = 0; e < HD / 32; ++e) {
    const int c = lane * (HD / 32) + e;
    if (sum[e] == 0.f) continue;
    if (part != nullptr) part[c] = add ? part[c] + sum[e] : sum[e];
    else out[c] = Elt<T>::from_f(add ? Elt<T>::to_f(out[c]) + sum[e] : sum[e]);
  }
}

cudaError_t launch_paged_attention_simt(const PagedAttnParams& p, cudaStream_t st);
cudaError_t launch_paged_attention_tokens(const PagedAttnParams& p, int copies, cudaStream_t st);
cudaError_t launch_paged_attention_chunk(const PagedAttnParams& p, cudaStream_t st);
cudaError_t launch_paged_merge(int dtype, const PagedAttnParams& p, cudaStream_t st);
cudaError_t launch_paged_mass_simt(const PagedMassParams& p, cudaStream_t st);
cudaError_t launch_paged_mass_tc(const PagedMassParams& p, cudaStream_t st);
cudaError_t launch_paged_mass_merge(const PagedMassParams& p, cudaStream_t st);

// {sequence, position} of every new token
struct PagedAppendParams {
  const void* k_new;
  const void* v_new;
  int64_t new_tok, new_head;
  PagedPool pool;
  const int32_t* tokens;            // [T][2]
  int T, Hkv, hd;
  int* err;
};
cudaError_t launch_paged_append(int dtype, const PagedAppendParams& p, cudaStream_t st);

struct PagedEvictParams {
  PagedPool pool;                   // table = the source table
  const int32_t* dst;               // destination table
  int64_t dst_stride;
  const int32_t* lens;              // [B][2]: cached keys, keys that stay
  int32_t* kept;                    // [B][Hkv][kept_stride]
  int kept_stride;
  int B, Hkv, hd, sinks, recent, max_len, max_keep, sms;
  int* err;
};
cudaError_t launch_paged_evict(int dtype, const PagedEvictParams& p, cudaStream_t st);

}  // namespace sf

// The paged cache's plan (how a step's work is split over the SMs) and its C entries.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <vector>

#include "paged.cuh"

using namespace sf;

namespace {

int bad(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return report(SF_ERR_ARG, buf);
}

constexpr int kItemWords = sizeof(PagedItem) / 4;
constexpr int kMergeWords = sizeof(PagedMerge) / 4;
constexpr int kMassWords = sizeof(PagedMassItem) / 4;
constexpr int kMassMergeWords = sizeof(PagedMassMerge) / 4;
constexpr int64_t kMaxWords = int64_t{1} << 30;

int64_t up4(int64_t x) { return (x + 3) & ~int64_t{3}; }

// Rows of a tile and of the two kernels' tiles.  bf16: one MMA tile of 128 rows (short chunks:
// single tokens, small blocks), two of them (long ones).  fp32: 16 and 64 rows.
struct Tiling {
  int rows[2], tokens[2], per_tile[2], workers[2], mass_workers, mass_rows;
  // A tile of at most `whole` key blocks is not cut where every tile can have a CTA: pieces need a
  // second launch for their join, which costs about what that many blocks take.  (One token over 7
  // blocks of 2 kv heads: 11.0 us on the device in 14 pieces, 18.2 in two, 2 us a block; the join's
  // launch takes the host 3 us.)
  int whole[2];
};
Tiling tiling(const sf_paged_plan& p) {
  const int G = p.H / p.Hkv;
  Tiling t{};
  if (p.dtype == SF_DTYPE_BF16) {
    t.rows[0] = 128;
    t.rows[1] = 256;
    t.tokens[0] = t.tokens[1] = 128 / G;
    t.per_tile[0] = t.tokens[0];
    t.per_tile[1] = 2 * t.tokens[1];
    t.workers[0] = t.workers[1] = p.sms;
    t.mass_workers = p.sms;
    t.mass_rows = 128;
    t.whole[0] = 4;
    t.whole[1] = 3;
    return t;
  }
  t.rows[0] = 16;
  t.rows[1] = 64;
  t.tokens[0] = 16 / G;
  t.tokens[1] = 64 / G;
  t.per_tile[0] = t.tokens[0];
  t.per_tile[1] = t.tokens[1];
  t.workers[0] = t.workers[1] = 2 * p.sms;
  t.mass_workers = 2 * p.sms;
  t.mass_rows = 64;
  t.whole[0] = 4;
  t.whole[1] = 2;
  return t;
}

int check_plan(const sf_paged_plan* p, const int32_t* q_lens, const int32_t* kv_lens) {
  if (!p || p->B < 0 || (p->B > 0 && (!q_lens || !kv_lens))) return bad("paged plan: null argument");
  if (p->dtype != SF_DTYPE_F32 && p->dtype != SF_DTYPE_BF16) return bad("paged plan: dtype %d not supported", p->dtype);
  if (p->hd != 64 && p->hd != 128) return bad("paged plan: head_dim %d must be 64 or 128", p->hd);
  if (p->H <= 0 || p->Hkv <= 0 || p->H % p->Hkv != 0 || p->H / p->Hkv > kPagedMaxGroup)
    return bad("paged plan: heads %d / kv heads %d unsupported", p->H, p->Hkv);
  if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return bad("paged plan: page size %d must be a power of two in [16, 256]", p->page_size);
  if (p->block < 0 || p->window < 0 || p->sinks < 0) return bad("paged plan: block, window and sinks must not be negative");
  if (p->window > (1 << 30)) return bad("paged plan: a window of %d is no limit: pass 0", p->window);
  int64_t T = 0;
  for (int b = 0; b < p->B; ++b) {
    if (q_lens[b] < 0 || kv_lens[b] < 0) return bad("paged plan: sequence %d has a negative length", b);
    if (kv_lens[b] > (1 << 30) || q_lens[b] > (1 << 30)) return bad("paged plan: sequence %d is too long", b);
    T += q_lens[b];
  }
  // rows of q and out are counted in 32 bits, as are a tensor map's coordinates
  if (T * p->H >= (int64_t{1} << 31)) return bad("paged plan: %lld query rows are too many", static_cast<long long>(T * p->H));
  return SF_OK;
}

int device_sms(int asked) {
  if (asked > 0) return asked;
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) == cudaSuccess &&
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0)
    return n;
  (void)cudaGetLastError();
  return 148;
}

int which(const Tiling& t, int q_len, int G) { return static_cast<int64_t>(q_len) * G <= t.rows[0] ? 0 : 1; }

// A share of something that is cut into units [0, units): the piece [i0, i1), and where its
// partial result goes (-1: it is whole)
struct Piece {
  int what, i0, i1, slot;
};
struct Cut {
  int what, slot0, n;
};

// Deals things out in order: each worker takes its share of their units (and `extra` per thing),
// and what does not fit goes on with the next one.
void deal(const std::vector<int>& units, int extra, int workers, int whole, std::vector<Piece>* pieces,
          std::vector<int32_t>* first, std::vector<Cut>* cuts, int* slots) {
  int64_t total = 0;
  int top = 0;
  for (int u : units) {
    total += u + extra;
    top = std::max(top, u);
  }
  *slots = 0;
  if (static_cast<int64_t>(units.size()) <= workers && top <= whole) {
    for (size_t x = 0; x < units.size(); ++x) {
      first->push_back(static_cast<int32_t>(x));
      pieces->push_back({static_cast<int>(x), 0, units[x], -1});
    }
    first->push_back(static_cast<int32_t>(units.size()));
    return;
  }
  const int64_t w = std::max<int64_t>(1, std::min<int64_t>(workers, total));
  first->push_back(0);
  int64_t done = 0, worker = 0;   // dealt out; this worker's share ends at (worker + 1) * total / w
  for (size_t x = 0; x < units.size(); ++x) {
    int at = 0, n = 0;
    const size_t from = pieces->size();
    do {
      // what is left of this worker's share; one too small to be worth a piece ends here
      int64_t room = (worker + 1) * total / w - done;
      while (room <= extra && worker + 1 < w) {
        first->push_back(static_cast<int32_t>(pieces->size()));
        ++worker;
        room = (worker + 1) * total / w - done;
      }
      const int need = units[x] - at;
      int take = need;
      if (worker + 1 < w && need + extra > room)
        take = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(need, room - extra)));
      pieces->push_back({static_cast<int>(x), at, at + take, -1});
      at += take;
      done += take + (n == 0 ? extra : 0);
      ++n;
    } while (at < units[x]);
    if (n > 1) {
      cuts->push_back({static_cast<int>(x), *slots, n});
      for (size_t i = from; i < pieces->size(); ++i) (*pieces)[i].slot = (*slots)++;
    }
  }
  while (static_cast<int64_t>(first->size()) <= w) first->push_back(static_cast<int32_t>(pieces->size()));
  first->back() = static_cast<int32_t>(pieces->size());
}

size_t list_ws(const sf_paged_list& l, int hd) {
  return (static_cast<size_t>(l.slots) * l.rows * (hd + 2) * 4 + 255) / 256 * 256;
}
size_t mass_ws(const sf_paged_list& l) { return static_cast<size_t>(l.slots) * kMassBlocks * kPagedKB * 4; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

PagedPool pool_of(const sf_paged_pool& s, int page_size) {
  PagedPool p{};
  p.k = s.k_pages;
  p.v = s.v_pages;
  p.mass = s.mass_pages;
  p.page_stride = s.page_stride;
  p.head_stride = s.head_stride;
  p.row_stride = s.row_stride;
  p.num_pages = s.num_pages;
  p.page_shift = __builtin_ctz(page_size);
  p.table = s.table;
  p.table_stride = s.table_stride;
  p.table_width = s.table_width;
  return p;
}

int check_pool(const char* who, const sf_paged_pool* s, int dtype, int hd, int page_size, int64_t max_kv,
               bool values, bool mass) {
  if (!s) return bad("%s: null pool", who);
  const int vec = dtype == SF_DTYPE_BF16 ? 8 : 4;
  if (static_cast<int64_t>(s->table_width) * page_size < max_kv || s->table_stride < s->table_width)
    return bad("%s: a table of %d pages does not hold %lld keys", who, s->table_width,
               static_cast<long long>(max_kv));
  if (!s->k_pages || (values && !s->v_pages) || (mass && !s->mass_pages) || (max_kv > 0 && !s->table) || s->num_pages < 1)
    return bad("%s: null pool pointer or empty pool", who);
  if (!aligned16(s->k_pages) || !aligned16(s->v_pages) || s->page_stride % vec || s->head_stride % vec ||
      s->row_stride % vec)
    return bad("%s: the pools need 16-byte aligned rows", who);
  if (s->row_stride < hd || s->head_stride < hd || s->page_stride < hd)
    return bad("%s: pool strides must be positive and at least head_dim", who);
  return SF_OK;
}

int check_ready(const char* who, const sf_paged_plan* p) {
  if (!p) return bad("%s: null plan", who);
  if (p->words <= 0 || (p->dtype != SF_DTYPE_F32 && p->dtype != SF_DTYPE_BF16) || (p->hd != 64 && p->hd != 128) ||
      p->page_size < 16)
    return bad("%s: the plan was not built", who);
  if (!p->dev || !p->err || (p->ws_bytes > 0 && !p->ws)) return bad("%s: the plan has no device memory", who);
  return SF_OK;
}

int check_rows(const char* who, const sf_paged_plan* p, const void* q, int64_t tok, int64_t head) {
  const int vec = p->dtype == SF_DTYPE_BF16 ? 8 : 4;
  if (!q || !aligned16(q) || tok % vec || head % vec || tok < 0 || head < p->hd)
    return bad("%s: rows must be 16-byte aligned, head stride at least head_dim", who);
  return SF_OK;
}

int status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return SF_OK;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
  return report(SF_ERR_CUDA, buf);
}

}  // namespace

extern "C" {

int64_t sf_paged_plan_words(const sf_paged_plan* plan, const int32_t* q_lens, const int32_t* kv_lens) {
  if (check_plan(plan, q_lens, kv_lens) != SF_OK) return 0;
  sf_paged_plan p = *plan;
  p.sms = device_sms(p.sms);
  const Tiling t = tiling(p);
  int64_t items = 0, mass = 0, tokens = 0;
  for (int b = 0; b < p.B; ++b) {
    const int k = which(t, q_lens[b], p.H / p.Hkv);
    items += static_cast<int64_t>((q_lens[b] + t.per_tile[k] - 1) / t.per_tile[k]) * p.Hkv;
    if (q_lens[b] > 0) mass += static_cast<int64_t>(kv_lens[b] / (kMassBlocks * kPagedKB) + 1) * p.Hkv;
    tokens += q_lens[b];
  }
  const int64_t w = t.workers[0] + t.workers[1];
  const int64_t m = t.mass_workers;
  const int64_t words = (items + 2 * w) * kItemWords + w * kMergeWords + 2 * (w + 16) + (mass + m) * kMassWords +
                        m * kMassMergeWords + m + 16 + 2 * tokens + 64;
  if (words > kMaxWords) {
    bad("paged plan: the step is too large");
    return 0;
  }
  return words;
}

int sf_paged_plan_build(sf_paged_plan* plan, const int32_t* q_lens, const int32_t* kv_lens, int32_t* words,
                        int64_t cap) {
  const int64_t need = sf_paged_plan_words(plan, q_lens, kv_lens);
  if (need == 0) return SF_ERR_ARG;
  if (!words || cap < need)
    return bad("paged plan: %lld words given, %lld needed", static_cast<long long>(cap), static_cast<long long>(need));
  try {
    sf_paged_plan& p = *plan;
    p.sms = device_sms(p.sms);
    const int G = p.H / p.Hkv;
    const Tiling t = tiling(p);
    p.T = 0;
    p.max_kv = 0;
    p.short_chunk = 0;
    int64_t at = 0;
    // {sequence, position} of every new token
    p.tokens = 0;
    for (int b = 0; b < p.B; ++b) {
      for (int i = 0; i < q_lens[b]; ++i) {
        words[at++] = b;
        words[at++] = kv_lens[b] - q_lens[b] + i;
      }
      p.T += q_lens[b];
      if (q_lens[b] > 0) p.max_kv = std::max(p.max_kv, kv_lens[b]);
      if (q_lens[b] > kv_lens[b]) p.short_chunk = 1;
    }
    at = up4(at);
    p.ws_bytes = 0;
    const int keys = p.dtype == SF_DTYPE_BF16 ? kPagedKB : kPagedKeysF32;   // of a block
    for (int k = 0; k < 2; ++k) {
      std::vector<PagedItem> tiles;
      std::vector<int> units;
      std::vector<Piece> pieces;
      std::vector<Cut> cuts;
      std::vector<int32_t> first;
      int q0 = 0;
      for (int b = 0; b < p.B; q0 += q_lens[b], ++b) {
        if (q_lens[b] == 0 || which(t, q_lens[b], G) != k) continue;
        const PagedMask mask{p.block, p.window, p.sinks, q_lens[b], kv_lens[b]};
        for (int h = 0; h < p.Hkv; ++h)
          for (int t0 = 0; t0 < q_lens[b]; t0 += t.per_tile[k]) {
            PagedItem it{};
            it.seq = b;
            it.kvh = h;
            it.tok0 = t0;
            it.ntok = std::min(t.per_tile[k], q_lens[b] - t0);
            it.slot = -1;
            const int hi = std::max(0, mask.hi(t0 + it.ntok - 1));
            const int end = (hi + keys - 1) / keys;
            it.lo_blk = std::min(mask.lo(t0) / keys, end);
            it.sink_blks = std::min((std::min(p.sinks, hi) + keys - 1) / keys, it.lo_blk);
            it.i1 = it.sink_blks + end - it.lo_blk;
            it.q0 = q0;
            it.q_len = q_lens[b];
            it.kv_len = kv_lens[b];
            tiles.push_back(it);
            units.push_back(it.i1);
          }
      }
      sf_paged_list& l = p.attn[k];
      l = sf_paged_list{};
      l.rows = t.rows[k];
      l.tile_tokens = t.tokens[k];
      for (const PagedItem& it : tiles) l.max_rows = std::max(l.max_rows, it.ntok * G);
      if (!tiles.empty()) {
        int slots = 0;
        deal(units, 1, t.workers[k], t.whole[k], &pieces, &first, &cuts, &slots);
        l.slots = slots;
        l.n_items = static_cast<int32_t>(pieces.size());
        l.workers = static_cast<int32_t>(first.size()) - 1;
        l.n_merges = static_cast<int32_t>(cuts.size());
      }
      l.items = static_cast<int32_t>(at);
      for (const Piece& x : pieces) {
        PagedItem it = tiles[x.what];
        it.i0 = x.i0;
        it.i1 = x.i1;
        it.slot = x.slot;
        memcpy(words + at, &it, sizeof(it));
        at += kItemWords;
      }
      // (a CTA finds its first item without knowing its index)
      l.heads = static_cast<int32_t>(at);
      for (int x = 0; x < l.workers; ++x) {
        memcpy(words + at, words + l.items + static_cast<int64_t>(std::min(first[x], l.n_items - 1)) * kItemWords, sizeof(PagedItem));
        at += kItemWords;
      }
      l.merges = static_cast<int32_t>(at);
      for (const Cut& c : cuts) {
        const PagedItem& it = tiles[c.what];
        const PagedMerge m{it.kvh, it.tok0, it.ntok, c.slot0, c.n, it.q0, 0, 0};
        memcpy(words + at, &m, sizeof(m));
        at += kMergeWords;
      }
      l.first = static_cast<int32_t>(at);
      memcpy(words + at, first.data(), first.size() * 4);
      at = up4(at + static_cast<int64_t>(first.size()));
      p.ws_bytes += list_ws(l, p.hd);
    }
    // weight accumulation: pairs of key blocks, their unit a tile of tokens
    {
      std::vector<PagedMassItem> pairs;
      std::vector<int> units;
      std::vector<Piece> pieces;
      std::vector<Cut> cuts;
      std::vector<int32_t> first;
      const int tile = std::max(1, t.mass_rows / G);
      int q0 = 0;
      for (int b = 0; b < p.B; q0 += q_lens[b], ++b) {
        if (q_lens[b] == 0 || p.skip_mass) continue;
        const PagedMask mask{p.block, p.window, p.sinks, q_lens[b], kv_lens[b]};
        for (int h = 0; h < p.Hkv; ++h)
          for (int kb = 0; kb * kPagedKB < kv_lens[b]; kb += kMassBlocks) {
            PagedMassItem it{};
            mask.pair_tokens(kb, &it.t0, &it.t1);
            if (it.t0 >= it.t1) continue;
            it.seq = b;
            it.kvh = h;
            it.kb0 = kb;
            it.q0 = q0;
            it.q_len = q_lens[b];
            it.kv_len = kv_lens[b];
            pairs.push_back(it);
            units.push_back((it.t1 - it.t0 + tile - 1) / tile);
          }
      }
      sf_paged_list& l = p.mass;
      l = sf_paged_list{};
      if (!pairs.empty()) {
        int slots = 0;
        // loading two key blocks takes about as long as two tiles
        deal(units, 2, t.mass_workers, 1, &pieces, &first, &cuts, &slots);
        l.slots = slots;
        l.n_items = static_cast<int32_t>(pieces.size());
        l.workers = static_cast<int32_t>(first.size()) - 1;
        l.n_merges = static_cast<int32_t>(cuts.size());
      }
      l.items = static_cast<int32_t>(at);
      for (const Piece& x : pieces) {
        PagedMassItem it = pairs[x.what];
        it.i0 = x.i0;
        it.i1 = x.i1;
        it.slot = x.slot;
        memcpy(words + at, &it, sizeof(it));
        at += kMassWords;
      }
      l.merges = static_cast<int32_t>(at);
      for (const Cut& c : cuts) {
        const PagedMassItem& it = pairs[c.what];
        const PagedMassMerge m{it.seq, it.kvh, it.kb0, c.slot0, c.n, it.q_len, it.kv_len, 0};
        memcpy(words + at, &m, sizeof(m));
        at += kMassMergeWords;
      }
      l.first = static_cast<int32_t>(at);
      memcpy(words + at, first.data(), first.size() * 4);
      at = up4(at + static_cast<int64_t>(first.size()));
      p.ws_bytes = std::max(p.ws_bytes, mass_ws(l));
    }
    p.words = std::max<int64_t>(at, 4);
    p.dev = nullptr;
    p.ws = nullptr;
    p.err = nullptr;
    return SF_OK;
  } catch (const std::exception& e) {
    return bad("paged plan: %s", e.what());
  }
}

int sf_paged_kv_append(const sf_paged_plan* plan, const sf_paged_pool* pool, const void* k_new, const void* v_new,
                       int64_t new_tok_stride, int64_t new_head_stride, void* stream) {
  int rc = check_ready("paged_kv_append", plan);
  if (rc == SF_OK && plan->short_chunk) rc = bad("paged_kv_append: a sequence has more new tokens than cached keys");
  if (rc != SF_OK || plan->T == 0) return rc;
  if ((rc = check_pool("paged_kv_append", pool, plan->dtype, plan->hd, plan->page_size, plan->max_kv, true, false)) != SF_OK ||
      (rc = check_rows("paged_kv_append", plan, k_new, new_tok_stride, new_head_stride)) != SF_OK ||
      (rc = check_rows("paged_kv_append", plan, v_new, new_tok_stride, new_head_stride)) != SF_OK)
    return rc;
  PagedAppendParams p{};
  p.k_new = k_new;
  p.v_new = v_new;
  p.new_tok = new_tok_stride;
  p.new_head = new_head_stride;
  p.pool = pool_of(*pool, plan->page_size);
  p.tokens = plan->dev + plan->tokens;
  p.T = plan->T;
  p.Hkv = plan->Hkv;
  p.hd = plan->hd;
  p.err = plan->err;
  return status(launch_paged_append(plan->dtype, p, static_cast<cudaStream_t>(stream)), "paged_kv_append");
}

int sf_paged_attention(const sf_paged_plan* plan, const sf_paged_pool* pool, const void* q, int64_t q_tok_stride,
                       int64_t q_head_stride, void* out, float* lse, float scale, void* stream) {
  int rc = check_ready("paged_attention", plan);
  if (rc != SF_OK || plan->T == 0) return rc;
  if ((rc = check_pool("paged_attention", pool, plan->dtype, plan->hd, plan->page_size, plan->max_kv, true, false)) != SF_OK ||
      (rc = check_rows("paged_attention", plan, q, q_tok_stride, q_head_stride)) != SF_OK)
    return rc;
  if (!out || !lse || !aligned16(out)) return bad("paged_attention: out and lse must be given, out 16-byte aligned");
  if (!(scale > 0.f) || scale > 3.0e38f) return bad("paged_attention: scale must be positive");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  size_t off = 0;
  for (int k = 0; k < 2; ++k) {
    const sf_paged_list& l = plan->attn[k];
    if (l.n_items == 0) continue;
    PagedAttnParams p{};
    p.q = q;
    p.q_tok = q_tok_stride;
    p.q_head = q_head_stride;
    p.pool = pool_of(*pool, plan->page_size);
    p.out = out;
    p.lse = lse;
    p.items = reinterpret_cast<const PagedItem*>(plan->dev + l.items);
    p.heads = reinterpret_cast<const PagedItem*>(plan->dev + l.heads);
    p.first = plan->dev + l.first;
    p.workers = l.workers;
    p.merges = reinterpret_cast<const PagedMerge*>(plan->dev + l.merges);
    p.n_merges = l.n_merges;
    p.part_O = reinterpret_cast<float*>(static_cast<char*>(plan->ws) + off);
    p.part_ml = p.part_O + static_cast<size_t>(l.slots) * l.rows * plan->hd;
    off += list_ws(l, plan->hd);
    p.rows = l.rows;
    p.tile_tokens = l.tile_tokens;
    p.H = plan->H;
    p.Hkv = plan->Hkv;
    p.G = plan->H / plan->Hkv;
    p.hd = plan->hd;
    p.T = plan->T;
    p.block = plan->block;
    p.window = plan->window;
    p.sinks = plan->sinks;
    p.scale = scale;
    p.err = plan->err;
    cudaError_t e;
    if (plan->dtype == SF_DTYPE_BF16 && k == 0)
      e = launch_paged_attention_tokens(p, l.max_rows <= 32 ? 4 : l.max_rows <= 64 ? 2 : 1, st);
    else if (plan->dtype == SF_DTYPE_BF16)
      e = launch_paged_attention_chunk(p, st);
    else
      e = launch_paged_attention_simt(p, st);
    if (e == cudaSuccess) e = launch_paged_merge(plan->dtype, p, st);
    if (e != cudaSuccess) return status(e, "paged_attention");
  }
  return SF_OK;
}

int sf_paged_attention_mass(const sf_paged_plan* plan, const sf_paged_pool* pool, const void* q, int64_t q_tok_stride,
                            int64_t q_head_stride, const float* lse, float scale, void* stream) {
  int rc = check_ready("paged_attention_mass", plan);
  if (rc == SF_OK && plan->skip_mass) rc = bad("paged_attention_mass: the plan was made without it");
  if (rc != SF_OK || plan->mass.n_items == 0) return rc;
  if ((rc = check_pool("paged_attention_mass", pool, plan->dtype, plan->hd, plan->page_size, plan->max_kv, false, true)) != SF_OK ||
      (rc = check_rows("paged_attention_mass", plan, q, q_tok_stride, q_head_stride)) != SF_OK)
    return rc;
  if (!lse) return bad("paged_attention_mass: null lse");
  if (!(scale > 0.f) || scale > 3.0e38f) return bad("paged_attention_mass: scale must be positive");
  PagedMassParams p{};
  p.q = q;
  p.q_tok = q_tok_stride;
  p.q_head = q_head_stride;
  p.pool = pool_of(*pool, plan->page_size);
  p.lse = lse;
  p.items = reinterpret_cast<const PagedMassItem*>(plan->dev + plan->mass.items);
  p.first = plan->dev + plan->mass.first;
  p.workers = plan->mass.workers;
  p.merges = reinterpret_cast<const PagedMassMerge*>(plan->dev + plan->mass.merges);
  p.n_merges = plan->mass.n_merges;
  p.part = static_cast<float*>(plan->ws);
  p.H = plan->H;
  p.Hkv = plan->Hkv;
  p.G = plan->H / plan->Hkv;
  p.hd = plan->hd;
  p.T = plan->T;
  p.block = plan->block;
  p.window = plan->window;
  p.sinks = plan->sinks;
  p.scale = scale;
  p.err = plan->err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = plan->dtype == SF_DTYPE_BF16 ? launch_paged_mass_tc(p, st) : launch_paged_mass_simt(p, st);
  if (e == cudaSuccess) e = launch_paged_mass_merge(p, st);
  return status(e, "paged_attention_mass");
}

int sf_paged_evict(int dtype, const sf_paged_pool* pool, const int32_t* dst_table, int64_t dst_stride,
                   int32_t dst_width, const int32_t* lens, int32_t max_len, int32_t max_keep, int B, int Hkv, int hd,
                   int page_size, int sinks, int recent, int32_t* kept, int64_t kept_stride, int* err, void* stream) {
  if (dtype != SF_DTYPE_F32 && dtype != SF_DTYPE_BF16) return bad("paged_evict: dtype %d not supported", dtype);
  if (hd != 64 && hd != 128) return bad("paged_evict: head_dim %d must be 64 or 128", hd);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return bad("paged_evict: page size %d must be a power of two in [16, 256]", page_size);
  if (B < 0 || Hkv < 1 || B > 65535 || static_cast<int64_t>(B) * Hkv > 65535) return bad("paged_evict: %d sequences of %d heads", B, Hkv);
  if (sinks < 0 || recent < 0 || max_len < 0 || max_keep < 0 || static_cast<int64_t>(sinks) + recent > max_keep)
    return bad("paged_evict: sinks %d + recent %d do not fit the %d keys that stay", sinks, recent, max_keep);
  if (B == 0) return SF_OK;
  const int stay = std::min(max_len, max_keep);
  if (stay == 0) return SF_OK;
  if (!lens || !kept || !err || kept_stride < stay || kept_stride > INT32_MAX)
    return bad("paged_evict: null argument or kept rows shorter than %d", stay);
  int rc = check_pool("paged_evict", pool, dtype, hd, page_size, max_len, true, true);
  if (rc != SF_OK) return rc;
  if (static_cast<int64_t>(dst_width) * page_size < stay || dst_stride < dst_width)
    return bad("paged_evict: a destination table of %d pages does not hold %d keys", dst_width, stay);
  if (!dst_table) return bad("paged_evict: null destination table");
  PagedEvictParams p{};
  p.pool = pool_of(*pool, page_size);
  p.dst = dst_table;
  p.dst_stride = dst_stride;
  p.lens = lens;
  p.kept = kept;
  p.kept_stride = static_cast<int>(kept_stride);
  p.B = B;
  p.Hkv = Hkv;
  p.hd = hd;
  p.sinks = sinks;
  p.recent = recent;
  p.max_len = max_len;
  p.max_keep = max_keep;
  p.sms = device_sms(0);
  p.err = err;
  return status(launch_paged_evict(dtype, p, static_cast<cudaStream_t>(stream)), "paged_evict");
}

}  // extern "C"

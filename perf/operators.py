"""The paged-cache operators as measured workloads.

Five operators over a pool of pages that many sequences share: the append of new keys and
values, the attention of each sequence's new tokens over its pages (single tokens, blocks and
long chunks; causal, block-causal or without a mask, optionally with a sliding window and a few
first tokens that stay visible), the accumulation of each cached key's attention weight, and the
eviction that keeps the keys with the largest accumulated weight.

``run`` computes them in plain torch (``own`` false) or through ``specfold_b200`` (``own``
true).  Head counts are those of the shapes in ``specfold_b200/synthetic.py`` (Qwen2.5-1.5B:
12/2 heads, Qwen2.5-7B: 28/4, Llama 8B: 32/8, Llama 14B: 40/8, the tiny test shapes 4/2);
the prefix lengths are those its bench and sweep use (1024 ... 32768) and odd ones around them.
"""

import math

import torch

own = False

#: (query heads, kv heads, head dim) of the framework's shapes
HEADS = {"tiny": (4, 2, 64), "qwen1.5b": (12, 2, 128), "qwen7b": (28, 4, 128),
         "llama8b": (32, 8, 128), "llama14b": (40, 8, 128)}
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(op, shape, dtype, seqs, q, kv, page, block=1, window=0, sinks=0, idle=0, keep=0,
          recent=0):
    """``seqs`` sequences; new tokens per sequence spread over q = (lo, hi), cached tokens
    (the new ones included) over kv = (lo, hi); every ``idle``-th sequence has no new token."""
    H, Hkv, hd = HEADS[shape]
    return {"op": op, "shape": shape, "heads": H, "kv_heads": Hkv, "head_dim": hd,
            "dtype": dtype, "seqs": seqs, "q_lo": q[0], "q_hi": q[1], "kv_lo": kv[0],
            "kv_hi": kv[1], "page": page, "block": block, "window": window, "sinks": sinks,
            "idle": idle, "keep": keep, "recent": recent}


def listed():
    def named(name, c):
        return dict(c, name=name)

    return [
        # the step of a server under load: one new row per running request
        named("append_tokens", _case("append", "qwen7b", "bf16", 64, (1, 1), (900, 9000), 64)),
        # four prompts enter the cache, their rows sliced out of a fused QKV output
        named("append_prompts", _case("append", "llama8b", "bf16", 4, (3000, 4100), (3000, 8200), 64)),
        # one request alone, a short context: nothing but latency
        named("attend_token", _case("attend", "qwen1.5b", "bf16", 1, (1, 1), (777, 777), 16)),
        # the decode step of a full batch, contexts of every length
        named("attend_tokens", _case("attend", "llama8b", "bf16", 64, (1, 1), (1100, 16384), 64)),
        # a chunk of a long prompt over what is already cached
        named("attend_prompt", _case("attend", "llama8b", "bf16", 1, (4096, 4096), (16384, 16384), 128)),
        # blocks of a diffusion model's verify pass (bidirectional within 32) in fp32
        named("attend_blocks_f32", _case("attend", "qwen1.5b", "f32", 3, (32, 320), (700, 2100), 32,
                                         block=32)),
        # streaming requests: long histories of which a window and the first tokens stay visible
        named("window_tokens", _case("attend", "qwen7b", "bf16", 32, (1, 1), (5000, 32768), 64,
                                     window=4096, sinks=4, idle=9)),
        # ragged chunks under the same kind of window, narrower than the chunk
        named("window_chunks", _case("attend", "llama14b", "bf16", 4, (500, 2048), (2048, 8000), 32,
                                     window=1000, sinks=16)),
        # weight accumulation after a decode step, and after a prompt chunk
        named("mass_tokens", _case("mass", "llama8b", "bf16", 32, (1, 1), (1000, 8192), 64)),
        named("mass_chunks", _case("mass", "qwen7b", "bf16", 2, (1500, 2048), (5000, 8192), 64)),
        # one long request cut to its budget; a batch of requests cut to theirs
        named("evict_one", _case("evict", "llama8b", "bf16", 1, (1, 1), (32768, 32768), 64, sinks=4,
                                 keep=8192, recent=256)),
        named("evict_batch", _case("evict", "qwen7b", "bf16", 24, (1, 1), (1500, 8200), 64, sinks=4,
                                   keep=2048, recent=128)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "window", "window", "mass", "mass", "evict"))
    shape = rng.choice(tuple(HEADS))
    dtype = "f32" if rng.random() < 0.2 else "bf16"
    page = rng.choice((16, 32, 64, 128))
    if op == "evict":
        seqs = _log(rng, 1, 32)
        hi = _log(rng, 600, 32768)
        sinks = rng.choice((0, 1, 4, 16))
        recent = _log(rng, 1, 256)
        return _case("evict", shape, dtype, seqs, (1, 1), (max(1, int(hi * rng.uniform(0.1, 1))), hi),
                     page, sinks=sinks, recent=recent, keep=sinks + recent + _log(rng, 1, max(2, hi // 2)))
    kind = rng.choice(("token", "block", "chunk"))
    seqs = _log(rng, 1, 64) if kind == "token" else _log(rng, 1, 12) if kind == "block" else _log(rng, 1, 4)
    q_hi = 1 if kind == "token" else rng.choice((8, 17, 32, 33, 64)) if kind == "block" else _log(rng, 65, 4096)
    if dtype == "f32":
        q_hi = min(q_hi, 512)
    q_lo = max(1, int(q_hi * rng.uniform(0.3, 1)))
    kv_hi = max(q_hi, _log(rng, 40, 32768 if kind == "token" else 16384))
    kv_lo = max(q_hi, int(kv_hi * rng.uniform(0.1, 1)))
    block = rng.choice((1, 1, 1, 32, 0)) if kind != "token" else 1
    window, sinks = (_log(rng, 16, 8192), rng.choice((0, 1, 4, 16))) if op == "window" else (0, 0)
    return _case("attend" if op == "window" else op, shape, dtype, seqs, (q_lo, q_hi), (kv_lo, kv_hi),
                 page, block=block, window=window, sinks=sinks,
                 idle=rng.choice((0, 0, 3)) if seqs > 3 else 0)


def _padded(c):
    """Elements of the plain form's padded scores: what its time goes by."""
    return c["seqs"] * c["heads"] * c["q_hi"] * c["kv_hi"]


def draw(rng):
    tops = {}
    for c in listed():
        w = work(c)
        for k, v in (("bytes", w["bytes"]), ("flops", w["flops"]), ("padded", _padded(c))):
            tops[k] = max(tops.get(k, 0), v)
    while True:
        c = _draw(rng)
        w = work(c)
        slow = 16 if c["dtype"] == "f32" else 1    # fp32 products cost more per operation
        if w["bytes"] <= tops["bytes"] and w["flops"] * slow <= tops["flops"] and _padded(c) <= tops["padded"]:
            return c


# ---------------------------------------------------------------------------- lengths
def _spread(lo, hi, n, phase):
    """n lengths over [lo, hi], spread over their logarithm, the largest first."""
    f = [((b * 0.6180339887 + phase) % 1.0) for b in range(n)]
    out = [int(round(lo * (hi / lo) ** x)) for x in f]
    out[0] = hi
    return out


def _lens(c):
    n = _spread(c["kv_lo"], c["kv_hi"], c["seqs"], 0.5)
    q = _spread(c["q_lo"], c["q_hi"], c["seqs"], 0.31)
    q = [min(a, b) for a, b in zip(q, n)]
    if c["idle"]:
        q = [0 if (b % c["idle"]) == c["idle"] - 1 else x for b, x in enumerate(q)]
    return q, n


def _pairs(c, q, n):
    """(query token, key) pairs that the mask leaves, and keys seen by any token."""
    if q == 0:
        return 0, 0
    i = torch.arange(q, dtype=torch.int64)
    p = n - q + i
    hi = torch.full_like(p, n) if c["block"] == 0 else ((i // c["block"] + 1) * c["block"] + n - q).clamp(max=n)
    lo = (p - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(p)
    first = torch.minimum(torch.full_like(lo, c["sinks"]), lo)
    pairs = int(((hi - lo).clamp(min=0) + torch.minimum(first, hi)).sum())
    low = int(lo.min())
    return pairs, int(hi.max()) - low + min(c["sinks"], low)


def work(case):
    c = case
    q, n = _lens(c)
    e = 2 if c["dtype"] == "bf16" else 4
    H, Hkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    T = sum(q)
    if c["op"] == "append":
        return {"bytes": 2 * T * Hkv * hd * 2 * e + T * Hkv * 4, "flops": 0}
    if c["op"] == "evict":
        kept = sum(min(x, c["keep"]) for x in n)
        return {"bytes": Hkv * (4 * sum(n) + kept * (2 * 2 * hd * e + 4 + 4)), "flops": 0}
    got = [_pairs(c, a, b) for a, b in zip(q, n)]
    pairs, keys = sum(g[0] for g in got), sum(g[1] for g in got)
    if c["op"] == "mass":
        return {"bytes": T * H * (hd * e + 4) + keys * Hkv * (hd * e + 8), "flops": 2 * hd * H * pairs}
    return {"bytes": T * H * (2 * hd * e + 4) + keys * Hkv * 2 * hd * e, "flops": 4 * hd * H * pairs}


# ---------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    dev, dt = "cuda", DT[c["dtype"]]
    H, Hkv, hd, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    q_lens, kv_lens = _lens(c)
    T, B = sum(q_lens), c["seqs"]
    need = [-(-n // ps) for n in kv_lens]
    into = [-(-min(n, c["keep"]) // ps) for n in kv_lens] if c["op"] == "evict" else [0] * B
    pool = sum(need) + sum(into) + 3
    # pages are handed out in no order, as in a pool that has been running for a while
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device=dev)
    dst = torch.full((B, max(1, max(into))), -1, dtype=torch.int32, device=dev)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        dst[b, :into[b]] = order[at + need[b]:at + need[b] + into[b]]
        at += need[b] + into[b]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    s = {"case": c, "q_lens": q_lens, "kv_lens": kv_lens, "table": table, "dst": dst,
         "k": randn(pool, Hkv, ps, hd), "v": randn(pool, Hkv, ps, hd), "scale": hd ** -0.5}
    # queries and new rows are slices of one fused projection's output
    qkv = randn(T, (H + 2 * Hkv) * hd)
    s["q"] = qkv[:, :H * hd].view(T, H, hd)
    s["k_new"] = qkv[:, H * hd:(H + Hkv) * hd].view(T, Hkv, hd)
    s["v_new"] = qkv[:, (H + Hkv) * hd:].view(T, Hkv, hd)
    # every sequence's first key draws much of the attention, as first tokens do
    u = torch.nn.functional.normalize(torch.randn(Hkv, hd, generator=g, device=dev), dim=-1)
    s["q"] += (4 * u.to(dt)).repeat_interleave(H // Hkv, 0)
    s["k"][table[:, 0].long(), :, 0] += (14 * u).to(dt)
    # accumulated weights: heavy-tailed, some equal, some still zero
    if c["op"] != "attend":
        mass = torch.exp(2 * torch.randn(pool, Hkv, ps, generator=g, device=dev))
        coarse = (mass * 4).round() / 4
        pick = torch.rand(pool, Hkv, ps, generator=g, device=dev)
        s["mass"] = torch.where(pick < 0.3, coarse, mass) * (pick < 0.95)
    if c["op"] == "mass":
        s["lse"] = _attend(s)[1]
    if own:
        from specfold_b200 import kernels as K
        if c["op"] == "evict":
            s["plan"] = K.EvictPlan(kv_lens, c["keep"], kv_heads=Hkv, page_size=ps, sinks=c["sinks"],
                                    recent=c["recent"], device=dev)
        else:
            s["plan"] = K.PagedPlan(q_lens, kv_lens, heads=H, kv_heads=Hkv, head_dim=hd,
                                    page_size=ps, dtype=dt, block=c["block"], window=c["window"],
                                    sinks=c["sinks"], device=dev)
    return s


# ---------------------------------------------------------------------------- plain forms
def _rows(s):
    """(sequence, index in its chunk, position) of every new token."""
    q = torch.tensor(s["q_lens"], device="cuda")
    n = torch.tensor(s["kv_lens"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(q), device="cuda"), q)
    i = torch.arange(len(seq), device="cuda") - (q.cumsum(0) - q)[seq]
    return seq, i, (n - q)[seq] + i


def _keys(pages, table):
    """[B, Hkv, keys, hd] in fp32 of the sequences' pages."""
    x = pages[table.clamp(min=0).long()].float()
    B, W, Hkv, ps = x.shape[:4]
    return x.transpose(1, 2).reshape(B, Hkv, W * ps, *x.shape[4:])


def _scores(s):
    """(scores [B, Hkv, q * group, keys], nothing-visible fill -inf; where each token sits)."""
    c = s["case"]
    H, Hkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    G, B, mq = H // Hkv, c["seqs"], max(1, max(s["q_lens"]))
    seq, i, pos = _rows(s)
    q = torch.zeros(B, mq, H, hd, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(B, mq, Hkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, Hkv, mq * G, hd)
    k = _keys(s["k"], s["table"])
    j = torch.arange(k.shape[2], device="cuda")
    ql = torch.tensor(s["q_lens"], device="cuda")[:, None]
    n = torch.tensor(s["kv_lens"], device="cuda")[:, None]
    t = torch.arange(mq, device="cuda")[None]
    p = n - ql + t
    hi = n.expand_as(p) if c["block"] == 0 else torch.minimum(n, n - ql + (t // c["block"] + 1) * c["block"])
    see = (j < hi[..., None]) & (t < ql)[..., None]
    if c["window"]:
        see &= (j > p[..., None] - c["window"]) | (j < c["sinks"])
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"])
    x.view(B, Hkv, mq, G, -1).masked_fill_(~see[:, None, :, None], -math.inf)
    return x, seq, i


def _tokens(x, seq, i, G):
    """[B, Hkv, q * group, ...] -> [tokens, H, ...]"""
    B, Hkv = x.shape[:2]
    x = x.view(B, Hkv, -1, G, *x.shape[3:]).transpose(1, 2)[seq, i]
    return x.reshape(x.shape[0], Hkv * G, *x.shape[3:])


def _attend(s):
    c = s["case"]
    G = c["heads"] // c["kv_heads"]
    x, seq, i = _scores(s)
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x = x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    o = torch.matmul(x, _keys(s["v"], s["table"])) / torch.where(l > 0, l, 1)
    lse = (m + l.log()).squeeze(-1)
    return _tokens(o, seq, i, G).to(s["q"].dtype), _tokens(lse, seq, i, G)


def _slots(table, ps):
    """Flat page * page_size + offset of every position [B, positions]."""
    off = torch.arange(ps, device="cuda")
    return (table.clamp(min=0).long()[..., None] * ps + off).flatten(1)


def _mass(s):
    c = s["case"]
    ps, mq = c["page"], max(1, max(s["q_lens"]))
    x, seq, i = _scores(s)
    B, Hkv, R = x.shape[:3]
    lse = torch.full((B, mq, c["heads"]), math.inf, device="cuda")
    lse[seq, i] = torch.where(s["lse"] == -math.inf, math.inf, s["lse"])
    lse = lse.view(B, mq, Hkv, -1).permute(0, 2, 1, 3).reshape(B, Hkv, R, 1)
    add = x.sub_(lse).exp_().sum(2)                                    # [B, Hkv, keys]
    live = torch.arange(add.shape[-1], device="cuda") < torch.tensor(s["kv_lens"], device="cuda")[:, None]
    slot = _slots(s["table"], ps)[live]
    mass = s["mass"]
    mass[slot // ps, :, slot % ps] += add.transpose(1, 2)[live]
    return mass


def _append(s):
    ps = s["case"]["page"]
    seq, _, pos = _rows(s)
    page = s["table"][seq, pos // ps].long()
    s["k"][page, :, pos % ps] = s["k_new"]
    s["v"][page, :, pos % ps] = s["v_new"]
    s["mass"][page, :, pos % ps] = 0
    return s["k"], s["v"], s["mass"]


def _evict(s):
    c = s["case"]
    ps, Hkv = c["page"], c["kv_heads"]
    n = torch.tensor(s["kv_lens"], device="cuda")[:, None, None]
    keep = n.clamp(max=c["keep"])
    a = _keys(s["mass"], s["table"])
    j = torch.arange(a.shape[-1], device="cuda")
    a = a.masked_fill((j < c["sinks"]) | (j >= n - c["recent"]), math.inf).masked_fill(j >= n, -math.inf)
    top = a.sort(dim=-1, descending=True, stable=True)[1][..., :max(min(x, c["keep"]) for x in s["kv_lens"])]
    rank = torch.arange(top.shape[-1], device="cuda")
    kept = top.masked_fill(rank >= keep, 1 << 30).sort(dim=-1)[0]
    live = (rank < keep).expand_as(kept)                                # [B, Hkv, kept]
    b, h, r = live.nonzero(as_tuple=True)
    src = _slots(s["table"], ps)[b, kept[b, h, r]]
    to = _slots(s["dst"], ps)[b, r]
    for x in (s["k"], s["v"], s["mass"]):
        x[to // ps, h, to % ps] = x[src // ps, h, src % ps]
    return s["k"], s["v"], s["mass"], kept.masked_fill(~live, -1).to(torch.int32)


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"attend": _attend, "mass": _mass, "append": _append, "evict": _evict}[op](s)
    from specfold_b200 import kernels as K
    if op == "attend":
        return K.paged_attention(s["q"], s["k"], s["v"], s["table"], s["plan"], scale=s["scale"])
    if op == "mass":
        K.paged_attention_mass(s["q"], s["k"], s["table"], s["lse"], s["mass"], s["plan"], scale=s["scale"])
        return s["mass"]
    if op == "append":
        K.paged_kv_append(s["k"], s["v"], s["k_new"], s["v_new"], s["table"], s["plan"], mass_pages=s["mass"])
        return s["k"], s["v"], s["mass"]
    kept = K.paged_evict(s["k"], s["v"], s["mass"], s["table"], s["dst"], s["plan"])
    return s["k"], s["v"], s["mass"], kept


# ---------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """From the definitions, one sequence and kv head at a time, in float64."""
    c = case
    if c["op"] in ("append", "evict"):
        return None                              # moved values, not computed ones
    s = prepare(case, seed)
    H, Hkv, hd, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    G, T = H // Hkv, sum(s["q_lens"])
    out = torch.zeros(T, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if c["op"] == "mass" else None
    t0 = 0
    for b, (ql, n) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        pages = s["table"][b, :-(-n // ps)].long()
        key = torch.arange(n, device="cuda")
        for h in range(Hkv):
            k = s["k"][pages, h].reshape(-1, hd)[:n].double()
            v = s["v"][pages, h].reshape(-1, hd)[:n].double()
            for i0 in range(0, ql, 512):
                i = torch.arange(i0, min(ql, i0 + 512), device="cuda")
                p = n - ql + i
                see = torch.ones(len(i), n, dtype=torch.bool, device="cuda")
                if c["block"]:
                    see &= key < ((i // c["block"] + 1) * c["block"] + n - ql)[:, None]
                if c["window"]:
                    see &= ((p[:, None] - key) < c["window"]) | (key < c["sinks"])
                rows = slice(t0 + i0, t0 + i0 + len(i))
                for g in range(h * G, (h + 1) * G):
                    x = (s["q"][rows, g].double() @ k.T) * s["scale"]
                    x = x.masked_fill(~see, -math.inf)
                    if mass is None:
                        top = x.amax(1, keepdim=True)
                        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
                        e = (x - top).exp()
                        z = e.sum(1, keepdim=True)
                        out[rows, g] = torch.where(z > 0, (e @ v) / z, torch.zeros_like(top))
                        lse[rows, g] = (top + z.log())[:, 0]
                    else:
                        w = (x - s["lse"][rows, g].double()[:, None]).exp().sum(0)
                        full = torch.zeros(len(pages) * ps, dtype=torch.float64, device="cuda")
                        full[:n] = w.masked_fill(~see.any(0), 0.0)
                        mass[pages, h] += full.view(-1, ps)
        t0 += ql
    return (out, lse) if mass is None else mass

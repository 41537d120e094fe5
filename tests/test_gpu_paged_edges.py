"""The paged cache's kernels where their pipelines and their inputs have edges: steps of many key
blocks and items against the definitions in float64 on the device."""
import math

import pytest
import torch

from specfold_b200 import kernels as K
from tests.paged_reference import U32, UB, UW, evict_positions

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


class Step:
    """One step's inputs on the device.  Pages are dealt in no order; ``q``, ``k[b]`` and ``v[b]``
    (rows of sequence b, in order) may be changed before ``pages()`` is called."""

    def __init__(self, q_lens, kv_lens, H, Hkv, hd=128, ps=64, dtype=BF, block=1, window=0, sinks=0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_lens, self.kv_lens, self.H, self.Hkv, self.hd, self.ps = q_lens, kv_lens, H, Hkv, hd, ps
        self.dtype, self.block, self.window, self.sinks, self.scale = dtype, block, window, sinks, hd ** -0.5
        self.q = torch.randn(sum(q_lens), H, hd, generator=g, device="cuda").to(dtype)
        self.k = [torch.randn(n, Hkv, hd, generator=g, device="cuda").to(dtype) for n in kv_lens]
        self.v = [torch.randn(n, Hkv, hd, generator=g, device="cuda").to(dtype) for n in kv_lens]
        need = [-(-n // ps) for n in kv_lens]
        order = torch.randperm(sum(need) + 1, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(kv_lens), max(need + [1])), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.num_pages = sum(need) + 1

    def pages(self):
        """(k_pages, v_pages); slots that hold no key are NaN."""
        out = []
        for rows in (self.k, self.v):
            p = torch.full((self.num_pages, self.Hkv, self.ps, self.hd), math.nan, dtype=self.dtype, device="cuda")
            for b, r in enumerate(rows):
                j = torch.arange(len(r), device="cuda")
                p[self.table[b, j // self.ps].long(), :, j % self.ps] = r
            out.append(p)
        return out

    def plan(self, **kw):
        return K.PagedPlan(self.q_lens, self.kv_lens, heads=self.H, kv_heads=self.Hkv, head_dim=self.hd,
                           page_size=self.ps, dtype=self.dtype, block=self.block, window=self.window,
                           sinks=self.sinks, **kw)

    def sees(self, b):
        """[q_len, kv_len]: which keys each token of sequence b sees"""
        q, n = self.q_lens[b], self.kv_lens[b]
        i, j = torch.arange(q, device="cuda")[:, None], torch.arange(n, device="cuda")
        see = (j < n - q + (i // self.block + 1) * self.block) if self.block else (j < n).expand(q, n)
        if self.window:
            see = see & ((j > n - q + i - self.window) | (j < self.sinks))
        return see

    def exact(self):
        """(out, lse, bound on out, bound on lse) in float64; the bounds as in paged_reference."""
        T, G, bf = sum(self.q_lens), self.H // self.Hkv, self.dtype == BF
        out = torch.zeros(T, self.H, self.hd, dtype=torch.float64, device="cuda")
        lse = torch.full((T, self.H), -math.inf, dtype=torch.float64, device="cuda")
        tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
        t0 = 0
        for b, ql in enumerate(self.q_lens):
            see, rows = self.sees(b), slice(t0, t0 + ql)
            t0 += ql
            some = see.any(1)
            for h in range(self.H if see.numel() else 0):
                q, k, v = self.q[rows, h].double(), self.k[b][:, h // G].double(), self.v[b][:, h // G].double()
                s = (q @ k.T * self.scale).masked_fill(~see, -math.inf)
                top = s.amax(1, keepdim=True).masked_fill(~some[:, None], 0)
                w = (s - top).exp()
                z = w.sum(1, keepdim=True)
                w = w / z.clamp(min=1e-300)
                fin = v.isfinite()
                o = w @ v.masked_fill(~fin, 0)
                # a value that is not finite decides its column for the tokens that see it
                x = see.double()
                pos, neg, nan = (x @ m.double() > 0 for m in (v == math.inf, v == -math.inf, v.isnan()))
                o = o.masked_fill(pos, math.inf).masked_fill(neg, -math.inf).masked_fill(nan | (pos & neg), math.nan)
                out[rows, h] = o.masked_fill(z.isnan(), math.nan)
                lse[rows, h] = torch.where(some, (top + z.log())[:, 0], -math.inf)
                e = self.hd * U32 * self.scale * (q.abs() @ k.abs().T).masked_fill(~see, 0).amax(1)
                e += 8 * U32 * s.abs().masked_fill(~see, 0).amax(1) + see.sum(1) * U32
                a = w @ v.masked_fill(~fin, 0).abs()
                tol_o[rows, h] = (2 * e + (2 * UW + 2.1 * UB if bf else 4 * U32))[:, None] * a
                tol_l[rows, h] = e + (UW if bf else 4 * U32) + 4 * U32 * lse[rows, h].abs().masked_fill(~some, 0)
        return out, lse, tol_o, tol_l

    def exact_mass(self, lse, mass):
        """(accumulated weights, bound) in float64 after the step's are added to ``mass``, from the
        given lse; the bound as in paged_reference, its parts added up over a page's holders."""
        G, acc = self.H // self.Hkv, mass.double()
        off, adds, terms = (torch.zeros_like(acc) for _ in range(3))
        t0 = 0
        for b, ql in enumerate(self.q_lens):
            see, rows, j = self.sees(b), slice(t0, t0 + ql), torch.arange(self.kv_lens[b], device="cuda")
            t0 += ql
            page, at = self.table[b, j // self.ps].long(), j % self.ps
            for h in range(self.H if ql else 0):
                q, k, ls = self.q[rows, h].double(), self.k[b][:, h // G].double(), lse[rows, h].double()[:, None]
                ls = ls.masked_fill(ls == -math.inf, math.inf)         # saw nothing: weight 0
                x = q @ k.T * self.scale
                w = (x - ls).exp().masked_fill(~see, 0)
                e = self.hd * U32 * self.scale * (q.abs() @ k.abs().T) + 8 * U32 * (x.abs() + ls.abs()) + 8 * U32
                where = (page, torch.full_like(page, h // G), at)
                for into, what in ((adds, w.sum(0)), (off, (w * e).masked_fill(~see | (w == 0), 0).sum(0)), (terms, see.double().sum(0))):
                    into.index_put_(where, what, accumulate=True)
        tol = off + (terms + 2 * len(self.q_lens)) * U32 * (adds + acc.abs())
        return acc + adds, tol.masked_fill(terms == 0, 0)


def within(got, want, tol, what):
    got = got.double()
    fin = want.isfinite()
    assert torch.equal(got.isfinite(), fin), f"{what}: finite elsewhere"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    over = ((got - want).abs() - tol)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max()):.3e} over its bound"


# ---------------------------------------------------------------------------- rescaled accumulators
def check_repeatedly(st, what, times=40):
    """Against float64, and the same bits every time."""
    k, v = st.pages()
    plan = st.plan()
    first = K.paged_attention(st.q, k, v, st.table, plan)
    o, l, tol_o, tol_l = st.exact()
    within(first[0], o, tol_o, f"{what}: out")
    within(first[1], l, tol_l, f"{what}: lse")
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for _ in range(times):
        again = K.paged_attention(st.q, k, v, st.table, plan)
        same &= (again[0] == first[0]).all() & (again[1] == first[1]).all()
    plan.check()
    assert bool(same), what


@pytest.mark.parametrize("hd", [128, 64])
def test_rows_that_outgrow_their_reference(hd):
    """One head's scores rise by more than 2^60 from each half block to the next, so that its rows
    move their reference and rescale what they have accumulated in every half; the rows beside
    them do not, and must lose nothing."""
    st = Step([64, 128], [1600, 1400], 8, 2, hd=hd, seed=1)
    for k in st.k:
        # 64 keys further on, 80 more: 50 nats (72 powers of two) at a scaled query of 8
        k[:, :, 0] = (torch.arange(len(k), device="cuda") * (80 / 64))[:, None].to(k.dtype)
    st.q[:, :, 0] = 0
    st.q[:, [1, 6], 0] = 50 / 80 * hd ** 0.5
    check_repeatedly(st, "growing scores")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_large_values_under_growing_scores(dtype):
    """Scores that rise by 2^2 to 2^50 over the sequence, in steps of any size, and values near 2^100:
    the accumulators hold them, whatever the softmax's reference was."""
    st = Step([64, 128, 1, 20], [900, 1400, 3000, 500], 8, 2, dtype=dtype, seed=6)
    for k in st.k:
        k[:, :, 0] = (torch.arange(len(k), device="cuda") / len(k))[:, None].to(dtype)
    st.v = [(v.float() * 2.0 ** 100).to(dtype) for v in st.v]
    st.q[:, :, 0] = (torch.linspace(2, 50, 213, device="cuda") * math.log(2) * st.hd ** 0.5)[:, None].to(dtype)
    check_repeatedly(st, "large values", times=5)


@pytest.mark.parametrize("window,sinks,block", [(24, 0, 1), (70, 3, 1), (5, 200, 1), (40, 0, 32)])
def test_windows_narrower_than_a_tile(window, sinks, block):
    """Rows of a tile see their first key in different half blocks."""
    st = Step([256, 128], [1500, 900], 8, 2, window=window, sinks=sinks, block=block, seed=2)
    check_repeatedly(st, "narrow window")


# ---------------------------------------------------------------------------- many items a CTA
@pytest.mark.parametrize("hd,window,sinks", [(128, 100, 4), (128, 0, 0), (64, 300, 0), (64, 0, 0)])
def test_ragged_chunks_whose_last_tiles_are_half_empty(hd, window, sinks):
    """Chunks that end within the first half of a tile pair, several of them in every CTA's share:
    the pair's second tile sits an item out and begins the next one with keys that no row sees."""
    g = torch.Generator().manual_seed(hd + window)
    q = (70 + 64 * torch.randint(0, 3, (48,), generator=g) + torch.randint(0, 20, (48,), generator=g)).tolist()
    n = [x + int(m) for x, m in zip(q, torch.randint(0, 700 if window else 40, (48,), generator=g))]
    st = Step(q, n, 32, 8, hd=hd, ps=32, window=window, sinks=sinks, seed=3)
    check_repeatedly(st, "half-empty tiles")


# ---------------------------------------------------------------------------- many pieces of a tile
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q,n,H,pieces", [(1, 32768, 4, 70), (1, 9000, 2, 33), (5, 40000, 12, 70), (48, 20000, 6, 40)])
def test_one_request_over_a_long_cache(q, n, H, pieces, dtype):
    """One tile per kv head, cut into more pieces than a warp has lanes, whose join takes several turns."""
    st = Step([q], [n], H, 2 if H > 2 else 1, ps=128, dtype=dtype, seed=9)
    st.k[0][::97] *= 2                                       # maxima in every piece
    plan = st.plan()._c
    assert max(x.slots / x.n_merges for x in plan.attn if x.n_merges) >= pieces
    check_repeatedly(st, "long cache", times=5)


# ---------------------------------------------------------------------------- shared pages
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("q", [1, 40, 150])
def test_weights_of_a_shared_prefix_add_up(dtype, q):
    """Every sequence's table begins with the same pages; the weights that all of them give those keys
    are there afterwards, those of a sequence's own pages in the same bits every time."""
    B, shared, ps = 12, 10, 32
    st = Step([q] * B, [400 + q + 13 * b for b in range(B)], 8, 2, ps=ps, dtype=dtype, seed=4)
    st.table[:, :shared] = st.table[0, :shared]
    for b in range(1, B):
        st.k[b][:shared * ps], st.v[b][:shared * ps] = st.k[0][:shared * ps], st.v[0][:shared * ps]
    k, v = st.pages()
    plan = st.plan()
    out, lse = K.paged_attention(st.q, k, v, st.table, plan)
    o, l, tol_o, tol_l = st.exact()
    within(out, o, tol_o, "out")
    within(lse, l, tol_l, "lse")
    start = torch.rand(k.shape[:3], generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    want, tol = st.exact_mass(lse, start)
    own = torch.ones(len(k), dtype=torch.bool, device="cuda")
    own[st.table[0, :shared].long()] = False
    first = None
    for _ in range(8):
        mass = start.clone()
        K.paged_attention_mass(st.q, k, st.table, lse, mass, plan)
        within(mass, want, tol, "weights")
        first = mass if first is None else first
        assert torch.equal(mass[own], first[own])
    plan.check()


# ---------------------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("window,block", [(0, 1), (0, 8), (30, 1)])
def test_a_token_that_is_not_finite_spoils_the_keys_it_sees_only(dtype, window, block):
    """Next to it in the tile are tokens that see other keys; a token whose lse is -inf adds nothing."""
    st = Step([1, 90, 24], [150, 200, 170], 8, 2, ps=16, dtype=dtype, window=window, block=block, seed=5)
    st.q[30, 5], st.q[100, 2, 7] = math.nan, math.inf
    k, v = st.pages()
    plan = st.plan()
    out, lse = K.paged_attention(st.q, k, v, st.table, plan)
    hit = torch.zeros(lse.shape, dtype=torch.bool, device="cuda")
    hit[30, 5] = hit[100, 2] = True
    assert torch.equal(lse.isnan(), hit) and torch.equal(out.isnan().all(2), hit) and torch.equal(out.isnan().any(2), hit)
    lse[50, 1] = lse[0] = -math.inf
    start = torch.rand(k.shape[:3], generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    mass = start.clone()
    K.paged_attention_mass(st.q, k, st.table, lse, mass, plan)
    plan.check()
    want, tol = st.exact_mass(lse, start)
    assert bool(want.isnan().any())
    within(mass, want, tol, "weights")


@pytest.mark.parametrize("dtype,hd", [(BF, 128), (BF, 64), (F32, 128), (F32, 64)])
@pytest.mark.parametrize("q,n,mask", [
    ([100, 20, 1, 33], [400, 150, 300, 33], {}), ([100, 64, 7], [300, 64, 500], dict(block=32)),
    ([70, 9], [200, 90], dict(block=0)), ([150, 20, 1], [500, 300, 90], dict(window=30, sinks=2)),
    ([40], [3000], {}), ([7, 5], [2000, 1500], {}), ([300], [2600], dict(window=700, sinks=1))])
def test_values_that_are_not_finite_stay_out_of_tokens_that_do_not_see_them(q, n, mask, dtype, hd):
    """Infinite and NaN values in keys that some tokens of a tile see and others do not: the ones
    have what the formula gives, the others finite outputs."""
    st = Step(q, n, 8, 2, hd=hd, ps=32, dtype=dtype, seed=7, **mask)
    for b, (ql, nl) in enumerate(zip(q, n)):
        base, v = nl - ql, st.v[b]
        v[base + ql // 3, :, 3] = math.nan
        v[base + ql // 2, 1, 5], v[base + ql // 2, :, 6] = math.inf, -math.inf
        v[base + 2 * ql // 3, 0, 6] = math.inf
        v[nl - 1, 0] = math.inf
        v[1, 1, 11] = -math.inf
        if base > 10:
            v[base - 5, :, 9] = math.nan
    k, v = st.pages()
    plan = st.plan()
    out, lse = K.paged_attention(st.q, k, v, st.table, plan)
    plan.check()
    want, l, tol_o, tol_l = st.exact()
    within(out, want, tol_o, "out")
    within(lse, l, tol_l, "lse")


# ---------------------------------------------------------------------------- eviction
def evict(lens, keep, ps=64, Hkv=2, hd=64, sinks=0, recent=0, dtype=BF, seed=0, mass=None, room=0):
    """An eviction against a sort of the weights: positions kept, rows and weights moved.  The
    destination table holds what stays, and ``room`` pages more."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    budget = [keep] * len(lens) if isinstance(keep, int) else keep
    stay = [min(n, m) for n, m in zip(lens, budget)]
    need, into = ([-(-n // ps) for n in x] for x in (lens, stay))
    order = torch.randperm(sum(need) + sum(into), generator=g, device="cuda").to(torch.int32)
    src = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    dst = torch.full((len(lens), max(into) + room), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (x, y) in enumerate(zip(need, into)):
        src[b, :x], dst[b, :y] = order[at:at + x], order[at + x:at + x + y]
        at += x + y
    k, v = (torch.randn(len(order), Hkv, ps, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
    if mass is None:
        mass = (torch.rand(len(order), Hkv, ps, generator=g, device="cuda") * 4000).round() / 8
    else:
        mass = mass(torch.rand(len(order), Hkv, ps, generator=g, device="cuda"))
    plan = K.EvictPlan(lens, keep, kv_heads=Hkv, page_size=ps, sinks=sinks, recent=recent)
    gk, gv, gm = k.clone(), v.clone(), mass.clone()
    kept = K.paged_evict(gk, gv, gm, src, dst, plan)
    plan.check()
    assert kept.shape == (len(lens), Hkv, max(stay))
    kept = kept.cpu()
    for b, n in enumerate(lens):
        j, r = torch.arange(n), torch.arange(stay[b])
        for h in range(Hkv):
            w = mass[src[b, j // ps].long().cpu(), h, j % ps].cpu()
            rank = torch.where(w.isnan(), math.inf, w.double().clamp(max=1e300)).tolist()
            want = evict_positions(rank, budget[b], sinks, recent)
            assert kept[b, h].tolist() == want + [-1] * (kept.shape[2] - len(want))
            x = torch.tensor(want, dtype=torch.long)
            a, c = (src[b, x // ps].long(), h, x % ps), (dst[b, r // ps].long(), h, r % ps)
            k[c], v[c], mass[c] = k[a], v[a], mass[a]
    assert torch.equal(gk, k) and torch.equal(gv, v)
    assert torch.equal(gm.view(torch.int32), mass.view(torch.int32))


@pytest.mark.parametrize("lens,keep,sinks,recent", [
    ([800, 100], [33, 500], 4, 8), ([10, 5000], [4096, 100], 0, 0), ([64, 65, 3], [64, 3, 900], 1, 1),
    ([50, 700], [1 << 30, 40], 0, 40), ([20, 30], [500, 40], 90, 90)])
def test_budgets_that_are_larger_on_shorter_sequences(lens, keep, sinks, recent):
    evict(lens, keep, sinks=sinks, recent=recent)
    evict(lens, keep, sinks=sinks, recent=recent, ps=16, room=3)


@pytest.mark.parametrize("kind", ["zeros", "nan"])
@pytest.mark.parametrize("n,keep", [(300, 120), (9000, 3000)])
def test_zeros_and_nans_of_either_sign(kind, n, keep):
    """-0 and 0 are equal weights, of which the lowest positions stay; a NaN ranks above +inf
    whatever its sign."""
    def mass(u):
        if kind == "zeros":
            return torch.where(u < 0.1, u, torch.where(u < 0.5, 0.0, -0.0))
        bad = torch.where(u < 0.1, 0x7fc00000, torch.where(u < 0.2, -0x400000, 0x7f800000))    # NaN, -NaN, inf
        return torch.where(u < 0.5, bad.to(torch.int32).view(torch.float32), u)
    evict([n, n // 2], keep, sinks=2, recent=7, mass=mass)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_more_keys_than_a_selecting_block_holds(dtype):
    """So many heads that each is one CTA's, some with more keys than its registers hold (8192)."""
    lens = [20000, 8300, 16385, 9000, 12000, 700, 8192, 8193, 30000, 1]
    evict(lens, 5000, Hkv=8, sinks=3, recent=100, dtype=dtype)


# ---------------------------------------------------------------------------- the cache
def filled_cache(lens, num_pages, layers=2, H=4, Hkv=2, hd=64, seed=0):
    """A cache whose sequences have these lengths, with random keys, values and weights."""
    from specfold_b200 import PagedKVCache
    cache = PagedKVCache(layers, Hkv, hd, num_pages=num_pages, page_size=16, dtype=F32, track_mass=True)
    g = torch.Generator(device="cuda").manual_seed(seed)
    seqs = [cache.add() for _ in lens]
    step = cache.step(seqs, lens, heads=H)
    for x in range(layers):
        k, v = (torch.randn(sum(lens), Hkv, hd, generator=g, device="cuda") for _ in range(2))
        cache.append(x, k, v, step)
    step.check()
    cache._mass.copy_(torch.rand(cache._mass.shape, generator=g, device="cuda"))
    return cache, seqs


def contents(cache, seq):
    """[layers, keys and values, Hkv, length, hd] and the weights of a sequence"""
    pages, n = torch.tensor(cache.pages(seq), dtype=torch.long, device="cuda"), cache.length(seq)
    rows = cache._store[:, :, pages].transpose(2, 3).flatten(3, 4)[:, :, :, :n]
    return rows.clone(), cache._mass[:, pages].transpose(1, 2).flatten(2, 3)[..., :n].clone()


def test_pages_are_not_lost_when_a_call_fails(monkeypatch):
    cache, (a, b) = filled_cache([100, 40], 30)
    free, pages, before = cache.free_pages, cache.pages(a), contents(cache, a)
    real, calls = K.paged_evict, []

    def fails_in_the_second_layer(*args):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("no")
        return real(*args)

    monkeypatch.setattr(K, "paged_evict", fails_in_the_second_layer)
    with pytest.raises(RuntimeError):
        cache.evict([a, b], 32)
    monkeypatch.setattr(K, "paged_evict", real)
    monkeypatch.setattr(cache, "_table", lambda rows: 1 / 0)
    for call in (lambda: cache.evict([a], 32), lambda: cache.step([a, b], [70, 1], heads=4)):
        with pytest.raises(ZeroDivisionError):
            call()
    monkeypatch.undo()
    assert cache.free_pages == free and cache.pages(a) == pages and cache.length(a) == 100
    assert all(torch.equal(x, y) for x, y in zip(contents(cache, a), before))
    cache.evict([a, b], 32)
    cache.step([a, b], [70, 1], heads=4).check()
    assert len(set(cache._free + cache.pages(a) + cache.pages(b))) == 30


def test_sequences_within_their_budget_stay_where_they_are():
    """An eviction moves, and needs room for, the sequences that are over the budget alone."""
    lens = [100, 40, 32, 0, 33]                              # 7 + 3 + 2 + 0 + 3 pages
    cache, seqs = filled_cache(lens, 15 + 4)                 # room for the two that are cut
    before, pages = [contents(cache, s) for s in seqs], [cache.pages(s) for s in seqs]
    kept = cache.evict(seqs, 40, sinks=2, recent=4)
    assert [cache.length(s) for s in seqs] == [40, 40, 32, 0, 33]
    assert all(cache.pages(s) == p for s, p in zip(seqs[1:], pages[1:])) and cache.free_pages == 19 - 11
    for x in range(2):
        assert kept[x].shape == (5, 2, 40) and kept[x].dtype == torch.int32
        for i, n in enumerate(lens):
            for h in range(2):
                want = evict_positions(before[i][1][x, h].tolist(), 40, 2, 4)
                assert kept[x][i, h].tolist() == want + [-1] * (40 - len(want))
                now = contents(cache, seqs[i])
                assert torch.equal(now[0][x, :, h], before[i][0][x, :, h][:, want])
                assert torch.equal(now[1][x, h], before[i][1][x, h][want])
    kept = cache.evict(seqs, 60, recent=100)                 # nothing to cut: nothing to hold
    assert [k.tolist()[4][0] for k in kept] == [list(range(33)) + [-1] * 7] * 2
    released = cache.add()
    cache.step([released], [70], heads=4).check()
    cache.release(released, 20)
    assert [k.shape for k in cache.evict([released], 80)] == [(1, 2, 70)] * 2
    with pytest.raises(ValueError, match="released"):
        cache.evict([released], 60)
    a, b = seqs[0], seqs[2]
    kept = cache.evict([a, b], [50, 7])                      # budgets of their own
    assert (cache.length(a), cache.length(b)) == (40, 7)
    assert kept[0].shape == (2, 2, 40) and kept[0][0, 1].tolist() == list(range(40)) and int(kept[0][1, 0, 7]) == -1
    with pytest.raises(ValueError, match="budgets"):
        cache.evict([a, b], [50])


def test_a_value_that_is_not_finite_holds_nobody_up():
    """One NaN late in a chunk over a long cache, and one in a long cache of single tokens: no wait of
    the kernels runs out, and the tokens before it stay finite."""
    st = Step([2048, 1, 1], [131072, 3000, 131072], 16, 8, ps=256, seed=8)
    st.v[0][131072 - 1000, :, 3] = math.nan
    st.v[2][700, :, 5] = math.nan
    k, v = st.pages()
    plan = st.plan()
    out, lse = K.paged_attention(st.q, k, v, st.table, plan)
    plan.check()
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[1048:2048, :, 3] = hit[2049, :, 5] = True
    assert torch.equal(out.isnan(), hit) and bool(lse.isfinite().all())

"""The paged cache's kernels against their definitions in float64 (paged_reference.py)."""
import math

import pytest
import torch

from specfold_b200 import _lib
from specfold_b200 import kernels as K
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32

# name: (q_lens, kv_lens, H, Hkv, more)
SHAPES = {
    "one token": ([1], [1], 4, 2, {}),
    "one key more than a block": ([1], [129], 4, 2, {}),
    "tokens": ([1, 1, 1, 1], [777, 128, 1, 300], 12, 2, dict(ps=16)),
    "tokens, idle sequences": ([0, 1, 0, 1], [50, 60, 0, 700], 28, 4, {}),
    "all idle": ([0, 0], [50, 0], 4, 2, {}),
    "two tokens, 16 heads a group": ([2], [333], 16, 1, {}),
    "block-causal": ([32, 64], [700, 64], 28, 4, dict(block=32, ps=32)),
    "a block cut by the chunk's end": ([33, 17], [200, 17], 4, 4, dict(block=32, ps=16)),
    "no mask": ([40, 3], [150, 260], 8, 2, dict(block=0)),
    "chunk": ([150], [400], 28, 4, {}),
    "ragged chunks": ([130, 1, 61, 7], [130, 513, 300, 7], 12, 2, dict(ps=128)),
    "chunk, group of 5": ([129], [257], 40, 8, dict(ps=256)),
    "more tokens than keys": ([9, 70], [4, 30], 4, 2, {}),
    "more tokens than keys, no mask": ([9, 70], [4, 0], 4, 2, dict(block=0)),
    "window": ([1, 1, 1], [1000, 90, 513], 28, 4, dict(window=100)),
    "window of one": ([1, 20], [300, 290], 4, 2, dict(window=1, ps=16)),
    "window and sinks": ([1, 150, 33], [900, 700, 35], 12, 2, dict(window=130, sinks=4, ps=16)),
    "sinks past a block": ([70], [900], 4, 1, dict(window=64, sinks=200)),
    "sinks meet the window": ([100], [260], 8, 2, dict(window=150, sinks=40)),
    "window, block-causal": ([64], [640], 8, 2, dict(window=40, sinks=1, block=32)),
    "token-major pool": ([1, 66], [200, 190], 8, 2, dict(layout="token")),
    "head_dim 64": ([1, 1, 140], [300, 64, 450], 4, 2, dict(hd=64, ps=32)),
    "head_dim 64, window": ([200, 2], [450, 300], 8, 1, dict(hd=64, window=77, sinks=3)),
    "sharp softmax": ([3, 80], [400, 300], 8, 2, dict(spread=40.0)),
}


def plan_of(bt, **kw):
    return K.PagedPlan(bt.q_lens, bt.kv_lens, heads=bt.H, kv_heads=bt.Hkv, head_dim=bt.hd,
                       page_size=bt.ps, dtype=bt.dtype, block=bt.block, window=bt.window,
                       sinks=bt.sinks, device="cuda", **kw)


def batch(name, dtype):
    q, n, H, Hkv, kw = SHAPES[name]
    return ref.make_batch(q, n, H, Hkv, dtype=dtype, seed=len(name), **kw)


def within(got, want, tol, what):
    got = got.double().cpu()
    assert bool((torch.isfinite(got) == torch.isfinite(want)).all()), f"{what}: finite elsewhere"
    inf = ~torch.isfinite(want)
    assert torch.equal(got[inf], want[inf]), what
    over = ((got - want).abs() - tol)[~inf]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float(over.max()):.3e} over its bound"


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", list(SHAPES))
def test_attention_and_mass(name, dtype):
    bt = batch(name, dtype)
    plan = plan_of(bt)
    q, k, v, table = bt.queries(bt.wide.cuda()), bt.k.cuda(), bt.v.cuda(), bt.table.cuda()
    assert q.shape[0] < 2 or not q.is_contiguous()
    out, lse = K.paged_attention(q, k, v, table, plan)
    plan.check()
    o, l, tol_o, tol_l = ref.attention(bt)
    within(out, o, tol_o, f"{name}: out")
    within(lse, l, tol_l, f"{name}: lse")
    mass = bt.mass.cuda()
    K.paged_attention_mass(q, k, table, lse, mass, plan)
    plan.check()
    m, tol = ref.mass(bt, lse.cpu())
    within(mass, m, tol, f"{name}: mass")
    # what no token sees keeps its bits, and the same call gives the same ones
    assert torch.equal(mass.cpu()[tol == 0], bt.mass[tol == 0])
    again, mass2 = K.paged_attention(q, k, v, table, plan), bt.mass.cuda()
    K.paged_attention_mass(q, k, table, lse, mass2, plan)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse) and torch.equal(mass2, mass)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_long_cache_past_32_bit_offsets(dtype):
    """Pages whose rows start beyond 2^31 elements of the pool."""
    hd, ps, Hkv = 128, 256, 8
    pages = (1 << 31) // (hd * ps * Hkv) + 40
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.empty(pages, Hkv, ps, hd, dtype=dtype, device="cuda")
    v = torch.empty_like(k)
    ids = torch.tensor([[pages - 1, 0, pages - 30, pages - 7]], dtype=torch.int32, device="cuda")
    small = torch.randn(4, 2, Hkv, ps, hd, generator=g, device="cuda").to(dtype)
    k[ids[0].long()], v[ids[0].long()] = small[:, 0], small[:, 1]
    q = torch.randn(2, 16, hd, generator=g, device="cuda").to(dtype)
    kw = dict(heads=16, kv_heads=Hkv, head_dim=hd, page_size=ps, dtype=dtype)
    plan = K.PagedPlan([2], [4 * ps - 3], **kw)
    far = K.paged_attention(q, k, v, ids, plan)
    near_ids = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    near = K.paged_attention(q, small[:, 0].contiguous(), small[:, 1].contiguous(), near_ids, plan)
    assert torch.equal(far[0], near[0]) and torch.equal(far[1], near[1])
    K.paged_kv_append(k, v, q[:, :Hkv], q[:, Hkv:], ids, plan)
    plan.check()
    assert torch.equal(k[pages - 7, :, ps - 5:ps - 3], q[:, :Hkv].transpose(0, 1))
    assert torch.equal(v[pages - 7, :, ps - 5:ps - 3], q[:, Hkv:].transpose(0, 1))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("hd,ps,layout", [(128, 64, "page"), (64, 16, "page"), (128, 32, "token")])
def test_append(dtype, hd, ps, layout):
    bt = ref.make_batch([5, 0, 1, 40], [5, 9, 65, 100], 4, 2, hd=hd, ps=ps, dtype=dtype, layout=layout,
                        block=0)
    plan = plan_of(bt)
    T = plan.tokens
    wide = torch.randn(T, 3, 2, hd, generator=torch.Generator().manual_seed(1)).to(dtype)
    k, v, mass = bt.k.clone(), bt.v.clone(), bt.mass.clone()
    gk, gv, gm = bt.k.cuda(), bt.v.cuda(), bt.mass.cuda()
    if layout == "token":
        gk, gv = (x.cuda().transpose(1, 2).contiguous().transpose(1, 2) for x in (bt.k, bt.v))
    dev = wide.cuda()
    K.paged_kv_append(gk, gv, dev[:, 0], dev[:, 2], bt.table.cuda(), plan, mass_pages=gm)
    plan.check()
    t = 0
    for b, (ql, n) in enumerate(zip(bt.q_lens, bt.kv_lens)):
        for i in range(ql):
            pos = n - ql + i
            page = bt.table[b, pos // ps]
            k[page, :, pos % ps], v[page, :, pos % ps] = wide[t, 0], wide[t, 2]
            mass[page, :, pos % ps] = 0
            t += 1
    for got, want in ((gk, k), (gv, v), (gm, mass)):
        assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))


EVICT = {
    "ties and zeros": ([300, 40, 0, 1000], 64, 4, 16, "coarse"),
    "all equal": ([500, 129], 100, 0, 10, "equal"),
    "only sinks and recent": ([300], 20, 4, 16, "any"),
    "only the heaviest": ([700, 64], 50, 0, 0, "any"),
    "one stays": ([90], 1, 0, 0, "any"),
    "none stays": ([90], 0, 0, 0, "any"),
    "all but one": ([257], 256, 3, 7, "any"),
    "nothing to evict": ([30, 64], 64, 60, 60, "any"),
    "negative, infinite and NaN weights": ([400], 100, 1, 5, "odd"),
    "long": ([5000, 40000], 3000, 16, 256, "coarse"),
    "budgets of their own": ([800, 800, 300], [500, 33, 300], 4, 8, "any"),
}


@pytest.mark.parametrize("dtype,hd,ps", [(BF, 128, 64), (BF, 64, 16), (F32, 128, 32), (F32, 64, 256)])
@pytest.mark.parametrize("name", list(EVICT))
def test_evict(name, dtype, hd, ps):
    lens, keep, sinks, recent, kind = EVICT[name]
    Hkv, B = 2, len(lens)
    budget = keep if isinstance(keep, list) else [keep] * B
    g = torch.Generator().manual_seed(len(name) + hd)
    need = [-(-n // ps) for n in lens]
    into = [-(-min(n, m) // ps) for n, m in zip(lens, budget)]
    pool = sum(need) + sum(into) + 2
    order = torch.randperm(pool, generator=g).to(torch.int32)
    src = torch.full((B, max(need) + 1), -1, dtype=torch.int32)
    dst = torch.full((B, max(into + [1])), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        src[b, :need[b]] = order[at:at + need[b]]
        dst[b, :into[b]] = order[at + need[b]:at + need[b] + into[b]]
        at += need[b] + into[b]
    k = torch.randn(pool, Hkv, ps, hd, generator=g).to(dtype)
    v = torch.randn(pool, Hkv, ps, hd, generator=g).to(dtype)
    mass = torch.rand(pool, Hkv, ps, generator=g).exp()
    if kind == "coarse":
        mass = (mass * 8).round() / 8 * (torch.rand(mass.shape, generator=g) < 0.7)
    elif kind == "equal":
        mass.fill_(0.25)
    elif kind == "odd":
        mass = torch.where(torch.rand(mass.shape, generator=g) < 0.3, -mass, mass)
        mass[torch.rand(mass.shape, generator=g) < 0.05] = math.inf
        mass[torch.rand(mass.shape, generator=g) < 0.05] = -math.inf
        mass[torch.rand(mass.shape, generator=g) < 0.02] = math.nan
    plan = K.EvictPlan(lens, keep, kv_heads=Hkv, page_size=ps, sinks=sinks, recent=recent)
    gk, gv, gm = k.cuda(), v.cuda(), mass.cuda()
    kept = K.paged_evict(gk, gv, gm, src.cuda(), dst.cuda(), plan).cpu()
    plan.check()
    assert kept.shape == (B, Hkv, max(min(n, m) for n, m in zip(lens, budget)))
    for b in range(B):
        for h in range(Hkv):
            w = [float(mass[src[b, j // ps], h, j % ps]) for j in range(lens[b])]
            rank = [math.inf if math.isnan(x) else min(x, 1e300) for x in w]
            want = ref.evict_positions(rank, budget[b], sinks, recent)
            assert kept[b, h].tolist() == want + [-1] * (kept.shape[2] - len(want))
            for r, j in enumerate(want):
                a, c = (src[b, j // ps], h, j % ps), (dst[b, r // ps], h, r % ps)
                k[c], v[c], mass[c] = k[a], v[a], mass[a]
    assert torch.equal(gk.cpu(), k) and torch.equal(gv.cpu(), v)
    assert torch.equal(gm.cpu().nan_to_num(9.0), mass.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_a_page_outside_the_pool_is_reported(dtype):
    bt = ref.make_batch([1, 70], [200, 130], 8, 2, dtype=dtype)
    plan = plan_of(bt)
    table = bt.table.clone()
    table[0, 1] = bt.k.shape[0]
    k, v, mass = (x.nan_to_num(0.0).cuda() for x in (bt.k, bt.v, bt.mass))
    K.paged_attention(bt.queries(bt.wide.cuda()), k, v, table.cuda(), plan)
    with pytest.raises(_lib.SpecFoldError, match="index out of range"):
        plan.check()
    table = bt.table.clone()
    table[1, 2] = -5
    plan = plan_of(bt)
    before = k.clone()
    K.paged_kv_append(k, v, k.new_ones(71, 2, 128), k.new_ones(71, 2, 128), table.cuda(), plan)
    with pytest.raises(_lib.SpecFoldError, match="index out of range"):
        plan.check()
    assert torch.equal(k[bt.table[1, 2]], before[bt.table[1, 2]])     # nothing was written there
    # weights: those of the keys on the missing page are left out, no other page gets them
    plan, want, got = plan_of(bt), mass.clone(), mass.clone()
    q, lse = bt.queries(bt.wide.cuda()), torch.full((71, 8), 3.0, device="cuda")
    K.paged_attention_mass(q, k, bt.table.cuda(), lse, want, plan_of(bt))
    K.paged_attention_mass(q, k, table.cuda(), lse, got, plan)
    with pytest.raises(_lib.SpecFoldError, match="index out of range"):
        plan.check()
    gone = bt.table[1, 2].item()
    assert torch.equal(got[gone], mass[gone])
    keep = torch.arange(mass.shape[0]) != gone
    assert torch.equal(got[keep], want[keep])


def test_eviction_lengths_beyond_the_hosts_bounds_are_cut():
    """Lengths on the device that contradict what the call was sized for are reported, and
    nothing outside its buffers is touched."""
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(16, 2, 16, 64, generator=g, device="cuda")
    v, mass = torch.randn_like(k), torch.rand(16, 2, 16, generator=g, device="cuda")
    src = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    dst = torch.arange(8, 14, dtype=torch.int32, device="cuda").view(2, 3)
    for lens in ([[900, 40], [64, 40]], [[64, 900], [64, 40]], [[64, 3], [64, 40]], [[-5, 40], [64, 40]]):
        plan = K.EvictPlan([64, 64], 40, kv_heads=2, page_size=16, sinks=4, recent=4)
        plan._lens.copy_(torch.tensor(lens, dtype=torch.int32))
        spare = k[14:].clone()
        kept = K.paged_evict(k, v, mass, src, dst, plan)
        with pytest.raises(_lib.SpecFoldError, match="index out of range"):
            plan.check()
        assert torch.equal(k[14:], spare)
        assert int(kept.max()) < 64 and int(kept.min()) >= -1
        assert kept[1, 0].tolist()[:4] == [0, 1, 2, 3]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_infinite_scores_stay_in_their_rows(dtype):
    """A key of one kv head that overflows makes the rows that see it NaN or infinite, as the
    formula does, and no others."""
    bt = ref.make_batch([40, 1], [200, 200], 8, 2, dtype=dtype)
    clean = K.paged_attention(bt.queries(bt.wide.cuda()), bt.k.cuda(), bt.v.cuda(), bt.table.cuda(), plan_of(bt))
    k = bt.k.clone()
    k[bt.table[0, 180 // bt.ps], 1, 180 % bt.ps] = math.inf          # token 20 on sees key 180
    out, lse = K.paged_attention(bt.queries(bt.wide.cuda()), k.cuda(), bt.v.cuda(), bt.table.cuda(), plan_of(bt))
    hit = torch.zeros(41, 8, dtype=torch.bool, device="cuda")
    hit[20:40, 4:] = True
    assert torch.equal(out[~hit], clean[0][~hit]) and torch.equal(lse[~hit], clean[1][~hit])
    assert not bool(torch.isfinite(lse[hit]).any()) or not bool(torch.isfinite(out[hit]).all())


def test_another_stream_and_given_outputs():
    bt = ref.make_batch([1, 100], [900, 400], 12, 2)
    q, k, v, table = bt.queries(bt.wide.cuda()), bt.k.cuda(), bt.v.cuda(), bt.table.cuda()
    want = K.paged_attention(q, k, v, table, plan_of(bt))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    plan = plan_of(bt)                       # made on the current stream, used on another
    with torch.cuda.stream(side):
        out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
        got = K.paged_attention(q, k, v, table, plan, out=out, lse=lse)
    side.synchronize()
    assert got[0] is out and got[1] is lse
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_captured_step_is_replayed_on_new_values():
    """The calls neither allocate nor synchronise when their outputs are given."""
    bt = ref.make_batch([1, 1, 90], [300, 31, 190], 12, 2)
    q, k, v, table = bt.queries(bt.wide.cuda()), bt.k.cuda(), bt.v.cuda(), bt.table.cuda()
    mass = bt.mass.cuda()
    plan = plan_of(bt)
    out, lse = K.paged_attention(q, k, v, table, plan)
    K.paged_attention_mass(q, k, table, lse, mass, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.paged_attention(q, k, v, table, plan, out=out, lse=lse)
        K.paged_attention_mass(q, k, table, lse, mass, plan)
    q2 = torch.randn(q.shape, generator=torch.Generator().manual_seed(9)).to(q.dtype).cuda()
    want = K.paged_attention(q2, k, v, table, plan)
    want_mass = bt.mass.cuda()
    K.paged_attention_mass(q2, k, table, want[1], want_mass, plan)
    q.copy_(q2)
    mass.copy_(bt.mass)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(mass, want_mass)


def test_refusals():
    bt = ref.make_batch([1, 9], [90, 30], 4, 2, block=0)
    q, k, v, table, plan = bt.queries(bt.wide.cuda()), bt.k.cuda(), bt.v.cuda(), bt.table.cuda(), plan_of(bt)
    mass, lse = bt.mass.cuda(), torch.zeros(10, 4, device="cuda")
    with pytest.raises(ValueError):
        K.paged_attention(q[:5], k, v, table, plan)                   # tokens
    with pytest.raises(ValueError):
        K.paged_attention(q.float(), k, v, table, plan)               # dtype
    with pytest.raises(ValueError):
        K.paged_attention(q, k, v[:, :1], table, plan)                # pools differ
    with pytest.raises(ValueError):
        K.paged_attention(q, k, v, table.long(), plan)                # table dtype
    with pytest.raises(ValueError):
        K.paged_attention(q.cpu(), k, v, table, plan)                 # device
    with pytest.raises(_lib.SpecFoldError, match="does not hold"):
        K.paged_attention(q, k, v, table[:, :1], plan)                # table too narrow
    with pytest.raises(_lib.SpecFoldError, match="scale"):
        K.paged_attention(q, k, v, table, plan, scale=0.0)
    with pytest.raises(_lib.SpecFoldError, match="aligned"):
        wide = torch.zeros(10, 4 * 128 + 1, dtype=BF, device="cuda")
        K.paged_attention(wide[:, 1:].view(10, 4, 128), k, v, table, plan)
    with pytest.raises(ValueError):
        K.paged_attention_mass(q, k, table, lse, mass.double(), plan)
    with pytest.raises(ValueError):
        K.paged_attention_mass(q, k, table, lse.half(), mass, plan)
    light = K.PagedPlan([1, 9], [90, 30], heads=4, kv_heads=2, head_dim=128, page_size=64, block=0, mass=False)
    K.paged_attention(q, k, v, table, light)
    with pytest.raises(_lib.SpecFoldError, match="made without"):
        K.paged_attention_mass(q, k, table, lse, mass, light)
    more = K.PagedPlan([5], [3], heads=4, kv_heads=2, head_dim=128, page_size=64)
    new = torch.zeros(5, 2, 128, dtype=BF, device="cuda")
    with pytest.raises(_lib.SpecFoldError, match="more new tokens"):
        K.paged_kv_append(k, v, new, new, table[:1], more)
    evict = K.EvictPlan([90, 30], 70, kv_heads=2, page_size=64)
    with pytest.raises(_lib.SpecFoldError, match="destination"):
        K.paged_evict(k, v, mass, table, table[:, :1], evict)


# ---------------------------------------------------------------------------- the cache and its use
def test_cache_steps_match_a_contiguous_cache():
    """Chunks, tokens and idle sequences over several steps, against attention over the sequence's
    whole history; pages come back when a sequence ends."""
    from specfold_b200 import PagedKVCache
    H, Hkv, hd = 8, 2, 64
    cache = PagedKVCache(2, Hkv, hd, num_pages=40, page_size=16, dtype=F32)
    g = torch.Generator(device="cuda").manual_seed(0)
    a, b, c = cache.add(), cache.add(), cache.add()
    past = {s: [[torch.empty(0, Hkv, hd, device="cuda")] * 2 for _ in range(2)] for s in (a, b, c)}
    for seqs, q_lens in (([a], [70]), ([b, a], [33, 1]), ([a, c, b], [1, 5, 0]), ([c, a, b], [20, 1, 1])):
        step = cache.step(seqs, q_lens, heads=H)
        T = sum(q_lens)
        for layer in range(2):
            q, k, v = (torch.randn(T, n, hd, generator=g, device="cuda") for n in (H, Hkv, Hkv))
            cache.append(layer, k, v, step)
            out, _ = cache.attend(layer, q, step)
            t = 0
            for s, n in zip(seqs, q_lens):
                kk, vv = (torch.cat((p, x[t:t + n])) for p, x in zip(past[s][layer], (k, v)))
                past[s][layer] = [kk, vv]
                if n:
                    want = torch.nn.functional.scaled_dot_product_attention(
                        q[t:t + n].transpose(0, 1).double()[None],
                        kk.transpose(0, 1).repeat_interleave(H // Hkv, 0).double()[None],
                        vv.transpose(0, 1).repeat_interleave(H // Hkv, 0).double()[None],
                        attn_mask=torch.ones(n, len(kk), dtype=torch.bool, device="cuda").tril(len(kk) - n))
                    assert (out[t:t + n].double() - want[0].transpose(0, 1)).abs().max() < 1e-5
                t += n
        step.check()
    assert [cache.length(s) for s in (a, b, c)] == [73, 34, 25]
    assert cache.free_pages == 40 - 5 - 3 - 2
    cache.remove(b)
    assert cache.free_pages == 40 - 5 - 2
    with pytest.raises(MemoryError):
        cache.step([c], [40 * 16], heads=H)
    assert cache.length(c) == 25 and cache.free_pages == 40 - 5 - 2
    with pytest.raises(ValueError):
        cache.step([a, a], [1, 1], heads=H)
    with pytest.raises(ValueError):
        cache.evict([a], 10)                               # made without track_mass


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
def test_released_pages_are_not_missed(dtype):
    """Pages that fell out of the window are taken by another sequence; the window's results stay
    bit for bit."""
    from specfold_b200 import PagedKVCache
    H, Hkv, hd, window, sinks = 8, 2, 128, 100, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = [torch.randn(500, n, hd, generator=g, device="cuda").to(dtype) for n in (H, Hkv, Hkv)]
    outs = []
    for free in (False, True):
        cache = PagedKVCache(1, Hkv, hd, num_pages=64, page_size=16, dtype=dtype)
        s, at, got = cache.add(), 0, []
        for n in (300, 1, 150, 1, 40):
            step = cache.step([s], [n], heads=H, window=window, sinks=sinks)
            q, k, v = (x[at:at + n] for x in rows)
            cache.append(0, k, v, step)
            got.append(cache.attend(0, q, step))
            step.check()
            at += n
            if free:
                before = cache.free_pages
                assert cache.release(s, window, sinks) == cache.free_pages - before
                other = cache.add()                        # whoever gets the pages fills them
                filler = cache.step([other], [cache.free_pages * 16], heads=H)
                junk = torch.full((filler.plan.tokens, Hkv, hd), float("nan"), device="cuda").to(dtype)
                cache.append(0, junk, junk, filler)
                filler.check()
                cache.remove(other)
        outs.append(got)
        assert not free or (-1 in cache.pages(s) and cache.pages(s)[0] >= 0)
    for (o1, l1), (o2, l2) in zip(*outs):
        assert torch.equal(o1, o2) and torch.equal(l1, l2)


def test_cache_eviction_keeps_what_was_looked_at():
    from specfold_b200 import PagedKVCache
    H, Hkv, hd = 4, 2, 64
    cache = PagedKVCache(2, Hkv, hd, num_pages=40, page_size=16, dtype=F32, track_mass=True)
    g = torch.Generator(device="cuda").manual_seed(2)
    a, b = cache.add(), cache.add()
    step = cache.step([a, b], [200, 30], heads=H)
    for layer in range(2):
        q, k, v = (torch.randn(230, n, hd, generator=g, device="cuda") for n in (H, Hkv, Hkv))
        cache.append(layer, k, v, step)
        _, lse = cache.attend(layer, q, step)
        cache.accumulate(layer, q, lse, step)
    step.check()
    # all rows' weights add up to one each
    total = sum(float(cache._mass[0, p].sum()) for s in (a, b) for p in cache.pages(s))
    assert abs(total - 230 * H) < 1e-2
    free = cache.free_pages
    old = [cache._mass[layer][cache.pages(a)].transpose(0, 1).reshape(Hkv, -1)[:, :200].clone() for layer in range(2)]
    kept = cache.evict([a, b], 64, sinks=4, recent=8)
    assert cache.length(a) == 64 and cache.length(b) == 30 and cache.free_pages == free + 13 - 4
    for layer in range(2):
        for h in range(Hkv):
            want = ref.evict_positions(old[layer][h].tolist(), 64, 4, 8)
            assert kept[layer][0, h].tolist() == want
            assert kept[layer][1, h].tolist() == list(range(30)) + [-1] * 34
            now = cache._mass[layer][cache.pages(a), h].flatten()
            assert torch.equal(now, old[layer][h][want])
    with pytest.raises(ValueError):
        cache.evict([a], 10, sinks=6, recent=5)
    step = cache.step([a, b], [1, 1], heads=H)                # and the sequences go on
    k = torch.randn(2, Hkv, hd, generator=g, device="cuda")
    cache.append(0, k, k, step)
    cache.attend(0, torch.randn(2, H, hd, generator=g, device="cuda"), step)
    step.check()
    assert cache.length(a) == 65


@pytest.mark.parametrize("shape,dtype,tol", [("tiny", F32, 1e-4), ("tiny128", BF, 2e-2)])
def test_serving_example_matches_the_dense_model(shape, dtype, tol):
    """examples/paged_serving.py's decoder, chunk by chunk and token by token next to other
    requests, against the model's own forward over the whole text (fp32 on the CPU)."""
    import importlib.util
    import os
    from specfold_b200 import synthetic as syn
    path = os.path.join(os.path.dirname(os.path.dirname(__file__)), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    dims = syn.SHAPES[shape]
    model = syn.build_model(dims, family="fastdllm", dtype=dtype, seed=3)
    dense = syn.build_model(dims, family="fastdllm", dtype=dtype, seed=3).float()
    g = torch.Generator().manual_seed(4)
    texts = [torch.randint(0, dims.vocab, (n,), generator=g).tolist() for n in (150, 21)]
    dec = ex.PagedDecoder(model.cuda(), dims, num_pages=32, page_size=16)
    a, b = dec.add(), dec.add()
    dec.step([a], [texts[0][:100]])
    dec.step([a, b], [texts[0][100:149], texts[1][:20]])
    got = dec.step([b, a], [texts[1][20:], texts[0][149:]])
    for row, text in ((1, texts[0]), (0, texts[1])):
        with torch.no_grad():
            want = dense(torch.tensor([text])).logits[0, -1]
        off = (got[row].float().cpu() - want).abs().max() / want.abs().max()
        assert off <= tol, float(off)
    out = ex.serve(ex.PagedDecoder(model, dims, num_pages=64, page_size=16, track_mass=True),
                   texts + [texts[0][:7]], 12, budget=64)
    assert [len(o) for o in out] == [12] * 3

"""The paged cache without a device: how a plan covers its step, and what is refused."""
import ctypes
import random

import pytest
import torch

from specfold_b200 import _lib
from specfold_b200 import kernels as K
from tests import paged_reference as ref

ITEM, MERGE, MASS, MASS_MERGE = 12, 8, 12, 8                      # words of the plan's records


def build(q_lens, kv_lens, **kw):
    lib = _lib.load()
    c = _lib.SfPagedPlan(B=len(q_lens), **kw)
    q, n = (torch.tensor(x, dtype=torch.int32) for x in (q_lens, kv_lens))
    cap = lib.sf_paged_plan_words(ctypes.byref(c), q.data_ptr(), n.data_ptr())
    assert cap > 0, lib.sf_last_error()
    words = torch.full((cap,), -77, dtype=torch.int32)
    assert lib.sf_paged_plan_build(ctypes.byref(c), q.data_ptr(), n.data_ptr(), words.data_ptr(), cap) == 0
    assert c.words <= cap
    return c, words.tolist()


def visible_blocks(q, n, i, block, window, sinks, keys=128):
    """Blocks of 128 (or ``keys``) keys that token i sees a key of."""
    hi = n if block == 0 else min(n, n - q + (i // block + 1) * block)
    lo = max(0, n - q + i - window + 1) if window else 0
    out = set()
    for b in range(-(-max(hi, 0) // keys)):
        a, e = b * keys, min(hi, b * keys + keys)
        if max(a, lo) < e or (window and a < min(sinks, e)):
            out.add(b)
    return out


@pytest.mark.parametrize("seed", range(60))
def test_a_plan_covers_every_row_and_key_once(seed):
    rng = random.Random(seed)
    Hkv, G = rng.choice([1, 2, 4]), rng.choice([1, 2, 5, 6, 7, 8, 16])
    block, window = rng.choice([0, 1, 1, 7, 32]), rng.choice([0, 0, 1, 50, 300, 1000])
    sinks = rng.choice([0, 1, 4, 200]) if window else 0
    q = [rng.choice([0, 1, 1, 5, 64, rng.randint(1, 700)]) for _ in range(rng.randint(0, 6))]
    n = [rng.choice([0, 1, 127, 128, 129, 3000]) if rng.random() < 0.3 else x + rng.randint(0, 2500)
         for x in q]
    c, w = build(q, n, dtype=rng.choice([0, 1]), H=Hkv * G, Hkv=Hkv, hd=128, page_size=64, block=block,
                 window=window, sinks=sinks, sms=rng.choice([1, 4, 148]))
    assert c.T == sum(q) and bool(c.short_chunk) == any(a > b for a, b in zip(q, n))
    assert w[c.tokens:c.tokens + 2 * c.T] == [x for b in range(len(q)) for i in range(q[b])
                                              for x in (b, n[b] - q[b] + i)]
    rows, keys = set(), 128 if c.dtype else 64
    for part in c.attn:
        if part.n_items == 0:
            continue
        first = w[part.first:part.first + part.workers + 1]
        assert first[0] == 0 and first[-1] == part.n_items and first == sorted(first)
        for x, at in enumerate(first[:-1]):
            if at < first[x + 1]:
                assert w[part.heads + ITEM * x:][:ITEM] == w[part.items + ITEM * at:][:ITEM]
            # only a share's first and last item can be pieces of a cut tile
            assert all(w[part.items + ITEM * i + 6] < 0 for i in range(at + 1, first[x + 1] - 1))
        tiles, used = {}, []
        for x in range(part.n_items):
            seq, kvh, t0, nt, i0, i1, slot, sink, lo, q0, ql, kv = w[part.items + ITEM * x:][:ITEM]
            assert (ql, kv, q0) == (q[seq], n[seq], sum(q[:seq])) and 0 < nt * G <= part.rows
            tiles.setdefault((seq, kvh, t0, nt), []).append((i0, i1, slot, sink, lo))
        for (seq, kvh, t0, nt), pieces in tiles.items():
            at = 0
            for i0, i1, slot, _, _ in pieces:
                assert i0 == at and (i1 > i0 or len(pieces) == 1)
                assert (slot >= 0) == (len(pieces) > 1)
                at = i1
                used += [slot] if slot >= 0 else []
            sink, lo = pieces[0][3:]
            blocks = [i if i < sink else i - sink + lo for i in range(at)]
            assert len(set(blocks)) == len(blocks) and all(b * keys < n[seq] for b in blocks)
            for t in range(t0, t0 + nt):
                assert (seq, kvh, t) not in rows
                rows.add((seq, kvh, t))
                assert visible_blocks(q[seq], n[seq], t, block, window, sinks, keys) <= set(blocks)
        assert used == list(range(part.slots))
        merged = [w[part.merges + MERGE * x:][:MERGE] for x in range(part.n_merges)]
        assert [s for m in merged for s in range(m[3], m[3] + m[4])] == used
    assert len(rows) == sum(q) * Hkv
    # weights: pairs of key blocks against tiles of tokens
    per, seen, used = max(1, (128 if c.dtype else 64) // G), {}, []
    for x in range(c.mass.n_items):
        seq, kvh, kb, t0, t1, i0, i1, slot, q0, ql, kv, _ = w[c.mass.items + MASS * x:][:MASS]
        assert (ql, kv, q0) == (q[seq], n[seq], sum(q[:seq])) and kb % 2 == 0 and kb * 128 < kv
        seen.setdefault((seq, kvh, kb), []).append((i0, i1, slot, t0, t1))
        used += [slot] if slot >= 0 else []
    assert used == list(range(c.mass.slots))
    for pieces in seen.values():
        at = 0
        for i0, i1, slot, t0, t1 in pieces:
            assert i0 == at and i1 > i0 and (slot >= 0) == (len(pieces) > 1)
            at = i1
        assert at == -(-(t1 - t0) // per)
    merged = [w[c.mass.merges + MASS_MERGE * x:][:MASS_MERGE] for x in range(c.mass.n_merges)]
    assert [s for m in merged for s in range(m[3], m[3] + m[4])] == used
    for b in range(len(q)):
        for t in range(q[b]):
            for kb in visible_blocks(q[b], n[b], t, block, window, sinks):
                for h in range(Hkv):
                    t0, t1 = seen[b, h, kb // 2 * 2][0][3:]
                    assert t0 <= t < t1


GOOD = dict(dtype=1, H=8, Hkv=2, hd=128, page_size=64, block=1)


@pytest.mark.parametrize("wrong,said", [
    (dict(dtype=2), b"dtype"), (dict(hd=96), b"head_dim"), (dict(H=7), b"heads"), (dict(H=34), b"heads"),
    (dict(Hkv=0), b"heads"), (dict(page_size=8), b"page size"), (dict(page_size=48), b"page size"),
    (dict(page_size=512), b"page size"), (dict(block=-1), b"negative"), (dict(window=-1), b"negative"),
    (dict(sinks=-1), b"negative"), (dict(window=(1 << 30) + 1), b"window")])
def test_plan_refusals(wrong, said):
    lib = _lib.load()
    q = torch.tensor([1], dtype=torch.int32)
    c = _lib.SfPagedPlan(B=1, sms=148, **{**GOOD, **wrong})
    assert lib.sf_paged_plan_words(ctypes.byref(c), q.data_ptr(), q.data_ptr()) == 0
    assert said in lib.sf_last_error()


def test_plan_refuses_lengths_and_room():
    lib = _lib.load()
    c = _lib.SfPagedPlan(B=1, sms=148, **GOOD)
    one, neg, long = (torch.tensor([x], dtype=torch.int32) for x in (1, -1, (1 << 30) + 1))
    ref_ = ctypes.byref(c)
    assert lib.sf_paged_plan_words(ref_, neg.data_ptr(), one.data_ptr()) == 0
    assert lib.sf_paged_plan_words(ref_, one.data_ptr(), long.data_ptr()) == 0
    assert lib.sf_paged_plan_words(ref_, None, one.data_ptr()) == 0
    room = lib.sf_paged_plan_words(ref_, one.data_ptr(), one.data_ptr())
    words = torch.empty(room, dtype=torch.int32)
    assert lib.sf_paged_plan_build(ref_, one.data_ptr(), one.data_ptr(), words.data_ptr(), room - 1) == 1
    assert lib.sf_paged_plan_build(ref_, one.data_ptr(), one.data_ptr(), None, room) == 1
    # a plan that was not built, or has no device memory, is refused before anything is launched
    pool = _lib.SfPagedPool()
    assert lib.sf_paged_attention(ref_, ctypes.byref(pool), 16, 1024, 128, 16, 16, 1.0, None) == 1
    assert lib.sf_paged_plan_build(ref_, one.data_ptr(), one.data_ptr(), words.data_ptr(), room) == 0
    assert lib.sf_paged_attention(ref_, ctypes.byref(pool), 16, 1024, 128, 16, 16, 1.0, None) == 1
    assert b"device memory" in lib.sf_last_error()


def test_evict_refusals():
    lib = _lib.load()
    pool = _lib.SfPagedPool(0x1000, 0x1000, 0x1000, 2 * 64 * 128, 64 * 128, 128, 0x1000, 8, 16, 8)

    def call(dtype=1, dst_width=4, max_len=500, max_keep=200, hd=128, ps=64, sinks=4, recent=16, kept=200):
        return lib.sf_paged_evict(dtype, ctypes.byref(pool), 0x1000, dst_width, dst_width, 0x1000, max_len,
                                  max_keep, 1, 2, hd, ps, sinks, recent, 0x1000, kept, 0x1000, None)

    for wrong in (dict(dtype=5), dict(hd=80), dict(ps=24), dict(sinks=190, recent=20), dict(kept=199),
                  dict(dst_width=3), dict(max_len=513)):
        assert call(**wrong) == 1, wrong
        assert b"paged_evict" in lib.sf_last_error()


def test_the_python_layer_is_device_only():
    kw = dict(heads=4, kv_heads=2, head_dim=128, page_size=64)
    with pytest.raises(ValueError):
        K.PagedPlan([1], [1], device="cpu", **kw)
    with pytest.raises(ValueError):
        K.PagedPlan([1, 1], [1], **kw)
    with pytest.raises(ValueError):
        K.PagedPlan([-1], [1], **kw)
    with pytest.raises(TypeError):
        K.PagedPlan([1], [1], dtype=torch.float16, **kw)
    with pytest.raises(ValueError):
        K.EvictPlan([100], 10, kv_heads=2, page_size=64, sinks=6, recent=5)
    with pytest.raises(ValueError):
        K.EvictPlan([100], 10, kv_heads=2, page_size=64, device="cpu")


def test_reference_eviction_order():
    assert ref.evict_positions([3, 1, 2, 2, 9, 0], 4, 1, 1) == [0, 2, 4, 5]
    assert ref.evict_positions([1, 1, 1, 1], 2, 0, 0) == [0, 1]
    assert ref.evict_positions([1, 1], 5, 9, 9) == [0, 1]

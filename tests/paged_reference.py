"""The paged cache's operators in float64, one sequence, token and head at a time from their
definitions, with bounds on how far a kernel may be off; and batches to run them on."""
import dataclasses
from typing import List

import torch

# Rounding units.  U32: one fp32 rounding.  UW: what a bf16 kernel may lose in a softmax weight
# before it is rounded to bf16 (an exponential good to 14 bits).  UB: one bf16 rounding (8
# significant bits: half a unit of the last one is 2^-8 of the value at most).
U32, UW, UB = 2.0 ** -24, 2.0 ** -14, 2.0 ** -8


@dataclasses.dataclass
class Batch:
    q_lens: List[int]
    kv_lens: List[int]
    H: int
    Hkv: int
    hd: int
    ps: int
    dtype: torch.dtype
    block: int
    window: int
    sinks: int
    wide: torch.Tensor     # [T, (H + 2) * hd]: q is a slice of its rows
    k: torch.Tensor
    v: torch.Tensor
    mass: torch.Tensor
    table: torch.Tensor
    scale: float

    @property
    def q(self) -> torch.Tensor:
        return self.queries(self.wide)

    def queries(self, wide: torch.Tensor) -> torch.Tensor:
        return wide[:, self.hd:(self.H + 1) * self.hd].unflatten(1, (self.H, self.hd))

    def keys(self, pages: torch.Tensor, b: int, h: int) -> torch.Tensor:
        """The cached rows of sequence b, kv head h, in order."""
        n = self.kv_lens[b]
        rows = [pages[self.table[b, j // self.ps], h, j % self.ps] for j in range(n)]
        return torch.stack(rows) if rows else pages[0, h, :0]

    def sees(self, b: int, i: int) -> torch.Tensor:
        """Which of sequence b's keys token i of its chunk sees."""
        q, n = self.q_lens[b], self.kv_lens[b]
        p = n - q + i
        hi = n if self.block == 0 else min(n, n - q + (i // self.block + 1) * self.block)
        j = torch.arange(n)
        see = j < hi
        if self.window:
            see &= (j > p - self.window) | (j < self.sinks)
        return see


def make_batch(q_lens, kv_lens, H, Hkv, hd=128, ps=64, dtype=torch.bfloat16, block=1, window=0, sinks=0,
               seed=0, spread=1.5, layout="page") -> Batch:
    """CPU tensors.  Every slot that no token may touch holds NaN, the table's unused entries
    -1, and pages are dealt out in no order.  layout "token": pools whose tokens' heads lie side
    by side; queries are slices of a wider row."""
    g = torch.Generator().manual_seed(seed)
    T, B = sum(q_lens), len(q_lens)
    need = [-(-n // ps) for n in kv_lens]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=g).to(torch.int32)
    width = max(need + [1])
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    shape = (pool, Hkv, ps, hd) if layout == "page" else (pool, ps, Hkv, hd)
    k = torch.randn(shape, generator=g).to(dtype)
    v = torch.randn(shape, generator=g).to(dtype)
    if layout != "page":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    wide = (torch.randn(T, (H + 2) * hd, generator=g) * spread).to(dtype)
    mass = torch.rand(pool, Hkv, ps, generator=g)
    out = Batch(list(q_lens), list(kv_lens), H, Hkv, hd, ps, dtype, block, window, sinks, wide, k, v, mass,
                table, hd ** -0.5)
    dead = torch.ones(pool, ps, dtype=torch.bool)
    for b in range(B):
        seen = torch.zeros(kv_lens[b], dtype=torch.bool)
        for i in range(q_lens[b]):
            seen |= out.sees(b, i)
        for j in seen.nonzero().flatten().tolist():
            dead[table[b, j // ps], j % ps] = False
        if q_lens[b]:
            for w in range(need[b]):      # a page that no token sees may be gone
                if not seen[w * ps:(w + 1) * ps].any():
                    table[b, w] = -1
    for t in (k, v):
        t.masked_fill_(dead[:, None, :, None], float("nan"))
    return out


def attention(bt: Batch):
    """(out, lse, bound on out, bound on lse), float64."""
    T, G = sum(bt.q_lens), bt.H // bt.Hkv
    out = torch.zeros(T, bt.H, bt.hd, dtype=torch.float64)
    lse = torch.full((T, bt.H), float("-inf"), dtype=torch.float64)
    tol_o, tol_l = torch.zeros_like(out), torch.zeros(T, bt.H, dtype=torch.float64)
    t = 0
    for b in range(len(bt.q_lens)):
        k = [bt.keys(bt.k, b, h).double() for h in range(bt.Hkv)]
        v = [bt.keys(bt.v, b, h).double() for h in range(bt.Hkv)]
        for i in range(bt.q_lens[b]):
            see = bt.sees(b, i)
            for h in range(bt.H):
                if see.any():
                    kk, vv, q = k[h // G][see], v[h // G][see], bt.q[t, h].double()
                    s = bt.scale * (kk @ q)
                    w = (s - s.max()).exp()
                    z = w.sum()
                    out[t, h] = (w @ vv) / z
                    lse[t, h] = s.max() + z.log()
                    # a score of hd products summed in fp32; the sums over the keys; a weight
                    # and its sum; then, in bf16, the weight's and the output's rounding
                    e = bt.hd * U32 * bt.scale * float((kk.abs() @ q.abs()).max()) + 8 * U32 * float(s.abs().max())
                    e += len(w) * U32
                    bf = bt.dtype == torch.bfloat16
                    a = (w @ vv.abs()) / z
                    tol_o[t, h] = (2 * e + (2 * UW + 2.1 * UB if bf else 4 * U32)) * a
                    tol_l[t, h] = e + (UW if bf else 4 * U32) + 4 * U32 * lse[t, h].abs()
            t += 1
    return out, lse, tol_o, tol_l


def mass(bt: Batch, lse: torch.Tensor):
    """(accumulated weights, bound), float64, from the given lse [T, H]."""
    acc, tol = bt.mass.double(), torch.zeros(bt.mass.shape, dtype=torch.float64)
    G, t = bt.H // bt.Hkv, 0
    for b in range(len(bt.q_lens)):
        n = bt.kv_lens[b]
        for h in range(bt.Hkv):
            k = bt.keys(bt.k, b, h).double()
            add, off = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
            for i in range(bt.q_lens[b]):
                see = bt.sees(b, i)
                for g in range(h * G, (h + 1) * G):
                    q = bt.q[t + i, g].double()
                    x = bt.scale * (k[see] @ q)
                    w = (x - lse[t + i, g].double()).exp()
                    e = (bt.hd * U32 * bt.scale * (k[see].abs() @ q.abs())
                         + 8 * U32 * (x.abs() + lse[t + i, g].double().abs()) + 8 * U32)
                    add[see] += w
                    off[see] += w * e
            for j in range(n):
                if bool((add[j] != 0) | (off[j] != 0)):
                    page, o = bt.table[b, j // bt.ps], j % bt.ps
                    tol[page, h, o] = off[j] + (bt.q_lens[b] * G + 2) * U32 * (add[j] + acc[page, h, o].abs())
                    acc[page, h, o] += add[j]
        t += bt.q_lens[b]
    return acc, tol


def evict_positions(weights: List[float], keep: int, sinks: int, recent: int) -> List[int]:
    """Which positions of one (sequence, kv head) stay, in order."""
    n = len(weights)
    if n <= keep:
        return list(range(n))
    middle = sorted(range(sinks, n - recent), key=lambda j: (-weights[j], j))[:keep - sinks - recent]
    return list(range(sinks)) + sorted(middle) + list(range(n - recent, n))

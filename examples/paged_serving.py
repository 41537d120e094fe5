"""Continuous batching on the paged cache: prompts of different lengths enter in chunks while
earlier requests decode, sequences that grow past their budget are cut by accumulated weight.

    python examples/paged_serving.py [--shape tiny128] [--requests 6] [--tokens 24] [--budget 96]

Runs a random-init model of one of the framework's shapes (specfold_b200/synthetic.py): the
projections are torch's, the cache, attention, weight accumulation, eviction and greedy sampling
are this library's.
"""

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from specfold_b200 import PagedKVCache  # noqa: E402
from specfold_b200 import kernels as K  # noqa: E402
from specfold_b200 import synthetic as syn  # noqa: E402


class PagedDecoder:
    """A Qwen2-style decoder stack whose sequences live in a ``PagedKVCache``."""

    def __init__(self, model, dims, num_pages: int, page_size: int = 64, track_mass: bool = False):
        self.model, self.dims = model, dims
        p = next(model.parameters())
        self.cache = PagedKVCache(dims.layers, dims.kv_heads, dims.head_dim, num_pages, page_size,
                                  dtype=p.dtype, device=p.device, track_mass=track_mass)
        self.inv_freq = dims.theta ** (-torch.arange(0, dims.head_dim, 2, device=p.device).float()
                                       / dims.head_dim)
        self.seen = {}                       # tokens a sequence has had: its rotary position

    def add(self) -> int:
        seq = self.cache.add()
        self.seen[seq] = 0
        return seq

    def _rotate(self, x, cos, sin):
        a, b = x.float().chunk(2, -1)
        return (x.float() * cos + torch.cat((-b, a), -1) * sin).to(x.dtype)

    @torch.no_grad()
    def step(self, seqs, tokens, **mask):
        """New tokens (a list of ids) of each sequence through the model; the logits of every
        sequence's last one."""
        d, dev = self.dims, self.cache.device
        q_lens = [len(t) for t in tokens]
        step = self.cache.step(seqs, q_lens, heads=d.heads, **mask)
        pos = torch.cat([torch.arange(self.seen[s], self.seen[s] + n) for s, n in zip(seqs, q_lens)])
        for s, n in zip(seqs, q_lens):
            self.seen[s] += n
        angle = pos.to(dev)[:, None].float() * self.inv_freq
        angle = torch.cat((angle, angle), -1)[:, None]
        cos, sin = angle.cos(), angle.sin()
        base = self.model.model
        x = base.embed_tokens(torch.tensor([t for ts in tokens for t in ts], device=dev))
        for li, layer in enumerate(base.layers):
            a, y = layer.self_attn, layer.input_layernorm(x)
            q = self._rotate(a.q_proj(y).view(-1, d.heads, d.head_dim), cos, sin)
            k = self._rotate(a.k_proj(y).view(-1, d.kv_heads, d.head_dim), cos, sin)
            v = a.v_proj(y).view(-1, d.kv_heads, d.head_dim)
            self.cache.append(li, k, v, step)
            out, lse = self.cache.attend(li, q, step)
            if self.cache._mass is not None:
                self.cache.accumulate(li, q, lse, step)
            x = x + a.o_proj(out.flatten(1))
            x = x + layer.mlp(layer.post_attention_layernorm(x))
        last = torch.tensor(q_lens, device=dev).cumsum(0) - 1
        logits = self.model.lm_head(base.norm(x[last]))
        step.check()
        return logits


def serve(decoder, prompts, new_tokens: int, chunk: int = 64, budget: int = 0, sinks: int = 4, recent: int = 16):
    """Every prompt's continuation: one request joins per step, prompts enter ``chunk`` tokens at a
    time, next to the requests that already decode."""
    todo = [list(p) for p in prompts]
    seqs, out = [], [[] for _ in prompts]
    while any(len(o) < new_tokens for o in out):
        if len(seqs) < len(prompts):
            seqs.append(decoder.add())
        live = [i for i in range(len(seqs)) if len(out[i]) < new_tokens]
        feed = [todo[i][:chunk] if todo[i] else out[i][-1:] for i in live]
        logits = decoder.step([seqs[i] for i in live], feed)
        tokens, _ = K.sample_top_p_greedy(logits)
        for i, t in zip(live, tokens.tolist()):
            todo[i] = todo[i][chunk:]
            if not todo[i]:
                out[i].append(t)
                if len(out[i]) == new_tokens:
                    decoder.cache.remove(seqs[i])
        if budget:
            # a quarter over before a cut, so that not every step moves the whole cache
            over = [seqs[i] for i in live if len(out[i]) < new_tokens
                    and decoder.cache.length(seqs[i]) > budget + budget // 4]
            if over:
                decoder.cache.evict(over, budget, sinks=sinks, recent=recent)
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--shape", default="tiny128", choices=sorted(syn.SHAPES))
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--budget", type=int, default=96)
    a = ap.parse_args()
    dims = syn.SHAPES[a.shape]
    model = syn.build_model(dims, family="fastdllm", dtype=torch.bfloat16, seed=0).cuda()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, dims.vocab, (40 + 37 * i,), generator=g).tolist() for i in range(a.requests)]
    decoder = PagedDecoder(model, dims, num_pages=64 * a.requests, page_size=16, track_mass=a.budget > 0)
    t0 = time.perf_counter()
    out = serve(decoder, prompts, a.tokens, budget=a.budget)
    dt = time.perf_counter() - t0
    for p, o in zip(prompts, out):
        print(f"prompt of {len(p):4d}: {o[:8]} ...")
    print(f"{sum(map(len, out))} tokens in {dt:.2f} s; {decoder.cache.free_pages} of "
          f"{decoder.cache.num_pages} pages free at the end")


if __name__ == "__main__":
    main()

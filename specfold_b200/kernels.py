"""Tensor-level wrappers of the C-ABI entry points, one per launch of the reference's
fused path (specfold/generate/triton_kernels.py, launched from
fastdllm_v2_folded.py:306-361).  They take torch CUDA tensors, launch on the current
stream and return without synchronising.  Used by the per-kernel parity tests; the
generator calls the whole-forward entry point instead.
"""

from __future__ import annotations

import ctypes
from typing import Dict, Optional, Sequence, Tuple, Union

import torch

from . import _lib

_WS: Dict[int, torch.Tensor] = {}


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _lib.SF_DTYPE_BF16
    if t.dtype == torch.float32:
        return _lib.SF_DTYPE_F32
    raise TypeError(f"unsupported dtype {t.dtype}; the kernels take float32 or bfloat16")


def _check_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("specfold_b200 kernels take CUDA tensors")
        if t is not None and not t.is_contiguous():
            raise ValueError("specfold_b200 kernels take contiguous tensors")


_DRAFT_WS = {}


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Zero-initialised scratch shared by the GEMM entry points (split-K partials and
    tile counters; the kernels leave the counters at zero)."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    ws = _WS.get(idx)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _WS[idx] = ws
    return ws


def error_word(device) -> torch.Tensor:
    return torch.zeros(1, dtype=torch.int32, device=device)


def raise_device_error(err: torch.Tensor) -> None:
    bits = int(err.item())
    if bits:
        raise _lib.SpecFoldError("device error: " + _lib.describe_device_error(bits))


def residual_delta_gate(Hf: torch.Tensor, par_idx: torch.Tensor, delta: float, B1: int, N: int,
                        bucket: int, eps: float, ln_w: Optional[torch.Tensor] = None,
                        err: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
    _check_cuda(Hf, par_idx, ln_w)
    dev = Hf.device
    BN, D = B1 * N, Hf.shape[-1]
    out = {
        "rstd": torch.empty(BN, dtype=torch.float32, device=dev),
        "f": torch.empty(BN, dtype=torch.int64, device=dev),
        "rec": torch.empty(BN, dtype=torch.int8, device=dev),
        "rows": torch.zeros(bucket, dtype=torch.int64, device=dev),
        "count": torch.zeros(1, dtype=torch.int32, device=dev),
        "seg": torch.zeros(BN, dtype=torch.int64, device=dev),
        "segcnt": torch.zeros(B1, dtype=torch.int32, device=dev),
        "src": torch.empty(BN, dtype=torch.int64, device=dev),
        "xn": torch.zeros(bucket, D, dtype=Hf.dtype, device=dev) if ln_w is not None else None,
    }
    err = err if err is not None else error_word(dev)
    lib = _lib.load()
    _lib.check(lib.sf_residual_delta_gate(
        dtype_code(Hf), Hf.data_ptr(), par_idx.data_ptr(), out["rstd"].data_ptr(),
        out["f"].data_ptr(), out["rec"].data_ptr(), out["rows"].data_ptr(),
        out["count"].data_ptr(), out["seg"].data_ptr(), out["segcnt"].data_ptr(),
        out["src"].data_ptr(), _ptr(out["xn"]), _ptr(ln_w), float(delta), B1, N, D, bucket,
        float(eps), err.data_ptr(), _stream()), "residual_delta_gate")
    out["err"] = err
    return out


def parent_map(ids: torch.Tensor) -> torch.Tensor:
    """par_idx [B1] int64 of a [B1, N] int64 token block, on the device
    (SpecFold*Generation._build_parent_map, fastdllm_v2_folded.py:55-75)."""
    _check_cuda(ids)
    ids = ids.contiguous()
    B1, N = ids.shape
    out = torch.empty(B1, dtype=torch.int64, device=ids.device)
    _lib.check(_lib.load().sf_parent_map(ids.data_ptr(), B1, N, out.data_ptr(), _stream()),
               "parent map")
    return out


def src_resolve(f: torch.Tensor, B1: int, N: int, err: Optional[torch.Tensor] = None):
    _check_cuda(f)
    src = torch.empty_like(f)
    err = err if err is not None else error_word(f.device)
    _lib.check(_lib.load().sf_src_resolve(f.data_ptr(), src.data_ptr(), B1, N, err.data_ptr(),
                                          _stream()), "src_resolve")
    return src


def _ws_args(device, BN, D, H, Hkv, hd, I, V):
    need = _lib.load().sf_workspace_bytes(BN, D, H, Hkv, hd, I, V)
    ws = workspace(device, need)
    return ws.data_ptr(), ws.numel()


def fused_ln_qkv_rope_scatter(xn, w_qkv, b_qkv, rows, count, cos, sin, q_buf, kv_buf, N, bucket,
                              H, Hkv, hd, q_scale=None, err=None):
    _check_cuda(xn, w_qkv, b_qkv, rows, count, cos, sin, q_buf, kv_buf, q_scale)
    D = xn.shape[-1]
    err = err if err is not None else error_word(xn.device)
    wp, wn = _ws_args(xn.device, bucket, D, H, Hkv, hd, 64, 64)
    _lib.check(_lib.load().sf_fused_ln_qkv_rope_scatter(
        dtype_code(xn), xn.data_ptr(), w_qkv.data_ptr(), _ptr(b_qkv), rows.data_ptr(),
        count.data_ptr(), cos.data_ptr(), sin.data_ptr(), _ptr(q_scale), q_buf.data_ptr(),
        kv_buf.data_ptr(), D, N, bucket, H, Hkv, hd, wp, wn, err.data_ptr(), _stream()),
        "fused_ln_qkv_rope_scatter")
    return err


def flash_attn_gqa(q_buf, pk, pv, kv_head_stride, kv_buf, src, rows, count, O, M, Z, P, N, scale,
                   bucket, B1, H, Hkv, hd, err=None):
    _check_cuda(q_buf, kv_buf, src, rows, count, O, M, Z)
    err = err if err is not None else error_word(q_buf.device)
    lib = _lib.load()
    need = lib.sf_attn_workspace_bytes(dtype_code(q_buf), bucket, H, Hkv, hd, P)
    ws = workspace(q_buf.device, need + (16 << 10)) if need else None
    # the scratch follows the GEMM tile counters, which must stay untouched
    wp = None if ws is None else ws.data_ptr() + (16 << 10)
    _lib.check(lib.sf_flash_attn_gqa(
        dtype_code(q_buf), q_buf.data_ptr(), _ptr(pk), _ptr(pv), int(kv_head_stride),
        kv_buf.data_ptr(), src.data_ptr(), rows.data_ptr(), count.data_ptr(), O.data_ptr(),
        M.data_ptr(), Z.data_ptr(), P, N, float(scale), bucket, B1, H, Hkv, hd, wp, need,
        err.data_ptr(), _stream()), "flash_attn_gqa")
    return err


def chain_correction_gqa(q_buf, kv_buf, src, par_idx, rec, seg, segcnt, O, M, Z, B1, N, scale, H,
                         Hkv, hd, err=None):
    _check_cuda(q_buf, kv_buf, src, par_idx, rec, seg, segcnt, O, M, Z)
    err = err if err is not None else error_word(q_buf.device)
    _lib.check(_lib.load().sf_chain_correction_gqa(
        dtype_code(q_buf), q_buf.data_ptr(), kv_buf.data_ptr(), src.data_ptr(), par_idx.data_ptr(),
        rec.data_ptr(), seg.data_ptr(), segcnt.data_ptr(), O.data_ptr(), M.data_ptr(),
        Z.data_ptr(), B1, N, float(scale), H, Hkv, hd, err.data_ptr(), _stream()),
        "chain_correction_gqa")
    return err


def o_proj_residual(Hf, O_tab, w_o, err=None):
    _check_cuda(Hf, O_tab, w_o)
    BN, D = Hf.shape
    q_dim = O_tab.shape[1]
    hp = torch.empty_like(Hf)
    err = err if err is not None else error_word(Hf.device)
    wp, wn = _ws_args(Hf.device, BN, D, q_dim // 64, 1, 64, 64, 64)
    _lib.check(_lib.load().sf_o_proj_residual(
        dtype_code(Hf), Hf.data_ptr(), O_tab.data_ptr(), w_o.data_ptr(), hp.data_ptr(), BN, D,
        q_dim, wp, wn, err.data_ptr(), _stream()), "o_proj_residual")
    return hp, err


def fused_ffn_scatter(hp_all, ln_w, w_gate, w_up, w_down, rows, count, ffn_buf, bucket, eps,
                      err=None):
    _check_cuda(hp_all, ln_w, w_gate, w_up, w_down, rows, count, ffn_buf)
    D = hp_all.shape[-1]
    I = w_gate.shape[0]
    dev = hp_all.device
    act = torch.zeros(bucket, I, dtype=hp_all.dtype, device=dev)
    xn = torch.zeros(bucket, D, dtype=hp_all.dtype, device=dev)
    rstd = torch.zeros(bucket, dtype=torch.float32, device=dev)
    err = err if err is not None else error_word(dev)
    wp, wn = _ws_args(dev, bucket, D, 1, 1, 64, I, 64)
    _lib.check(_lib.load().sf_fused_ffn_scatter(
        dtype_code(hp_all), hp_all.data_ptr(), ln_w.data_ptr(), w_gate.data_ptr(),
        w_up.data_ptr(), w_down.data_ptr(), rows.data_ptr(), count.data_ptr(), ffn_buf.data_ptr(),
        bucket, act.data_ptr(), xn.data_ptr(), rstd.data_ptr(), float(eps), D, I, wp, wn,
        err.data_ptr(), _stream()), "fused_ffn_scatter")
    return {"act": act, "xn": xn, "rstd": rstd, "err": err}


def combine(hp_all, ffn_buf, src, B1, N, err=None):
    _check_cuda(hp_all, ffn_buf, src)
    D = hp_all.shape[-1]
    hidden = torch.empty(B1 * N, D, dtype=hp_all.dtype, device=hp_all.device)
    err = err if err is not None else error_word(hp_all.device)
    _lib.check(_lib.load().sf_combine(dtype_code(hp_all), hp_all.data_ptr(), ffn_buf.data_ptr(),
                                      src.data_ptr(), hidden.data_ptr(), B1, N, D,
                                      err.data_ptr(), _stream()), "combine")
    return hidden, err


def final_norm_lm_head(hidden, norm_w, lm_w, B1, N, eps, shift, err=None):
    _check_cuda(hidden, norm_w, lm_w)
    D = hidden.shape[-1]
    V = lm_w.shape[0]
    dev = hidden.device
    logits = torch.empty(B1, N, V, dtype=hidden.dtype, device=dev)
    xn = torch.empty(B1 * N, D, dtype=hidden.dtype, device=dev)
    err = err if err is not None else error_word(dev)
    wp, wn = _ws_args(dev, B1 * N, D, 1, 1, 64, 64, V)
    _lib.check(_lib.load().sf_final_norm_lm_head(
        dtype_code(hidden), hidden.data_ptr(), norm_w.data_ptr(), lm_w.data_ptr(),
        logits.data_ptr(), xn.data_ptr(), B1, N, D, V, float(eps), int(shift), wp, wn,
        err.data_ptr(), _stream()), "final_norm_lm_head")
    return logits, err


def sample_top_p_greedy(logits: torch.Tensor, top_p: float = 0.95):
    """Greedy top-p sampling over the last dimension on the GPU: (tokens int64, the
    tokens' top-p filtered probabilities in the logits' dtype), both shaped
    logits.shape[:-1] (sf_sample_top_p_greedy; the reference's
    FastDLLMModelExecutor.sample_with_top_p at temperature 0)."""
    if not logits.is_cuda:
        raise ValueError("specfold_b200 kernels take CUDA tensors")
    V = logits.shape[-1]
    x = logits.reshape(-1, V)
    if x.stride(-1) != 1:
        x = x.contiguous()
    rows = x.shape[0]
    tokens = torch.empty(rows, dtype=torch.int64, device=x.device)
    conf = torch.empty(rows, dtype=x.dtype, device=x.device)
    _lib.check(_lib.load().sf_sample_top_p_greedy(
        dtype_code(x), x.data_ptr(), rows, V, x.stride(0), float(top_p), tokens.data_ptr(),
        conf.data_ptr(), _stream()), "sample_top_p_greedy")
    return tokens.view(logits.shape[:-1]), conf.view(logits.shape[:-1])


def draft_blocks(logits: torch.Tensor, mask: torch.Tensor, block: torch.Tensor, pos_offset: int,
                 pairs: torch.Tensor, node_off: torch.Tensor, K: int, conf_fp32: bool):
    """Draft blocks from the calibration graph on the GPU (sf_draft_blocks): logits
    [n_pos, V] of the positions [pos_offset, pos_offset + n_pos) of ``block`` (int64
    [L]), mask bool [n_pos], pairs int32 [n_pairs, 2] (pos_rank, vocab_rank), node_off
    int32 [n_nodes + 1].  Returns (drafts int64 [n_nodes, L], valid int32 [n_nodes])."""
    for t in (logits, mask, block, pairs, node_off):
        if not t.is_cuda:
            raise ValueError("specfold_b200 kernels take CUDA tensors")
    n_pos, V = logits.shape
    x = logits if logits.stride(-1) == 1 else logits.contiguous()
    m = mask.contiguous().view(torch.uint8) if mask.dtype == torch.bool else mask.to(torch.uint8)
    blk = block.contiguous()
    n_nodes = node_off.numel() - 1
    drafts = torch.empty(max(n_nodes, 1), blk.numel(), dtype=torch.int64, device=x.device)[:n_nodes]
    valid = torch.empty(max(n_nodes, 1), dtype=torch.int32, device=x.device)[:n_nodes]
    lib = _lib.load()
    nbytes = lib.sf_draft_workspace_bytes(n_pos, K)
    # scratch of its own: the GEMM workspace's counters must stay zero
    idx = x.device.index if x.device.index is not None else torch.cuda.current_device()
    ws = _DRAFT_WS.get(idx)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 16), dtype=torch.uint8, device=x.device)
        _DRAFT_WS[idx] = ws
    _lib.check(lib.sf_draft_blocks(
        dtype_code(x), x.data_ptr(), x.stride(0), n_pos, V, K, 1 if conf_fp32 else 0,
        m.data_ptr(), pairs.data_ptr(), node_off.data_ptr(), n_nodes, blk.data_ptr(), blk.numel(),
        int(pos_offset), drafts.data_ptr(), valid.data_ptr(), ws.data_ptr(), ws.numel(), _stream()),
        "draft_blocks")
    return drafts, valid


def kv_append(cache_k, cache_v, new_k, new_v, P):
    """cache_{k,v}: [Hkv, cap, hd] (any head stride, inner dims contiguous); new_{k,v}:
    [Hkv, n, hd].  Writes positions [P, P+n)."""
    Hkv, cap, hd = cache_k.shape
    n = new_k.shape[1]
    for t in (cache_k, cache_v):
        if t.stride(2) != 1 or t.stride(1) != hd:
            raise ValueError("cache rows must be contiguous [cap, hd] per head")
    if cache_v.stride(0) != cache_k.stride(0):
        raise ValueError("cache_k and cache_v must share one head stride")
    for t in (new_k, new_v):
        if t.stride(2) != 1 or (n > 1 and t.stride(1) != hd):
            raise ValueError("new rows must be contiguous [n, hd] per head")
    if new_v.stride(0) != new_k.stride(0):
        raise ValueError("new_k and new_v must share one head stride")
    if P + n > cap:
        raise ValueError(f"cache capacity {cap} < {P + n}")
    _lib.check(_lib.load().sf_kv_append(
        dtype_code(cache_k), cache_k.data_ptr(), cache_v.data_ptr(), cache_k.stride(0),
        new_k.data_ptr(), new_v.data_ptr(), new_k.stride(0), Hkv, hd, P, n, _stream()),
        "kv_append")


# ---------------------------------------------------------------------------- paged cache
def _int32(lens) -> torch.Tensor:
    t = torch.as_tensor(lens, dtype=torch.int64).reshape(-1)
    if t.is_cuda:
        raise ValueError("lengths are host integers (the split of the work is made on the host)")
    if t.numel() and (int(t.min()) < 0 or int(t.max()) > 1 << 30):
        raise ValueError("lengths must lie in [0, 2^30]")
    return t.to(torch.int32)


def _cuda_device(device) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("specfold_b200 kernels run on a CUDA device")
    return torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)


class _OnStream:
    """Device buffers made on one stream and used on others: a use on another stream waits for
    their making and keeps them from being handed out again while it runs."""

    def _made(self, device: torch.device, *tensors: torch.Tensor) -> None:
        self.device = device
        self._tensors = tensors
        self._home = torch.cuda.current_stream(device)
        self._home_raw = self._home.cuda_stream
        self._ready = self._home.record_event()

    def _call(self, fn, what: str, *args) -> None:
        """fn(*args, the current stream) on the plan's device"""
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._call(fn, what, *args)
        raw = torch._C._cuda_getCurrentRawStream(self.device.index)
        # (a capture begins after a synchronisation and may not wait for what it did not record)
        if raw != self._home_raw and not torch.cuda.is_current_stream_capturing():
            st = torch.cuda.current_stream(self.device)
            st.wait_event(self._ready)
            for t in self._tensors:
                t.record_stream(st)
        status = fn(*args, raw)
        if status:
            _lib.check(status, what)

    def check(self) -> None:
        """Raises what the kernels reported (a page id outside the pool, a wait that ran out).
        Synchronises with the device."""
        raise_device_error(self.err)


class PagedPlan(_OnStream):
    """One step of a batch over a paged cache: how its work is split over the SMs, the scratch
    and the error word of its calls.  Made once per step from the lengths on the host and used
    by every layer; calls that share a plan must not overlap on the GPU.

    ``q_lens[b]`` new tokens of sequence b see its ``kv_lens[b]`` cached keys (the new ones
    included): all up to the end of their own block of ``block`` tokens (1: causal, N:
    block-causal, 0: all), and with ``window`` > 0 only those less than ``window`` positions
    back and the first ``sinks``.  ``mass`` False leaves out what paged_attention_mass needs (for
    a large batch of single tokens most of a plan)."""

    def __init__(self, q_lens: Sequence[int], kv_lens: Sequence[int], *, heads: int, kv_heads: int,
                 head_dim: int, page_size: int, dtype: torch.dtype = torch.bfloat16, block: int = 1,
                 window: int = 0, sinks: int = 0, mass: bool = True, device="cuda"):
        q, n = _int32(q_lens), _int32(kv_lens)
        if q.numel() != n.numel():
            raise ValueError(f"{q.numel()} chunk lengths for {n.numel()} cache lengths")
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"unsupported dtype {dtype}; the kernels take float32 or bfloat16")
        lib = _lib.load()
        c = _lib.SfPagedPlan(dtype=_lib.SF_DTYPE_BF16 if dtype == torch.bfloat16 else _lib.SF_DTYPE_F32,
                             B=q.numel(), H=heads, Hkv=kv_heads, hd=head_dim, page_size=page_size,
                             block=block, window=window, sinks=sinks, skip_mass=not mass)
        device = _cuda_device(device)
        c.sms = torch.cuda.get_device_properties(device).multi_processor_count
        cap = lib.sf_paged_plan_words(ctypes.byref(c), q.data_ptr(), n.data_ptr())
        if cap <= 0:
            _lib.check(_lib.SF_ERR_ARG, "paged plan")
        words = torch.empty(cap, dtype=torch.int32)
        _lib.check(lib.sf_paged_plan_build(ctypes.byref(c), q.data_ptr(), n.data_ptr(),
                                           words.data_ptr(), cap), "paged plan")
        self.dtype, self.tokens, self.sequences = dtype, c.T, c.B
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        self._dev = words[:c.words].to(device)
        self._ws = torch.empty(max(c.ws_bytes, 256), dtype=torch.uint8, device=device)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)
        c.dev, c.ws, c.err = self._dev.data_ptr(), self._ws.data_ptr(), self.err.data_ptr()
        self._f32 = self.err.view(torch.float32)
        self._c = c
        self._ref = ctypes.byref(c)
        self._made(device, self._dev, self._ws, self.err)


class EvictPlan(_OnStream):
    """What an eviction needs on the device: of ``kv_lens[b]`` cached keys ``keep`` (or
    ``keep[b]``) stay, the first ``sinks`` and the last ``recent`` among them."""

    def __init__(self, kv_lens: Sequence[int], keep: Union[int, Sequence[int]], *, kv_heads: int,
                 page_size: int, sinks: int = 0, recent: int = 0, device="cuda"):
        n = _int32(kv_lens)
        k = _int32([keep] * n.numel() if isinstance(keep, int) else keep)
        if k.numel() != n.numel():
            raise ValueError(f"{k.numel()} budgets for {n.numel()} cache lengths")
        if sinks < 0 or recent < 0:
            raise ValueError("sinks and recent must not be negative")
        if bool(((n > k) & (k < sinks + recent)).any()):
            raise ValueError(f"sinks {sinks} + recent {recent} do not fit a budget that evicts")
        device = _cuda_device(device)
        self.sequences, self.kv_heads, self.page_size = n.numel(), kv_heads, page_size
        self.sinks, self.recent = sinks, recent
        # a budget above its length evicts nothing: what stays is then the length, and a budget that
        # only a short sequence has does not size the others' rows and tables
        k = torch.minimum(n, k)
        self.stay = k.tolist()
        self.max_len = int(n.max()) if n.numel() else 0
        self.kept = max(self.stay, default=0)
        # (where nothing is evicted sinks + recent may be more than stays: it bounds nothing)
        self.max_keep = max(self.kept, sinks + recent)
        self._lens = torch.stack((n, k), 1).contiguous().to(device)
        self.err = torch.zeros(1, dtype=torch.int32, device=device)
        self._made(device, self._lens, self.err)


def _paged_pool(k_pages, v_pages, table, mass_pages, plan, dtype):
    shape, dev = k_pages.shape, plan.device
    if len(shape) != 4:
        raise ValueError("pools are [pages, kv heads, page size, head_dim]")
    N, Hkv, ps, hd = shape
    stride = k_pages.stride()
    if Hkv != plan.kv_heads or ps != plan.page_size or k_pages.dtype != dtype or stride[3] != 1:
        raise ValueError(f"the plan is for {dtype} pools of {plan.kv_heads} kv heads and pages of "
                         f"{plan.page_size}, got {k_pages.dtype} {tuple(shape)}")
    if v_pages is None:
        v_ptr = None
    elif v_pages.shape != shape or v_pages.dtype != dtype or v_pages.stride() != stride:
        raise ValueError("k_pages and v_pages must share shape, dtype and strides")
    else:
        v_ptr = v_pages.data_ptr()
    if mass_pages is None:
        m_ptr = None
    elif (mass_pages.shape != (N, Hkv, ps) or mass_pages.dtype != torch.float32
          or not mass_pages.is_contiguous() or mass_pages.device != dev):
        raise ValueError(f"mass_pages must be contiguous float32 {(N, Hkv, ps)} on {dev}")
    else:
        m_ptr = mass_pages.data_ptr()
    rows, width = table.shape if table.dim() == 2 else (-1, 0)
    if rows != plan.sequences or table.dtype != torch.int32 or (width > 1 and table.stride(1) != 1):
        raise ValueError(f"the table must be int32 [{plan.sequences}, pages], rows contiguous")
    if k_pages.device != dev or table.device != dev or (v_pages is not None and v_pages.device != dev):
        raise ValueError(f"the plan lives on {dev}, got a tensor elsewhere")
    # the stride of an axis of one element is not used (torch keeps odd ones)
    return _lib.SfPagedPool(
        k_pages.data_ptr(), v_ptr, m_ptr, stride[0] if N > 1 else Hkv * ps * hd,
        stride[1] if Hkv > 1 else ps * hd, stride[2], table.data_ptr(),
        table.stride(0) if rows > 1 else width, N, width)


def _paged_rows(t: torch.Tensor, heads: int, plan: PagedPlan, what: str) -> Tuple[int, int]:
    """(token, head) strides of the new tokens' rows"""
    if t.shape != (plan.tokens, heads, plan.head_dim) or t.dtype != plan.dtype or t.device != plan.device:
        raise ValueError(f"{what} must be {plan.dtype} {(plan.tokens, heads, plan.head_dim)} on "
                         f"{plan.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    tok, head, one = t.stride()
    if one != 1:
        raise ValueError(f"{what}: head_dim must be contiguous")
    if heads == 1:
        head = plan.head_dim
    return (tok if plan.tokens > 1 else heads * head), head


def paged_kv_append(k_pages: torch.Tensor, v_pages: torch.Tensor, k_new: torch.Tensor,
                    v_new: torch.Tensor, table: torch.Tensor, plan: PagedPlan,
                    mass_pages: Optional[torch.Tensor] = None) -> None:
    """The new tokens' keys and values [T, Hkv, hd] (strided rows, e.g. slices of a fused
    projection's output) into their sequences' pages (sf_paged_kv_append); their accumulated
    weights start at zero.  Sequences may share pages, but not those of their new positions."""
    pool = _paged_pool(k_pages, v_pages, table, mass_pages, plan, plan.dtype)
    tok, head = _paged_rows(k_new, plan.kv_heads, plan, "k_new")
    if _paged_rows(v_new, plan.kv_heads, plan, "v_new") != (tok, head):
        raise ValueError("k_new and v_new must share their strides")
    plan._call(_lib.load().sf_paged_kv_append, "paged_kv_append", plan._ref, ctypes.byref(pool),
               k_new.data_ptr(), v_new.data_ptr(), tok, head)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, plan: PagedPlan, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of every sequence's new tokens q [T, H, hd] over its pages, under the plan's
    mask (sf_paged_attention).  Returns (out [T, H, hd], lse [T, H] float32); a token that sees
    no key gets zeros and -inf.  ``scale`` defaults to head_dim ** -0.5."""
    pool = _paged_pool(k_pages, v_pages, table, None, plan, plan.dtype)
    tok, head = _paged_rows(q, plan.heads, plan, "q")
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != q.device:
        raise ValueError("out must be contiguous, of q's shape, dtype and device")
    if lse is None:
        lse = plan._f32.new_empty((plan.tokens, plan.heads))
    elif lse.shape != q.shape[:2] or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError("lse must be contiguous float32 [T, H] on q's device")
    plan._call(_lib.load().sf_paged_attention, "paged_attention", plan._ref, ctypes.byref(pool),
               q.data_ptr(), tok, head, out.data_ptr(), lse.data_ptr(),
               plan.head_dim ** -0.5 if scale is None else scale)
    return out, lse


def paged_attention_mass(q: torch.Tensor, k_pages: torch.Tensor, table: torch.Tensor,
                         lse: torch.Tensor, mass_pages: torch.Tensor, plan: PagedPlan,
                         scale: Optional[float] = None) -> None:
    """Adds to every cached key's accumulated weight what the new tokens' softmax gave it,
    summed over tokens and the query heads of its kv head (sf_paged_attention_mass); ``lse`` is
    paged_attention's.  A page that several sequences of the step hold gets the weights of all
    (whose order, and so the last bits, may then differ from call to call)."""
    pool = _paged_pool(k_pages, None, table, mass_pages, plan, plan.dtype)
    tok, head = _paged_rows(q, plan.heads, plan, "q")
    if lse.shape != q.shape[:2] or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != q.device:
        raise ValueError("lse must be contiguous float32 [T, H] on q's device")
    plan._call(_lib.load().sf_paged_attention_mass, "paged_attention_mass", plan._ref,
               ctypes.byref(pool), q.data_ptr(), tok, head, lse.data_ptr(),
               plan.head_dim ** -0.5 if scale is None else scale)


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, mass_pages: torch.Tensor,
                table: torch.Tensor, dst_table: torch.Tensor, plan: EvictPlan) -> torch.Tensor:
    """Cuts every sequence to its budget, per kv head by accumulated weight, and moves what
    stays, in order, to the pages of ``dst_table``, which no source table may hold
    (sf_paged_evict).  Returns the old positions of what stayed, int32 [B, Hkv, most kept],
    -1 after the last."""
    dtype = k_pages.dtype
    code = dtype_code(k_pages)
    pool = _paged_pool(k_pages, v_pages, table, mass_pages, plan, dtype)
    if (dst_table.dim() != 2 or dst_table.shape[0] != plan.sequences or dst_table.dtype != torch.int32
            or (dst_table.shape[1] > 1 and dst_table.stride(1) != 1) or dst_table.device != plan.device):
        raise ValueError(f"dst_table must be int32 [{plan.sequences}, pages] on {plan.device}")
    kept = plan._lens.new_empty((plan.sequences, plan.kv_heads, plan.kept))
    plan._call(_lib.load().sf_paged_evict, "paged_evict", code, ctypes.byref(pool), dst_table.data_ptr(),
               dst_table.stride(0) if plan.sequences > 1 else dst_table.shape[1], dst_table.shape[1],
               plan._lens.data_ptr(), plan.max_len, plan.max_keep, plan.sequences, plan.kv_heads,
               k_pages.shape[3], plan.page_size, plan.sinks, plan.recent, kept.data_ptr(), plan.kept,
               plan.err.data_ptr())
    return kept

"""Torch-tensor front end of the HIP kernels (one function per C entry point).

Tensors stay torch tensors; this module only extracts pointers, strides and the
current stream and calls libomnikv_hip.so.  K / V are accepted in the reference's
shape (bsz, num_kv_heads, tokens, head_dim) with ANY strides whose last dimension
is contiguous, so both the reference's contiguous cache tensors and views of a
token-major store are read in place.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from dataclasses import dataclass
from typing import Dict, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import KVLayout, Shape, check, lib

_DTYPES = {torch.float32: _lib.OKV_F32, torch.bfloat16: _lib.OKV_BF16, torch.float16: _lib.OKV_F16}
_REDUCE = {"max": _lib.OKV_REDUCE_MAX, "sum": _lib.OKV_REDUCE_SUM}
_NORM = {"raw": _lib.OKV_NORM_RAW, "softmax": _lib.OKV_NORM_SOFTMAX}

# selector name -> (normalise, head_reduce); modeling/omnikv.py:40-58 plus the
# benchmark's softmax-sum variant.
SELECTOR_MODES = {
    "last": ("raw", "max"),
    "softmax_before_last": ("softmax", "max"),
    "softmax_sum_last": ("softmax", "sum"),
}


@dataclass
class PagedKV:
    """A paged K/V pool: pool_k / pool_v (num_pages, page_size, Hkv, D) and
    page_table (bsz, max_pages) int32.  page_size == 1 is a token-slot table."""

    pool_k: torch.Tensor
    pool_v: torch.Tensor
    page_table: torch.Tensor
    page_size: int

    def slot_index(self, idx: torch.Tensor) -> torch.Tensor:
        """Token positions (bsz, k) int32 -> rows of the pool seen as one flat array of token
        slots: page_table[b, t // page_size] * page_size + t % page_size.  Composed once per
        selection (the reference's serving stack keeps exactly such a table per request,
        req_to_imp_token_indexs, common/req_manager.py:12-17), every sparse layer of the
        group then reads its rows with one lookup instead of two.  Padding entries (< 0)
        stay padding."""
        if self.pool_k.stride(0) != self.page_size * self.pool_k.stride(1):
            raise ValueError("the pool's pages must lie back to back")
        t = idx.clamp(min=0).to(torch.int64)
        page = (t // self.page_size).clamp(max=self.page_table.shape[1] - 1)  # a stray entry never reads outside the table
        slots = self.page_table.gather(1, page).to(torch.int64) * self.page_size + t % self.page_size
        return torch.where(idx < 0, idx, slots.to(torch.int32))


_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _stream_ptr(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_retired: list = []  # outgrown scratch buffers: captured graphs may still hold their addresses


def _workspace(device, nbytes: int) -> torch.Tensor:
    """One growing scratch buffer per (device, stream).  It at least doubles when it grows and
    the buffer it replaces stays allocated (a HIP graph captured earlier keeps launching with
    the old address), so what is held in total is bounded by twice the largest request."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream_ptr(device))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _retired.append(ws)
        ws = torch.empty(max(nbytes, 1 << 20, 2 * ws.numel() if ws is not None else 0), dtype=torch.uint8,
                         device=device)
        _workspaces[key] = ws
    return ws


def workspace_bytes(op: int, batch: int, hq: int, hkv: int, d: int, max_seq_len: int,
                    max_tail_len: int = 0, with_scores: bool = False) -> int:
    shape = Shape(batch, hq, hkv, d, max_seq_len, max_tail_len, int(with_scores))
    out = C.c_size_t(0)
    check(lib().okv_workspace_bytes(op, C.byref(shape), C.byref(out)))
    return out.value


def _require_gpu(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (the HIP path has no CPU fallback)")


def _layout(k, v, hq: int):
    """(layout struct, k ptr, v ptr, batch, tokens) for tensors or a PagedKV."""
    if isinstance(k, PagedKV):
        pk = k
        pool_k, pool_v = pk.pool_k, pk.pool_v
        if pool_k.dim() != 4 or pool_k.stride(-1) != 1:
            raise ValueError("pool_k must be (pages, page_size, Hkv, D) with contiguous D")
        if pool_v is not None and pool_v.stride() != pool_k.stride():
            raise ValueError("pool_k and pool_v must share strides")
        pt = pk.page_table
        if pt.dtype != torch.int32 or pt.dim() != 2 or pt.stride(1) != 1:
            raise ValueError("page_table must be (bsz, max_pages) int32, rows contiguous")
        lay = KVLayout(
            _DTYPES[pool_k.dtype], hq, pool_k.shape[2], pool_k.shape[3],
            pool_k.stride(1), pool_k.stride(2), 0,
            pt.data_ptr(), pk.page_size, pt.stride(0), pool_k.stride(0),
        )
        return lay, pool_k.data_ptr(), (pool_v.data_ptr() if pool_v is not None else pool_k.data_ptr()), pt.shape[0], None
    if k.dim() != 4 or k.stride(-1) != 1:
        raise ValueError("K must be (bsz, Hkv, tokens, D) with a contiguous last dimension")
    if v is not None and (v.shape != k.shape or v.stride() != k.stride() or v.dtype != k.dtype):
        raise ValueError("K and V must share shape, strides and dtype")
    lay = KVLayout(
        _DTYPES[k.dtype], hq, k.shape[1], k.shape[3],
        k.stride(2), k.stride(1), k.stride(0), None, 0, 0, 0,
    )
    return lay, k.data_ptr(), (v.data_ptr() if v is not None else k.data_ptr()), k.shape[0], k.shape[2]


def _q3(q: torch.Tensor) -> torch.Tensor:
    if q.dim() == 4:
        if q.shape[2] != 1:
            raise ValueError("q must hold one query row per head")
        q = q[:, :, 0, :]
    return q.contiguous()


def _same_dtype(q: torch.Tensor, lay) -> None:
    if _DTYPES.get(q.dtype) != lay.dtype:
        raise ValueError("q and K/V must have the same dtype (float32, bfloat16 or float16)")


def _lens(t: Optional[torch.Tensor], batch: int, name: str) -> int:
    if t is None:
        return 0
    if t.dtype != torch.int32 or not t.is_cuda or t.numel() != batch or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 GPU tensor of {batch} entries")
    return t.data_ptr()


def score(q, k, score_len: Optional[int] = None, selector: str = "last", scale: Optional[float] = None,
          score_lens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(bsz, score_len) fp32 filter-layer scores; okv_score."""
    q = _q3(q)
    _require_gpu(q, "q")
    hq, d = q.shape[1], q.shape[2]
    lay, kp, _, batch, n = _layout(k, None, hq)
    _same_dtype(q, lay)
    if score_len is None:
        if n is None:
            raise ValueError("score_len is required with a paged pool")
        score_len = n
    norm, red = SELECTOR_MODES[selector]
    if out is None:
        out = torch.empty((batch, score_len), dtype=torch.float32, device=q.device)
    nbytes = workspace_bytes(_lib.OKV_OP_SCORE, batch, hq, lay.num_kv_heads, d, score_len)
    ws = _workspace(q.device, nbytes)
    check(lib().okv_score(
        q.data_ptr(), kp, C.byref(lay), _lens(score_lens, batch, "score_lens"), score_len, batch,
        _REDUCE[red], _NORM[norm], scale if scale is not None else 1.0 / math.sqrt(d),
        out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), _stream_ptr(q.device)))
    return out


def window_supported(q: torch.Tensor, k) -> bool:
    """Whether score_window takes these operands (else: one `score` call per position)."""
    if isinstance(k, PagedKV) or q.dim() != 4 or q.dtype not in (torch.bfloat16, torch.float16):
        return False
    hq, w = q.shape[1], q.shape[2]
    hkv = k.shape[1]
    if k.dtype != q.dtype or hkv > 8 or hq % hkv:
        return False
    return hq // hkv in (1, 2, 4, 8) and w * (hq // hkv) <= 64  # the kernel's max over a kv head's q heads pairs lanes


def score_window(q, k, score_len: Optional[int] = None, selector: str = "uniform", scale: Optional[float] = None,
                 score_lens: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(bsz, score_len) fp32 scores of the window selectors; okv_score_window.
    q: (bsz, Hq, W, D), the last W query positions, oldest first."""
    _require_gpu(q, "q")
    if selector not in ("uniform", "exp"):
        raise ValueError(f"selector {selector!r} is not a window selector")
    if q.dim() != 4 or q.stride(3) != 1:
        raise ValueError("q must be (bsz, Hq, W, D) with contiguous D")
    hq, w, d = q.shape[1], q.shape[2], q.shape[3]
    lay, kp, _, batch, n = _layout(k, None, hq)
    _same_dtype(q, lay)
    if score_len is None:
        score_len = n
    if out is None:
        out = torch.empty((batch, score_len), dtype=torch.float32, device=q.device)
    nbytes = workspace_bytes(_lib.OKV_OP_SCORE_WINDOW, batch, hq, lay.num_kv_heads, d, score_len)
    ws = _workspace(q.device, nbytes)
    check(lib().okv_score_window(
        q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), w, int(selector == "exp"), kp, C.byref(lay),
        _lens(score_lens, batch, "score_lens"), score_len, batch,
        scale if scale is not None else 1.0 / math.sqrt(d),
        out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), _stream_ptr(q.device)))
    return out


def dense_attn_window(q, q_window, k, v, selector: str = "uniform", seq_len: Optional[int] = None,
                      seq_lens: Optional[torch.Tensor] = None, score_len: Optional[int] = None,
                      score_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                      scores_out: Optional[torch.Tensor] = None):
    """A window-selector filter layer in two passes over K: (out, scores) = (dense_attn(q, k, v),
    score_window(q_window, k, score_len)) with the first scoring pass done inside the attention's;
    okv_dense_attn_window.  q: (bsz, Hq, D) or (bsz, Hq, 1, D); q_window: (bsz, Hq, W, D), oldest first."""
    q = _q3(q)
    _require_gpu(q, "q")
    _require_gpu(q_window, "q_window")
    if selector not in ("uniform", "exp"):
        raise ValueError(f"selector {selector!r} is not a window selector")
    if q_window.dim() != 4 or q_window.stride(3) != 1 or q_window.dtype != q.dtype:
        raise ValueError("q_window must be (bsz, Hq, W, D) with contiguous D and q's dtype")
    hq, d = q.shape[1], q.shape[2]
    if q_window.shape[0] != q.shape[0] or q_window.shape[1] != hq or q_window.shape[3] != d:
        raise ValueError("q_window does not match q")
    lay, kp, vp, batch, n = _layout(k, v, hq)
    _same_dtype(q, lay)
    if seq_len is None:
        seq_len = n
    if score_len is None:
        score_len = seq_len
    out = torch.empty_like(q)
    scores = scores_out
    if scores is None:
        scores = torch.empty((batch, score_len), dtype=torch.float32, device=q.device)
    elif scores.shape != (batch, score_len) or scores.dtype != torch.float32 or scores.stride(1) != 1:
        raise ValueError("scores_out must be (bsz, score_len) float32 with contiguous rows")
    nbytes = workspace_bytes(_lib.OKV_OP_DENSE_ATTN_WINDOW, batch, hq, lay.num_kv_heads, d, seq_len)
    ws = _workspace(q.device, nbytes)
    check(lib().okv_dense_attn_window(
        q.data_ptr(), q_window.data_ptr(), q_window.stride(0), q_window.stride(1), q_window.stride(2),
        q_window.shape[2], int(selector == "exp"), kp, vp, C.byref(lay), _lens(seq_lens, batch, "seq_lens"), seq_len,
        batch, scale if scale is not None else 1.0 / math.sqrt(d), out.data_ptr(),
        _lens(score_lens, batch, "score_lens"), score_len, scores.data_ptr(), scores.stride(0),
        ws.data_ptr(), ws.numel(), _stream_ptr(q.device)))
    return out, scores


def topk(scores: torch.Tensor, k: int, seq_lens: Optional[torch.Tensor] = None,
         k_per_seg: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(bsz, min(k, N)) int32 ascending indices of the k largest scores; okv_topk."""
    return _topk(scores, k, seq_lens, k_per_seg, out, _workspace)


def _topk(scores, k, seq_lens, k_per_seg, out, scratch) -> torch.Tensor:
    """topk with its scratch from scratch(device, bytes)."""
    _require_gpu(scores, "scores")
    if scores.dtype != torch.float32 or scores.dim() != 2 or scores.stride(1) != 1:
        raise ValueError("scores must be (bsz, N) float32 with contiguous rows")
    batch, n = scores.shape
    kk = min(k, n)
    if out is None:
        if seq_lens is None and k_per_seg is None:
            out = torch.empty((batch, kk), dtype=torch.int32, device=scores.device)
        else:  # ragged: the kernels leave entries beyond a request's own k untouched -> padding is -1
            out = torch.full((batch, kk), -1, dtype=torch.int32, device=scores.device)
    if kk == 0:
        return out
    ws = scratch(scores.device, workspace_bytes(_lib.OKV_OP_TOPK, batch, 0, 0, 0, n))
    check(lib().okv_topk(
        scores.data_ptr(), scores.stride(0), _lens(seq_lens, batch, "seq_lens"), n,
        _lens(k_per_seg, batch, "k_per_seg"), k, batch, out.data_ptr(), out.stride(0),
        ws.data_ptr(), ws.numel(), _stream_ptr(scores.device)))
    return out


def dense_attn(q, k, v=None, seq_len: Optional[int] = None, seq_lens: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, selector: Optional[str] = None,
               score_len: Optional[int] = None, score_lens: Optional[torch.Tensor] = None,
               scores_out: Optional[torch.Tensor] = None, select_k: Optional[int] = None,
               k_per_seg: Optional[torch.Tensor] = None, idx_out: Optional[torch.Tensor] = None):
    """Dense GQA decode attention; with `selector` also returns the filter-layer
    scores of the first score_len tokens from the same pass (okv_dense_attn), and with
    `select_k` on top of that the ascending indices of the select_k largest of them, as
    topk(scores, select_k, score_lens, k_per_seg) would: (out, scores, idx), the whole filter
    layer in one call (okv_dense_attn_select)."""
    q = _q3(q)
    _require_gpu(q, "q")
    hq, d = q.shape[1], q.shape[2]
    lay, kp, vp, batch, n = _layout(k, v, hq)
    _same_dtype(q, lay)
    if seq_len is None:
        if n is None:
            raise ValueError("seq_len is required with a paged pool")
        seq_len = n
    out = torch.empty_like(q)
    scores = None
    sp, ss, red, norm = None, 0, 0, 0
    if select_k is not None and selector is None:
        raise ValueError("select_k needs a selector")
    if selector is not None:
        norm_s, red_s = SELECTOR_MODES[selector]
        red, norm = _REDUCE[red_s], _NORM[norm_s]
        if score_len is None:
            score_len = seq_len
        scores = scores_out
        if scores is None:
            scores = torch.empty((batch, score_len), dtype=torch.float32, device=q.device)
        elif scores.shape != (batch, score_len) or scores.dtype != torch.float32 or scores.stride(1) != 1:
            raise ValueError("scores_out must be (bsz, score_len) float32 with contiguous rows")
        sp, ss = scores.data_ptr(), scores.stride(0)
    sc = scale if scale is not None else 1.0 / math.sqrt(d)
    if select_k is None:
        nbytes = workspace_bytes(_lib.OKV_OP_DENSE_ATTN, batch, hq, lay.num_kv_heads, d, seq_len,
                                 with_scores=selector is not None)
        ws = _workspace(q.device, nbytes)
        check(lib().okv_dense_attn(
            q.data_ptr(), kp, vp, C.byref(lay), _lens(seq_lens, batch, "seq_lens"), seq_len, batch,
            sc, out.data_ptr(), _lens(score_lens, batch, "score_lens"), score_len or 0, red, norm, sp, ss,
            ws.data_ptr(), ws.numel(), _stream_ptr(q.device)))
        return (out, scores) if selector is not None else out
    kk = min(select_k, score_len)
    idx = idx_out
    if idx is None:
        if score_lens is None and k_per_seg is None:
            idx = torch.empty((batch, kk), dtype=torch.int32, device=q.device)
        else:  # ragged: entries beyond a request's own k are left untouched -> padding is -1
            idx = torch.full((batch, kk), -1, dtype=torch.int32, device=q.device)
    elif idx.shape != (batch, kk) or idx.dtype != torch.int32 or idx.stride(1) != 1:
        raise ValueError("idx_out must be (bsz, min(select_k, score_len)) int32 with contiguous rows")
    nbytes = workspace_bytes(_lib.OKV_OP_DENSE_ATTN_SELECT, batch, hq, lay.num_kv_heads, d, seq_len,
                             with_scores=True)
    ws = _workspace(q.device, nbytes)
    check(lib().okv_dense_attn_select(
        q.data_ptr(), kp, vp, C.byref(lay), _lens(seq_lens, batch, "seq_lens"), seq_len, batch,
        sc, out.data_ptr(), _lens(score_lens, batch, "score_lens"), score_len, red, norm, sp, ss,
        _lens(k_per_seg, batch, "k_per_seg"), select_k, idx.data_ptr(), idx.stride(0),
        ws.data_ptr(), ws.numel(), _stream_ptr(q.device)))
    return out, scores, idx


def sparse_attn(q, k, v=None, idx: Optional[torch.Tensor] = None, sel_len: Optional[int] = None,
                sel_lens: Optional[torch.Tensor] = None, tail_k: Optional[torch.Tensor] = None,
                tail_v: Optional[torch.Tensor] = None, tail_len: Optional[int] = None,
                tail_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention over rows idx of K/V followed by the tail rows; okv_sparse_attn.

    idx (bsz, k) int32 ascending, or None for rows [0, sel_len).  tail_k / tail_v
    are (bsz, Hkv, T, D) with any strides (last dimension contiguous)."""
    q = _q3(q)
    _require_gpu(q, "q")
    hq, d = q.shape[1], q.shape[2]
    if slots is not None:
        # rows of a paged pool addressed as token slots (PagedKV.slot_index): no page table
        if not isinstance(k, PagedKV) or idx is not None:
            raise ValueError("slots go with a PagedKV and replace idx")
        pool_k, pool_v = k.pool_k, k.pool_v
        lay = KVLayout(_DTYPES[pool_k.dtype], hq, pool_k.shape[2], pool_k.shape[3], pool_k.stride(1),
                       pool_k.stride(2), 0, None, 0, 0, 0)
        kp, vp, batch, n, idx = pool_k.data_ptr(), pool_v.data_ptr(), slots.shape[0], None, slots
    else:
        lay, kp, vp, batch, n = _layout(k, v, hq)
    _same_dtype(q, lay)
    ip, istride = None, 0
    if idx is not None:
        if idx.dtype != torch.int32 or idx.dim() != 2 or idx.stride(1) != 1 or not idx.is_cuda:
            raise ValueError("idx must be a (bsz, k) int32 GPU tensor with contiguous rows")
        ip, istride = idx.data_ptr(), idx.stride(0)
        if sel_len is None:
            sel_len = idx.shape[1]
    elif sel_len is None:
        sel_len = n
    tkp = tvp = None
    tts = ths = tbs = 0
    if tail_k is not None:
        if tail_k.dim() != 4 or tail_k.stride(-1) != 1 or tail_v.stride() != tail_k.stride():
            raise ValueError("tail_k / tail_v must be (bsz, Hkv, T, D), same strides, contiguous D")
        if tail_k.dtype != q.dtype:
            raise ValueError("tail dtype differs from q")
        if tail_len is None:
            tail_len = tail_k.shape[2]
        tkp, tvp = tail_k.data_ptr(), tail_v.data_ptr()
        tts, ths, tbs = tail_k.stride(2), tail_k.stride(1), tail_k.stride(0)
    tail_len = tail_len or 0
    out = torch.empty_like(q)
    nbytes = workspace_bytes(_lib.OKV_OP_SPARSE_ATTN, batch, hq, lay.num_kv_heads, d, sel_len, tail_len)
    ws = _workspace(q.device, nbytes)
    check(lib().okv_sparse_attn(
        q.data_ptr(), kp, vp, C.byref(lay), ip, istride, _lens(sel_lens, batch, "sel_lens"), sel_len,
        tkp, tvp, tts, ths, tbs, _lens(tail_lens, batch, "tail_lens"), tail_len, batch,
        scale if scale is not None else 1.0 / math.sqrt(d), out.data_ptr(),
        ws.data_ptr(), ws.numel(), _stream_ptr(q.device)))
    return out


def gather_rows(src, idx: torch.Tensor, out: Optional[torch.Tensor] = None,
                sel_lens: Optional[torch.Tensor] = None, hq: Optional[int] = None) -> torch.Tensor:
    """out[b, g, j, :] = src[b, g, idx[b, j], :]; okv_gather_rows.

    `out` may be any (bsz, Hkv, k, D) tensor with a contiguous last dimension;
    by default it is token-major storage viewed in that shape."""
    if idx.dtype != torch.int32 or idx.dim() != 2 or idx.stride(1) != 1 or not idx.is_cuda:
        raise ValueError("idx must be a (bsz, k) int32 GPU tensor with contiguous rows")
    probe = src.pool_k if isinstance(src, PagedKV) else src
    hkv = probe.shape[2] if isinstance(src, PagedKV) else probe.shape[1]
    lay, sp, _, batch, _ = _layout(src, None, hq or hkv)
    ksel = idx.shape[1]
    d = probe.shape[-1]
    if out is None:
        out = torch.empty((batch, ksel, hkv, d), dtype=probe.dtype, device=idx.device).permute(0, 2, 1, 3)
    if out.stride(-1) != 1 or out.shape != (batch, hkv, ksel, d):
        raise ValueError("out must be (bsz, Hkv, k, D) with a contiguous last dimension")
    check(lib().okv_gather_rows(
        sp, C.byref(lay), idx.data_ptr(), idx.stride(0), _lens(sel_lens, batch, "sel_lens"), ksel,
        batch, out.data_ptr(), out.stride(2), out.stride(1), out.stride(0), _stream_ptr(idx.device)))
    return out


# ---------------------------------------------------------------- per-token layer operations
def _same(*ts):
    t0 = ts[0]
    for t in ts:
        _require_gpu(t, "tensor")
        if t.dtype != t0.dtype or not t.is_contiguous():
            raise ValueError("operands must be contiguous GPU tensors of one dtype")
    if t0.dtype not in _DTYPES:
        raise ValueError("dtype must be float32, bfloat16 or float16")
    return _DTYPES[t0.dtype]


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None):
    """weight * rms_normalise(x [+ residual]) over the last dimension; okv_rmsnorm.  Returns the
    normalised tensor, or (normalised, x + residual) when a residual is given."""
    dt = _same(x, weight) if residual is None else _same(x, weight, residual)
    hidden = x.shape[-1]
    rows = x.numel() // hidden
    out = torch.empty_like(x)
    total = torch.empty_like(x) if residual is not None else None
    check(lib().okv_rmsnorm(x.data_ptr(), residual.data_ptr() if residual is not None else None, weight.data_ptr(),
                            float(eps), rows, hidden, dt, total.data_ptr() if total is not None else None,
                            out.data_ptr(), _stream_ptr(x.device)))
    return out if residual is None else (out, total)


def _check_rope_tables(cos: torch.Tensor, sin: torch.Tensor, bsz: int, d: int) -> None:
    """The kernels read one row of d cos / sin values per request, back to back: a broadcast (1, 1, d) table
    next to bsz > 1 would be read past its end."""
    if d != 128:
        raise ValueError("the rotary kernels are built for head_dim 128")
    if tuple(cos.shape) != (bsz, 1, d) or tuple(sin.shape) != (bsz, 1, d):
        raise ValueError(f"cos / sin must be (bsz, 1, head_dim) = ({bsz}, 1, {d}), one row per request; "
                         f"got {tuple(cos.shape)} and {tuple(sin.shape)} (expand a shared row first)")


def rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, num_q_heads: int,
         num_kv_heads: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rotary embedding of one position per request: q (bsz, 1, Hq*D) and k (bsz, 1, Hkv*D) as the
    projections leave them, cos / sin (bsz, 1, D); returns (bsz, Hq, 1, D) and (bsz, Hkv, 1, D).  okv_rope."""
    dt = _same(q, k, cos, sin)
    bsz = q.shape[0]
    d = cos.shape[-1]
    if q.shape[1] != 1 or q.shape[-1] != num_q_heads * d or k.shape[-1] != num_kv_heads * d:
        raise ValueError("q / k must be (bsz, 1, heads * head_dim)")
    _check_rope_tables(cos, sin, bsz, d)
    q_out = torch.empty((bsz, num_q_heads, 1, d), dtype=q.dtype, device=q.device)
    k_out = torch.empty((bsz, num_kv_heads, 1, d), dtype=q.dtype, device=q.device)
    check(lib().okv_rope(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), cos.data_ptr(), sin.data_ptr(), bsz,
                         num_q_heads, num_kv_heads, d, dt, q_out.data_ptr(), k_out.data_ptr(), _stream_ptr(q.device)))
    return q_out, k_out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                num_q_heads: int, num_kv_heads: int, k_store: torch.Tensor, v_store: torch.Tensor,
                pos) -> torch.Tensor:
    """`rope` whose rotated k row and the v row are written into k_store / v_store (bsz, Hkv, capacity, D) at
    token position `pos` (an int, or a one-element int64 GPU tensor read by the kernel); returns the rotated
    q (bsz, Hq, 1, D).  Every request of the batch is written at the SAME position (the static decode
    path advances all requests together); nothing on the device checks a device position against the
    store's capacity -- the cache's host-side step count does.  okv_rope_append."""
    dt = _same(q, k, v, cos, sin)
    bsz, d = q.shape[0], cos.shape[-1]
    _check_rope_tables(cos, sin, bsz, d)
    if k_store.dtype != q.dtype or k_store.stride() != v_store.stride() or k_store.stride(-1) != 1:
        raise ValueError("k_store / v_store must share dtype with q and strides with each other")
    if k_store.shape[0] != bsz or k_store.shape[1] != num_kv_heads or k_store.shape[3] != d:
        raise ValueError("stores must be (bsz, Hkv, capacity, D)")
    q_out = torch.empty((bsz, num_q_heads, 1, d), dtype=q.dtype, device=q.device)
    on_dev = isinstance(pos, torch.Tensor)
    if on_dev and (pos.dtype != torch.int64 or not pos.is_cuda or pos.numel() != 1):
        raise ValueError("a device position must be a one-element int64 GPU tensor")
    if not on_dev and not 0 <= int(pos) < k_store.shape[2]:
        raise ValueError("position outside the store")
    check(lib().okv_rope_append(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                cos.data_ptr(), sin.data_ptr(), bsz, num_q_heads, num_kv_heads, d, dt, q_out.data_ptr(),
                                k_store.data_ptr(), v_store.data_ptr(), k_store.stride(2), k_store.stride(1),
                                k_store.stride(0), pos.data_ptr() if on_dev else None, 0 if on_dev else int(pos),
                                _stream_ptr(q.device)))
    return q_out


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up; okv_silu_mul."""
    dt = _same(gate, up)
    out = torch.empty_like(gate)
    check(lib().okv_silu_mul(gate.data_ptr(), up.data_ptr(), gate.numel(), dt, out.data_ptr(), _stream_ptr(gate.device)))
    return out


# ---------------------------------------------------------------- 8-bit K/V cache
KV8_FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_SCALE128 = 1.0 / math.sqrt(128)
_KV8_CODES = {torch.float8_e4m3fn: _lib.OKV_E4M3, torch.int8: _lib.OKV_I8}
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice  # (torch.cuda.current_device() less its check that the GPU is in use: tensors are)


def _launch(device: torch.device, fn, *args) -> None:
    """fn(*args, current stream of `device`), with that device current: a launch goes to the current one."""
    i = device.index
    if i != _current_device():
        with torch.cuda.device(i):
            check(fn(*args, _raw_stream(i)))
        return
    rc = fn(*args, _raw_stream(i))
    if rc:
        check(rc)


def _scratch(device, nbytes: int) -> torch.Tensor:
    """Scratch of one call, from torch's allocator: it may be reused by what the same stream runs next, two threads
    never hold the same piece, and a captured graph keeps a piece of its own pool, so two graphs do not share one."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _dev_i32(t: Optional[torch.Tensor], n: int, device, name: str):
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.numel() != n or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} entries on {device}")
    return t.data_ptr()


def _overlaps(t: torch.Tensor) -> bool:
    """Whether two indices of t may name one element (an expanded tensor, say)."""
    reach = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride < reach:
            return True
        reach = stride * (size - 1) + reach
    return False


class KV8:
    """An 8-bit K/V cache: codes (torch.float8_e4m3fn or torch.int8) with one fp32 scale per `block` tokens and kv
    head (include/omnikv_hip.h, okv_kv8_cache_t, has the format).

    contiguous: k, v (bsz, Hkv, capacity, 128), scales (bsz, Hkv, capacity / block)
    paged:      k, v (pages, page_size, Hkv, 128), scales (pages, page_size / block, Hkv), page_table (bsz, max_pages) int32
    open_k, open_v (bsz, Hkv, block, 128), bfloat16 or float16: the rows of each request's last, not yet full block; without them the
    cache is closed (it takes no more rows).  K and V share strides, and so do the two scales.  The
    handle keeps the tensors; the lengths are the caller's."""

    def __init__(self, k, v, k_scale, v_scale, block: int, open_k=None, open_v=None,
                 page_table: Optional[torch.Tensor] = None):
        paged = page_table is not None
        if k.dtype not in _KV8_CODES or v.dtype != k.dtype:
            raise ValueError("codes must be torch.float8_e4m3fn or torch.int8, K and V alike")
        if k.dim() != 4 or k.shape[-1] != 128 or k.stride(-1) != 1 or v.shape != k.shape or v.stride() != k.stride():
            raise ValueError("K and V codes must be 4-d with 128 contiguous elements last, same shape and strides")
        if any(s % 16 and n > 1 for s, n in zip(k.stride()[:3], k.shape)):
            raise ValueError("code strides must be multiples of 16")
        if block not in (16, 32, 64, 128):
            raise ValueError("block must be 16, 32, 64 or 128 tokens")
        tokens = k.shape[1] if paged else k.shape[2]
        hkv = k.shape[2] if paged else k.shape[1]
        if tokens < block or tokens % block:
            raise ValueError(f"{'page_size' if paged else 'capacity'} must be a multiple of block")
        want = (k.shape[0], tokens // block, hkv) if paged else (k.shape[0], hkv, tokens // block)
        for s in (k_scale, v_scale):
            if tuple(s.shape) != want or s.dtype != torch.float32 or s.stride() != k_scale.stride():
                raise ValueError(f"scales must be float32 {want}, same strides for K and V")
        devices = {t.device for t in (k, v, k_scale, v_scale, open_k, open_v, page_table) if t is not None}
        if len(devices) != 1 or not k.is_cuda:
            raise ValueError("every tensor of the cache must be on one GPU (the HIP path has no CPU fallback)")
        self.bsz = page_table.shape[0] if paged else k.shape[0]
        if paged and (page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1):
            raise ValueError("page_table must be (bsz, max_pages) int32, rows contiguous")
        if (open_k is None) != (open_v is None):
            raise ValueError("open_k and open_v go together")
        if open_k is not None:
            if (tuple(open_k.shape) != (self.bsz, hkv, block, 128) or open_k.dtype not in (torch.bfloat16, torch.float16)
                    or open_v.shape != open_k.shape or open_v.dtype != open_k.dtype or open_v.stride() != open_k.stride()
                    or open_k.stride(-1) != 1 or any(s % 8 and n > 1 for s, n in zip(open_k.stride()[:3], open_k.shape))):
                raise ValueError(f"open_k / open_v must be ({self.bsz}, {hkv}, {block}, 128) in bfloat16 or float16, "
                                 "same strides (multiples of 8), contiguous last dimension")
        self.k, self.v, self.k_scale, self.v_scale, self.block = k, v, k_scale, v_scale, block
        self.open_k, self.open_v, self.page_table = open_k, open_v, page_table
        self.device, self.num_kv_heads = k.device, hkv
        self.page_size = tokens if paged else 0
        self.capacity = page_table.shape[1] * tokens if paged else tokens  # tokens a request has room for
        self.dtype = open_k.dtype if open_k is not None else None
        st, ss = [s if n > 1 or s % 16 == 0 else 0 for s, n in zip(k.stride(), k.shape)], k_scale.stride()
        self._c = {}
        for dt in (torch.bfloat16, torch.float16):
            if self.dtype not in (None, dt):
                continue
            c = _lib.KV8Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), _KV8_CODES[k.dtype],
                              _DTYPES[dt], hkv, 128, block, 0 if paged else tokens)
            if paged:
                c.token_stride, c.head_stride, c.page_stride = st[1], st[2], st[0]
                c.scale_block_stride, c.scale_head_stride, c.scale_page_stride = ss[1], ss[2], ss[0]
                c.page_table, c.page_size = page_table.data_ptr(), tokens
                c.page_table_stride, c.num_pages = page_table.shape[1], k.shape[0]
                if self.bsz > 1 and page_table.stride(0) != page_table.shape[1]:
                    raise ValueError("page_table rows must lie back to back")
            else:
                c.batch_stride, c.head_stride, c.token_stride = st[:3]
                c.scale_batch_stride, c.scale_head_stride, c.scale_block_stride = ss
            if open_k is not None:
                c.open_k, c.open_v = open_k.data_ptr(), open_v.data_ptr()
                c.open_batch_stride, c.open_head_stride, c.open_token_stride = [
                    s if n > 1 else 0 for s, n in zip(open_k.stride()[:3], open_k.shape)]
            self._c[dt] = c
        self._ref = {dt: C.byref(c) for dt, c in self._c.items()}
        self._ws_bytes = {}  # scratch of a call, by its sizes
        # an expanded cache (one prompt shared by several requests) can be attended to, not written
        self._writable = not any(_overlaps(t) for t in (k, k_scale, open_k) if t is not None)

    @classmethod
    def empty(cls, bsz: int, num_kv_heads: int, capacity: int, fmt: str = "e4m3", block: int = 64,
              dtype: Optional[torch.dtype] = torch.bfloat16, device="cuda") -> "KV8":
        """A contiguous cache with room for `capacity` tokens per request (rounded up to whole blocks); dtype None: closed."""
        cap = -(-capacity // block) * block
        k, v = (torch.zeros((bsz, num_kv_heads, cap, 128), dtype=torch.uint8, device=device).view(KV8_FORMATS[fmt])
                for _ in "kv")
        s = torch.zeros((2, bsz, num_kv_heads, cap // block), dtype=torch.float32, device=device)
        o = [None, None] if dtype is None else torch.zeros((2, bsz, num_kv_heads, block, 128), dtype=dtype, device=device)
        return cls(k, v, s[0], s[1], block, o[0], o[1])

    @classmethod
    def empty_paged(cls, page_table: torch.Tensor, num_pages: int, page_size: int, num_kv_heads: int, fmt: str = "e4m3",
                    block: int = 16, dtype: Optional[torch.dtype] = torch.bfloat16) -> "KV8":
        """A pool of `num_pages` pages read and written through `page_table` (bsz, max_pages); dtype None: closed."""
        dev = page_table.device
        k, v = (torch.zeros((num_pages, page_size, num_kv_heads, 128), dtype=torch.uint8, device=dev).view(KV8_FORMATS[fmt])
                for _ in "kv")
        s = torch.zeros((2, num_pages, page_size // block, num_kv_heads), dtype=torch.float32, device=dev)
        o = [None, None] if dtype is None else torch.zeros((2, page_table.shape[0], num_kv_heads, block, 128), dtype=dtype,
                                                           device=dev)
        return cls(k, v, s[0], s[1], block, o[0], o[1], page_table)

    def slot_index(self, idx: torch.Tensor) -> torch.Tensor:
        """Token positions (bsz, k) int32 -> rows of the pool seen as one array of token slots, as
        PagedKV.slot_index; positions and pages outside the request's table stay out (-1)."""
        if self.page_table is None:
            raise ValueError("slots address a paged pool")
        t = idx.clamp(min=0, max=self.capacity - 1).to(torch.int64)
        page = self.page_table.gather(1, t // self.page_size).to(torch.int64)
        slots = page * self.page_size + t % self.page_size
        ok = (idx >= 0) & (idx < self.capacity) & (page >= 0) & (page < self.k.shape[0])
        return torch.where(ok, slots.to(torch.int32), -1)

    def _struct(self, dtype: torch.dtype):
        c = self._ref.get(dtype)
        if c is None:
            raise ValueError(f"{dtype} next to this cache: it takes " + " and ".join(str(d) for d in self._c))
        return c


def _kv8_workspace_bytes(cache: KV8, hq: int, rows: int, score_len: int, indexed: bool) -> int:
    n = cache._ws_bytes.get((hq, rows, score_len, indexed))
    if n is None:
        out = C.c_size_t(0)
        check(lib().okv_kv8_workspace_bytes(next(iter(cache._ref.values())), hq, cache.bsz, rows, score_len, int(indexed),
                                            C.byref(out)))
        if len(cache._ws_bytes) >= 4096:  # lengths that grow by one per call
            cache._ws_bytes.clear()
        n = cache._ws_bytes[(hq, rows, score_len, indexed)] = out.value
    return n


def kv8_append(cache: KV8, k: torch.Tensor, v: torch.Tensor, start: Union[int, torch.Tensor] = 0,
               new_lens: Optional[torch.Tensor] = None, close: bool = False) -> None:
    """Appends k, v (bsz, Hkv, n, 128; strides multiples of 8, contiguous last dimension) behind the first `start` rows of each
    request: an int, or an int32 GPU tensor (bsz,) of the requests' lengths.  new_lens (bsz,) int32: rows per request,
    at most n.  Blocks that fill become codes, the other rows wait in the open buffers; close=True quantises a
    short last block as well (start then an int at a block's border) and leaves the open buffers alone: such rows are
    read by an index, or through a KV8 of the same tensors without open buffers.  A request whose rows would not
    fit is left as it was.  okv_kv8_append."""
    c = cache._struct(k.dtype)
    shape, dev = k.shape, cache.device
    if len(shape) != 4:
        raise ValueError(f"new rows must be ({cache.bsz}, {cache.num_kv_heads}, n, 128)")
    b, h, n, d = shape
    if b != cache.bsz or h != cache.num_kv_heads or d != 128:
        raise ValueError(f"new rows must be ({cache.bsz}, {cache.num_kv_heads}, n, 128)")
    if v.shape != shape or v.dtype is not k.dtype:
        raise ValueError("new K and V must share shape and dtype, with a contiguous last dimension")
    (kb, kg, kt, k1), (vb, vg, vt, v1) = k.stride(), v.stride()
    if k1 != 1 or v1 != 1:
        raise ValueError("new K and V must share shape and dtype, with a contiguous last dimension")
    if k.device != dev or v.device != dev:
        raise ValueError("new rows and cache must be on one GPU")
    if not cache._writable:
        raise ValueError("rows of this cache share memory: it can be read only")
    if n == 0:
        return
    if b == 1:  # (whatever a view left as the stride of a single entry)
        kb = vb = 0
    if h == 1:
        kg = vg = 0
    if n == 1:
        kt = vt = 0
    on_dev = isinstance(start, torch.Tensor)
    if not on_dev and not 0 <= start <= cache.capacity:
        raise ValueError(f"invalid start {start}: the cache has room for {cache.capacity} tokens")
    starts = _dev_i32(start, cache.bsz, cache.device, "start") if on_dev else None
    _launch(cache.device, lib().okv_kv8_append, c, k.data_ptr(), kt, kg, kb, v.data_ptr(), vt, vg, vb, starts,
            0 if on_dev else int(start), _dev_i32(new_lens, cache.bsz, cache.device, "new_lens"), n, int(close), cache.bsz)


def _kv8_query(q: torch.Tensor, cache: KV8):
    if q.dim() != 3 or not q.is_contiguous():
        q = _q3(q)
    if q.dim() != 3 or q.shape[0] != cache.bsz or q.shape[2] != 128:
        raise ValueError(f"q must be ({cache.bsz}, Hq, 128) or ({cache.bsz}, Hq, 1, 128)")
    if q.device != cache.device:
        raise ValueError("q and cache must be on one GPU")
    return q, cache._struct(q.dtype)


def kv8_dense_attn(q: torch.Tensor, cache: KV8, seq_len: Optional[int] = None, seq_lens: Optional[torch.Tensor] = None,
                   scale: Optional[float] = None, selector: Optional[str] = None, score_len: Optional[int] = None,
                   score_lens: Optional[torch.Tensor] = None, scores_out: Optional[torch.Tensor] = None,
                   select_k: Optional[int] = None, k_per_seg: Optional[torch.Tensor] = None,
                   idx_out: Optional[torch.Tensor] = None):
    """dense_attn over an 8-bit cache: q (bsz, Hq, 128) attends to the seq_len rows that each request holds (seq_lens: per
    request, on the GPU, seq_len their bound) -> (bsz, Hq, 128).  The rows behind the last full block of that length are taken
    from the open buffers: what is shorter than a request ends at a block's border, or goes through a KV8 of the same tensors
    without them.  With `selector` also the filter layer's scores of the first score_len rows, from the same
    pass, and with `select_k` the ascending indices of the largest ones, as topk gives them: of a request's own rows alone,
    -1 (in idx_out: what was there) behind the last of them.  A request without rows gets zeros.  okv_kv8_dense_attn."""
    q, c = _kv8_query(q, cache)
    hq, dev, bsz = q.shape[1], cache.device, cache.bsz
    if seq_len is None:
        seq_len = cache.capacity
    elif seq_len > cache.capacity:
        raise ValueError(f"invalid seq_len {seq_len}: the cache has room for {cache.capacity} tokens")
    if select_k is not None and selector is None:
        raise ValueError("select_k needs a selector")
    out = torch.empty_like(q)
    scores, sp, ss, red, norm, slen, sl = None, None, 0, 0, 0, 0, None
    if selector is not None:
        norm_s, red_s = SELECTOR_MODES[selector]
        red, norm = _REDUCE[red_s], _NORM[norm_s]
        slen = seq_len if score_len is None else score_len
        if not 0 <= slen <= seq_len:
            raise ValueError(f"score_len {slen} must lie in [0, seq_len]")
        scores = scores_out
        if scores is None:
            scores = torch.empty((bsz, slen), dtype=torch.float32, device=dev)
        elif scores.shape != (bsz, slen) or scores.dtype != torch.float32 or scores.stride(1) != 1 or scores.device != dev:
            raise ValueError("scores_out must be (bsz, score_len) float32 with contiguous rows, on the cache's GPU")
        sp, ss, sl = scores.data_ptr(), scores.stride(0) if bsz > 1 else max(slen, scores.stride(0)), _dev_i32(score_lens, bsz, dev, "score_lens")
    if select_k is not None and idx_out is not None:
        kk = min(select_k, slen)
        if (idx_out.shape != (bsz, kk) or idx_out.dtype != torch.int32 or idx_out.stride(1) != 1 or idx_out.device != dev
                or (bsz > 1 and idx_out.stride(0) < kk)):
            raise ValueError("idx_out must be (bsz, min(select_k, score_len)) int32 with contiguous rows, on the cache's GPU")
    nbytes = _kv8_workspace_bytes(cache, hq, seq_len, slen, False)
    ws = _scratch(dev, nbytes) if nbytes else None
    _launch(dev, lib().okv_kv8_dense_attn, q.data_ptr(), hq, c, _dev_i32(seq_lens, bsz, dev, "seq_lens"), seq_len, bsz,
            scale if scale is not None else _SCALE128, out.data_ptr(), sl, slen, red, norm, sp, ss,
            ws.data_ptr() if nbytes else None, nbytes)
    if selector is None:
        return out
    if select_k is None:
        return out, scores
    with torch.cuda.device(dev):
        # only a request's own rows have scores: its length bounds the ranking too (topk itself holds lengths to slen)
        if seq_lens is None or score_lens is seq_lens:
            ranked = score_lens
        else:
            ranked = seq_lens if score_lens is None else torch.minimum(seq_lens.view(-1), score_lens.view(-1))
        return out, scores, _topk(scores, select_k, ranked, k_per_seg, idx_out, _scratch)


def kv8_sparse_attn(q: torch.Tensor, cache: KV8, idx: Optional[torch.Tensor] = None, sel_len: Optional[int] = None,
                    sel_lens: Optional[torch.Tensor] = None, tail_k: Optional[torch.Tensor] = None,
                    tail_v: Optional[torch.Tensor] = None, tail_len: Optional[int] = None,
                    tail_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """sparse_attn over an 8-bit cache: rows idx (bsz, k) int32 of the codes (None: rows [0, sel_len)) followed by
    16-bit tail rows (bsz, Hkv, T, 128) in q's dtype; slots: KV8.slot_index(idx) instead of idx.  Entries outside the
    request's room (padding, -1) take no part.  They name rows that are codes: the place of an open row holds whatever was there before
    (open_k / open_v themselves can be the tail).  okv_kv8_sparse_attn."""
    q, c = _kv8_query(q, cache)
    hq, hkv, dev, bsz = q.shape[1], cache.num_kv_heads, cache.device, cache.bsz
    if slots is not None:
        if cache.page_table is None or idx is not None:
            raise ValueError("slots go with a paged cache and replace idx")
        idx = slots
    ip, istride = None, 0
    if idx is not None:
        if idx.dtype is not torch.int32 or idx.dim() != 2 or idx.device != dev:
            raise ValueError(f"idx must be a ({bsz}, k) int32 tensor with contiguous rows on the cache's GPU")
        (ib, width), (istride, unit) = idx.shape, idx.stride()
        if ib != bsz or unit != 1:
            raise ValueError(f"idx must be a ({bsz}, k) int32 tensor with contiguous rows on the cache's GPU")
        if sel_len is None:
            sel_len = width
        elif sel_len > width:
            raise ValueError("sel_len exceeds idx")
        if istride < width:
            if bsz > 1:
                raise ValueError("idx rows must not overlap")
            istride = width
        ip = idx.data_ptr()
    elif sel_len is None:
        sel_len = cache.capacity
    elif sel_len > cache.capacity:
        raise ValueError(f"invalid sel_len {sel_len}: the cache has room for {cache.capacity} tokens")
    tkp = tvp = None
    tts = ths = tbs = 0
    if tail_k is not None:
        shape, strides = tail_k.shape, tail_k.stride()
        if len(strides) != 4 or tail_v is None or shape != tail_v.shape or strides != tail_v.stride():
            raise ValueError("tail_k / tail_v must be (bsz, Hkv, T, 128), same strides, contiguous last dimension")
        (tb, th, rows, td), (tbs, ths, tts, unit) = shape, strides
        if tb != bsz or th != hkv or td != 128 or unit != 1:
            raise ValueError("tail_k / tail_v must be (bsz, Hkv, T, 128), same strides, contiguous last dimension")
        if tb == 1:
            tbs = 0
        if th == 1:
            ths = 0
        if rows == 1:
            tts = 0
        dt = q.dtype
        if tail_k.dtype is not dt or tail_v.dtype is not dt or tail_k.device != dev or tail_v.device != dev:
            raise ValueError("tail and q differ in dtype or GPU")
        if tail_len is None:
            tail_len = rows
        elif tail_len > rows:
            raise ValueError("tail_len exceeds the tail")
        tkp, tvp = tail_k.data_ptr(), tail_v.data_ptr()
    elif tail_len:
        raise ValueError("tail_len without a tail")
    tail_len = tail_len or 0
    out = torch.empty_like(q)
    nbytes = _kv8_workspace_bytes(cache, hq, sel_len + tail_len, 0, idx is not None)
    ws = _scratch(dev, nbytes) if nbytes else None
    _launch(dev, lib().okv_kv8_sparse_attn, q.data_ptr(), hq, c, ip, istride, int(slots is not None),
            _dev_i32(sel_lens, bsz, dev, "sel_lens"), sel_len, tkp, tvp, tts, ths, tbs,
            _dev_i32(tail_lens, bsz, dev, "tail_lens"), tail_len, bsz, scale if scale is not None else _SCALE128,
            out.data_ptr(), ws.data_ptr() if nbytes else None, nbytes)
    return out


def kv8_read(cache: KV8, dtype: torch.dtype, idx: Optional[torch.Tensor] = None, seq_len: Optional[int] = None,
             seq_lens: Optional[torch.Tensor] = None):
    """The cached values as 16-bit tensors (bsz, Hkv, n, 128): rows idx (bsz, n) int32, or the first seq_len; rows outside a
    request (seq_lens, seq_len; default: the whole room) are zeros.  okv_kv8_read."""
    c, dev, bsz = cache._struct(dtype), cache.device, cache.bsz
    if seq_len is None:
        seq_len = cache.capacity
    elif seq_len > cache.capacity:
        raise ValueError(f"invalid seq_len {seq_len}: the cache has room for {cache.capacity} tokens")
    n = seq_len
    if idx is not None:
        if idx.dtype != torch.int32 or idx.dim() != 2 or idx.shape[0] != bsz or not idx.is_contiguous() or idx.device != dev:
            raise ValueError(f"idx must be a contiguous ({bsz}, n) int32 tensor on the cache's GPU")
        n = idx.shape[1]
    k, v = (torch.empty((bsz, cache.num_kv_heads, n, 128), dtype=dtype, device=dev) for _ in "kv")
    sb, sg, st, _ = k.stride()
    _launch(dev, lib().okv_kv8_read, c, idx.data_ptr() if idx is not None else None, n, n,
            _dev_i32(seq_lens, bsz, dev, "seq_lens"), seq_len, bsz, k.data_ptr(), v.data_ptr(), st, sg, sb)
    return k, v


# ---------------------------------------------------------------- pages of a cache
_MOST = 1 << 30  # pages, sequences, entries of a call (a larger number would be cut to 32 bits on its way)


class PageBuffers:
    """The arrays whose pages move together (every layer's K, V and scales): contiguous tensors
    (num_pages, ...) on one GPU, their page a multiple of 4 bytes.  Listed once, used by every call."""

    def __init__(self, tensors: Sequence[torch.Tensor]):
        self.tensors = list(tensors)
        if not self.tensors:
            raise ValueError("no buffers")
        self.device, self.num_pages = self.tensors[0].device, self.tensors[0].shape[0]
        if self.num_pages > _MOST:
            raise ValueError("more than 2^30 pages")
        self._c = (_lib.PageBuffer * len(self.tensors))()
        for t, b in zip(self.tensors, self._c):
            if not t.is_cuda or t.device != self.device or not t.is_contiguous() or t.shape[0] != self.num_pages:
                raise ValueError("buffers must be contiguous (num_pages, ...) tensors on one GPU")
            b.base, b.page_bytes = t.data_ptr(), t.numel() // max(1, self.num_pages) * t.element_size()

    def __len__(self) -> int:
        return len(self.tensors)


def _buffers(buffers) -> PageBuffers:
    return buffers if isinstance(buffers, PageBuffers) else PageBuffers(buffers)


def _page_pool(table, lens, refs, page_size):
    rows, width = table.shape
    stride, unit = table.stride()
    if max(rows, width, refs.numel()) > _MOST:
        raise ValueError("more than 2^30 sequences or pages")
    if table.dtype is not torch.int32 or unit != 1 or not table.is_cuda:
        raise ValueError("table must be a (num_seqs, max_pages) int32 GPU tensor with contiguous rows")
    if stride < width:
        if rows > 1:
            raise ValueError("table rows must not overlap")
        stride = width
    dev, pages = table.device, refs.numel()
    return dev, _lib.PagePool(table.data_ptr(), _dev_i32(lens, rows, dev, "lens"), _dev_i32(refs, pages, dev, "refs"), stride,
                              rows, width, pages, page_size)


def _entries(t, n, device, name):
    if t.dim() != 1 or not 1 <= n <= _MOST:
        raise ValueError(f"{name} must be a list of at least one entry (and at most 2^30)")
    return _dev_i32(t, n, device, name)


@functools.lru_cache(maxsize=4096)
def _pages_workspace_bytes(num_seqs: int, num_pages: int, n: int) -> int:
    out = C.c_size_t(0)
    check(lib().okv_pages_workspace_bytes(C.byref(_lib.PagePool(None, None, None, 0, num_seqs, 0, num_pages, 0)), n, C.byref(out)))
    return out.value


def _pages_scratch(pool, n, device):
    return _scratch(device, _pages_workspace_bytes(pool.num_seqs, pool.num_pages, n))


def pages_free(table, lens, refs, seqs, page_size: int, status: Optional[torch.Tensor] = None) -> None:
    """Sequences `seqs` give their pages back, in place: reference counts drop, table rows become -1, lengths 0.  table
    (num_seqs, max_pages), lens (num_seqs,), refs (num_pages,), seqs (n,): int32 on the GPU; status (2,) int32
    receives [0, entries outside the table].  okv_pages_free."""
    dev, pool = _page_pool(table, lens, refs, page_size)
    n = seqs.numel()
    _launch(dev, lib().okv_pages_free, pool, _entries(seqs, n, dev, "seqs"), n, _dev_i32(status, 2, dev, "status"))


def pages_fork(table, lens, refs, parents, children, page_size: int, buffers, status: Optional[torch.Tensor] = None,
               rows: Optional[PageBuffers] = None) -> None:
    """Sequence children[i] (empty) becomes a continuation of parents[i], in place: it shares the full pages and gets a copy
    of a partly filled last one in every buffer (a PageBuffers or a list of tensors; the lowest free pages).  rows: tensors
    (num_seqs, ...) whose row is copied from parent to child (an 8-bit cache's open buffers).  status
    (2,) int32 receives [pages short, pairs refused]; short of pages, nothing changes.  At most 1024 pairs.  okv_pages_fork."""
    dev, pool = _page_pool(table, lens, refs, page_size)
    bufs = _buffers(buffers)
    if bufs.device != dev or bufs.num_pages != refs.numel():
        raise ValueError("buffers must hold refs.numel() pages on the table's GPU")
    if rows is not None and (rows.device != dev or rows.num_pages != table.shape[0]):
        raise ValueError("rows must hold one row per sequence on the table's GPU")
    n = parents.numel()
    parents, children = _entries(parents, n, dev, "parents"), _entries(children, n, dev, "children")
    ws = _pages_scratch(pool, n, dev)
    _launch(dev, lib().okv_pages_fork, pool, parents, children, n, bufs._c, len(bufs), rows._c if rows else None,
            len(rows) if rows else 0, _dev_i32(status, 2, dev, "status"), ws.data_ptr(), ws.numel())


def pages_extend(table, lens, refs, seqs, more, page_size: int, status: Optional[torch.Tensor] = None) -> None:
    """Sequence seqs[i] grows by more[i] tokens, in place: it takes the pages it lacks from the lowest free ones.  status as in
    pages_fork.  okv_pages_extend."""
    dev, pool = _page_pool(table, lens, refs, page_size)
    n = seqs.numel()
    _launch(dev, lib().okv_pages_extend, pool, _entries(seqs, n, dev, "seqs"), _entries(more, n, dev, "more"), n,
            _dev_i32(status, 2, dev, "status"))


def pages_copy(buffers, src: torch.Tensor, dst: torch.Tensor, count: Optional[torch.Tensor] = None) -> None:
    """Pages dst[i] = pages src[i] of every buffer; count (1,) int32 on the GPU: only the first count.  No page may be
    both a source and a destination, and the destinations are distinct.  okv_pages_copy."""
    bufs, n = _buffers(buffers), src.numel()
    dev = bufs.device
    if n == 0:
        return
    _launch(dev, lib().okv_pages_copy, bufs._c, len(bufs), bufs.num_pages, _entries(src, n, dev, "src"),
            _entries(dst, n, dev, "dst"), _dev_i32(count, 1, dev, "count"), n)


def pages_compact(table, refs, buffers, table_out: Optional[torch.Tensor] = None, refs_out: Optional[torch.Tensor] = None):
    """Moves the pool's U used pages to pages 0 .. U-1 (those at or above U go to the free ones below, in order) and returns
    (table, refs, used): the renamed table and counts (new tensors, or table_out / refs_out, which may be the inputs) and
    U as a (1,) int32 GPU tensor.  okv_pages_compact."""
    dev, pool = _page_pool(table, None, refs, 1)
    bufs = _buffers(buffers)
    if bufs.device != dev or bufs.num_pages != refs.numel():
        raise ValueError("buffers must hold refs.numel() pages on the table's GPU")
    if table_out is None:
        table_out = torch.empty_like(table)
    elif table_out.shape != table.shape or table_out.dtype != torch.int32 or table_out.stride(1) != 1 or table_out.device != dev:
        raise ValueError("table_out must look like table")
    if refs_out is None:
        refs_out = torch.empty_like(refs)
    used = refs.new_empty(1)
    ws = _pages_scratch(pool, 0, dev)
    _launch(dev, lib().okv_pages_compact, pool, table_out.data_ptr(), max(table_out.stride(0), table_out.shape[1]),
            _dev_i32(refs_out, refs.numel(), dev, "refs_out"), used.data_ptr(), bufs._c, len(bufs), ws.data_ptr(), ws.numel())
    return table_out, refs_out, used

"""Attention whose mask is a sparse matrix: each query row attends to the key rows that its row of A lists.

``sparse_attention`` takes part in autograd; ``sparse_attention_forward`` / ``sparse_attention_backward`` are the same
kernels called directly; ``sparse_attention_decode`` is the form for single tokens over a cache, whose lists are a CSR in
device memory that may change with every call. Scores, softmax statistics and sums are fp32 in every case.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import call, dsp_attn_decode_desc, dsp_attn_desc, dsp_attn_grad_desc, lib
from .pattern import DTYPES, SparsePattern, need, no_tangents, on_device, ptr, stream_of, wants_grad, workspace


def _heads(t: torch.Tensor):
    """(tensor, (address, row stride, head stride)): t itself where the kernels can read it in place (dim contiguous, address
    and strides multiples of 16 bytes, no axis expanded), else a contiguous copy. Strides of axes of length one are free and
    are set to what the alignment rule accepts."""
    n, h, w = t.shape
    at = t.data_ptr()
    if t.is_contiguous() and at % 16 == 0:
        return t, (at, h * w, w)
    rs, hs, ws = t.stride()
    e = t.element_size()
    if (ws == 1 or w == 1) and at % 16 == 0 and (n <= 1 or (rs > 0 and rs * e % 16 == 0)) and (
            h <= 1 or (hs > 0 and hs * e % 16 == 0)):
        return t, (at, rs if n > 1 else h * w, hs if h > 1 else w)
    t = t.contiguous()
    if t.data_ptr() % 16:  # contiguous already, at an odd address
        t = t.clone()
    return t, (t.data_ptr(), h * w, w)


def _desc(q, k, v, out, lse, scale, softcap, slopes, row_offset):
    """q, k, v, out: as _heads gives them."""
    (n, heads, dim), kv_heads = q[0].shape, k[0].shape[1]
    return dsp_attn_desc(DTYPES[q[0].dtype], heads, kv_heads, dim, scale, softcap, ptr(slopes), row_offset, *q[1], *k[1], *v[1],
                         *out[1], ptr(lse))


def _check(device, rows, keys, q, k, v, scale, softcap, slopes):
    on_device("q", q, device)
    t = q.dtype
    if t not in DTYPES or q.dim() != 3 or q.shape[0] != rows:
        need(t in DTYPES, f"q must be fp32, bf16 or fp16, is {t}")
        need(False, f"q must have shape ({rows}, heads, dim), has {tuple(q.shape)}")
    on_device("k", k, device, t)
    heads, dim = q.shape[1:]
    if k.dim() != 3 or (keys is not None and k.shape[0] != keys) or k.shape[2] != dim:
        need(False, f"k must have shape ({'keys' if keys is None else keys}, kv_heads, {dim}), has {tuple(k.shape)}")
    on_device("v", v, device, t, k.shape)
    if k.shape[1] == 0 or heads == 0 or heads % k.shape[1]:
        need(False, f"{heads} query heads over {k.shape[1]} key/value heads")
    scale = 1.0 / math.sqrt(max(dim, 1)) if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    if not (math.isfinite(scale) and math.isfinite(softcap) and softcap >= 0):
        need(False, f"scale {scale}, softcap {softcap}")
    if slopes is not None:
        on_device("slopes", slopes, device, torch.float32, (heads,))
        need(not slopes.requires_grad, "slopes are constants: they get no gradient")
        slopes = slopes.contiguous()
    return _heads(q), _heads(k), _heads(v), scale, softcap, slopes


def _pattern(p, grad=False):
    need(isinstance(p, SparsePattern), "the first argument must be a SparsePattern")
    need(p.attention, "attention needs a SparsePattern(..., attention=True)")
    need(not grad or p.grad, "gradients need a SparsePattern(..., grad=True)")


def sparse_attention_forward(p: SparsePattern, q, k, v, scale=None, softcap=0.0, slopes=None, row_offset: int = 0):
    """(out, lse): out [rows, heads, dim] in q's type, lse [rows, heads] fp32."""
    _pattern(p)
    q, k, v, scale, softcap, slopes = _check(p.device, p.rows, p.cols, q, k, v, scale, softcap, slopes)
    out = torch.empty(q[0].shape, dtype=q[0].dtype, device=q[0].device)
    lse = torch.empty(out.shape[:2], dtype=torch.float32, device=out.device)
    d = _desc(q, k, v, _heads(out), lse, scale, softcap, slopes, row_offset)
    nbytes = lib().dsp_attn_workspace(p._h, ctypes.byref(d))
    ws = workspace(nbytes, out.device)
    call("dsp_attn", p._h, ctypes.byref(d), ptr(ws), nbytes, stream_of(p.device))
    return out, lse


def sparse_attention_backward(p: SparsePattern, dout, q, k, v, out, lse, scale=None, softcap=0.0, slopes=None,
                              row_offset: int = 0):
    """(dq, dk, dv) for the gradient ``dout`` of out; out and lse as the forward returned them, the other arguments as it
    took them."""
    _pattern(p, grad=True)
    q, k, v, scale, softcap, slopes = _check(p.device, p.rows, p.cols, q, k, v, scale, softcap, slopes)
    shape, t = q[0].shape, q[0].dtype
    on_device("dout", dout, p.device, t, shape)
    on_device("out", out, p.device, t, shape)
    on_device("lse", lse, p.device, torch.float32, shape[:2])
    dout, out, lse = _heads(dout), _heads(out), lse.contiguous()
    res = [torch.empty(x.shape, dtype=t, device=lse.device) for x, _ in (q, k, v)]
    g = dsp_attn_grad_desc(_desc(q, k, v, out, lse, scale, softcap, slopes, row_offset), *dout[1], *_heads(res[0])[1],
                           *_heads(res[1])[1], *_heads(res[2])[1])
    nbytes = lib().dsp_attn_grad_workspace(p._h, ctypes.byref(g.fwd))
    ws = workspace(nbytes, lse.device)
    call("dsp_attn_grad", p._h, ctypes.byref(g), ptr(ws), nbytes, stream_of(p.device))
    return tuple(res)


class _SparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, p, q, k, v, scale, softcap, slopes, row_offset):
        _pattern(p, grad=any(ctx.needs_input_grad))
        out, lse = sparse_attention_forward(p, q, k, v, scale, softcap, slopes, row_offset)
        ctx.p, ctx.opt = p, (scale, softcap)
        ctx.row_offset = row_offset
        ctx.save_for_backward(q, k, v, out, lse, slopes)  # slopes too: a change in place before the backward pass is noticed
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, lse, slopes = ctx.saved_tensors
        dq, dk, dv = sparse_attention_backward(ctx.p, dout, q, k, v, out, lse, *ctx.opt, slopes, ctx.row_offset)
        return None, dq, dk, dv, None, None, None, None


def sparse_attention(p: SparsePattern, q, k, v, scale=None, softcap=0.0, slopes=None, row_offset: int = 0,
                     return_lse: bool = False):
    """Attention of q [rows, heads, dim] over k, v [cols, kv_heads, dim] under the mask that p's entries are; differentiable
    in q, k and v (p needs grad=True then).

    scale: of the scores (None: 1 / sqrt(dim)); softcap: scores become softcap tanh(score / softcap); slopes [heads] fp32: a
    bias of -slope |i + row_offset - j|, a constant; heads a multiple of kv_heads. Rows without entries give 0 (lse:
    -infinity). fp32, bf16 or fp16; dim a multiple of 8 up to 256. return_lse: (out, lse) (lse has no gradient). Forward-mode derivatives are refused."""
    need(slopes is None or not slopes.requires_grad, "slopes are constants: they get no gradient")
    no_tangents(q, k, v, slopes)
    if not wants_grad(q, k, v):
        out, lse = sparse_attention_forward(p, q, k, v, scale, softcap, slopes, row_offset)
        return (out, lse) if return_lse else out
    out, lse = _SparseAttention.apply(p, q, k, v, scale, softcap, slopes, row_offset)
    return (out, lse) if return_lse else out


def sparse_attention_decode(q, k_cache, v_cache, indptr, indices, scale=None, softcap=0.0, slopes=None,
                            return_lse: bool = False):
    """One query token per sequence, q [rows, heads, dim], over the cache rows indices[indptr[r]:indptr[r+1]] of k_cache and
    v_cache [keys, kv_heads, dim], listed oldest first (int64 CSR on the device, read when the kernel runs: a captured
    graph sees the lists of its replay; their lengths, and so len(indices), are those of the capture at most).

    The last listed token is the newest: entry t of n is at distance n - 1 - t for ``slopes``. An entry outside the cache
    makes its row NaN. No gradient (forward-mode derivatives are refused)."""
    no_tangents(q, k_cache, v_cache, slopes)
    need(isinstance(q, torch.Tensor) and q.is_cuda and q.dim() == 3, "q must be a CUDA tensor [rows, heads, dim]")
    dev, rows = q.get_device(), q.shape[0]
    on_device("indptr", indptr, dev, torch.int64)
    on_device("indices", indices, dev, torch.int64)
    if indptr.dim() != 1 or indices.dim() != 1 or indptr.shape[0] != rows + 1:
        need(False, f"indptr must have {rows + 1} entries, has {tuple(indptr.shape)}")
    q, k, v, scale, softcap, slopes = _check(dev, rows, None, q, k_cache, v_cache, scale, softcap, slopes)
    indptr, indices = indptr.contiguous(), indices.contiguous()
    out = torch.empty(q[0].shape, dtype=q[0].dtype, device=q[0].device)
    lse = torch.empty(out.shape[:2], dtype=torch.float32, device=out.device) if return_lse else None
    g = dsp_attn_decode_desc(_desc(q, k, v, _heads(out), lse, scale, softcap, slopes, 0), rows, indices.numel(), k[0].shape[0],
                             indptr.data_ptr(), indices.data_ptr(), dev)
    nbytes = lib().dsp_attn_decode_workspace(ctypes.byref(g))
    ws = workspace(nbytes, out.device)
    call("dsp_attn_decode", ctypes.byref(g), ptr(ws), nbytes, stream_of(dev))
    return (out, lse) if return_lse else out

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
from .pattern import DTYPES, SparsePattern, need, on_device, ptr, workspace


def _heads(t: torch.Tensor) -> torch.Tensor:
    """t itself where the kernels can read it in place (dim contiguous, address and strides multiples of 16 bytes, no axis
    expanded), else a contiguous copy."""
    e = t.element_size()
    ok = t.stride(2) == 1 and t.data_ptr() % 16 == 0 and all(
        n <= 1 or (s > 0 and (s * e) % 16 == 0) for n, s in zip(t.shape[:2], t.stride()[:2]))
    return t if ok else t.contiguous()


def _strides(t: torch.Tensor):
    """(row, head) strides; those of axes of length one are free and are set to what the alignment rule accepts."""
    return (t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2], t.stride(1) if t.shape[1] > 1 else t.shape[2])


def _desc(q, k, v, out, lse, scale, softcap, slopes, row_offset):
    d = dsp_attn_desc(DTYPES[q.dtype], q.shape[1], k.shape[1], q.shape[2], scale, softcap, ptr(slopes), row_offset)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        setattr(d, name, t.data_ptr())
        row, head = _strides(t)
        setattr(d, name + "_row", row)
        setattr(d, name + "_head", head)
    d.lse = ptr(lse)
    return d


def _check(device, rows, keys, q, k, v, scale, softcap, slopes):
    on_device("q", q, device)
    need(q.dtype in DTYPES, f"q must be fp32, bf16 or fp16, is {q.dtype}")
    need(q.dim() == 3 and q.shape[0] == rows, f"q must have shape ({rows}, heads, dim), has {tuple(q.shape)}")
    on_device("k", k, device, q.dtype)
    need(k.dim() == 3 and (keys is None or k.shape[0] == keys) and k.shape[2] == q.shape[2],
         f"k must have shape ({'keys' if keys is None else keys}, kv_heads, {q.shape[2]}), has {tuple(k.shape)}")
    on_device("v", v, device, q.dtype, k.shape)
    need(k.shape[1] > 0 and q.shape[1] > 0 and q.shape[1] % k.shape[1] == 0,
         f"{q.shape[1]} query heads over {k.shape[1]} key/value heads")
    scale = 1.0 / math.sqrt(max(q.shape[2], 1)) if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    need(math.isfinite(scale) and math.isfinite(softcap) and softcap >= 0, f"scale {scale}, softcap {softcap}")
    if slopes is not None:
        on_device("slopes", slopes, device, torch.float32, (q.shape[1],))
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
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    d = _desc(q, k, v, out, lse, scale, softcap, slopes, row_offset)
    ws = workspace(lib().dsp_attn_workspace(p._h, ctypes.byref(d)), q.device)
    call("dsp_attn", p._h, ctypes.byref(d), ptr(ws), ws.numel(), torch.cuda.current_stream(q.device).cuda_stream)
    return out, lse


def sparse_attention_backward(p: SparsePattern, dout, q, k, v, out, lse, scale=None, softcap=0.0, slopes=None,
                              row_offset: int = 0):
    """(dq, dk, dv) for the gradient ``dout`` of out; out and lse as the forward returned them, the other arguments as it
    took them."""
    _pattern(p, grad=True)
    q, k, v, scale, softcap, slopes = _check(p.device, p.rows, p.cols, q, k, v, scale, softcap, slopes)
    on_device("dout", dout, p.device, q.dtype, q.shape)
    on_device("out", out, p.device, q.dtype, q.shape)
    on_device("lse", lse, p.device, torch.float32, q.shape[:2])
    dout, out, lse = _heads(dout), _heads(out), lse.contiguous()
    g = dsp_attn_grad_desc(_desc(q, k, v, out, lse, scale, softcap, slopes, row_offset))
    res = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)]
    for name, t in zip(("dout", "dq", "dk", "dv"), [dout] + res):
        setattr(g, name, t.data_ptr())
        row, head = _strides(t)
        setattr(g, name + "_row", row)
        setattr(g, name + "_head", head)
    ws = workspace(lib().dsp_attn_grad_workspace(p._h, ctypes.byref(g.fwd)), q.device)
    call("dsp_attn_grad", p._h, ctypes.byref(g), ptr(ws), ws.numel(), torch.cuda.current_stream(q.device).cuda_stream)
    return tuple(res)


class _SparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, p, q, k, v, scale, softcap, slopes, row_offset):
        _pattern(p, grad=any(ctx.needs_input_grad))
        out, lse = sparse_attention_forward(p, q, k, v, scale, softcap, slopes, row_offset)
        ctx.p, ctx.opt = p, (scale, softcap, slopes, row_offset)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = sparse_attention_backward(ctx.p, dout, q, k, v, out, lse, *ctx.opt)
        return None, dq, dk, dv, None, None, None, None


def sparse_attention(p: SparsePattern, q, k, v, scale=None, softcap=0.0, slopes=None, row_offset: int = 0,
                     return_lse: bool = False):
    """Attention of q [rows, heads, dim] over k, v [cols, kv_heads, dim] under the mask that p's entries are; differentiable
    in q, k and v (p needs grad=True then).

    scale: of the scores (None: 1 / sqrt(dim)); softcap: scores become softcap tanh(score / softcap); slopes [heads] fp32: a
    bias of -slope |i + row_offset - j|, a constant; heads a multiple of kv_heads. Rows without entries give 0 (lse:
    -infinity). fp32, bf16 or fp16; dim a multiple of 8 up to 256. return_lse: (out, lse) (lse has no gradient)."""
    need(slopes is None or not slopes.requires_grad, "slopes are constants: they get no gradient")
    out, lse = _SparseAttention.apply(p, q, k, v, scale, softcap, slopes, row_offset)
    return (out, lse) if return_lse else out


def sparse_attention_decode(q, k_cache, v_cache, indptr, indices, scale=None, softcap=0.0, slopes=None,
                            return_lse: bool = False):
    """One query token per sequence, q [rows, heads, dim], over the cache rows indices[indptr[r]:indptr[r+1]] of k_cache and
    v_cache [keys, kv_heads, dim], listed oldest first (int64 CSR on the device, read when the kernel runs: a captured
    graph sees the lists of its replay; their lengths, and so len(indices), are those of the capture at most).

    The last listed token is the newest: entry t of n is at distance n - 1 - t for ``slopes``. An entry outside the cache
    makes its row NaN. No gradient."""
    need(isinstance(q, torch.Tensor) and q.is_cuda, "q must be a CUDA tensor")
    dev = q.device.index
    on_device("indptr", indptr, dev, torch.int64)
    on_device("indices", indices, dev, torch.int64)
    need(indptr.dim() == 1 and indices.dim() == 1 and q.dim() == 3 and indptr.shape[0] == q.shape[0] + 1,
         f"indptr must have {q.shape[0] + 1} entries, has {tuple(indptr.shape)}")
    q, k, v, scale, softcap, slopes = _check(dev, q.shape[0], None, q, k_cache, v_cache, scale, softcap, slopes)
    indptr, indices = indptr.contiguous(), indices.contiguous()
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    g = dsp_attn_decode_desc(_desc(q, k, v, out, lse, scale, softcap, slopes, 0), q.shape[0], indices.numel(), k.shape[0],
                             ptr(indptr), ptr(indices))
    ws = workspace(lib().dsp_attn_decode_workspace(ctypes.byref(g)), q.device)
    with torch.cuda.device(q.device):
        call("dsp_attn_decode", ctypes.byref(g), ptr(ws), ws.numel(), torch.cuda.current_stream(q.device).cuda_stream)
    return (out, lse) if return_lse else out

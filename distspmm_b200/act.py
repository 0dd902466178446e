"""out = act(A.B + bias) + residual with A sparse, and its gradients.

``spmm_act`` takes part in autograd; ``spmm_act_forward`` / ``spmm_act_backward`` are the same
kernels called directly (for code that runs its own backward pass or captures it into a graph).
Dense operands are fp32, bf16 or fp16; A's values, the bias and their gradients are fp32; sums
are fp32 in every case.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import call, dsp_act_desc, dsp_act_grad_desc, lib
from .pattern import DTYPES, SparsePattern, ld, need, no_tangents, on_device, ptr, rows_of, stream_of, wants_grad, workspace

ACTS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _act(act):
    if act not in ACTS:
        need(False, f"act must be one of {sorted(k for k in ACTS if k)}, is {act!r}")
    return ACTS[act]


def _check(p: SparsePattern, B, values):
    need(isinstance(p, SparsePattern), "the first argument must be a SparsePattern")
    on_device("B", B, p.device)
    if B.dtype not in DTYPES or B.dim() != 2 or B.shape[0] != p.cols:
        need(B.dtype in DTYPES, f"B must be fp32, bf16 or fp16, is {B.dtype}")
        need(False, f"B must have shape ({p.cols}, N), has {tuple(B.shape)}")
    values = p.values if values is None else values
    on_device("values", values, p.device, torch.float32, (p.nnz,))
    return rows_of(B), values.contiguous()


def spmm_act_forward(p: SparsePattern, B: torch.Tensor, values=None, bias=None, residual=None, act=None,
                     save: bool = False):
    """(out, pre): pre is z = A.B + bias in fp32 where ``save`` asks for it and act is not none
    (what the backward pass needs; it stays fp32 because act' of a rounded z would cost the
    fp32 gradients their last 16 bits), else None."""
    code = _act(act)
    B, values = _check(p, B, values)
    N = B.shape[1]
    if bias is not None:
        on_device("bias", bias, p.device, torch.float32, (N,))
        bias = bias.contiguous()
    if residual is not None:
        on_device("residual", residual, p.device, B.dtype, (p.rows, N))
        residual = rows_of(residual)
    out = torch.empty((p.rows, N), dtype=B.dtype, device=B.device)
    pre = torch.empty((p.rows, N), dtype=torch.float32, device=B.device) if save and code else None
    d = dsp_act_desc(DTYPES[B.dtype], code, N, ptr(values), ptr(B), ld(B), ptr(bias), ptr(residual),
                     ld(residual) if residual is not None else 0, ptr(out), N, ptr(pre), N)
    nbytes = lib().dsp_spmm_act_workspace(p._h, N)
    ws = workspace(nbytes, B.device)
    call("dsp_spmm_act", p._h, ctypes.byref(d), ptr(ws), nbytes, stream_of(p.device))
    return out, pre


def spmm_act_backward(p: SparsePattern, dout: torch.Tensor, B: torch.Tensor, pre, values=None, act=None,
                      need_B: bool = True, need_values: bool = True, need_bias: bool = True):
    """(dB, dvalues, dbias) for the gradient ``dout`` of out; a result that is not asked for is None.
    The gradient of the residual is ``dout`` itself."""
    code = _act(act)
    B, values = _check(p, B, values)
    N = B.shape[1]
    on_device("dout", dout, p.device, B.dtype, (p.rows, N))
    dout = rows_of(dout)
    if code:
        need(pre is not None, "the activation's gradient needs pre (spmm_act_forward(..., save=True))")
        on_device("pre", pre, p.device, torch.float32, (p.rows, N))
        pre = rows_of(pre)
    need(not need_B or p.grad, "dB needs a SparsePattern(..., grad=True)")
    dev = B.device
    dB = torch.empty((p.cols, N), dtype=B.dtype, device=dev) if need_B else None
    dvalues = torch.empty(p.nnz, dtype=torch.float32, device=dev) if need_values else None
    dbias = torch.empty(N, dtype=torch.float32, device=dev) if need_bias else None
    d = dsp_act_grad_desc(DTYPES[B.dtype], code, N, ptr(values), ptr(B), ld(B), ptr(pre) if code else None,
                          ld(pre) if code else 0, ptr(dout), ld(dout), ptr(dB), N, ptr(dvalues), ptr(dbias))
    nbytes = lib().dsp_spmm_act_grad_workspace(p._h, ctypes.byref(d))
    ws = workspace(nbytes, dev)
    call("dsp_spmm_act_grad", p._h, ctypes.byref(d), ptr(ws), nbytes, stream_of(p.device))
    return dB, dvalues, dbias


class _SpmmAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, p, act, B, values, bias, residual):
        # z is kept only where its activation's gradient will be asked for
        out, pre = spmm_act_forward(p, B, values, bias, residual, act, save=any(ctx.needs_input_grad[2:5]))
        ctx.p, ctx.act = p, act
        ctx.save_for_backward(B, values, pre)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        B, values, pre = ctx.saved_tensors
        nB, nv, nb, nr = ctx.needs_input_grad[2:]
        dB = dvalues = dbias = None
        if nB or nv or nb:
            dB, dvalues, dbias = spmm_act_backward(ctx.p, dout, B, pre, values, ctx.act, nB, nv, nb)
        return None, None, dB, dvalues, dbias, dout if nr else None


def spmm_act(p: SparsePattern, B: torch.Tensor, values=None, bias=None, residual=None, act=None) -> torch.Tensor:
    """act(A.B + bias) + residual, [rows, N] in B's type, differentiable in B, values, bias and
    residual (dB needs a pattern with grad=True).

    values: [nnz] fp32 in CSR order (None: A's own); bias: [N] fp32; residual: [rows, N] in B's
    type; act: None, "relu", "silu" or "gelu" (erf form). Runs on the current stream. Forward-mode derivatives are refused."""
    no_tangents(B, values, bias, residual)
    if not wants_grad(B, values, bias, residual):
        return spmm_act_forward(p, B, values, bias, residual, act)[0]
    need(isinstance(p, SparsePattern), "the first argument must be a SparsePattern")
    need(p.grad or not B.requires_grad, "a gradient of B needs a SparsePattern(..., grad=True)")
    if values is None:
        values = p.values
    return _SpmmAct.apply(p, act, B, values, bias, residual)

"""A CSR matrix prepared on one GPU for the sparse-layer operators.

``SparsePattern`` holds A's entries in device memory as the fused product (``spmm_act``) and
attention (``sparse_attention``) read them: 32-bit ids, chunks of equal work and, for
gradients, the transposed lists. It is read-only: several streams and captured graphs may use
one pattern at a time.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from ._lib import c_vp, call, dsp_pattern_info, lib
from .matrix import Csr

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class SparsePattern:
    """grad: keep the transposed lists that gradients need. attention: check that no row lists a
    column twice and prepare the forms that attention reads. form: "tiles" or "rows" force how
    attention reads the pattern (None: tiles where they are filled well enough)."""

    GRAD, ATTENTION = 1, 2
    FORMS = {None: 0, "tiles": 4, "rows": 8}

    def __init__(self, a: Csr, device: int = 0, grad: bool = False, attention: bool = False, form: str | None = None):
        need(form in self.FORMS, f"form must be one of {sorted(k for k in self.FORMS if k)}, is {form!r}")
        self.device = device
        self.rows = a.num_rows
        self.cols = a.num_cols
        self.nnz = a.nnz
        self.grad = bool(grad)
        self.attention = bool(attention)
        c = a.to_c()
        h = c_vp()
        call("dsp_pattern_create", device, ctypes.byref(c), self.GRAD * self.grad + self.ATTENTION * self.attention +
             self.FORMS[form], ctypes.byref(h))
        self._h = h
        self._host_values = a.values.copy()  # those of now, whatever becomes of a
        self._values = None

    @property
    def values(self) -> torch.Tensor:
        """A's own values on the device (fp32, CSR order), uploaded on first use (so use it once
        before capturing a graph that relies on it)."""
        if self._values is None:
            self._values = torch.from_numpy(self._host_values).to(torch.device("cuda", self.device))
        return self._values

    def info(self) -> dict:
        i = dsp_pattern_info()
        call("dsp_pattern_info_get", self._h, ctypes.byref(i))
        return {k: int(getattr(i, k)) for k, _ in dsp_pattern_info._fields_}

    def check_error(self) -> None:
        """After the streams were synchronised: raise DspError if an attention kernel's bounded wait
        gave up (its rows are NaN; the flag is cleared)."""
        call("dsp_pattern_check_error", self._h)

    def close(self) -> None:
        """Free the device memory; no call that uses the pattern may still be running."""
        if getattr(self, "_h", None):
            lib().dsp_pattern_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def on_device(name: str, t: torch.Tensor, device: int, dtype=None, shape=None) -> None:
    """The checks that every dense operand goes through."""
    if (type(t) is torch.Tensor and t.is_cuda and t.get_device() == device and (dtype is None or t.dtype == dtype)
            and (shape is None or t.shape == shape)):
        return
    need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    need(t.is_cuda and t.get_device() == device, f"{name} must be on cuda:{device}, is on {t.device}")
    need(dtype is None or t.dtype == dtype, f"{name} must be {dtype}, is {t.dtype}")
    need(shape is None or tuple(t.shape) == tuple(shape), f"{name} must have shape {shape}, has {tuple(t.shape)}")


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """t itself where its rows are contiguous and do not overlap, else a contiguous copy."""
    if t.is_contiguous():
        return t
    return t if (t.stride(1) == 1 or t.shape[1] <= 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


def ld(t: torch.Tensor) -> int:
    """Leading dimension of rows_of(t)."""
    n, w = t.shape
    return max(t.stride(0), w) if n > 1 else max(w, 1)


def ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    """Workspace of one call, from torch's allocator on the current stream (so that calls on other
    streams and captured graphs never share it)."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def stream_of(device: int) -> int:
    """The current stream of the device (cudaStream_t as int)."""
    return torch._C._cuda_getCurrentRawStream(device)


def no_tangents(*tensors) -> None:
    """Refuse dual tensors: only reverse-mode gradients are provided, and a tangent would be lost without a word."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            need(not isinstance(t, torch.Tensor) or forward_ad.unpack_dual(t).tangent is None,
                 "forward-mode derivatives are not provided")


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)

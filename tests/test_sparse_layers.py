"""Refusals of the sparse-layer entry points that need no GPU: the checks come before any CUDA call."""
import ctypes

import numpy as np
import pytest
import torch

import distspmm_b200 as d
from distspmm_b200._lib import DspError, c_vp, dsp_act_desc, dsp_act_grad_desc, dsp_pattern_info
from sparse_reference import csr_of


def status(name, *args):
    return getattr(d.lib(), name)(*args)


def test_pattern_refuses_bad_matrices():
    with pytest.raises(DspError, match="lists a column twice"):
        d.SparsePattern(csr_of([[0, 1], [2, 0, 2]], 3), attention=True)
    with pytest.raises(DspError, match="DSP_ERR_FORMAT"):
        d.SparsePattern(csr_of([[0, 3]], 3))
    with pytest.raises(DspError, match="DSP_ERR_FORMAT"):
        d.SparsePattern(csr_of([[0, -1]], 3))
    bad = csr_of([[0], [1], [2]], 3)
    bad.indptr[1] = 3
    with pytest.raises(DspError, match="DSP_ERR_FORMAT"):
        d.SparsePattern(bad)
    big = csr_of([[0]], 1)
    big.num_cols = 1 << 31
    with pytest.raises(DspError, match="DSP_ERR_UNSUPPORTED"):
        d.SparsePattern(big)
    c = csr_of([[0]], 1).to_c()
    h = c_vp()
    assert status("dsp_pattern_create", 0, ctypes.byref(c), 64, ctypes.byref(h)) == -1
    assert status("dsp_pattern_create", 0, ctypes.byref(c), 2 + 4 + 8, ctypes.byref(h)) == -1
    with pytest.raises(ValueError, match="form must be"):
        d.SparsePattern(csr_of([[0]], 1), attention=True, form="columns")
    assert status("dsp_pattern_create", 0, None, 0, ctypes.byref(h)) == -1
    assert status("dsp_pattern_info_get", None, ctypes.byref(dsp_pattern_info())) == -1
    d.lib().dsp_pattern_destroy(None)


def test_null_arguments():
    assert status("dsp_spmm_act", None, ctypes.byref(dsp_act_desc()), None, 0, None) == -1
    assert status("dsp_spmm_act_grad", None, ctypes.byref(dsp_act_grad_desc()), None, 0, None) == -1
    assert d.lib().dsp_spmm_act_workspace(None, 8) == 0
    assert d.lib().dsp_spmm_act_grad_workspace(None, None) == 0


def test_python_refuses_what_is_no_pattern():
    with pytest.raises(ValueError, match="SparsePattern"):
        d.spmm_act("A", torch.ones(2, 2))
    with pytest.raises(ValueError, match="act must be"):
        d.spmm_act_forward("A", torch.ones(2, 2), act="swish")


def test_attention_null_arguments():
    from distspmm_b200._lib import dsp_attn_decode_desc, dsp_attn_desc, dsp_attn_grad_desc
    assert status("dsp_attn", None, ctypes.byref(dsp_attn_desc()), None, 0, None) == -1
    assert status("dsp_attn_grad", None, ctypes.byref(dsp_attn_grad_desc()), None, 0, None) == -1
    assert status("dsp_attn_decode", None, None, 0, None) == -1
    assert d.lib().dsp_attn_workspace(None, None) == 0
    assert d.lib().dsp_attn_grad_workspace(None, None) == 0
    assert d.lib().dsp_attn_decode_workspace(None) == 0


def decode_desc(**kw):
    from distspmm_b200._lib import dsp_attn_decode_desc, dsp_attn_desc
    f = dict(dtype=1, heads=4, kv_heads=2, dim=64, scale=0.125, softcap=0.0, slopes=None, row_offset=0, q=1 << 12, q_row=256, q_head=64,
             k=1 << 13, k_row=128, k_head=64, v=1 << 14, v_row=128, v_head=64, out=1 << 15, out_row=256, out_head=64, lse=None)
    g = dict(rows=1, nnz=5, keys=5, indptr=1 << 16, indices=1 << 17, device=0)
    for k, v in kw.items():
        (f if k in f else g)[k] = v
    return dsp_attn_decode_desc(dsp_attn_desc(*f.values()), *g.values())


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=3), -1), (dict(heads=0), -1), (dict(kv_heads=3), -1), (dict(kv_heads=0), -1), (dict(dim=0), -6), (dict(dim=20), -6),
    (dict(dim=264), -6), (dict(softcap=-1.0), -1), (dict(softcap=float("inf")), -1), (dict(softcap=1e-9), -1), (dict(scale=float("inf")), -1), (dict(scale=float("nan")), -1), (dict(q=None), -1),
    (dict(q=(1 << 12) + 2), -1), (dict(k_row=129), -1), (dict(k_row=-128), -1), (dict(v_row=1 << 30), -6), (dict(out=None), -1), (dict(indptr=None), -1), (dict(indices=None), -1),
    (dict(rows=-1), -1), (dict(nnz=-1), -1), (dict(rows=1 << 25), -6), (dict(nnz=1 << 31), -6), (dict(), -1)])
def test_decode_refuses(bad, code):
    """Bad arguments, and (last) a missing workspace: all refused before anything reaches a device."""
    assert status("dsp_attn_decode", ctypes.byref(decode_desc(**bad)), None, 0, None) == code


def test_act_refuses_wide_products():
    d1 = dsp_act_desc(0, 0, (1 << 22) + 1)
    p = 1 << 12  # never read: the check comes first
    assert status("dsp_spmm_act", p, ctypes.byref(d1), None, 0, None) == -6

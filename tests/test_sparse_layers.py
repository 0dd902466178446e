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

"""Attention tiles whose bounded waits run out: no copies are started (DSP_ATTN_WAIT_CYCLES=0), so that every wait gives up at once, with
nothing in flight. The rows are NaN, the pattern's error word says so, and calls after it are right."""
import pytest
import torch

import distspmm_b200 as d
from distspmm_b200._lib import DspError
from sparse_reference import csr_of, positional
from test_attention_gpu import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("split", [False, True])
def test_rows_of_a_wait_that_gave_up_are_nan(gpu, monkeypatch, split, dim, t):
    if split:  # one row tile over many keys, in pieces; the last rows have no entry
        a = csr_of([list(range(3000)) if i < 90 else [] for i in range(100)], 3000)
    else:
        a = positional("docs", 300, cuts=[0, 130, 290])
    empty = torch.from_numpy(a.indptr).diff() == 0
    q, k, v, dout = (x.cuda() for x in inputs(a.num_rows, a.num_cols, 2, 1, dim, t, 3))
    fine = d.SparsePattern(a, grad=True, attention=True, form="tiles")
    monkeypatch.setenv("DSP_ATTN_WAIT_CYCLES", "0")
    cut = d.SparsePattern(a, grad=True, attention=True, form="tiles")
    out, lse = d.sparse_attention_forward(cut, q, k, v)
    torch.cuda.synchronize()
    with pytest.raises(DspError, match="DSP_ERR_TIMEOUT"):
        cut.check_error()
    cut.check_error()  # cleared
    assert torch.isnan(out[~empty]).all() and torch.isnan(lse[~empty]).all()
    want = d.sparse_attention_forward(fine, q, k, v)
    dq, dk, dv = d.sparse_attention_backward(cut, dout, q, k, v, *want)
    listed = torch.zeros(a.num_cols, dtype=torch.bool)
    listed[torch.from_numpy(a.indices)] = True
    assert torch.isnan(dq[~empty]).all() and torch.isnan(dk[listed]).all() and torch.isnan(dv[listed]).all()
    torch.cuda.synchronize()
    with pytest.raises(DspError, match="DSP_ERR_TIMEOUT"):
        cut.check_error()
    fine.check_error()
    again = d.sparse_attention_forward(fine, q, k, v)
    assert all(torch.equal(x, y) for x, y in zip(again, want)) and torch.isfinite(want[0]).all()

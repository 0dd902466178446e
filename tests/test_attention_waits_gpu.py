"""The waits of the attention tiles."""
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
    """No copies are started (DSP_ATTN_WAIT_CYCLES=0), so that every wait gives up at once, with nothing in flight: the rows are NaN,
    the pattern's error word says so, and calls after it are right."""
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


def test_forward_beside_backward_of_another_stream(gpu):
    """Backward CTAs of dim 128 take all of an SM's tensor memory, forward ones half of it: side by side on two streams the later
    allocation waits for the earlier CTA's end. Results are those of calls one after another, bit for bit."""
    a = positional("window", 2500, window=400)
    p = d.SparsePattern(a, grad=True, attention=True, form="tiles")
    sets = []
    for s, dim in enumerate((128, 64)):
        x = [y.cuda() for y in inputs(2500, 2500, 8, 4, dim, torch.bfloat16, s)]
        fwd = d.sparse_attention_forward(p, *x[:3])
        sets.append((x, fwd, d.sparse_attention_backward(p, x[3], *x[:3], *fwd)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for (x, fwd, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(d.sparse_attention_backward(p, x[3], *x[:3], *fwd))
        with torch.cuda.stream(streams[2]):
            got.append(d.sparse_attention_forward(p, *sets[0][0][:3]))
            got.append(d.sparse_attention_forward(p, *sets[1][0][:3]))
    torch.cuda.synchronize()
    p.check_error()
    want = [sets[0][2], sets[1][2], sets[0][1], sets[1][1]]
    for i, g in enumerate(got):
        assert all(torch.equal(y, z) for y, z in zip(g, want[i % 4]))


@pytest.mark.parametrize("text", ["", "fast", "-1", "10 s"])
def test_limits_that_are_no_number_are_ignored(gpu, monkeypatch, text):
    monkeypatch.setenv("DSP_ATTN_WAIT_CYCLES", text)
    a = positional("window", 200, window=50)
    p = d.SparsePattern(a, attention=True, form="tiles")
    q, k, v, _ = (x.cuda() for x in inputs(200, 200, 2, 1, 64, torch.bfloat16, 3))
    assert torch.isfinite(d.sparse_attention(p, q, k, v)).all()
    p.check_error()

"""spmm_act (product with bias, activation, residual) and its gradients against 64-bit forms.

Tolerances, from the arithmetic: a sum of n products in fp32, in any order, is off by at most (n + 2) u sum|terms|, u = 2^-24
(2 more for the bias and the product's own rounding); the activations have slopes of at most 1.13 and are evaluated within
8 u max(|z|, 1); the result is rounded to its type once, half a step.
"""
import numpy as np
import pytest
import torch

import distspmm_b200 as d
from sparse_reference import HALF_STEP, TINY, U, act64, csr_of, matrix, product64, row_ids

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(a, n, t, seed=0, bias=True, residual=True, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    B = torch.randn((a.num_cols, n), generator=g).to(t)
    r = torch.randn((a.num_rows, n), generator=g).to(t) if residual else None
    b = torch.randn(n, generator=g) if bias else None
    dy = torch.randn((a.num_rows, n), generator=g).to(t)
    return B, b, r, dy


def cuda(x):
    return None if x is None else x.cuda()


def wide(x):
    return None if x is None else x.double()


def lens(a):
    return torch.from_numpy(np.diff(a.indptr)).double()


def near(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    bad = (got - want).abs() > tol
    assert not bad.any() and torch.isfinite(got).all(), \
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol).max():.2f} of the tolerance"


def forward_tolerance(a, y, z, size, residual, t):
    tol = 1.13 * (lens(a)[:, None] + 2) * U * size + 8 * U * z.abs().clamp(min=1)
    if residual is not None:
        tol = tol + U * (y.abs() + residual.abs())
    return tol + HALF_STEP[t] * (y.abs() + tol) + TINY[t]


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 3, 8, 33, 64, 100, 128, 129, 200, 256, 300, 520, 1030])
def test_widths(gpu, n, t):
    a = matrix("rmat")
    p = d.SparsePattern(a)
    B, b, r, _ = inputs(a, n, t, n)
    out = d.spmm_act(p, B.cuda(), None, cuda(b), cuda(r), "gelu")
    y, z, size = product64(a, wide(B), torch.from_numpy(a.values).double(), wide(b), wide(r), "gelu")
    assert out.dtype == t
    near(out, y, forward_tolerance(a, y, z, size, wide(r), t), "out")


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("kind", ["rmat", "hub", "empty", "row", "column", "one", "repeated", "gap"])
def test_matrices(gpu, kind, act):
    a = matrix(kind)
    p = d.SparsePattern(a)
    for t, n, bias, residual in ((F32, 64, True, False), (BF16, 96, False, True), (F16, 20, True, True), (BF16, 7, False, False)):
        B, b, r, _ = inputs(a, n, t, n, bias, residual)
        out = d.spmm_act(p, B.cuda(), None, cuda(b), cuda(r), act)
        y, z, size = product64(a, wide(B), torch.from_numpy(a.values).double(), wide(b), wide(r), act)
        near(out, y, forward_tolerance(a, y, z, size, wide(r), t), f"{kind} {t} {n}")


def grads64(a, B, values, bias, dy, act):
    """(dB, dvalues, dbias, dz, sizes) by the formulas."""
    rows, cols = row_ids(a), torch.from_numpy(a.indices)
    z = product64(a, B, values, bias, None, act)[1].detach().requires_grad_()
    (slope,) = torch.autograd.grad(act64(z, act).sum(), z)
    slope = torch.nan_to_num(slope)
    dz = dy * slope
    dB = torch.zeros_like(B).index_add(0, cols, values[:, None] * dz[rows])
    sB = torch.zeros_like(B).index_add(0, cols, values.abs()[:, None] * dz.abs()[rows])
    dv = (dz[rows] * B[cols]).sum(1)
    sv = (dz.abs()[rows] * B.abs()[cols]).sum(1)
    return dB, dv, dz.sum(0), dz, (sB, sv, dz.abs().sum(0))


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("t,n", [(F32, 64), (F32, 129), (F32, 260), (BF16, 128), (BF16, 40), (BF16, 600), (F16, 256), (F16, 33), (F16, 1)])
@pytest.mark.parametrize("kind", ["rmat", "hub", "empty", "row", "column", "repeated", "gap"])
def test_gradients(gpu, kind, t, n, act):
    a = matrix(kind)
    p = d.SparsePattern(a, grad=True)
    B, b, _, dy = inputs(a, n, t, n)
    values = torch.from_numpy(a.values)
    out, pre = d.spmm_act_forward(p, B.cuda(), None, cuda(b), None, act, save=True)
    dB, dv, db = d.spmm_act_backward(p, dy.cuda(), B.cuda(), pre, None, act)
    wB, wv, wb, dz, (sB, sv, sb) = grads64(a, wide(B), wide(values), wide(b), wide(dy), act)
    assert dB.dtype == t and dv.dtype == F32 and db.dtype == F32
    tol = grad_tolerances(a, B, values, b, dy, act, t, n, dz, wB, wv, wb, sB, sv, sb)
    near(dB, wB, tol[0], "dB")
    near(dv, wv, tol[1], "dvalues")
    near(db, wb, tol[2], "dbias")


def grad_tolerances(a, B, values, b, dy, act, t, n, dz, wB, wv, wb, sB, sv, sb):
    """z carries the forward sum's error e into act' (second derivatives are at most 0.8 for both activations); act' itself is
    evaluated within 8 u max(|z|, 1); so each dz is off by at most e_dz. dB sums dz rounded to t (half a step each, except with
    no activation: dz is dout itself)."""
    if act is None:
        e_dz = torch.zeros_like(dz)
    else:
        _, z, size = product64(a, wide(B), wide(values), wide(b), None, act)
        e_dz = wide(dy).abs() * (0.8 * (lens(a)[:, None] + 2) * U * size + 9 * U * z.abs().clamp(min=1))
    rows, cols = row_ids(a), torch.from_numpy(a.indices)
    count = torch.bincount(cols, minlength=a.num_cols).double()
    e_row = e_dz + (0 if act is None else HALF_STEP[t] * (dz.abs() + e_dz) + TINY[t])
    e_B = torch.zeros_like(wB).index_add(0, cols, wide(values).abs()[:, None] * e_row[rows]) + (count[:, None] + 2) * U * sB
    e_v = (e_dz[rows] * wide(B).abs()[cols]).sum(1) + (n + 2) * U * sv
    return (1.01 * e_B + HALF_STEP[t] * (wB.abs() + e_B) + TINY[t], 1.01 * e_v + 1e-37,
            1.01 * (e_dz.sum(0) + (a.num_rows + 2) * U * sb) + 1e-37)


def test_relu_gradient(gpu):
    """Small whole numbers: every sum is exact, so that z = 0 is 0 and its slope is 0."""
    a = matrix("rmat")
    values = torch.from_numpy(np.random.default_rng(1).integers(-2, 3, a.nnz)).float()
    g = torch.Generator().manual_seed(5)
    for t in (F32, BF16):
        B = torch.randint(-2, 3, (a.num_cols, 64), generator=g).to(t)
        dy = torch.randint(-3, 4, (a.num_rows, 64), generator=g).to(t)
        p = d.SparsePattern(a, grad=True)
        _, pre = d.spmm_act_forward(p, B.cuda(), values.cuda(), None, None, "relu", save=True)
        z = product64(a, wide(B), wide(values), None, None, None)[1]
        assert torch.equal(pre.cpu().double(), z) and (z == 0).any()
        dB, dv, db = d.spmm_act_backward(p, dy.cuda(), B.cuda(), pre, values.cuda(), "relu")
        dz = wide(dy) * (z > 0)
        rows, cols = row_ids(a), torch.from_numpy(a.indices)
        assert torch.equal(dv.cpu().double(), (dz[rows] * wide(B)[cols]).sum(1))
        assert torch.equal(db.cpu().double(), dz.sum(0))
        want = torch.zeros_like(wide(B)).index_add(0, cols, wide(values)[:, None] * dz[rows])
        assert torch.equal(dB.cpu().double(), want.to(t).double())


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_autograd_and_differences(gpu, act):
    """autograd's gradients are the backward entry's, and agree with differences of the 64-bit form: for the loss L = sum(out * dy)
    along random directions, central differences of step 1e-4 are off by O(1e-8) of the third derivatives, well below the 2e-5
    relative to the sum of magnitudes that fp32 gradients are held to here (64 terms and more of 2^-24 each)."""
    a = matrix("rmat")
    p = d.SparsePattern(a, grad=True)
    B, b, r, dy = inputs(a, 32, F32, 3)
    leaves = [x.cuda().requires_grad_() for x in (B, torch.from_numpy(a.values).clone(), b, r)]
    out = d.spmm_act(p, leaves[0], leaves[1], leaves[2], leaves[3], act)
    got = torch.autograd.grad(out, leaves, dy.cuda())
    _, pre = d.spmm_act_forward(p, leaves[0].detach(), leaves[1].detach(), leaves[2].detach(), None, act, save=True)
    direct = d.spmm_act_backward(p, dy.cuda(), leaves[0].detach(), pre, leaves[1].detach(), act)
    for x, y in zip(got, direct + (dy.cuda(),)):
        assert torch.equal(x, y)
    g = torch.Generator().manual_seed(9)
    base = [wide(x) for x in (B, torch.from_numpy(a.values), b, r)]
    loss = lambda v: (product64(a, v[0], v[1], v[2], v[3], act)[0] * wide(dy)).sum()  # noqa: E731
    for k in range(4):
        u = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        up, down = list(base), list(base)
        up[k], down[k] = base[k] + 1e-4 * u, base[k] - 1e-4 * u
        diff = float(loss(up) - loss(down)) / 2e-4
        terms = (got[k].cpu().double() * u).reshape(-1)
        assert abs(float(terms.sum()) - diff) <= 2e-5 * float(terms.abs().sum())


@pytest.mark.parametrize("t", [F32, BF16])
def test_strides_and_alignment(gpu, t):
    """Windows of wider buffers at every alignment, transposed and expanded operands; nothing outside is read (NaN there)."""
    a = matrix("rmat")
    p = d.SparsePattern(a, grad=True)
    n = 64
    B, b, r, dy = inputs(a, n, t, 2)
    want = d.spmm_act(p, B.cuda(), None, b.cuda(), r.cuda(), "silu")
    _, pre = d.spmm_act_forward(p, B.cuda(), None, b.cuda(), None, "silu", save=True)
    values = torch.from_numpy(a.values)
    y, z, size = product64(a, wide(B), wide(values), wide(b), wide(r), "silu")
    tol = forward_tolerance(a, y, z, size, wide(r), t)
    wB, wv, wb, dz, sizes = grads64(a, wide(B), wide(values), wide(b), wide(dy), "silu")
    tols = grad_tolerances(a, B, values, b, dy, "silu", t, n, dz, wB, wv, wb, *sizes)

    def window(x, left, right):
        w = torch.full((x.shape[0], left + n + right), float("nan"), dtype=x.dtype, device="cuda")
        w[:, left:left + n] = x.cuda()
        return w[:, left:left + n]

    for left, right in ((0, 8), (8, 0), (4, 4), (2, 1), (1, 0), (3, 6)):
        out = d.spmm_act(p, window(B, left, right), None, b.cuda(), window(r, right, left), "silu")
        near(out, y, tol, "out")  # alignment sets the vector width, and that the order of the sums
        grads = d.spmm_act_backward(p, window(dy, left, right), window(B, right, left), window(pre, left, 0), None, "silu")
        for x, w, e, name in zip(grads, (wB, wv, wb), tols, ("dB", "dvalues", "dbias")):
            near(x, w, e, name)
    Bt = B.t().contiguous().cuda().t()
    assert torch.equal(d.spmm_act(p, Bt, None, b.cuda(), r.cuda(), "silu"), want)
    one = torch.randn((1, n)).to(t).cuda()
    assert torch.equal(d.spmm_act(p, one.expand(a.num_cols, n)), d.spmm_act(p, one.expand(a.num_cols, n).contiguous()))
    with_r = d.spmm_act(p, B.cuda(), residual=one.expand(a.num_rows, n))
    assert torch.equal(with_r, d.spmm_act(p, B.cuda(), residual=one.expand(a.num_rows, n).contiguous()))


def test_broadcast_inputs_get_summed_gradients(gpu):
    a = matrix("rmat")
    p = d.SparsePattern(a, grad=True)
    one = torch.randn(1, 64, device="cuda", requires_grad=True)
    d.spmm_act(p, one.expand(a.num_cols, 64)).sum().backward()
    want = torch.zeros(64, dtype=torch.float64) + float(a.values.astype(np.float64).sum())
    near(one.grad[0], want, (a.nnz + 2) * U * np.abs(a.values).sum() + 0 * want, "gradient of a broadcast B")


def test_not_finite_values_stay_in_their_rows(gpu):
    """NaN and infinities in rows of B that a row of A does not list leave it as it was."""
    a = csr_of([[0, 2], [1], [], [3, 4, 5]], 6, [1.0, 2.0, 1.0, 1.0, 1.0, 1.0])
    p = d.SparsePattern(a)
    B = torch.ones(6, 40)
    B[1] = float("inf")
    B[4] = float("nan")
    out = d.spmm_act(p, B.cuda()).cpu()
    assert (out[0] == 3).all() and torch.isinf(out[1]).all() and (out[2] == 0).all() and torch.isnan(out[3]).all()
    for act in ("relu", "silu", "gelu"):
        assert torch.isnan(d.spmm_act(p, B.cuda(), act=act).cpu()[3]).all()


def test_same_bits_every_time(gpu):
    a = d.gen_rmat(13, seed=2)
    p = d.SparsePattern(a, grad=True)
    B, b, r, dy = inputs(a, 128, BF16, 1)
    runs = []
    for _ in range(2):
        out, pre = d.spmm_act_forward(p, B.cuda(), None, b.cuda(), r.cuda(), "gelu", save=True)
        runs.append((out, pre) + d.spmm_act_backward(p, dy.cuda(), B.cuda(), pre, None, "gelu"))
    for x, y in zip(*runs):
        assert torch.equal(x, y)


def test_graphs_and_streams(gpu):
    """Two captured graphs and an eager call of one pattern, replayed on two streams at once."""
    a = d.gen_rmat(11, seed=5)
    p = d.SparsePattern(a, grad=True)
    sets = []
    for k in range(2):
        B, b, r, dy = (x.cuda() for x in inputs(a, 128, BF16, k))
        v = torch.rand(a.nnz, device="cuda")

        def step(B=B, b=b, r=r, dy=dy, v=v):
            out, pre = d.spmm_act_forward(p, B, v, b, r, "silu", save=True)
            return (out,) + d.spmm_act_backward(p, dy, B, pre, v, "silu")

        want = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        sets.append((step, want, graph, got, (B, b, r, dy, v)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (_, _, graph, _, _) in zip(streams, sets):
            with torch.cuda.stream(s):
                graph.replay()
        eager = sets[0][0]()
        torch.cuda.synchronize()
        for _, want, _, got, _ in sets:
            for x, y in zip(got, want):
                assert torch.equal(x, y)
        for x, y in zip(eager, sets[0][1]):
            assert torch.equal(x, y)
    # new inputs in the captured buffers
    B = sets[0][4][0]
    B.mul_(2)
    sets[0][2].replay()
    torch.cuda.synchronize()
    for x, y in zip(sets[0][3], sets[0][0]()):
        assert torch.equal(x, y)


def test_residual_in_place_through_the_c_entry(gpu):
    import ctypes

    from distspmm_b200._lib import DspError, call, dsp_act_desc
    a = matrix("hub")
    p = d.SparsePattern(a)
    B, b, r, _ = inputs(a, 64, BF16, 4)
    B, b, r = B.cuda(), b.cuda(), r.cuda()
    want = d.spmm_act(p, B, None, b, r, "silu")
    io, v = r.clone(), p.values
    n = d.lib().dsp_spmm_act_workspace(p._h, 64)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    dd = dsp_act_desc(1, 2, 64, v.data_ptr(), B.data_ptr(), 64, b.data_ptr(), io.data_ptr(), 64, io.data_ptr(), 64, None, 0)
    with pytest.raises(DspError, match="workspace"):
        call("dsp_spmm_act", p._h, ctypes.byref(dd), ws.data_ptr(), n - 1, None)
    call("dsp_spmm_act", p._h, ctypes.byref(dd), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(io, want)


def test_empty_shapes(gpu):
    none = csr_of([], 5)
    p = d.SparsePattern(none, grad=True)
    assert d.spmm_act(p, torch.ones(5, 8, device="cuda")).shape == (0, 8)
    dB, dv, db = d.spmm_act_backward(p, torch.ones(0, 8, device="cuda"), torch.ones(5, 8, device="cuda"), None)
    torch.cuda.synchronize()
    assert (dB == 0).all() and dB.shape == (5, 8) and dv.numel() == 0 and (db == 0).all()
    a = matrix("rmat")
    p = d.SparsePattern(a, grad=True)
    assert d.spmm_act(p, torch.ones(a.num_cols, 0, device="cuda")).shape == (a.num_rows, 0)
    dB, dv, db = d.spmm_act_backward(p, torch.ones(a.num_rows, 0, device="cuda"), torch.ones(a.num_cols, 0, device="cuda"), None)
    assert (dv == 0).all() and dB.shape == (a.num_cols, 0) and db.numel() == 0
    no_cols = csr_of([[], []], 0)
    p = d.SparsePattern(no_cols, grad=True)
    out = d.spmm_act(p, torch.ones(0, 8, device="cuda"), bias=torch.ones(8, device="cuda"))
    assert (out == 1).all()


def test_agrees_with_the_plain_product(gpu):
    """fp32 without an epilogue is the plan's product (other summation order)."""
    from distspmm_b200.spmm import SpmmPlan
    a = d.gen_rmat(12, seed=8)
    B = torch.randn(a.num_cols, 128, device="cuda")
    x, y = d.spmm_act(d.SparsePattern(a), B), SpmmPlan(a, 0, 128)(B)
    size = product64(a, B.cpu().double(), torch.from_numpy(a.values).double(), None, None, None)[2]
    near(x, y.cpu().double(), 2 * (lens(a)[:, None] + 2) * U * size + 1e-37, "product")


def test_refusals(gpu):
    import ctypes

    from distspmm_b200._lib import dsp_act_desc, dsp_act_grad_desc
    a = matrix("rmat")
    p = d.SparsePattern(a)
    B = torch.ones(a.num_cols, 64, device="cuda")
    dy = torch.ones(a.num_rows, 64, device="cuda")
    with pytest.raises(ValueError, match="must be on cuda"):
        d.spmm_act(p, B.cpu())
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        d.spmm_act(p, B.double())
    with pytest.raises(ValueError, match="shape"):
        d.spmm_act(p, B[:-1])
    with pytest.raises(ValueError, match="values"):
        d.spmm_act(p, B, torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        d.spmm_act(p, B, bias=torch.ones(64, device="cuda", dtype=BF16))
    with pytest.raises(ValueError, match="residual"):
        d.spmm_act(p, B, residual=dy.to(BF16))
    with pytest.raises(ValueError, match="grad=True"):
        d.spmm_act_backward(p, dy, B, None)
    with pytest.raises(ValueError, match="grad=True"):
        d.spmm_act(p, B.clone().requires_grad_())
    with pytest.raises(ValueError, match="needs pre"):
        d.spmm_act_backward(p, dy, B, None, act="silu", need_B=False)
    ok = (0, 0, 64, p.values.data_ptr(), B.data_ptr(), 64, None, None, 0, dy.data_ptr(), 64, None, 0)
    for at, bad in ((0, 3), (0, -1), (1, 4), (2, -1), (3, None), (4, None), (5, 63), (9, None), (10, 63)):
        args = list(ok)
        args[at] = bad
        assert d.lib().dsp_spmm_act(p._h, ctypes.byref(dsp_act_desc(*args)), None, 0, None) == -1, at
    g = dsp_act_grad_desc(0, 0, 64, p.values.data_ptr(), B.data_ptr(), 64, None, 0, dy.data_ptr(), 64, B.data_ptr(), 64, None, None)
    assert d.lib().dsp_spmm_act_grad(p._h, ctypes.byref(g), None, 0, None) == -8
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("t", [F32, BF16])
def test_offsets_past_32_bits(gpu, t):
    """Rows of B and gradients behind 2^32 bytes (untouched rows in between are never read)."""
    n, cols = 256, (1 << 32) // 256 // (4 if t == F32 else 2) + 5000
    a = csr_of([[0, 7, cols - 1], [cols - 2], []], cols, [1.0, 2.0, 3.0, 4.0])
    p = d.SparsePattern(a)
    B = torch.empty(cols, n, dtype=t, device="cuda")
    used = {c: torch.randint(-4, 5, (n,)).float() for c in (0, 7, cols - 2, cols - 1)}
    for c, x in used.items():
        B[c] = x.to(t).cuda()
    out = d.spmm_act(p, B).cpu().float()
    assert torch.equal(out[0], used[0] + 2 * used[7] + 3 * used[cols - 1])
    assert torch.equal(out[1], 4 * used[cols - 2]) and (out[2] == 0).all()
    dv = d.spmm_act_backward(p, torch.ones(3, n, dtype=t, device="cuda"), B, None, need_B=False)[1].cpu()
    assert torch.equal(dv, torch.stack([used[0], used[7], used[cols - 1], used[cols - 2]]).sum(1))

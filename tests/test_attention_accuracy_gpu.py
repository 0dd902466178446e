"""What 16-bit attention keeps of fp32: weights and score gradients in two parts, gradients of any size in fp16, caps of any size,
infinite values (bounds: derived in attention_bounds.bounds)."""
import math

import pytest
import torch

import distspmm_b200 as d
from attention_bounds import bounds
from sparse_reference import attention64, csr_of, mask_of, matrix, positional
from test_attention_gpu import FORMS, inputs, lists, near, slopes_of

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def check(form, a, q, k, v, dout, cap=0.0, scale=None, slopes=None, names=("out", "lse", "dq", "dk", "dv"), depth=None, offset=0):
    t, dim = q.dtype, q.shape[2]
    p = d.SparsePattern(a, grad=True, attention=True, form=form)
    opt = dict(scale=scale, softcap=cap, slopes=None if slopes is None else slopes.cuda(), row_offset=offset)
    qc, kc, vc, dc = (x.cuda() for x in (q, k, v, dout))
    out, lse = d.sparse_attention_forward(p, qc, kc, vc, **opt)
    got = dict(out=out, lse=lse)
    got.update(zip(("dq", "dk", "dv"), d.sparse_attention_backward(p, dc, qc, kc, vc, out, lse, **opt)))
    w = [x.double().requires_grad_() for x in (q, k, v)]
    s = dim ** -0.5 if scale is None else scale
    mask = mask_of(a)
    o, l, pr = attention64(mask, *w, s, cap, slopes, offset)
    grads = torch.autograd.grad(o, w, dout.double())
    want = dict(out=o.detach(), lse=l.detach(), **dict(zip(("dq", "dk", "dv"), grads)))
    tol = bounds(mask, *(x.detach() for x in (*w, o, l, pr)), t, s, cap, slopes, offset, dout=dout.double(), grads=grads, depth=depth, once=form == "tiles")
    for name in names:
        near(got[name], want[name], tol[name], name)
    p.check_error()


MASKS = {"window": lambda: positional("window", 300, window=120, first=3), "docs": lambda: positional("docs", 260, cuts=[0, 90, 91, 250]),
         "rmat": lambda: d.gen_rmat(8, seed=3)}


def forms(dim):
    return FORMS if dim in (64, 128) else FORMS[1:]


@pytest.mark.parametrize("what", [("out", "lse"), ("dv",), ("dq",), ("dk",)])
@pytest.mark.parametrize("cap,scale", [(0.0, None), (8.0, None), (0.0, 1.0)])
@pytest.mark.parametrize("heads,kv,dim,t", [(2, 1, 64, BF16), (4, 2, 128, BF16), (2, 2, 64, F16), (2, 1, 128, F16), (2, 1, 32, BF16)])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("form", FORMS)
def test_weights_keep_16_bits(gpu, form, mask, heads, kv, dim, t, cap, scale, what):
    """A scale of 1 saturates the softmax: score gradients are small differences then."""
    if form not in forms(dim):
        pytest.skip("dims 64 and 128 have tiles")
    a = MASKS[mask]()
    check(form, a, *inputs(a.num_rows, a.num_cols, heads, kv, dim, t, 5), cap=cap, scale=scale, names=what)


def rows_of_sizes():
    """Rows of 1, 2 and 100 entries, one cut across chunks, rows without any."""
    rows = [[i] for i in range(20)] + [[i, i + 30] for i in range(20)] + [list(range(i, i + 100)) for i in range(20)] + [[]] * 3
    rows[25] = list(range(0, 1100))
    return csr_of(rows, 1100)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [BF16, F16])
def test_score_gradients_of_rows_with_few_entries(gpu, form, t):
    """A row of one entry has no score gradient: what is left is rounding of fp32, not of the type."""
    check(form, rows_of_sizes(), *inputs(63, 1100, 2, 1, 64, t, 6))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_one_entry_has_no_score_gradient(gpu, form, t):
    """dp of 18 bits, exact in fp32: dp - delta is 0, and what is left of dq has fp32's size, not that of dp in two 16-bit parts."""
    if t == F32 and form == "tiles":
        pytest.skip("16-bit operands have tiles")
    n = 70
    q, k, _, _ = inputs(n, n, 2, 2, 64, t, 12)
    v, dout = torch.zeros_like(q), torch.zeros_like(q)
    v[..., 0], dout[..., 0] = 256, 1
    v[..., 1], dout[..., 1] = (torch.arange(n)[:, None] % 7 + 1) / 512, 1
    v[..., 2], dout[..., 2] = 1, 1
    p = d.SparsePattern(csr_of([[i] for i in range(n)], n), grad=True, attention=True, form=form)
    qc, kc, vc, dc = (x.cuda() for x in (q, k, v, dout))
    out, lse = d.sparse_attention_forward(p, qc, kc, vc)
    assert torch.equal(out, vc)
    dq, dk, dv = d.sparse_attention_backward(p, dc, qc, kc, vc, out, lse)
    # p is 1 within the exponential's 2^-21, once or twice in a product
    zero, size = torch.zeros(q.shape, dtype=torch.float64), 258 * 64 ** -0.5 * 2.0 ** -20
    near(dq, zero, size * k.double().abs() + 1e-37, "dq")
    near(dk, zero, size * q.double().abs() + 1e-37, "dk")


@pytest.mark.parametrize("size", [100.0, 1000.0])
@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (3, 3, 128), (4, 1, 32)])
@pytest.mark.parametrize("form", FORMS)
def test_fp16_gradients_with_large_values(gpu, form, heads, kv, dim, size):
    """dout . v leaves fp16's range where neither dout nor v does, nor the results."""
    if form not in forms(dim):
        pytest.skip("dims 64 and 128 have tiles")
    a = rows_of_sizes()
    q, k, v, _ = inputs(63, 1100, heads, kv, dim, F16, 7)
    for values in (torch.full_like(v, size), (v.float() * size).to(F16)):
        dout = torch.ones_like(q)
        dout[5:] = 0.25
        check(form, a, (q.float() / 4).to(F16), k, values, dout)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("high", [1.0, 2.0 ** 11])
def test_fp16_gradients_of_different_sizes(gpu, form, high):
    """Rows whose gradient is small beside another's, documents apart and in one: each is right for itself."""
    a = positional("docs", 400, cuts=[0, 60, 190, 400])
    q, k, v, dout = inputs(400, 400, 2, 1, 64, F16, 8)
    dout = dout.float() * 2.0 ** -10
    dout[70] = high
    dout[300] = high * torch.randn(2, 64)
    check(form, a, q, k, v, dout.to(F16))
    dout[60:100] = 0  # the first rows that many keys see
    check(form, a, q, k, v, dout.to(F16))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [BF16, F16])
def test_long_row_of_equal_weights(gpu, form, t):
    """Weights of 2^-18 are subnormal in fp16; keys of nonzero mean add up their errors. Sums: by rows 512 entries of a chunk, then
    the chunks' in eight interleaved sums; by tiles 16 entries a step."""
    n = 300_000 if form == "rows" else 100_000
    a = csr_of([list(range(n)), [0, 1]], n)
    g = torch.Generator().manual_seed(3)
    q = (torch.randn((2, 1, 64), generator=g) / 16).to(t)
    k = (1 + torch.randn((n, 1, 64), generator=g) / 4).to(t)
    v = (1 + torch.randn((n, 1, 64), generator=g)).to(t)
    dout = (1 + torch.randn((2, 1, 64), generator=g)).to(t)
    check(form, a, q, k, v, dout, names=("out", "lse", "dq"), depth=540 + n // 4096 if form == "rows" else 64 + n // 16)


@pytest.mark.parametrize("cap", [1e3, 1e5, 1e8, 1e30])
@pytest.mark.parametrize("form,t,dim", [("tiles", BF16, 64), ("tiles", F16, 128), ("rows", BF16, 64), ("rows", F16, 32), ("rows", F32, 64)])
def test_large_caps(gpu, form, t, dim, cap):
    """A cap far above the scores leaves them as they are."""
    a = MASKS["window"]()
    check(form, a, *inputs(300, 300, 2, 1, dim, t, 9), cap=cap)


@pytest.mark.parametrize("cap", [1e3, 1e5, 1e8, 1e30])
@pytest.mark.parametrize("t,dim", [(BF16, 64), (F16, 128), (BF16, 96), (F32, 64)])
def test_large_caps_of_decode(gpu, t, dim, cap):
    q, k, v, _ = inputs(2, 500, 4, 2, dim, t, 9)
    ptr, idx = lists([333, 41], 500)
    out, lse = d.sparse_attention_decode(*(x.cuda() for x in (q, k, v, ptr, idx)), softcap=cap, return_lse=True)
    for r in range(2):
        at = idx[ptr[r]:ptr[r + 1]]
        mask = torch.ones(1, at.numel(), dtype=torch.bool)
        args = [x.double() for x in (q[r:r + 1], k[at], v[at])]
        o, l, p = attention64(mask, *args, dim ** -0.5, cap)
        tol = bounds(mask, *args, o, l, p, t, dim ** -0.5, cap)
        near(out[r:r + 1], o, tol["out"], "out")
        near(lse[r:r + 1], l, tol["lse"], "lse")


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t,dim", [(BF16, 64), (F16, 128), (BF16, 32), (F16, 96), (F32, 64)])
def test_infinite_values_that_are_listed(gpu, form, t, dim):
    """An infinity in a listed value is the row's result in that place (both signs: NaN), in short and in cut rows."""
    if form not in forms(dim):
        pytest.skip("dims 64 and 128 have tiles")
    a = rows_of_sizes()
    q, k, v, _ = inputs(63, 1100, 2, 1, dim, t, 10)
    v[5, :, 3] = math.inf  # row 5, row 25 and others
    v[31, :, 4] = -math.inf
    v[900, :, 5] = math.inf  # row 25 alone
    v[901, :, 5] = -math.inf
    want, lse, p = attention64(mask_of(a), q.double(), k.double(), v.double().nan_to_num(posinf=0, neginf=0), dim ** -0.5)
    tol = bounds(mask_of(a), q.double(), k.double(), v.double().nan_to_num(posinf=0, neginf=0), want, lse, p, t, dim ** -0.5)
    mask = mask_of(a)
    want[mask[:, 5], :, 3] = math.inf
    want[mask[:, 31], :, 4] = -math.inf
    got, got_lse = d.sparse_attention_forward(d.SparsePattern(a, attention=True, form=form), *(x.cuda() for x in (q, k, v)))
    got = got.cpu()
    assert torch.isnan(got[25, :, 5]).all()
    want[25, :, 5] = 0
    got[25, :, 5] = 0
    near(got, want, tol["out"], "out")
    near(got_lse, lse, tol["lse"], "lse")


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t,dim", [(BF16, 64), (F16, 128), (BF16, 32), (F16, 96), (F32, 64)])
def test_infinite_gradients(gpu, form, t, dim):
    """An infinity in dout is dv's in that place for every key of its row; row 25 is cut, and by columns key 5 is long."""
    if form not in forms(dim):
        pytest.skip("dims 64 and 128 have tiles")
    a = rows_of_sizes()
    q, k, v, dout = inputs(63, 1100, 2, 1, dim, t, 13)
    dout[25, :, 3] = math.inf
    dout[45, :, 4] = -math.inf
    mask = mask_of(a)
    w = [x.double().requires_grad_() for x in (q, k, v)]
    o, l, p = attention64(mask, *w, dim ** -0.5)
    fine = dout.double().nan_to_num(posinf=0, neginf=0)
    grads = torch.autograd.grad(o, w, fine)
    tol = bounds(mask, *(x.detach() for x in (*w, o, l, p)), t, dim ** -0.5, dout=fine, grads=grads)
    want = grads[2].clone()
    want[mask[25], :, 3] = math.inf
    want[mask[45], :, 4] = -math.inf
    pat = d.SparsePattern(a, grad=True, attention=True, form=form)
    qc, kc, vc, dc = (x.cuda() for x in (q, k, v, dout))
    dv = d.sparse_attention_backward(pat, dc, qc, kc, vc, *d.sparse_attention_forward(pat, qc, kc, vc))[2]
    near(dv, want, tol["dv"], "dv")


@pytest.mark.parametrize("t,dim", [(BF16, 64), (F16, 128), (BF16, 96), (F32, 64)])
def test_infinite_values_in_a_cache(gpu, t, dim):
    q, k, v, _ = inputs(3, 700, 8, 2, dim, t, 11)
    ptr, idx = lists([3, 600, 90], 700, 2)
    v[idx[1], :, 3] = math.inf
    v[idx[500], :, 4] = -math.inf
    fine = v.double().nan_to_num(posinf=0, neginf=0)
    got = d.sparse_attention_decode(*(x.cuda() for x in (q, k, v, ptr, idx)))
    for r in range(3):
        at = idx[ptr[r]:ptr[r + 1]]
        mask = torch.ones(1, at.numel(), dtype=torch.bool)
        args = q[r:r + 1].double(), k[at].double(), fine[at]
        o, l, p = attention64(mask, *args, dim ** -0.5)
        tol = bounds(mask, *args, o, l, p, t, dim ** -0.5)
        if (at == idx[1]).any():
            o[:, :, 3] = math.inf
        if (at == idx[500]).any():
            o[:, :, 4] = -math.inf
        near(got[r:r + 1], o, tol["out"], "out")


def test_slopes_changed_before_the_backward_pass(gpu):
    """The gradient of other slopes than the forward's is no gradient: autograd refuses, as for q, k and v."""
    a = positional("window", 40, window=9)
    p = d.SparsePattern(a, grad=True, attention=True)
    q, k, v, dout = (x.cuda() for x in inputs(40, 40, 2, 1, 64, BF16, 1))
    slopes = slopes_of(2).cuda()
    out = d.sparse_attention(p, q.requires_grad_(), k, v, slopes=slopes)
    out.backward(dout, retain_graph=True)
    slopes.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(dout)


@pytest.mark.parametrize("offset", [0, 100_000])
@pytest.mark.parametrize("form,t,dim", [("tiles", BF16, 64), ("tiles", F16, 128), ("rows", BF16, 64), ("rows", F16, 32), ("rows", F16, 8), ("rows", BF16, 96),
                                        ("rows", F32, 64), ("rows", F32, 8)])
def test_gradients_under_a_far_distance_bias(gpu, form, t, dim, offset):
    """lse is some -50000 there and rounded by 2^-9: the weights' sum is off by as much, and no share of delta may come into dq and dk."""
    a = positional("docs", 300, cuts=[0, 1, 2, 40, 41, 200, 290])
    q, k, v, dout = inputs(300, 300, 4, 2, dim, t, 14)
    check(form, a, q, k, v, dout, slopes=slopes_of(4), offset=offset)

"""Attention over a pattern's entries, its gradients and its single-token form, against 64-bit forms (tolerances: derived in
sparse_reference.attention_tolerances)."""
import math

import numpy as np
import pytest
import torch

import distspmm_b200 as d
from sparse_reference import attention64, attention_tolerances, csr_of, mask_of, matrix, positional

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(rows, keys, heads, kv, dim, t, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, dout = (torch.randn((rows, heads, dim), generator=g).to(t) for _ in range(2))
    k, v = (torch.randn((keys, kv, dim), generator=g).to(t) for _ in range(2))
    return q, k, v, dout


def slopes_of(heads):
    return torch.exp2(-torch.arange(1, heads + 1).float() * 8 / heads)


def near(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    same_inf = torch.isinf(want) & (got == want)
    bad = ~((got - want).abs() <= tol) & ~same_inf
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst " \
        f"{((got - want).abs() / tol)[bad].max():.2f} of the tolerance, first at {bad.nonzero()[0].tolist()}"


FORMS = ["tiles", "rows"]


def check(a, heads, kv, dim, t, cap=0.0, bias=False, offset=0, grad=True, seed=0, scale=None):
    """Both forms of the pattern, where the operands have two."""
    for form in FORMS if t != F32 and dim in (64, 128) else FORMS[1:]:
        check_form(form, a, heads, kv, dim, t, cap, bias, offset, grad, seed, scale)


def check_form(form, a, heads, kv, dim, t, cap, bias, offset, grad, seed, scale):
    p = d.SparsePattern(a, grad=grad, attention=True, form=form)
    q, k, v, dout = inputs(a.num_rows, a.num_cols, heads, kv, dim, t, seed)
    sl = slopes_of(heads) if bias else None
    opt = dict(scale=scale, softcap=cap, slopes=sl.cuda() if bias else None, row_offset=offset)
    qc, kc, vc, dc = (x.cuda() for x in (q, k, v, dout))
    out, lse = d.sparse_attention_forward(p, qc, kc, vc, **opt)
    w = [x.double().requires_grad_(grad) for x in (q, k, v)]
    mask, s = mask_of(a), 1 / math.sqrt(dim) if scale is None else scale
    wo, wl, wp = attention64(mask, *w, s, cap, sl, offset)
    grads = torch.autograd.grad(wo, w, dout.double()) if grad and a.nnz else [torch.zeros_like(x) for x in w]
    args = [x.detach() for x in (*w, wo, wl, wp)]
    tol = attention_tolerances(mask, *args, t, s, cap, sl, offset, dout=dout.double(), grads=grads)
    assert out.dtype == t
    near(out, args[3], tol["out"], "out")
    near(lse, args[4], tol["lse"], "lse")
    if grad:
        got = d.sparse_attention_backward(p, dc, qc, kc, vc, out, lse, **opt)
        for name, x, y in zip(("dq", "dk", "dv"), got, grads):
            assert x.dtype == t
            near(x, y, tol[name], name)
    p.check_error()  # no bounded wait gave up


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("kind", ["rmat", "hub", "empty", "row", "column", "one", "gap"])
def test_patterns(gpu, kind, t):
    check(matrix(kind), 4, 2, 64, t, cap=20.0 if kind == "rmat" else 0.0, bias=kind in ("hub", "gap"))


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("dim", [8, 16, 24, 32, 64, 80, 96, 128, 136, 256])
def test_dims(gpu, dim, t):
    check(d.gen_rmat(7, seed=4), 2, 1, dim, t, bias=True)


MASKS = {
    "window": lambda n: positional("window", n, window=70, first=5),
    "wide window": lambda n: positional("window", n, window=300),
    "prefix": lambda n: positional("prefix", n, prefix=min(n, 33)),
    "docs": lambda n: positional("docs", n, cuts=[0, n // 5, n // 5 + 1, n // 2, n - n // 7]),
    "full": lambda n: positional("full", n),
}


@pytest.mark.parametrize("heads,kv,dim,t", [(4, 4, 64, BF16), (8, 2, 128, BF16), (6, 2, 64, F16), (3, 3, 128, F16), (2, 2, 32, BF16), (2, 1, 64, F32)])
@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 127, 128, 129, 200, 385])
@pytest.mark.parametrize("mask", list(MASKS))
def test_positional_masks(gpu, mask, rows, heads, kv, dim, t):
    check(MASKS[mask](rows), heads, kv, dim, t, cap=15.0 if heads == 4 else 0.0, bias=heads == 8, seed=rows)


@pytest.mark.parametrize("t", [F32, BF16])
def test_rectangular_with_offset(gpu, t):
    """The last 130 rows of a causal window over 700 keys: a later piece of a prompt, or one rank's rows."""
    full = positional("window", 700, window=260, first=3)
    a = d.planner.partition(full, 570, 700)
    assert (a.num_rows, a.num_cols) == (130, 700)
    check(a, 4, 2, 64, t, bias=True, offset=570)
    # the same rows of the whole
    q, k, v, _ = inputs(700, 700, 4, 2, 64, t, 1)
    sl = slopes_of(4).cuda()
    whole = d.sparse_attention(d.SparsePattern(full, attention=True), q.cuda(), k.cuda(), v.cuda(), slopes=sl)
    part = d.sparse_attention(d.SparsePattern(a, attention=True), q[570:].cuda(), k.cuda(), v.cuda(), slopes=sl, row_offset=570)
    torch.testing.assert_close(part, whole[570:], rtol=0, atol=2e-2 if t == BF16 else 1e-5)


@pytest.mark.parametrize("t", [BF16, F32])
def test_large_scores(gpu, t):
    """Scores up to some +-80 (saturated softmax), and a scale of zero (plain means)."""
    check(positional("window", 150, window=64), 2, 2, 64, t, scale=2.0)
    check(positional("window", 150, window=64), 2, 2, 64, t, scale=2.0, cap=5.0)
    check(positional("window", 150, window=64), 2, 2, 64, t, scale=0.0)
    check(positional("window", 150, window=64), 2, 2, 64, t, scale=0.0, cap=5.0)
    check(positional("window", 150, window=64), 2, 2, 64, t, scale=0.125, cap=0.01)
    check(positional("window", 150, window=64), 2, 2, 64, t, scale=-0.125, cap=7.0, bias=True)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["window", "rmat"])
def test_unlisted_keys_never_count(gpu, kind, form, t):
    """NaN and infinities in k and v rows that a query row does not list, inside the same tiles as rows it does: its result and
    the other rows' gradients are those without them."""
    a = positional("window", 260, window=50, first=2) if kind == "window" else d.gen_rmat(8, seed=3)
    n = a.num_rows
    p = d.SparsePattern(a, grad=True, attention=True, form=form)
    q, k, v, dout = inputs(n, n, 4, 2, 64, t, 3)
    mask = mask_of(a)
    bad = torch.tensor([37, 100, 101, 200])
    hit = mask[:, bad].any(1)  # rows that list one of them
    assert hit.any() and not hit.all()
    kb, vb = k.clone(), v.clone()
    kb[bad[:2]] = float("nan")
    kb[bad[2:]] = float("inf")
    vb[bad[:3]] = float("inf")
    vb[bad[3:]] = float("nan")
    got, lse = (x.cpu() for x in d.sparse_attention(p, q.cuda(), kb.cuda(), vb.cuda(), return_lse=True))
    want, tol = want64(mask, q, k, v, dout)
    near(got[~hit], want["out"][~hit], tol["out"][~hit], "out")
    near(lse[~hit], want["lse"][~hit], tol["lse"][~hit], "lse")
    assert not torch.isfinite(got[hit]).all(-1).any()
    # gradients: the rows that see a bad key, and the keys that such rows see, are spoiled
    spoiled = mask[hit].any(0)
    dq, dk, dv = (x.cpu() for x in backward(p, dout, q, kb, vb))
    clean = ~spoiled & ~torch.isin(torch.arange(n), bad)
    assert clean.any()
    near(dq[~hit], want["dq"][~hit], tol["dq"][~hit], "dq")
    near(dk[clean], want["dk"][clean], tol["dk"][clean], "dk")
    near(dv[clean], want["dv"][clean], tol["dv"][clean], "dv")


def want64(mask, q, k, v, dout):
    """Results and tolerances for these inputs."""
    w = [x.double().requires_grad_() for x in (q, k, v)]
    scale = q.shape[2] ** -0.5
    o, l, p = attention64(mask, *w, scale)
    grads = torch.autograd.grad(o, w, dout.double())
    args = [x.detach() for x in (*w, o, l, p)]
    tol = attention_tolerances(mask, *args, q.dtype, scale, dout=dout.double(), grads=grads)
    return dict(out=args[3], lse=args[4], dq=grads[0], dk=grads[1], dv=grads[2]), tol


def backward(p, dout, q, k, v):
    q, k, v, dout = (x.cuda() for x in (q, k, v, dout))
    out, lse = d.sparse_attention_forward(p, q, k, v)
    return d.sparse_attention_backward(p, dout, q, k, v, out, lse)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("t", [F32, BF16])
def test_bad_query_rows_stay_alone(gpu, t, form):
    """A NaN query row spoils itself and the gradients of the keys it lists, nothing else."""
    a = positional("window", 260, window=50)
    p = d.SparsePattern(a, grad=True, attention=True, form=form)
    q, k, v, dout = inputs(260, 260, 2, 2, 64, t, 4)
    qb, db = q.clone(), dout.clone()
    qb[130] = float("nan")
    db[131] = float("inf")
    dq, dk, dv = (x.cpu() for x in backward(p, db, qb, k, v))
    mask = mask_of(a)
    rows = torch.ones(260, dtype=torch.bool)
    rows[130:132] = False
    keys = ~mask[130:132].any(0)
    want, tol = want64(mask, q, k, v, dout)
    near(dq[rows], want["dq"][rows], tol["dq"][rows], "dq")
    near(dk[keys], want["dk"][keys], tol["dk"][keys], "dk")
    near(dv[keys], want["dv"][keys], tol["dv"][keys], "dv")


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("size", [1.0, 2.0 ** -10, 2.0 ** 9])
def test_fp16_gradients_of_any_size(gpu, size, form):
    """Small and large gradients in fp16: what the type cannot hold in between is scaled, results keep the tolerance."""
    a = positional("window", 400, window=220)
    n = a.num_rows
    p = d.SparsePattern(a, grad=True, attention=True, form=form)
    assert (p.info()["tiles"] > 0) == (form == "tiles")
    q, k, v, dout = inputs(n, n, 2, 1, 64, F16, 11)
    dout = (dout.float() * size).to(F16)
    dq, dk, dv = (x.cpu() for x in backward(p, dout, q, k, v))
    want, tol = want64(mask_of(a), q, k, v, dout)
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        near(x, want[name], tol[name], name)


def test_split_rows(gpu):
    """One row tile over many keys, few heads: its list is cut into pieces that are joined; NaN in unlisted keys stays out."""
    rows, keys = 100, 4000
    a = csr_of([[j for j in range(keys) if j % 7 or j < i * 30] for i in range(rows)], keys)
    p = d.SparsePattern(a, attention=True)
    for t, dim in ((BF16, 128), (F16, 64)):
        q, k, v, _ = inputs(rows, keys, 2, 1, dim, t, 12)
        mask = mask_of(a)
        w = [x.double() for x in (q, k, v)]
        o, l, pr = attention64(mask, *w, dim ** -0.5)
        tol = attention_tolerances(mask, *w, o, l, pr, t, dim ** -0.5)
        out, lse = d.sparse_attention_forward(p, q.cuda(), k.cuda(), v.cuda())
        near(out, o, tol["out"], "out")
        near(lse, l, tol["lse"], "lse")
        v[3500] = float("nan")  # 3500 is a multiple of 7: row 0 does not list it
        out = d.sparse_attention(p, q.cuda(), k.cuda(), v.cuda()).cpu()
        free = ~mask[:, 3500]
        assert free.all()
        near(out, o, tol["out"], "out")


def test_forms_are_chosen_by_fill(gpu):
    assert d.SparsePattern(positional("window", 600, window=300), attention=True).info()["tiles"] > 0
    assert d.SparsePattern(d.gen_uniform(4096, 8, seed=1), attention=True).info()["tiles"] == 0
    assert d.SparsePattern(positional("window", 600, window=300)).info()["tiles"] == 0  # not asked for
    d.SparsePattern(matrix("one")).check_error()


def test_autograd_and_differences(gpu):
    a = d.gen_rmat(7, seed=9)
    p = d.SparsePattern(a, grad=True, attention=True)
    n = a.num_rows
    q, k, v, dout = inputs(n, n, 4, 2, 32, F32, 5)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    sl = slopes_of(4).cuda()
    out = d.sparse_attention(p, *leaves, softcap=3.0, slopes=sl)
    got = torch.autograd.grad(out, leaves, dout.cuda())
    o, lse = d.sparse_attention_forward(p, *[x.detach() for x in leaves], softcap=3.0, slopes=sl)
    direct = d.sparse_attention_backward(p, dout.cuda(), *[x.detach() for x in leaves], o, lse, softcap=3.0, slopes=sl)
    for x, y in zip(got, direct):
        assert torch.equal(x, y)
    # central differences in 64 bits: step 1e-4, error of the order 1e-8 of the third derivatives; fp32 gradients have 2e-5 of
    # the sum of magnitudes (sums of up to 128 terms of a few 2^-24 each, through two products)
    g = torch.Generator().manual_seed(1)
    base, mask = [x.double() for x in (q, k, v)], mask_of(a)
    loss = lambda z: float((attention64(mask, *z, 32 ** -0.5, 3.0, sl.cpu())[0] * dout.double()).sum())  # noqa: E731
    for i in range(3):
        u = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-4 * u, base[i] - 1e-4 * u
        terms = got[i].cpu().double() * u
        assert abs((loss(up) - loss(down)) / 2e-4 - float(terms.sum())) <= 2e-5 * float(terms.abs().sum())


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["window", "rmat"])
def test_strides(gpu, kind, form, t):
    """q, k, v as parts of one fused projection, head-major storage, odd offsets, expanded heads."""
    a = positional("window", 200, window=90) if kind == "window" else d.gen_rmat(8, seed=2)
    n = a.num_rows
    p = d.SparsePattern(a, grad=True, attention=True, form=form)
    q, k, v, dout = (x.cuda() for x in inputs(n, n, 4, 4, 64, t, 6))
    want = d.sparse_attention_forward(p, q, k, v)
    wg = d.sparse_attention_backward(p, dout, q, k, v, *want)
    fused = torch.full((n, 3, 4, 64), float("nan"), dtype=t, device="cuda")
    for i, x in enumerate((q, k, v)):
        fused[:, i] = x
    heads_first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731

    def odd(x):
        w = torch.full((n, 4, 67), float("nan"), dtype=t, device="cuda")
        w[:, :, 1:65] = x
        return w[:, :, 1:65]

    for parts in ([fused[:, i] for i in range(3)], [heads_first(x) for x in (q, k, v)], [odd(x) for x in (q, k, v)]):
        got = d.sparse_attention_forward(p, *parts)
        gg = d.sparse_attention_backward(p, heads_first(dout), *parts, *got)
        for x, y in zip(got + gg, want + wg):
            assert torch.equal(x, y)
    one = k[:, :1].contiguous()
    got = d.sparse_attention(p, q, one.expand(n, 4, 64), v[:, :1].expand(n, 4, 64))
    assert torch.equal(got, d.sparse_attention(p, q, one.expand(n, 4, 64).contiguous(), v[:, :1].repeat(1, 4, 1)))


def test_broadcast_keys_get_summed_gradients(gpu):
    a = positional("window", 150, window=40)
    p = d.SparsePattern(a, grad=True, attention=True)
    q, k, v, dout = (x.cuda() for x in inputs(150, 150, 4, 1, 64, F32, 7))
    k1, v1 = k.clone().requires_grad_(), v.clone().requires_grad_()
    d.sparse_attention(p, q, k1.expand(150, 4, 64), v1.expand(150, 4, 64)).backward(dout)
    k2, v2 = k.clone().requires_grad_(), v.clone().requires_grad_()
    d.sparse_attention(p, q, k2, v2).backward(dout)
    torch.testing.assert_close(k1.grad, k2.grad, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(v1.grad, v2.grad, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["window", "rmat"])
def test_same_bits_graphs_and_streams(gpu, kind, form):
    a = positional("window", 600, window=200, first=4) if kind == "window" else d.gen_rmat(10, seed=2)
    n = a.num_rows
    p = d.SparsePattern(a, grad=True, attention=True, form=form)
    sets = []
    for s in range(2):
        q, k, v, dout = (x.cuda() for x in inputs(n, n, 4, 2, 64, BF16, s))

        def step(q=q, k=k, v=v, dout=dout):
            out, lse = d.sparse_attention_forward(p, q, k, v)
            return (out, lse) + d.sparse_attention_backward(p, dout, q, k, v, out, lse)

        want = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        sets.append((step, want, graph, got, q))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                x[2].replay()
        eager = sets[0][0]()
        torch.cuda.synchronize()
        for _, want, _, got, _ in sets:
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(eager, sets[0][1]))
    sets[0][4].mul_(0.5)
    sets[0][2].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(sets[0][3], sets[0][0]()))


def test_empty_shapes(gpu):
    none = csr_of([], 5)
    p = d.SparsePattern(none, grad=True, attention=True)
    q, k, v, dout = (x.cuda() for x in inputs(0, 5, 2, 2, 64, BF16))
    out, lse = d.sparse_attention_forward(p, q, k, v)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    dq, dk, dv = d.sparse_attention_backward(p, dout, q, k, v, out, lse)
    assert dq.shape == (0, 2, 64) and (dk == 0).all() and (dv == 0).all()
    no_keys = csr_of([[], [], []], 0)
    p = d.SparsePattern(no_keys, grad=True, attention=True)
    q, k, v, dout = (x.cuda() for x in inputs(3, 0, 2, 2, 64, BF16))
    out, lse = d.sparse_attention_forward(p, q, k, v)
    assert (out == 0).all() and torch.isneginf(lse).all()
    dq, dk, dv = d.sparse_attention_backward(p, dout, q, k, v, out, lse)
    assert (dq == 0).all() and dk.shape == (0, 2, 64)


# ---------------------------------------------------------------------------------------------- single tokens


def lists(lens, slots, seed=0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.cat([torch.randperm(slots, generator=g)[:n] for n in lens] + [torch.zeros(0, dtype=torch.int64)])
    ptr = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int64)
    return ptr, idx


def decode64(q, k, v, ptr, idx, cap, slopes):
    """By rows, with the tolerance of each."""
    out, lse, to, tl = [], [], [], []
    t = q.dtype
    for r in range(q.shape[0]):
        at = idx[ptr[r]:ptr[r + 1]]
        n = at.numel()
        mask = torch.ones(1, n, dtype=torch.bool)
        dist = torch.arange(n - 1, -1, -1).double()[None]
        args = [x.double() for x in (q[r:r + 1], k[at], v[at])]
        o, l, p = attention64(mask, *args, q.shape[2] ** -0.5, cap, slopes, dist=dist)
        tol = attention_tolerances(mask, *args, o, l, p, t, q.shape[2] ** -0.5, cap, slopes, dist=dist)
        out.append(o), lse.append(l), to.append(tol["out"]), tl.append(tol["lse"])
    return torch.cat(out), torch.cat(lse), torch.cat(to), torch.cat(tl)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (4, 4, 128), (8, 1, 128), (8, 2, 64), (16, 1, 128), (24, 1, 64), (6, 2, 96), (5, 5, 256), (12, 4, 8)])
@pytest.mark.parametrize("lens", [[1], [0], [5, 0, 1, 64, 63, 65], [700], [3000, 1, 129, 0, 2000]])
def test_decode(gpu, lens, heads, kv, dim, t):
    if max(lens) > 700 and t == F16:
        pytest.skip("covered by the other types")
    slots = max(lens) + 40
    q, k, v, _ = inputs(len(lens), slots, heads, kv, dim, t, sum(lens))
    ptr, idx = lists(lens, slots)
    cap, sl = (10.0, slopes_of(heads)) if heads % 8 == 0 else (0.0, None)
    out, lse = d.sparse_attention_decode(*(x.cuda() for x in (q, k, v, ptr, idx)), softcap=cap,
                                         slopes=None if sl is None else sl.cuda(), return_lse=True)
    wo, wl, to, tl = decode64(q, k, v, ptr, idx, cap, sl)
    near(out, wo, to, "out")
    near(lse, wl, tl, "lse")


@pytest.mark.parametrize("t", [F32, BF16])
def test_decode_unlisted_slots_and_bad_entries(gpu, t):
    slots = 300
    q, k, v, _ = inputs(4, slots, 8, 2, 64, t, 2)
    ptr, idx = lists([100, 50, 90, 33], slots, 4)
    want = d.sparse_attention_decode(*(x.cuda() for x in (q, k, v, ptr, idx))).cpu()
    used = torch.zeros(slots, dtype=torch.bool)
    used[idx] = True
    kb, vb = k.clone(), v.clone()
    kb[~used] = float("nan")
    vb[~used] = float("inf")
    assert (~used).any()
    assert torch.equal(d.sparse_attention_decode(*(x.cuda() for x in (q, kb, vb, ptr, idx))).cpu(), want)
    for bad in (-1, slots, 1 << 40, -(1 << 62)):
        i2 = idx.clone()
        i2[120] = bad  # in row 1
        got, lse = (x.cpu() for x in d.sparse_attention_decode(*(x.cuda() for x in (q, k, v, ptr, i2)), return_lse=True))
        assert torch.isnan(got[1]).all() and torch.isnan(lse[1]).all()
        rest = torch.tensor([0, 2, 3])
        assert torch.equal(got[rest], want[rest])
    # a NaN in a listed slot is the row's own
    vb = v.clone()
    vb[idx[10]] = float("nan")
    got = d.sparse_attention_decode(*(x.cuda() for x in (q, k, vb, ptr, idx))).cpu()
    hit = torch.tensor([bool((idx[ptr[r]:ptr[r + 1]] == idx[10]).any()) for r in range(4)])
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


def test_decode_malformed_lists_stay_in_bounds(gpu):
    """Row pointers that fall, exceed the list or are negative: results are unspecified, nothing faults (every index is bounded
    in the kernel), and well-formed calls after it are right."""
    q, k, v, _ = (x.cuda() for x in inputs(3, 64, 4, 2, 64, BF16))
    idx = torch.arange(64, device="cuda")
    for p in ([0, 40, 20, 64], [0, 1 << 40, 5, 64], [-5, 10, 20, 1 << 50], [64, 0, 64, 0], [0, 0, 0, 0], [5, 10, 20, 30]):
        d.sparse_attention_decode(q, k, v, torch.tensor(p, device="cuda"), idx)
        torch.cuda.synchronize()
    got = d.sparse_attention_decode(q, k, v, torch.tensor([5, 10, 20, 30], device="cuda"), idx)
    want = d.sparse_attention_decode(q, k, v, torch.tensor([0, 5, 15, 25], device="cuda"), idx[5:30])
    torch.testing.assert_close(got, want, rtol=2 ** -7, atol=2 ** -7)


def test_decode_repeated_entry_counts_twice(gpu):
    q, k, v, _ = inputs(1, 8, 2, 1, 64, F32, 1)
    idx = torch.tensor([3, 3, 5])
    got = d.sparse_attention_decode(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, 3], device="cuda"), idx.cuda())
    wo, _, to, _ = decode64(q, k, v, torch.tensor([0, 3]), idx, 0.0, None)
    near(got, wo, to, "out")


def test_decode_follows_its_lists_in_a_graph(gpu):
    q, k, v, _ = (x.cuda() for x in inputs(2, 600, 8, 2, 128, BF16, 3))
    ptr, idx = (x.cuda() for x in lists([300, 200], 600, 1))
    d.sparse_attention_decode(q, k, v, ptr, idx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = d.sparse_attention_decode(q, k, v, ptr, idx)
    for lens, seed in (([300, 200], 5), ([100, 250], 6), ([0, 500], 7)):
        p2, i2 = lists(lens, 600, seed)
        ptr.copy_(p2)
        idx[:i2.numel()] = i2.cuda()
        graph.replay()
        torch.cuda.synchronize()
        wo, _, to, _ = decode64(q.cpu(), k.cpu(), v.cpu(), p2, i2, 0.0, None)
        near(got, wo, to, "out")


def test_decode_matches_prefill(gpu):
    """The last row of a causal prompt is the single-token form over the same keys."""
    n = 333
    a = positional("window", n, window=n)
    q, k, v, _ = (x.cuda() for x in inputs(n, n, 8, 2, 64, BF16, 8))
    sl = slopes_of(8).cuda()
    full = d.sparse_attention(d.SparsePattern(a, attention=True), q, k, v, softcap=9.0, slopes=sl)
    one = d.sparse_attention_decode(q[-1:].contiguous(), k, v, torch.tensor([0, n], device="cuda"), torch.arange(n, device="cuda"),
                                    softcap=9.0, slopes=sl)
    # each is within its own weights' rounding (2^-8 of a mean of |v|, 0.8) and the result's
    torch.testing.assert_close(one[0], full[-1], rtol=2 ** -7, atol=2 ** -7)


def test_refusals(gpu):
    a = positional("window", 64, window=9)
    q, k, v, dout = (x.cuda() for x in inputs(64, 64, 4, 2, 64, BF16))
    p = d.SparsePattern(a, attention=True)
    plain = d.SparsePattern(a)
    with pytest.raises(ValueError, match="attention=True"):
        d.sparse_attention(plain, q, k, v)
    out, lse = d.sparse_attention_forward(p, q, k, v)
    with pytest.raises(ValueError, match="grad=True"):
        d.sparse_attention_backward(p, dout, q, k, v, out, lse)
    with pytest.raises(ValueError, match="grad=True"):
        d.sparse_attention(p, q.clone().requires_grad_(), k, v)
    with pytest.raises(ValueError, match="query heads"):
        d.sparse_attention(p, q[:, :3], k, v)
    with pytest.raises(ValueError, match="shape"):
        d.sparse_attention(p, q[:-1], k, v)
    with pytest.raises(ValueError, match="must be torch.bfloat16"):
        d.sparse_attention(p, q, k.float(), v)
    with pytest.raises(ValueError, match="softcap"):
        d.sparse_attention(p, q, k, v, softcap=-1.0)
    with pytest.raises(ValueError, match="constants"):
        d.sparse_attention(p, q, k, v, slopes=torch.ones(4, device="cuda", requires_grad=True))
    from distspmm_b200._lib import DspError
    with pytest.raises(DspError, match="DSP_ERR_UNSUPPORTED"):
        d.sparse_attention(p, q[:, :, :20], k[:, :, :20], v[:, :, :20])
    with pytest.raises(DspError, match="DSP_ERR_UNSUPPORTED"):
        big = torch.zeros(64, 1, 264, dtype=BF16, device="cuda")
        d.sparse_attention(p, big, big, big)
    ptr, idx = torch.tensor([0, 5], device="cuda"), torch.arange(5, device="cuda")
    with pytest.raises(ValueError, match="indptr"):
        d.sparse_attention_decode(q, k, v, ptr, idx)
    with pytest.raises(ValueError, match="int64"):
        d.sparse_attention_decode(q[:1], k, v, ptr.int(), idx)


def test_a_graph_transformer_layer(gpu):
    """The operators together: attention over a graph's edges, then the mean over the neighbours with bias, activation and the
    residual around it; gradients of every input agree with the 64-bit composition by differences of autograd."""
    a = d.gen_rmat(8, seed=6)
    n, heads, dim = a.num_rows, 4, 16
    p = d.SparsePattern(a, grad=True, attention=True)
    q, k, v, _ = inputs(n, n, heads, heads, dim, F32, 2)
    g = torch.Generator().manual_seed(3)
    bias, dy = torch.randn(64, generator=g), torch.randn((n, 64), generator=g)
    values = torch.from_numpy(a.values).clone()

    def layer(attend, mix, q, k, v, values, bias):
        h = attend(q, k, v).reshape(n, 64)
        return mix(h, values, bias, q.reshape(n, 64))

    from sparse_reference import product64
    leaves = [x.cuda().requires_grad_() for x in (q, k, v, values, bias)]
    y = layer(lambda *x: d.sparse_attention(p, *x), lambda h, w, b, r: d.spmm_act(p, h, w, b, r, "silu"), *leaves)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    w = [x.double().requires_grad_() for x in (q, k, v, values, bias)]
    mask = mask_of(a)
    y64 = layer(lambda *x: attention64(mask, *x, dim ** -0.5)[0], lambda h, x, b, r: product64(a, h, x, b, r, "silu")[0], *w)
    want = torch.autograd.grad(y64, w, dy.double())
    # fp32 through two sparse sums (rows of up to 110 entries) and their transposes: some 500 roundings of 2^-24 of terms that
    # are larger than the result by cancellation; held to 1e-4 of each result's largest value
    for x, z in zip((y,) + got, (y64.detach(),) + want):
        assert (x.detach().cpu().double() - z).abs().max() <= 1e-4 * z.abs().max()


@pytest.mark.parametrize("t", [F32, BF16])
def test_decode_offsets_past_32_bits(gpu, t):
    """A cache whose last rows lie behind 2^32 bytes: the same tokens at its front and at its end give the same result."""
    dim, kv = 128, 4
    keys = (1 << 32) // (dim * kv * (4 if t == F32 else 2)) + 3000
    k, v = (torch.empty(keys, kv, dim, dtype=t, device="cuda") for _ in range(2))
    q, ks, vs, _ = (x.cuda() for x in inputs(2, 200, 8, kv, dim, t, 3))
    for cache, x in ((k, ks), (v, vs)):
        cache[:200] = x
        cache[-200:] = x
    idx = torch.cat([torch.arange(200), torch.arange(keys - 200, keys)]).cuda()
    both = torch.cat([q[:1], q[:1]])
    out = d.sparse_attention_decode(both, k, v, torch.tensor([0, 200, 400], device="cuda"), idx)
    want = d.sparse_attention_decode(q[:1], ks, vs, torch.tensor([0, 200], device="cuda"), torch.arange(200, device="cuda"))
    # chunk borders fall elsewhere: sums in another order
    torch.testing.assert_close(out, torch.cat([want, want]), rtol=0, atol=2 ** -8 if t == BF16 else 1e-6)


def test_tiles_of_rows_past_32_bits(gpu):
    """q, k and v as strided rows that reach past 2^32 bytes, by tiles and by rows."""
    n, stride = 300, (1 << 32) // 2 // 256
    base = torch.empty(n * stride + 8192, dtype=BF16, device="cuda")
    a = positional("window", n, window=90)
    q, k, v, dout = (x.cuda() for x in inputs(n, n, 2, 2, 64, BF16, 5))
    far = []
    for i, x in enumerate((q, k, v)):
        w = base.as_strided((n, 2, 64), (stride, 64, 1), i * 1024)
        w.copy_(x)
        far.append(w)
    for form in FORMS:
        p = d.SparsePattern(a, grad=True, attention=True, form=form)
        near_out = d.sparse_attention_forward(p, q, k, v)
        far_out = d.sparse_attention_forward(p, *far)
        for x, y in zip(near_out + d.sparse_attention_backward(p, dout, q, k, v, *near_out),
                        far_out + d.sparse_attention_backward(p, dout, *far, *far_out)):
            assert torch.equal(x, y)

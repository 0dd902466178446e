"""Plain 64-bit forms of the sparse-layer operators and matrices for their tests (CPU)."""
import numpy as np
import torch

import distspmm_b200 as d

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}  # half a step at the bottom (fp16: subnormals)
U = 2.0 ** -24


def csr_of(dense_rows, cols, values=None):
    """Csr from a list of column lists."""
    indptr = np.zeros(len(dense_rows) + 1, np.int64)
    indptr[1:] = np.cumsum([len(r) for r in dense_rows])
    indices = np.array([c for r in dense_rows for c in r], np.int64)
    if values is None:
        values = np.random.default_rng(indices.size).uniform(-1, 1, indices.size)
    return d.Csr(indptr, indices, np.asarray(values, np.float32), len(dense_rows), cols)


def matrix(kind):
    r = np.random.default_rng(7)
    if kind == "rmat":
        return d.gen_rmat(9, seed=3)
    if kind == "hub":  # one long row, one long column, empty rows and columns around them
        rows = [[] for _ in range(300)]
        rows[137] = list(range(5, 2600))
        for i in range(40, 300, 2):
            rows[i] = sorted(set(rows[i]) | {17})
        return csr_of(rows, 2700)
    if kind == "empty":
        return csr_of([[] for _ in range(70)], 33)
    if kind == "row":  # one row over everything
        return csr_of([list(range(1000))], 1000)
    if kind == "column":
        return csr_of([[0] for _ in range(500)], 1)
    if kind == "one":
        return csr_of([[0]], 1)
    if kind == "repeated":  # unordered columns, some twice
        return csr_of([list(r.integers(0, 40, r.integers(0, 30))) for _ in range(90)], 40)
    if kind == "gap":  # long runs of empty rows between short ones
        return csr_of([list(r.choice(64, 5, replace=False)) if i % 211 == 3 else [] for i in range(4000)], 64)
    raise ValueError(kind)


def row_ids(a):
    return torch.from_numpy(np.repeat(np.arange(a.num_rows), np.diff(a.indptr)))


def act64(z, act):
    return {None: lambda x: x, "none": lambda x: x, "relu": torch.relu, "silu": lambda x: x / (1 + torch.exp(-x)),
            "gelu": lambda x: 0.5 * x * torch.special.erfc(-x * 0.5 ** 0.5)}[act](z)


def product64(a, B, values, bias, residual, act):
    """(out, z, size): size = |A|.|B| + |bias|, what rounding errors of z are relative to."""
    rows, cols = row_ids(a), torch.from_numpy(a.indices)
    n = B.shape[1]
    z = torch.zeros((a.num_rows, n), dtype=torch.float64).index_add(0, rows, values[:, None] * B[cols])
    size = torch.zeros((a.num_rows, n), dtype=torch.float64).index_add(0, rows, values.detach().abs()[:, None] * B.detach().abs()[cols])
    if bias is not None:
        z = z + bias
        size = size + bias.detach().abs()
    y = act64(z, act)
    return (y if residual is None else y + residual), z, size


def mask_of(a):
    m = torch.zeros((a.num_rows, a.num_cols), dtype=torch.bool)
    m[row_ids(a), torch.from_numpy(a.indices)] = True
    return m


def positional(kind, rows, **kw):
    """Causal masks as a Csr: window (and first tokens), prefix, documents (and padding rows)."""
    i, j = np.arange(rows)[:, None], np.arange(rows)[None, :]
    if kind == "window":
        m = (j <= i) & ((i - j < kw["window"]) | (j < kw.get("first", 0)))
    elif kind == "prefix":
        m = (j <= i) | (j < kw["prefix"])
    elif kind == "full":
        m = i + j >= 0
    else:
        doc = np.full(rows, -1)
        for n, (b, e) in enumerate(zip(kw["cuts"], kw["cuts"][1:])):
            doc[b:e] = n
        m = (j <= i) & (doc[:, None] == doc[None, :]) & (doc[:, None] >= 0)
    return csr_of([list(np.flatnonzero(r)) for r in m], rows)


def attention64(mask, q, k, v, scale, cap=0.0, slopes=None, row_offset=0, dist=None):
    """(out, lse, p) in 64 bits: q [rows, heads, dim], k, v [keys, kv_heads, dim], mask [rows, keys]."""
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    u = torch.einsum("ihd,jhd->hij", q, k) * scale
    if cap:
        u = cap * torch.tanh(u / cap)
    if slopes is not None:
        if dist is None:
            dist = (torch.arange(q.shape[0])[:, None] + row_offset - torch.arange(k.shape[0])[None, :]).abs().double()
        u = u - slopes.double()[:, None, None] * dist
    u = u.masked_fill(~mask, -float("inf"))
    top = u.amax(-1, keepdim=True) if u.shape[-1] else torch.zeros(u.shape[:2] + (1,), dtype=u.dtype)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top).detach()
    e = torch.exp(u - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)).squeeze(-1).t()
    return torch.einsum("hij,jhd->ihd", p, v), lse, p


def attention_tolerances(mask, q, k, v, out, lse, p, t, scale, cap=0.0, slopes=None, row_offset=0, dist=None, dout=None, grads=None):
    """Bounds on the errors of out, lse (and dq, dk, dv), from the arithmetic, for 64-bit copies of the inputs.

    A score is a sum of dim products in fp32 (dim + 2 roundings of its magnitudes), the cap adds 2^-21 of the cap, the bias a
    rounding or two; a weight exp(u - max) is off by twice the scores' error and the exponential's own 2^-21 and argument
    rounding; sums of n terms add n + 10 roundings. Weights and score gradients of 16-bit types are rounded to the type before
    they enter a product (half a step each). Results are rounded once."""
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    m = mask.double()
    size = torch.einsum("ihd,jhd->hij", q.abs(), kk.abs()) * abs(scale)
    e_u = (dim + 4) * U * size + (cap * 2.0 ** -21 if cap else 0)
    if slopes is not None:
        if dist is None:
            dist = (torch.arange(q.shape[0])[:, None] + row_offset - torch.arange(k.shape[0])[None, :]).abs().double()
        e_u = e_u + 4 * U * slopes.double().abs()[:, None, None] * dist
    e_u = e_u + 6 * U * size.clamp(min=1)
    worst = (e_u * m).amax(-1, keepdim=True) if e_u.shape[-1] else e_u.sum(-1, keepdim=True)  # [h, i, 1]
    n = m.sum(-1).clamp(min=1)[None, :, None]
    rounded = 0.0 if t == torch.float32 else HALF_STEP[t]
    e_p = 2 * worst + (n + 10) * U + 2.0 ** -20 + 8 * U * lse.t().nan_to_num(neginf=0).abs()[:, :, None]  # relative
    h = HALF_STEP[t]
    e_out = torch.einsum("hij,jhd->ihd", p * (e_p + rounded), vv.abs())
    tol = {"out": e_out + h * (out.abs() + e_out) + TINY[t],
           "lse": (worst + (n + 10) * U + 2.0 ** -20).squeeze(-1).t() + 4 * U * lse.nan_to_num(neginf=0).abs()}
    if dout is None:
        return tol
    o_t = tol["out"]
    dp = torch.einsum("ihd,jhd->hij", dout, vv)
    delta = (dout * out).sum(-1).t()[:, :, None]
    e_delta = ((dout.abs() * o_t).sum(-1) + (dim + 2) * U * (dout * out).abs().sum(-1)).t()[:, :, None]
    e_dp = (dim + 2) * U * torch.einsum("ihd,jhd->hij", dout.abs(), vv.abs())
    slope = abs(scale)
    e_th = (4 * e_u / cap + 2.0 ** -19) if cap else 0.0
    ds = p * (dp - delta).abs() * slope
    e_ds = ds * (e_p + e_th + rounded + 8 * U) + p * slope * (e_dp + e_delta) * (1 + e_p + rounded)
    keys = k.shape[0]
    rows_n = m.sum(0).clamp(min=1)[None, None, :] * group

    def fold(x):
        return x.view(keys, k.shape[1], group, dim).sum(2)

    e_dq = torch.einsum("hij,jhd->ihd", e_ds + ds * n * U, kk.abs())
    e_dk = fold(torch.einsum("hij,ihd->jhd", e_ds + ds * rows_n * U, q.abs()))
    e_dv = fold(torch.einsum("hij,ihd->jhd", p * (e_p + rounded + rows_n * U), dout.abs()))
    for name, e, g in zip(("dq", "dk", "dv"), (e_dq, e_dk, e_dv), grads):
        tol[name] = e + h * (g.abs() + e) + TINY[t]
    return tol

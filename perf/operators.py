"""Cases and plain forms of the sparse-layer operators.

Three operators on a sparse matrix A in CSR form:

product    Y = act(A.B + bias) + residual; a training step also returns the gradients of B, A's values, the bias and
           the residual.
attention  O_i = sum over the entries (i, j) of A of softmax_j(u_ij) V_j with
           u_ij = cap tanh(scale q_i.k_j / cap) - slope_h |i - j|: A's pattern is the mask (sliding window, documents,
           prefix, a graph). A training step also returns dQ, dK, dV.
decode     one query token per sequence over cache rows listed in token order by a CSR in device memory.

``run`` computes the plain form in fp32 with elementary torch operations where ``own`` is false and calls the framework
where it is true.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # a small neighbourhood mix, as a step on a few hundred nodes: launch latency counts
        dict(name="product small", op="product", train=False, pattern="uniform", rows=300, per_row=8, width=64, type="bf16", act="silu", residual=True),
        # one layer of a graph network on a skewed graph, inference
        dict(name="product rmat", op="product", train=False, pattern="rmat", scale=18, width=128, type="bf16", act="gelu", residual=True),
        # the same layer trained, in the framework's own fp32
        dict(name="product rmat train f32", op="product", train=True, pattern="rmat", scale=16, width=128, type="f32", act="gelu", residual=True),
        # and trained in bf16 on a larger graph
        dict(name="product rmat train", op="product", train=True, pattern="rmat", scale=18, width=128, type="bf16", act="silu", residual=True),
        # odd width, no residual, regular rows: an uneven feature count. (No training case has relu: a sum that lands within
        # rounding of its corner has either slope, so that two right results may differ by a whole gradient.)
        dict(name="product odd train", op="product", train=True, pattern="uniform", rows=20011, per_row=27, width=101, type="f16", act="none", residual=False),
        # a short prompt with a bidirectional prefix
        dict(name="attention small", op="attention", train=False, pattern="prefix", rows=77, prefix=13, heads=4, kv_heads=4, dim=64, type="f16", cap=0.0, bias=False),
        # a long prompt under a sliding window with first tokens kept, grouped heads, distance bias
        dict(name="attention window", op="attention", train=False, pattern="window", rows=8192, window=1024, prefix=64, heads=32, kv_heads=8, dim=128, type="bf16", cap=0.0, bias=True),
        # training on packed documents with padding rows behind the last, capped scores
        dict(name="attention docs train", op="attention", train=True, pattern="docs", rows=6001, docs=7, pad=90, heads=16, kv_heads=16, dim=64, type="bf16", cap=30.0, bias=False),
        # a trained graph transformer layer: attention over a skewed graph's edges
        dict(name="attention graph train", op="attention", train=True, pattern="rmat", scale=15, heads=8, kv_heads=8, dim=64, type="bf16", cap=0.0, bias=False),
        # fp32 attention over a graph's edges, inference
        dict(name="attention graph f32", op="attention", train=False, pattern="rmat", scale=14, heads=4, kv_heads=4, dim=32, type="f32", cap=20.0, bias=False),
        # one sequence being answered
        dict(name="decode one", op="decode", seqs=1, context=2500, heads=16, kv_heads=4, dim=128, type="bf16", cap=0.0, bias=False),
        # a full serving batch of ragged contexts
        dict(name="decode batch", op="decode", seqs=64, context=6000, heads=32, kv_heads=8, dim=128, type="bf16", cap=50.0, bias=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "attention", "attention", "decode"])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "product":
        c = dict(op=op, train=rng.random() < 0.5, type=t, act=rng.choice(["none", "relu", "silu", "gelu"]), residual=rng.random() < 0.5)
        if c["train"] and c["act"] == "relu":
            c["act"] = "silu"
        if rng.random() < 0.5:
            c.update(pattern="rmat", graph=rng.randint(1, 1 << 20), scale=rng.randint(10, 17), width=rng.choice([32, 64, 96, 128, rng.randint(17, 128)]))
        else:
            c.update(pattern="uniform", graph=rng.randint(1, 1 << 20), rows=_spread(rng, 200, 50000), per_row=_spread(rng, 3, 60), width=rng.choice([8, 64, 128, 200, 256, rng.randint(1, 256)]))
        return c
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4])
    if op == "decode":
        return dict(op=op, seqs=_spread(rng, 1, 64), context=_spread(rng, 20, 6000), heads=heads, kv_heads=kv, dim=rng.choice([64, 128]), type=t,
                    cap=rng.choice([0.0, 30.0]), bias=rng.random() < 0.5)
    c = dict(op=op, train=rng.random() < 0.5, type=t, heads=heads, kv_heads=kv, dim=rng.choice([64, 128]), cap=rng.choice([0.0, 25.0]), bias=rng.random() < 0.5)
    kind = rng.choice(["window", "docs", "prefix", "rmat"])
    rows = _spread(rng, 65, 4500)
    if kind == "window":
        c.update(pattern=kind, rows=rows, window=min(rows, _spread(rng, 32, 1500)), prefix=rng.choice([0, 4, 64]))
    elif kind == "docs":
        c.update(pattern=kind, rows=rows, docs=rng.randint(1, 12), pad=rng.choice([0, rng.randint(1, 60)]))
    elif kind == "prefix":
        c.update(pattern=kind, rows=min(rows, 3000), prefix=rng.randint(1, 60))
    else:
        c.update(pattern=kind, graph=rng.randint(1, 1 << 20), scale=rng.randint(8, 13))
        c["dim"] = rng.choice([32, 64, 128])
    return c


# ------------------------------------------------------------------------------------------------ inputs


def _doc_cuts(c):
    """Cut points of the packed documents, a rule of the case alone."""
    n = c["rows"] - c["pad"]
    r = random.Random(n * 31 + c["docs"])
    return [0] + sorted(r.sample(range(1, n), min(c["docs"] - 1, n - 1))) + [n]


def _size(c):
    """Rows of A."""
    return 1 << c["scale"] if c["pattern"] == "rmat" else c["rows"]


def _mask(c):
    """The positional masks as a dense truth table [rows, rows]."""
    n = c["rows"]
    i = torch.arange(n, device="cuda")[:, None]
    j = torch.arange(n, device="cuda")[None, :]
    if c["pattern"] == "window":
        return (j <= i) & ((i - j < c["window"]) | (j < c["prefix"]))
    if c["pattern"] == "prefix":
        return (j <= i) | (j < c["prefix"])
    cuts = _doc_cuts(c)
    doc = torch.full((n,), -1, device="cuda")
    for d, (a, b) in enumerate(zip(cuts, cuts[1:])):
        doc[a:b] = d
    return (j <= i) & (doc[:, None] == doc[None, :]) & (doc[:, None] >= 0)


def _entries(c):
    """(row ids, column ids) of A's entries in row order, int64 on the GPU: the graph is the case's, as a plan is kept."""
    g = torch.Generator(device="cuda").manual_seed(c.get("graph", 1))
    if c["pattern"] == "rmat":  # edge factor 16, probabilities .57 .19 .19 .05, symmetric, no loops, no duplicates
        n, m = 1 << c["scale"], 16 << c["scale"]
        u = torch.zeros(m, dtype=torch.int64, device="cuda")
        v = torch.zeros_like(u)
        for _ in range(c["scale"]):
            p = torch.rand(m, device="cuda", generator=g)
            u = 2 * u + (p >= 0.76)
            v = 2 * v + (((p >= 0.57) & (p < 0.76)) | (p >= 0.95))
        u, v = torch.cat([u, v]), torch.cat([v, u])
        key = torch.unique((u * n + v)[u != v])
        return key // n, key % n
    if c["pattern"] == "uniform":  # distinct columns: a random start, then equal steps of a random length
        n, k = c["rows"], min(c["per_row"], c["rows"])
        start = torch.randint(n, (n, 1), device="cuda", generator=g)
        step = torch.randint(1, max(2, n // k + 1), (n, 1), device="cuda", generator=g)
        cols = torch.sort((start + step * torch.arange(k, device="cuda")) % n, dim=1).values
        return torch.arange(n, device="cuda").repeat_interleave(k), cols.reshape(-1)
    at = _mask(c).nonzero()
    return at[:, 0].contiguous(), at[:, 1].contiguous()


def _normal(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def prepare(case, seed):
    c, t = case, DTYPES[case["type"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "decode":
        r = random.Random(seed)
        lens = [max(1, int(c["context"] * r.uniform(0.6, 1.0))) for _ in range(c["seqs"])]
        total = sum(lens)
        slots = total + total // 8 + 16  # a cache with free rows between the used ones
        s["indptr"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int64, device="cuda")
        s["indices"] = torch.randperm(slots, device="cuda", generator=g)[:total].contiguous()
        s["q"] = _normal((c["seqs"], c["heads"], c["dim"]), g, t)
        s["k"] = _normal((slots, c["kv_heads"], c["dim"]), g, t)
        s["v"] = _normal((slots, c["kv_heads"], c["dim"]), g, t)
        s["slopes"] = _slopes(c)
        return s
    n = _size(c)
    s["rows"], s["cols"] = _entries(c)
    s["n"] = n
    count = torch.bincount(s["rows"], minlength=n)
    indptr = np.zeros(n + 1, np.int64)
    indptr[1:] = np.cumsum(count.cpu().numpy())
    if c["op"] == "product":
        w = c["width"]
        # a mean over the neighbours, each with its own weight
        s["values"] = (0.5 + torch.rand(s["cols"].numel(), device="cuda", generator=g)) / count.clamp(min=1)[s["rows"]].float().sqrt()
        s["B"] = _normal((n, w), g, t)
        s["bias"] = _normal((w,), g, torch.float32, 0.5)
        s["residual"] = _normal((n, w), g, t) if c["residual"] else None
        s["dY"] = _normal((n, w), g, t) if c["train"] else None
    else:
        s["q"] = _normal((n, c["heads"], c["dim"]), g, t)
        s["k"] = _normal((n, c["kv_heads"], c["dim"]), g, t)
        s["v"] = _normal((n, c["kv_heads"], c["dim"]), g, t)
        s["dO"] = _normal((n, c["heads"], c["dim"]), g, t) if c["train"] else None
        s["slopes"] = _slopes(c)
    if own:
        import distspmm_b200 as d
        values = s["values"].cpu().numpy() if c["op"] == "product" else np.zeros(s["cols"].numel(), np.float32)
        a = d.Csr(indptr, s["cols"].cpu().numpy(), values, n, n)
        s["plan"] = d.SparsePattern(a, grad=c["train"], attention=c["op"] == "attention")
    return s


def _slopes(c):
    """Distance-bias slopes, one for each head: 2^-1, 2^-2, ... spread over eight octaves."""
    if not c["bias"]:
        return None
    h = torch.arange(1, c["heads"] + 1, device="cuda", dtype=torch.float32)
    return torch.exp2(-8.0 * h / c["heads"])


# ------------------------------------------------------------------------------------------------ the pass


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "product":
        return _product(s, c)
    if c["op"] == "decode":
        rows = torch.repeat_interleave(s["indptr"].diff())
        dist = (s["indptr"][1:] - 1)[rows] - torch.arange(rows.numel(), device=rows.device)
        return _attention_edges(s, c, c["seqs"], rows, s["indices"], dist, False)
    if c["pattern"] == "rmat":
        return _attention_edges(s, c, s["n"], s["rows"], s["cols"], (s["rows"] - s["cols"]).abs(), c["train"])
    return _attention_dense(s, c)


def _run_own(s, c):
    import distspmm_b200 as d
    if c["op"] == "product":
        if not c["train"]:
            return dict(y=d.spmm_act(s["plan"], s["B"], values=s["values"], bias=s["bias"], residual=s["residual"], act=c["act"]))
        y, pre = d.spmm_act_forward(s["plan"], s["B"], values=s["values"], bias=s["bias"], residual=s["residual"], act=c["act"], save=True)
        dB, dvalues, dbias = d.spmm_act_backward(s["plan"], s["dY"], s["B"], pre, values=s["values"], act=c["act"])
        return dict(y=y, dB=dB, dvalues=dvalues, dbias=dbias)
    opt = dict(softcap=c["cap"], slopes=s["slopes"])
    if c["op"] == "decode":
        return dict(o=d.sparse_attention_decode(s["q"], s["k"], s["v"], s["indptr"], s["indices"], **opt))
    o, lse = d.sparse_attention_forward(s["plan"], s["q"], s["k"], s["v"], **opt)
    if not c["train"]:
        return dict(o=o, lse=lse)
    dq, dk, dv = d.sparse_attention_backward(s["plan"], s["dO"], s["q"], s["k"], s["v"], o, lse, **opt)
    return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)


def _act(z, act):
    """(act(z), act'(z))"""
    if act == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if act == "silu":
        e = 1 / (1 + torch.exp(-z))
        return z * e, e * (1 + z * (1 - e))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _product(s, c):
    t = s["B"].dtype
    B = s["B"].float()
    z = torch.zeros_like(B).index_add_(0, s["rows"], B[s["cols"]] * s["values"][:, None]) + s["bias"]
    y, slope = _act(z, c["act"])
    if c["residual"]:
        y = y + s["residual"].float()
    if not c["train"]:
        return dict(y=y.to(t))
    dz = s["dY"].float() * slope
    far = dz[s["rows"]]
    dB = torch.zeros_like(B).index_add_(0, s["cols"], far * s["values"][:, None])
    dvalues = (far * B[s["cols"]]).sum(1)
    return dict(y=y.to(t), dB=dB.to(t), dvalues=dvalues, dbias=dz.sum(0))


def _cap(x, cap):
    """The capped score and its derivative."""
    if not cap:
        return x, None
    th = torch.tanh(x / cap)
    return cap * th, 1 - th * th


def _attention_edges(s, c, n, rows, cols, dist, train):
    """Attention entry by entry: nnz x heads scores, sums over a row by indexed addition."""
    t, h, hk, dim = s["q"].dtype, c["heads"], c["kv_heads"], c["dim"]
    scale = 1 / math.sqrt(dim)
    q = s["q"].float().view(n, hk, h // hk, dim)[rows]
    k, v = s["k"].float()[cols], s["v"].float()[cols]
    u, dcap = _cap((q * k[:, :, None]).sum(-1) * scale, c["cap"])
    u = u.reshape(-1, h)
    if s["slopes"] is not None:
        u = u - s["slopes"] * dist[:, None].float()
    top = torch.full((n, h), -math.inf, device=u.device).index_reduce_(0, rows, u, "amax")
    top0 = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(u - top0[rows])
    total = torch.zeros_like(top).index_add_(0, rows, e)
    p = (e / total[rows]).view(-1, hk, h // hk)
    o = torch.zeros((n, hk, h // hk, dim), device=u.device).index_add_(0, rows, p[..., None] * v[:, :, None])
    o_t = o.view(n, h, dim).to(t)
    if c["op"] == "decode":
        return dict(o=o_t)
    lse = top0 + torch.log(total)
    if not train:
        return dict(o=o_t, lse=lse)
    dO = s["dO"].float().view(n, hk, h // hk, dim)
    dv = torch.zeros_like(s["v"], dtype=torch.float32).index_add_(0, cols, (p[..., None] * dO[rows]).sum(2))
    dp = (dO[rows] * v[:, :, None]).sum(-1)
    du = p * (dp - (dO * o).sum(-1)[rows])
    ds = (du if dcap is None else du * dcap) * scale
    dq = torch.zeros_like(o).index_add_(0, rows, ds[..., None] * k[:, :, None])
    dk = torch.zeros_like(dv).index_add_(0, cols, (ds[..., None] * q).sum(2))
    return dict(o=o_t, lse=lse, dq=dq.view(n, h, dim).to(t), dk=dk.to(t), dv=dv.to(t))


def _attention_dense(s, c):
    """Attention with the mask as a dense table."""
    t, n, h, hk, dim = s["q"].dtype, s["n"], c["heads"], c["kv_heads"], c["dim"]
    scale = 1 / math.sqrt(dim)
    mask = torch.zeros((n, n), dtype=torch.bool, device="cuda")
    mask[s["rows"], s["cols"]] = True
    q = s["q"].float().view(n, hk, h // hk, dim).permute(1, 2, 0, 3)  # [kv head, group, rows, dim]
    k = s["k"].float().permute(1, 0, 2)[:, None]
    v = s["v"].float().permute(1, 0, 2)[:, None]
    u, dcap = _cap(torch.matmul(q, k.transpose(-1, -2)) * scale, c["cap"])
    if s["slopes"] is not None:
        i = torch.arange(n, device="cuda", dtype=torch.float32)
        u = u - s["slopes"].view(hk, h // hk, 1, 1) * (i[:, None] - i[None, :]).abs()
    u = u.masked_fill(~mask, -math.inf)
    top = u.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(u - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, v)
    o_t = o.permute(2, 0, 1, 3).reshape(n, h, dim).to(t)
    lse = (top + torch.log(total)).squeeze(-1).permute(2, 0, 1).reshape(n, h)
    if not c["train"]:
        return dict(o=o_t, lse=lse)
    dO = s["dO"].float().view(n, hk, h // hk, dim).permute(1, 2, 0, 3)
    dv = torch.matmul(p.transpose(-1, -2), dO).sum(1)
    du = p * (torch.matmul(dO, v.transpose(-1, -2)) - (dO * o).sum(-1, keepdim=True))
    ds = (du if dcap is None else du * dcap) * scale
    dq = torch.matmul(ds, k).permute(2, 0, 1, 3).reshape(n, h, dim)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(1)
    return dict(o=o_t, lse=lse, dq=dq.to(t), dk=dk.permute(1, 0, 2).to(t), dv=dv.permute(1, 0, 2).to(t))


# ------------------------------------------------------------------------------------------------ work and exact values


def _count(c):
    """Entries of A."""
    if c["op"] == "decode":
        return int(c["seqs"] * max(1.0, 0.8 * c["context"]))
    if c["pattern"] == "uniform":
        return c["rows"] * min(c["per_row"], c["rows"])
    if c["pattern"] == "rmat":
        return _entries(c)[0].numel()
    n = c["rows"]
    if c["pattern"] == "window":
        w, f = min(c["window"], n), min(c["prefix"], n)
        return sum(min(i + 1, w) + min(max(0, i + 1 - w), f) for i in range(n))
    if c["pattern"] == "prefix":
        return sum(max(i + 1, min(c["prefix"], n)) for i in range(n))
    cuts = _doc_cuts(c)
    return sum((b - a) * (b - a + 1) // 2 for a, b in zip(cuts, cuts[1:]))


def work(case):
    c, nnz, t = case, _count(case), SIZE[case["type"]]
    if c["op"] == "decode":
        rows = c["seqs"] * c["heads"] * c["dim"] * t * 2 + (c["seqs"] + 1) * 8
        return dict(bytes=rows + nnz * (8 + 2 * c["kv_heads"] * c["dim"] * t), flops=4 * nnz * c["heads"] * c["dim"])
    n = _size(c)
    if c["op"] == "product":
        dense = n * c["width"] * t
        b = (n + 1) * 8 + nnz * 8 + c["width"] * 4 + dense * (3 if c["residual"] else 2)
        if not c["train"]:
            return dict(bytes=b, flops=2 * nnz * c["width"])
        return dict(bytes=b + 2 * dense + nnz * 4 + c["width"] * 4, flops=6 * nnz * c["width"])
    q, kv = n * c["heads"] * c["dim"] * t, n * c["kv_heads"] * c["dim"] * t
    b = (n + 1) * 8 + nnz * 4 + 2 * q + 2 * kv + n * c["heads"] * 4
    f = nnz * c["heads"] * c["dim"]
    if not c["train"]:
        return dict(bytes=b, flops=4 * f)
    return dict(bytes=b + 2 * q + 2 * kv, flops=14 * f)


def exact(case, seed):
    """The definitions in 64 bits; gradients by automatic differentiation."""
    c, s = case, prepare(case, seed)
    wide = lambda x: None if x is None else x.double()  # noqa: E731
    if c["op"] == "product":
        B, values, bias = (wide(s[x]).requires_grad_(c["train"]) for x in ("B", "values", "bias"))
        z = torch.zeros((s["n"], c["width"]), dtype=torch.float64, device="cuda")
        z = z.index_add(0, s["rows"], values[:, None] * B.index_select(0, s["cols"])) + bias
        y = {"none": lambda x: x, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[c["act"]](z)
        if c["residual"]:
            y = y + wide(s["residual"])
        if not c["train"]:
            return dict(y=y)
        g = torch.autograd.grad(y, [B, values, bias], wide(s["dY"]))
        return dict(y=y.detach(), dB=g[0], dvalues=g[1], dbias=g[2])
    group = c["heads"] // c["kv_heads"]
    if c["op"] == "decode":
        out = []
        ends = s["indptr"].tolist()
        for r, (a, b) in enumerate(zip(ends, ends[1:])):
            at = s["indices"][a:b]
            k, v = (wide(s[x][at]).repeat_interleave(group, 1) for x in ("k", "v"))
            u = torch.einsum("hd,thd->ht", wide(s["q"][r]), k) / math.sqrt(c["dim"])
            u = torch.tanh(u / c["cap"]) * c["cap"] if c["cap"] else u
            if s["slopes"] is not None:
                u = u - wide(s["slopes"])[:, None] * torch.arange(b - a - 1, -1, -1, device="cuda", dtype=torch.float64)
            out.append(torch.einsum("ht,thd->hd", torch.softmax(u, 1), v))
        return dict(o=torch.stack(out))
    n = s["n"]
    if n > 20000:  # entry by entry, a head at a time
        rows, cols = s["rows"], s["cols"]
        dist = (rows - cols).abs().double()
    else:
        far = torch.ones((n, n), dtype=torch.bool, device="cuda")
        far[s["rows"], s["cols"]] = False
        i = torch.arange(n, device="cuda", dtype=torch.float64)
        dist = (i[:, None] - i[None, :]).abs()
    o, lse, dq = [], [], []
    dk, dv = [[torch.zeros((n, c["dim"]), dtype=torch.float64, device="cuda") for _ in range(c["kv_heads"])] for _ in range(2)]
    for h in range(c["heads"]):
        q, k, v = (wide(x).requires_grad_(c["train"]) for x in (s["q"][:, h], s["k"][:, h // group], s["v"][:, h // group]))
        if n > 20000:
            u = (q[rows] * k[cols]).sum(1) / math.sqrt(c["dim"])
        else:
            u = q @ k.T / math.sqrt(c["dim"])
        if c["cap"]:
            u = torch.tanh(u / c["cap"]) * c["cap"]
        if s["slopes"] is not None:
            u = u - float(s["slopes"][h]) * dist
        if n > 20000:
            shift = u.detach().max()
            e = torch.exp(u - shift)
            total = torch.zeros(n, dtype=torch.float64, device="cuda").index_add(0, rows, e)
            one = torch.zeros((n, c["dim"]), dtype=torch.float64, device="cuda").index_add(0, rows, (e / total[rows])[:, None] * v[cols])
            lse.append((shift + torch.log(total)).detach())
        else:
            u = u.masked_fill(far, -math.inf)
            lse.append(torch.logsumexp(u.detach(), 1))
            live = ~torch.isinf(lse[-1])
            p = torch.exp(u - torch.where(live, lse[-1], torch.zeros_like(lse[-1]))[:, None])
            one = p @ v / torch.where(live, p.sum(1), torch.ones_like(lse[-1]))[:, None]
        o.append(one.detach())
        if c["train"]:
            g = torch.autograd.grad(one, [q, k, v], wide(s["dO"][:, h]))
            dq.append(g[0])
            dk[h // group] += g[1]
            dv[h // group] += g[2]
    res = dict(o=torch.stack(o, 1), lse=torch.stack(lse, 1))
    if c["train"]:
        res.update(dq=torch.stack(dq, 1), dk=torch.stack(dk, 1), dv=torch.stack(dv, 1))
    return res

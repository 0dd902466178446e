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

"""What spmm_act's gradients keep of fp32 in 16-bit training, and activations at their ends (tolerances: as derived in test_act_gpu,
without a rounding of dz to 16 bits)."""
import numpy as np
import pytest
import torch

import distspmm_b200 as d
from sparse_reference import HALF_STEP, TINY, U, csr_of, matrix, product64, row_ids
from test_act_gpu import grads64, inputs, lens, near, wide

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def dB_tolerance(a, B, values, b, dy, act, t, n, dz, wB, sB):
    """As grad_tolerances, with dz kept to 16 bits (2^-16) at least."""
    _, z, size = product64(a, wide(B), wide(values), wide(b), None, act)
    e_dz = wide(dy).abs() * (0.8 * (lens(a)[:, None] + 2) * U * size + 9 * U * z.abs().clamp(min=1)) + 2.0 ** -16 * dz.abs()
    rows, cols = row_ids(a), torch.from_numpy(a.indices)
    count = torch.bincount(cols, minlength=a.num_cols).double()
    e_B = torch.zeros_like(wB).index_add(0, cols, wide(values).abs()[:, None] * e_dz[rows]) + (count[:, None] + 2) * U * sB
    return 1.01 * e_B + HALF_STEP[t] * (wB.abs() + e_B) + TINY[t]


def check_dB(a, n, t, act, values=None, size=1.0):
    p = d.SparsePattern(a, grad=True)
    B, b, _, dy = inputs(a, n, t, n)
    dy = (dy.float() * size).to(t)
    values = torch.from_numpy(a.values) if values is None else values
    _, pre = d.spmm_act_forward(p, B.cuda(), values.cuda(), b.cuda(), None, act, save=True)
    dB = d.spmm_act_backward(p, dy.cuda(), B.cuda(), pre, values.cuda(), act)[0]
    wB, _, _, dz, (sB, _, _) = grads64(a, wide(B), wide(values), wide(b), wide(dy), act)
    assert dB.dtype == t
    near(dB, wB, dB_tolerance(a, B, values, b, dy, act, t, n, dz, wB, sB), "dB")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("n", [1, 7, 12, 20, 32, 40, 64, 128, 200, 256, 264, 520])
@pytest.mark.parametrize("t", [BF16, F16])
def test_dz_is_not_rounded_to_the_type(gpu, t, n, act):
    check_dB(matrix("rmat"), n, t, act)


@pytest.mark.parametrize("kind", ["hub", "repeated", "gap", "column", "row"])
@pytest.mark.parametrize("t,n", [(BF16, 64), (F16, 96), (F16, 33)])
def test_dz_of_other_matrices(gpu, kind, t, n):
    check_dB(matrix(kind), n, t, "silu")


@pytest.mark.parametrize("n", [20, 33, 64])
def test_small_dz_in_fp16(gpu, n):
    """dz near 1e-7 with values of 100: the products are far above fp16's smallest."""
    a = matrix("rmat")
    check_dB(a, n, F16, "silu", values=torch.full((a.nnz,), 100.0), size=2.0 ** -20)


@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_relu_gradient_of_infinities(gpu, t):
    """Where z <= 0 nothing flows, not even an infinity."""
    a = csr_of([[0], [1], [2]], 3, [1.0, 1.0, 1.0])
    p = d.SparsePattern(a, grad=True)
    B = torch.tensor([[1.0], [-1.0], [0.0]]).repeat(1, 40).to(t).cuda()
    _, pre = d.spmm_act_forward(p, B, act="relu", save=True)
    dy = torch.full((3, 40), float("inf"), dtype=t)
    dy[:, 1::2] = float("nan")
    dB, dv, db = d.spmm_act_backward(p, dy.cuda(), B, pre, act="relu")
    zero = torch.zeros(2, 40)
    assert torch.equal(dB[1:].cpu().float(), zero) and torch.isinf(dB[0, ::2]).all() and torch.isnan(dB[0, 1::2]).all()
    assert (dv[1:] == 0).all() and torch.isinf(db[::2]).all() and torch.isnan(db[1::2]).all()


def test_gelu_tail(gpu):
    """gelu keeps its relative accuracy in the negative tail: the exponent z^2 / 2 is rounded (2^-24 of z^2), the rest is 2^-20."""
    z = torch.linspace(-12, -0.5, 4000)
    a = csr_of([[i] for i in range(4000)], 4000, np.ones(4000))
    out = d.spmm_act(d.SparsePattern(a), z[:, None].cuda(), act="gelu")[:, 0].cpu().double()
    want = 0.5 * z.double() * torch.special.erfc(-z.double() * 0.5 ** 0.5)
    near(out, want, (z.double() ** 2 * U + 2.0 ** -20) * want.abs(), "gelu")


def test_a_pattern_keeps_the_values_it_was_made_with(gpu):
    a = csr_of([[0], [1]], 2, [1.0, 2.0])
    p = d.SparsePattern(a)
    a.values[:] = 5
    B = torch.ones(2, 4, device="cuda")
    assert torch.equal(d.spmm_act(p, B).cpu(), torch.tensor([[1.0] * 4, [2.0] * 4]))
    assert torch.equal(p.values.cpu(), torch.tensor([1.0, 2.0]))

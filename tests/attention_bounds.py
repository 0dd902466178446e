"""Bounds on the errors of 16-bit attention whose weights and score gradients enter the products in two parts (CPU, 64 bits)."""
import torch

from sparse_reference import HALF_STEP, TINY, U

PART = 2.0 ** -16  # x as bf16 hi + lo: hi is off by 2^-8 of x at most, lo by 2^-8 of that (fp16: 2^-22, where neither is subnormal)


def bounds(mask, q, k, v, out, lse, p, t, scale, cap=0.0, slopes=None, row_offset=0, dist=None, dout=None, grads=None, depth=None, once=True):
    """{"out", "lse"[, "dq", "dk", "dv"]}: how far a result of type t may be off, for 64-bit copies of the inputs.

    A score is a sum of dim products in fp32; the cap's tanh is within 2^-20 of itself, the bias a rounding or two. A normalised
    weight is off (relatively) by twice the row's worst score error, the exponential's 2^-21 and argument rounding, and the sums' n +
    10 roundings; as an operand by PART more. delta is delta0 + sum p (dp - delta0), delta0 = dout . out with the rounded out, so
    that it is off by what p and dp are off, applied to differences from delta0 (at most D away from delta) alone; once: the correction's
    weights may be rounded to t once, as they are multiplied by D. Results are rounded to t once. depth: roundings on a term's way
    through a row's sum, where fewer than the row has entries."""
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    m, h, s = mask.double(), HALF_STEP[t], abs(scale)
    part = 0.0 if t == torch.float32 else PART
    size = torch.einsum("ihd,jhd->hij", q.abs(), kk.abs()) * s
    e_u = (dim + 10) * U * size.clamp(min=1)
    if cap:
        e_u = e_u + 2.0 ** -20 * size
    if slopes is not None:
        if dist is None:
            dist = (torch.arange(q.shape[0])[:, None] + row_offset - torch.arange(k.shape[0])[None, :]).abs().double()
        e_u = e_u + 4 * U * slopes.double().abs()[:, None, None] * dist
    worst = (e_u * m).amax(-1, keepdim=True) if e_u.shape[-1] else e_u.sum(-1, keepdim=True)  # [h, i, 1]
    n = m.sum(-1).clamp(min=1, max=depth)[None, :, None]
    live = lse.t().nan_to_num(neginf=0).abs()[:, :, None]
    e_p = 2 * worst + (n + 10) * U + 2.0 ** -20 + 8 * U * live
    e_out = torch.einsum("hij,jhd->ihd", p * (e_p + part), vv.abs())
    tol = {"out": e_out + h * (out.abs() + e_out) + TINY[t],
           "lse": (worst + (n + 10) * U + 2.0 ** -20).squeeze(-1).t() + 4 * U * live.squeeze(-1).t()}
    if dout is None:
        return tol

    def row(x):  # [i, h] -> [h, i, 1]
        return x.t()[:, :, None]

    far = row((dout.abs() * tol["out"]).sum(-1))  # D
    dp = torch.einsum("ihd,jhd->hij", dout, vv)
    gap = (dp - row((dout * out).sum(-1))).abs()
    e_dp = (dim + 2) * U * torch.einsum("ihd,jhd->hij", dout.abs(), vv.abs())
    e_delta = (p * ((gap + far) * (e_p + (n + 10) * U) + e_dp)).sum(-1, keepdim=True) + row((dim + 2) * U * (dout * out).abs().sum(-1))
    e_c = (4 * e_u / cap + 2.0 ** -18) if cap else 0.0
    ds = p * gap * s
    e_ds = ds * (e_p + e_c + 8 * U) + p * s * (e_dp + e_delta) * (1 + e_p)
    keys = k.shape[0]
    rows_n = m.sum(0).clamp(min=1)[None, None, :] * group

    def fold(x):
        return x.view(keys, k.shape[1], group, dim).sum(2)

    near_q = p * s * (gap + far)
    rounded = h if t != torch.float32 and once else part
    e_dq = torch.einsum("hij,jhd->ihd", e_ds + near_q * (part + n * U) + p * s * far * (rounded + e_p + e_c), kk.abs())
    e_dk = fold(torch.einsum("hij,ihd->jhd", e_ds + ds * (part + rows_n * U), q.abs()))
    e_dv = fold(torch.einsum("hij,ihd->jhd", p * (e_p + part + rows_n * U), dout.abs()))
    for name, e, g in zip(("dq", "dk", "dv"), (e_dq, e_dk, e_dv), grads):
        tol[name] = e + h * (g.abs() + e) + TINY[t]
    return tol

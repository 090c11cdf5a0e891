"""Low-rank adapters beside a shared projection, in fp64 and token by token.  Test infrastructure only.

Next to every result stands a bound of what rounding may do to it: fp32 sums of n products are off by at most n 2^-24 of the sum
of their absolute values, an fp32 vector split into two bf16 parts by 2^-17 of it, and a result rounded to t by half a step.
"""
from __future__ import annotations

import torch

F32 = 2.0 ** -24


def _sums(n):
    return (n + 8) * F32


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _denormal(dtype):
    """Half the spacing of the smallest numbers of a type: what rounding costs near zero."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def forward(base, hidden, a, b, ids, scaling):
    """(out, u, bound of out, bound of u), fp64."""
    s, r, h = a.shape
    x, y = hidden.double(), base.double().clone()
    u = torch.zeros(x.shape[0], r, dtype=torch.float64)
    du = torch.zeros_like(u)
    slack = torch.zeros_like(y)
    for i in range(s):
        rows = torch.nonzero(ids == i).squeeze(1)
        if rows.numel() == 0:
            continue
        ai, bi, sc = a[i].double(), b[i].double(), float(scaling[i])
        u[rows] = sc * (x[rows] @ ai.t())
        du[rows] = abs(sc) * _sums(h) * (x[rows].abs() @ ai.abs().t()) + F32 * u[rows].abs()
        y[rows] += u[rows] @ bi.t()
        slack[rows] = (du[rows] + (2.0 ** -17 + 2 * _sums(r)) * u[rows].abs()) @ bi.abs().t() + 2 * F32 * base[rows].double().abs()
    bound = slack + _half_step(base.dtype) * (y.abs() + slack) + _denormal(base.dtype)
    return y, u, bound, du + 1e-38


def backward(dy, hidden, a, b, ids, scaling, u, dx_base):
    """((dx, dA, dB), their bounds), fp64; u as the kernel is given it."""
    s, r, h = a.shape
    o = b.shape[1]
    n = hidden.shape[0]
    g, x, u = dy.double(), hidden.double(), u.double()
    dx = torch.zeros(n, h, dtype=torch.float64) if dx_base is None else dx_base.double().clone()
    slack = 2 * F32 * dx.abs()
    da, db = torch.zeros(s, r, h, dtype=torch.float64), torch.zeros(s, o, r, dtype=torch.float64)
    ea, eb = torch.zeros_like(da), torch.zeros_like(db)
    for i in range(s):
        rows = torch.nonzero(ids == i).squeeze(1)
        if rows.numel() == 0:
            continue
        ai, bi, sc = a[i].double(), b[i].double(), float(scaling[i])
        du = sc * (g[rows] @ bi)
        e_du = abs(sc) * _sums(o) * (g[rows].abs() @ bi.abs()) + F32 * du.abs()
        dx[rows] += du @ ai
        slack[rows] += (e_du + (2.0 ** -17 + 2 * _sums(r)) * du.abs()) @ ai.abs()
        da[i] = du.t() @ x[rows]
        ea[i] = (e_du + 6 * _sums(rows.numel()) * du.abs()).t() @ x[rows].abs()
        db[i] = g[rows].t() @ u[rows]
        eb[i] = g[rows].abs().t() @ (6 * _sums(rows.numel()) * u[rows].abs())
    edx = slack + _half_step(hidden.dtype) * (dx.abs() + slack) + _denormal(hidden.dtype)
    return (dx, da, db), (edx, ea + 1e-38, eb + 1e-38)

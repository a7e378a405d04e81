"""64-bit definitions of the hidden-layer operators and what an evaluation with the kernels' roundings may be off by."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # smallest subnormal
U = 2.0 ** -24  # half a step of the fp32 sums


def close(got, ref, bound, what=""):
    """|got - ref| <= bound + half a step of got's type, element by element; the same elements finite."""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    ref = ref.detach()
    tol = bound + HALF[got.dtype] * (ref.abs() + bound) + TINY[got.dtype]
    err = (got.detach().double().cpu() - ref).abs()
    assert bool(torch.isfinite(err).all()), (what, "not finite")
    worst = float((err / tol).max()) if err.numel() else 0.0
    assert worst <= 1.0, (what, worst)


def layer_norm(x, w, b, dy, eps=1e-5):
    """-> {name: (value, bound of the fp32 evaluation)} on the CPU in 64 bits."""
    x, dy = x.double().cpu(), dy.double().cpu()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double().cpu()
    x, dy = x.reshape(-1, D), dy.reshape(-1, D)
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    # a sum over a row is at most 32 additions in a thread and 16 levels of a tree: 48 roundings of partial sums that the sum
    # of magnitudes bounds; the mean's error shifts a row, the variance's scales it by half as much
    n = 64 * U
    e_mean = n * x.abs().mean(1, keepdim=True)
    e_rel = n + e_mean * rstd * 2
    e_xh = e_rel * xh.abs() + (e_mean + U * (x - mean).abs()) * rstd
    e_y = e_xh * w.abs() + 4 * U * ((xh * w).abs() + b.abs())
    e_m0 = n * g.abs().mean(1, keepdim=True)
    e_m1 = n * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    m1 = (g * xh).mean(1, keepdim=True)
    e_dx = rstd * (e_m0 + xh.abs() * e_m1 + e_xh * m1.abs() + 8 * U * (g.abs() + g.mean(1, keepdim=True).abs() + (xh * m1).abs()))
    e_dx = e_dx + e_rel * dx.abs()
    R = x.shape[0]
    e_dw = (R + 32) * U * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    e_db = (R + 32) * U * dy.abs().sum(0)
    return {"y": (xh * w + b, e_y), "dx": (dx, e_dx), "dw": ((dy * xh).sum(0), e_dw), "db": (dy.sum(0), e_db),
            "mean": (mean[:, 0], e_mean[:, 0]), "rstd": (rstd[:, 0], (e_rel * rstd)[:, 0])}


def _act(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def gated_mlp(x, w_in, w_out, b_in, b_out, dy, act, residual=None):
    """-> {name: (value, bound)}: fp32 sums in any order (one rounding per term), h and [dg | du] rounded once to the type."""
    dt = x.dtype
    half = HALF[dt] + 4 * U  # (fp32: the operands' 24-bit planes and the dropped products, a few U per term)
    x, w_in, w_out, dy = (t.double().cpu() for t in (x.reshape(-1, x.shape[-1]), w_in, w_out, dy.reshape(-1, dy.shape[-1])))
    F, M = w_out.shape[1], x.shape[0]
    K, O = x.shape[1], w_out.shape[0]
    b_in = torch.zeros(2 * F, dtype=torch.float64) if b_in is None else b_in.double().cpu()
    b_out = torch.zeros(O, dtype=torch.float64) if b_out is None else b_out.double().cpu()
    res = torch.zeros(M, O, dtype=torch.float64) if residual is None else residual.double().cpu().reshape(M, O)
    gu = x @ w_in.t() + b_in
    e_gu = (K + 32) * U * (x.abs() @ w_in.abs().t() + b_in.abs())
    g, u, e_g, e_u = gu[:, :F], gu[:, F:], e_gu[:, :F], e_gu[:, F:]
    a, da = _act(act, g)
    e_a, e_da = 1.13 * e_g + 16 * U * (a.abs() + U), 0.8 * e_g + 16 * U  # |act'| <= 1.13, |act''| <= 0.8
    h = a * u
    e_h = e_a * u.abs() + a.abs() * e_u + half * h.abs() + TINY[dt]
    y = h @ w_out.t() + b_out + res
    e_y = e_h @ w_out.abs().t() + (F + 32) * U * (h.abs() @ w_out.abs().t()) + 4 * U * (b_out.abs() + res.abs() + y.abs())
    dh = dy @ w_out
    e_dh = (O + 32) * U * (dy.abs() @ w_out.abs())
    dgu = torch.cat([dh * u * da, dh * a], 1)
    e_d32 = torch.cat([e_dh * (u * da).abs() + dh.abs() * (e_u * da.abs() + u.abs() * e_da), e_dh * a.abs() + dh.abs() * e_a], 1)
    e_d = e_d32 + half * dgu.abs() + TINY[dt]
    out = {"y": (y, e_y)}
    out["dx"] = (dgu @ w_in, e_d @ w_in.abs() + (2 * F + 32) * U * (dgu.abs() @ w_in.abs()))
    out["dw_in"] = (dgu.t() @ x, e_d.t() @ x.abs() + (M + 32) * U * (dgu.abs().t() @ x.abs()))
    out["dw_out"] = (dy.t() @ h, dy.abs().t() @ e_h + (M + 32) * U * (dy.abs().t() @ h.abs()))
    out["db_in"] = (dgu.sum(0), e_d32.sum(0) + (M + 32) * U * dgu.abs().sum(0))
    out["db_out"] = (dy.sum(0), (M + 32) * U * dy.abs().sum(0))
    # root mean square of the roundings to the type, each uniform within half a step at the most: (half step)^2 / 3
    v = HALF[dt] ** 2 / 3
    rms = {"y": v * (h ** 2 @ (w_out ** 2).t() + y ** 2), "dx": v * (dgu ** 2 @ w_in ** 2 + out["dx"][0] ** 2),
           "dw_in": v * ((dgu ** 2).t() @ x ** 2 + out["dw_in"][0] ** 2),
           "dw_out": v * ((dy ** 2).t() @ h ** 2 + out["dw_out"][0] ** 2)}
    return out, {k: float(t.sum()) ** 0.5 for k, t in rms.items()}


def orthogonalize(g, steps, coeffs, eps=1e-7, dtype=torch.float64):
    a, b, c = coeffs
    x = g.to(dtype)
    flip = x.shape[-2] > x.shape[-1]
    x = x / (x.double().pow(2).sum((-2, -1), keepdim=True).sqrt().to(dtype) + eps)
    if flip:
        x = x.transpose(-2, -1)
    for _ in range(steps):
        s = x @ x.transpose(-2, -1)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(-2, -1) if flip else x

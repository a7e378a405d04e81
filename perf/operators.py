"""Sizes, inputs and plain forms of the network operators this package adds beside its likelihood and ELBO kernels:
layer normalisation, the gated feed-forward block, and the orthogonalised update of a weight matrix, each in the
direction and the types a training run or a single prediction calls it with.

``own`` chooses what ``run`` does: ``False`` evaluates the formulas with elementary torch operations in 32 bits, rounded
once at the end; ``True`` calls ``cradle_vae_amd.ops``.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NS_COEFFS = (3.4445, -4.7750, 2.0315)  # odd quintic a s + b s^3 + c s^5, applied to every singular value
NS_EPS = 1e-7


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one row of a 512-wide hidden layer: a single cell scored at inference, where only latency counts
        dict(name="layer_norm_one_row", op="layer_norm", rows=1, width=512, dtype="f32", train=False),
        # 5 particles x 512 cells at the hidden width of the Norman configuration, forward and backward
        dict(name="layer_norm_step", op="layer_norm", rows=2560, width=400, dtype="f32", train=True),
        # an odd number of rows of an odd width (no row but the first is aligned), bf16 with its own weights' type
        dict(name="layer_norm_odd", op="layer_norm", rows=4099, width=1001, dtype="bf16", train=True),
        # a large training batch of a wide hidden layer: pure streaming
        dict(name="layer_norm_large", op="layer_norm", rows=32768, width=4096, dtype="bf16", train=True),
        # one row through a wide block at inference: bound by reading the weights once
        dict(name="gated_mlp_one_row", op="gated_mlp", rows=1, width=4096, hidden=10240, dtype="bf16", act="silu", bias=False,
             train=False),
        # a training step's rows at the Norman configuration's hidden width, fp32 as the package's parameters are
        dict(name="gated_mlp_step", op="gated_mlp", rows=2560, width=400, hidden=800, dtype="f32", act="silu", bias=True,
             train=True),
        # odd rows and an odd hidden width in fp16: no leading dimension of the hidden axis is a multiple of a vector
        dict(name="gated_mlp_odd", op="gated_mlp", rows=1537, width=1000, hidden=2731, dtype="f16", act="gelu", bias=True,
             train=True),
        # a large training batch of a wide block: bound by the matrix cores
        dict(name="gated_mlp_large", op="gated_mlp", rows=8192, width=4096, hidden=10240, dtype="bf16", act="silu", bias=False,
             train=True),
        # the eight 128 x 128 hidden matrices of the demo configuration, updated together: bound by latency
        dict(name="orthogonalize_hidden", op="orthogonalize", batch=8, m=128, n=128, dtype="f32", steps=5),
        # the decoder's output layer, genes x hidden, of the Norman configuration
        dict(name="orthogonalize_decoder", op="orthogonalize", batch=1, m=5000, n=400, dtype="f32", steps=5),
        # two odd matrices of 16-bit gradients
        dict(name="orthogonalize_odd", op="orthogonalize", batch=2, m=513, n=1001, dtype="f16", steps=5),
        # one large hidden matrix of 16-bit gradients: bound by the matrix cores
        dict(name="orthogonalize_large", op="orthogonalize", batch=1, m=4096, n=8192, dtype="bf16", steps=5),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; a third of them made a multiple of 64, as widths often are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 128 and rng.random() < 0.33:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    op = rng.choice(["layer_norm", "gated_mlp", "orthogonalize"])
    if op == "layer_norm":
        width = _spread(rng, 16, 32768)
        return dict(op=op, rows=_spread(rng, 1, min(65536, (1 << 27) // width)), width=width, dtype=dtype,
                    train=rng.random() < 0.7)
    if op == "gated_mlp":
        width, hidden = _spread(rng, 16, 4096), _spread(rng, 16, 10240)
        rows = _spread(rng, 1, 8192)
        if dtype == "f32":  # (keeps the 32-bit products of the plain form and the 64-bit ones within the largest case)
            rows = min(rows, max(1, int(1.5e10 / (width * hidden))))
        return dict(op=op, rows=rows, width=width, hidden=hidden, dtype=dtype, act=rng.choice(["silu", "gelu"]),
                    bias=rng.random() < 0.5, train=rng.random() < 0.7)
    small = rng.random() < 0.5
    m, n = (_spread(rng, 16, 512), _spread(rng, 16, 512)) if small else (_spread(rng, 256, 4096), _spread(rng, 256, 8192))
    return dict(op=op, batch=rng.randint(1, 12) if small else rng.randint(1, 2), m=m, n=n, dtype=dtype, steps=rng.choice([3, 5]))


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dt)

    st = dict(case=dict(case))
    if case["op"] == "layer_norm":
        R, D = case["rows"], case["width"]
        # hidden activations: rows of different scale around a mean that is not zero, scales near one, small shifts
        row_scale = torch.exp(0.5 * torch.randn(R, 1, generator=gen, device=dev))
        st["x"] = (torch.randn(R, D, generator=gen, device=dev) * row_scale + 0.5 * row_scale).to(dt)
        st["w"], st["b"] = normal(D, scale=0.2, shift=1.0), normal(D, scale=0.1)
        if case["train"]:
            st["dy"] = normal(R, D)
    elif case["op"] == "gated_mlp":
        R, K, F = case["rows"], case["width"], case["hidden"]
        st["x"] = normal(R, K)
        st["w_in"], st["w_out"] = normal(2 * F, K, scale=K ** -0.5), normal(K, F, scale=F ** -0.5)
        st["b_in"] = normal(2 * F, scale=0.1) if case["bias"] else None
        st["b_out"] = normal(K, scale=0.1) if case["bias"] else None
        if case["train"]:
            st["dy"] = normal(R, K)
    else:
        B, m, n = case["batch"], case["m"], case["n"]
        # a momentum-averaged gradient: noise plus a few directions that stand out of it
        r = max(1, min(m, n) // 16)
        u = torch.randn(B, m, r, generator=gen, device=dev)
        v = torch.randn(B, r, n, generator=gen, device=dev)
        scale = 1e-3 if case["dtype"] != "f16" else 1e-1
        st["g"] = ((torch.randn(B, m, n, generator=gen, device=dev) + torch.matmul(u, v) / r ** 0.5) * scale).to(dt)
    return st


# ---------------------------------------------------------------------------------------------------------------
# plain forms (32 bits, rounded once at the end)
# ---------------------------------------------------------------------------------------------------------------
def _plain_layer_norm(st):
    x, w, b = st["x"].float(), st["w"].float(), st["b"].float()
    dt = st["x"].dtype
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xh = xc * rstd
    y = (xh * w + b).to(dt)
    if not st["case"]["train"]:
        return {"y": y}
    dy = st["dy"].float()
    g = dy * w
    dx = (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * rstd
    return {"y": y, "dx": dx.to(dt), "dw": (dy * xh).sum(0).to(dt), "db": dy.sum(0).to(dt)}


def _act(name, g):
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    cdf = 0.5 * (1.0 + torch.erf(g * 0.7071067811865476))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * 0.3989422804014327


def _plain_gated_mlp(st):
    c = st["case"]
    F, dt = c["hidden"], st["x"].dtype
    x, w_in, w_out = st["x"].float(), st["w_in"].float(), st["w_out"].float()
    gu = x @ w_in.t()
    if st["b_in"] is not None:
        gu = gu + st["b_in"].float()
    g, u = gu[:, :F], gu[:, F:]
    a, da = _act(c["act"], g)
    h = a * u
    y = h @ w_out.t()
    if st["b_out"] is not None:
        y = y + st["b_out"].float()
    if not c["train"]:
        return {"y": y.to(dt)}
    dy = st["dy"].float()
    dh = dy @ w_out
    dgu = torch.cat([dh * u * da, dh * a], dim=1)
    out = {"y": y.to(dt), "dx": (dgu @ w_in).to(dt), "dw_in": (dgu.t() @ x).to(dt), "dw_out": (dy.t() @ h).to(dt)}
    if c["bias"]:
        out["db_in"], out["db_out"] = dgu.sum(0).to(dt), dy.sum(0).to(dt)
    return out


def _plain_orthogonalize(st):
    g = st["g"].float()
    a, b, c = NS_COEFFS
    x = g / ((g * g).sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    flip = x.shape[-2] > x.shape[-1]
    if flip:
        x = x.transpose(-2, -1).contiguous()
    for _ in range(st["case"]["steps"]):
        s = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    if flip:
        x = x.transpose(-2, -1)
    return {"o": x.to(st["g"].dtype).contiguous()}


# ---------------------------------------------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------------------------------------------
def _own_layer_norm(st):
    from cradle_vae_amd import ops

    y, mean, rstd = ops.layer_norm(st["x"], st["w"], st["b"], eps=1e-5)
    if not st["case"]["train"]:
        return {"y": y}
    dx, dw, db = ops.layer_norm_bwd(st["dy"], st["x"], st["w"], mean, rstd)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _own_gated_mlp(st):
    from cradle_vae_amd import ops

    c = st["case"]
    if not c["train"]:
        return {"y": ops.gated_mlp(st["x"], st["w_in"], st["w_out"], st["b_in"], st["b_out"], act=c["act"])}
    y, saved = ops.gated_mlp(st["x"], st["w_in"], st["w_out"], st["b_in"], st["b_out"], act=c["act"], save=True)
    dx, dw_in, dw_out, db_in, db_out = ops.gated_mlp_bwd(st["dy"], st["x"], st["w_in"], st["w_out"], saved, act=c["act"],
                                                         bias=c["bias"])
    out = {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out}
    if c["bias"]:
        out["db_in"], out["db_out"] = db_in, db_out
    return out


def _own_orthogonalize(st):
    from cradle_vae_amd import ops

    return {"o": ops.orthogonalize(st["g"], steps=st["case"]["steps"], coeffs=NS_COEFFS, eps=NS_EPS)}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "gated_mlp": _own_gated_mlp, "orthogonalize": _own_orthogonalize}[op](state)
    return {"layer_norm": _plain_layer_norm, "gated_mlp": _plain_gated_mlp, "orthogonalize": _plain_orthogonalize}[op](state)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "layer_norm":
        R, D = case["rows"], case["width"]
        fwd = (2 * R * D + 2 * D) * e  # x, weight, bias in; y out
        bwd = (2 * R * D + 2 * D) * e  # dy in (x is read already); dx, dweight, dbias out
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": (8 + (14 if case["train"] else 0)) * R * D}
    if case["op"] == "gated_mlp":
        R, K, F = case["rows"], case["width"], case["hidden"]
        bias = 2 * F + K if case["bias"] else 0
        fwd = (2 * R * K + 3 * F * K + bias) * e  # x, both weights in; y out
        bwd = (2 * R * K + 3 * F * K + bias) * e  # dy in; dx, the weights' gradients out
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": (18 if case["train"] else 6) * R * K * F}
    B, m, n = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    # per step: the symmetric x x^T and its square need half of their elements, the product with x all of them
    return {"bytes": 2 * B * m * n * e, "flops": B * case["steps"] * (m * m * n + m * m * m + 2 * m * m * n)}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "orthogonalize":
        a, b, c = NS_COEFFS
        done = []
        for g in st["g"].double():
            x = g / (torch.linalg.matrix_norm(g) + NS_EPS)
            for _ in range(case["steps"]):  # p(x) = x (a + b x^T x + c (x^T x)^2) or its mirror: the same singular values
                left = x.shape[0] <= x.shape[1]
                s = torch.mm(x, x.t()) if left else torch.mm(x.t(), x)
                q = torch.addmm(torch.eye(s.shape[0], dtype=s.dtype, device=s.device) * a + b * s, s, s, alpha=c)
                x = torch.mm(q, x) if left else torch.mm(x, q)
            done.append(x)
        return {"o": torch.stack(done)}
    f64 = {k: v.double().requires_grad_(case["train"]) for k, v in st.items() if torch.is_tensor(v) and k != "dy"}
    if case["op"] == "layer_norm":
        x = f64["x"]
        var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
        y = (x - mean) / (var + 1e-5).sqrt() * f64["w"] + f64["b"]
        names = {"dx": "x", "dw": "w", "db": "b"}
    else:
        gu = torch.nn.functional.linear(f64["x"], f64["w_in"], f64.get("b_in"))
        gate, up = gu.chunk(2, dim=1)
        act = torch.nn.functional.silu if case["act"] == "silu" else torch.nn.functional.gelu
        y = torch.nn.functional.linear(act(gate) * up, f64["w_out"], f64.get("b_out"))
        names = {"dx": "x", "dw_in": "w_in", "dw_out": "w_out"}
        if case["bias"]:
            names.update(db_in="b_in", db_out="b_out")
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [f64[k] for k in names.values()], st["dy"].double())
    return {"y": y.detach(), **dict(zip(names, grads))}

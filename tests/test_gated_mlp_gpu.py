"""The gated feed-forward block, forward / backward, against the 64-bit definition."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("dx", "dw_in", "dw_out", "db_in", "db_out")


def _inputs(M, K, F, O, dtype, bias=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=gen) * scale).to(dtype)
    x, w_in, w_out = n(M, K), n(2 * F, K, scale=K ** -0.5), n(O, F, scale=F ** -0.5)
    b_in, b_out = (n(2 * F, scale=0.3), n(O, scale=0.3)) if bias else (None, None)
    return x, w_in, w_out, b_in, b_out, n(M, O)


def _rms(name, got, want, rms):
    # the roundings are independent: with this many elements their root mean square is within a quarter of its expectation
    if got.dtype != torch.float32 and got.numel() >= 2000:
        err = float((got.double().cpu() - want).norm())
        assert err <= 1.25 * rms, (name, err / rms)


def _check(x, w_in, w_out, b_in, b_out, dy, act="silu", residual=None):
    want, rms = ref.gated_mlp(x, w_in, w_out, b_in, b_out, dy, act, residual)
    c = lambda t: None if t is None else t.cuda()
    gx, gi, go = c(x), c(w_in), c(w_out)
    y0 = ops.gated_mlp(gx, gi, go, c(b_in), c(b_out), act=act, residual=c(residual))
    y, saved = ops.gated_mlp(gx, gi, go, c(b_in), c(b_out), act=act, residual=c(residual), save=True)
    ref.close(y0, want["y"][0], want["y"][1], "y (inference)")
    ref.close(y, want["y"][0], want["y"][1], "y")
    _rms("y", y, want["y"][0], rms["y"])
    grads = ops.gated_mlp_bwd(c(dy), gx, gi, go, saved, act=act, bias=b_in is not None)
    for name, got in zip(NAMES, grads):
        if b_in is None and name.startswith("db"):
            assert got is None
            continue
        ref.close(got, want[name][0], want[name][1], name)
        if name in rms:
            _rms(name, got, want[name][0], rms[name])


SIZES = [(1, 1, 1, 1), (1, 16, 24, 16), (2, 40, 8, 40), (5, 7, 9, 11), (64, 64, 64, 64), (33, 100, 51, 100), (130, 72, 136, 72),
         (257, 200, 300, 96), (129, 129, 127, 131), (300, 33, 520, 33)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,F,O", SIZES)
def test_against_definition(M, K, F, O, dtype):
    _check(*_inputs(M, K, F, O, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_without_bias(act, dtype):
    _check(*_inputs(70, 88, 120, 56, dtype, bias=False), act=act)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sums_split_along_k(dtype):
    # weight gradients over 3001 rows and a hidden axis of 2100: few output tiles, so the products are split along K
    _check(*_inputs(3001, 40, 24, 48, dtype))
    _check(*_inputs(20, 48, 2100, 40, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_tiles(dtype):
    # enough tiles for the 256-wide kernels
    x, w_in, w_out, b_in, b_out, dy = _inputs(4100, 264, 4104, 264, dtype)
    gx, gi, go, gb, gdy = (t.cuda() for t in (x, w_in, w_out, b_in, dy))
    y, saved = ops.gated_mlp(gx, gi, go, gb, None, save=True)
    grads = ops.gated_mlp_bwd(gdy, gx, gi, go, saved, bias=True)
    xd, wi, wo, d = (t.double().cuda() for t in (x, w_in, w_out, dy))
    gu = xd @ wi.t() + b_in.double().cuda()
    g, u = gu.chunk(2, 1)
    s = torch.sigmoid(g)
    h = g * s * u
    dh = d @ wo
    dgu = torch.cat([dh * u * s * (1 + g * (1 - s)), dh * g * s], 1)
    # normwise: two roundings to the type (fp32: sums of up to 4104 terms, each off by a few 2^-24 of a random walk)
    tol = 1.25 * (2 * ref.HALF[dtype] ** 2 / 3) ** 0.5 if dtype != torch.float32 else 16 * ref.U
    for name, got, want in (("y", y, h @ wo.t()), ("dx", grads[0], dgu @ wi), ("dw_in", grads[1], dgu.t() @ xd),
                            ("dw_out", grads[2], d.t() @ h), ("db_in", grads[3], dgu.sum(0))):
        err = float((got.double() - want).norm() / want.norm())
        assert err <= tol, (name, err, tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_residual_strides_and_leading_axes(dtype):
    x, w_in, w_out, b_in, b_out, dy = _inputs(24, 40, 56, 48, dtype)
    res = torch.randn(24, 48, generator=torch.Generator().manual_seed(9)).to(dtype)
    _check(x, w_in, w_out, b_in, b_out, dy, residual=res)
    want, _ = ref.gated_mlp(x, w_in, w_out, b_in, b_out, dy, "silu", res)

    def strided(t, pad):  # rows inside a wider buffer of NaN
        buf = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=dtype, device="cuda")
        view = buf[:, pad // 2:pad // 2 + t.shape[1]]
        view.copy_(t)
        return view

    sx, si, so, sr, sd = (strided(t, p) for t, p in ((x, 16), (w_in, 6), (w_out, 16), (res, 5), (dy, 16)))
    y, saved = ops.gated_mlp(sx, si, so, b_in.cuda(), b_out.cuda(), residual=sr, save=True)
    ref.close(y, want["y"][0], want["y"][1], "y")
    for name, got in zip(NAMES, ops.gated_mlp_bwd(sd, sx, si, so, saved, bias=True)):
        ref.close(got, want[name][0], want[name][1], name)
    y3 = ops.gated_mlp(x.cuda().reshape(2, 3, 4, 40), w_in.cuda(), w_out.cuda(), b_in.cuda(), b_out.cuda(),
                       residual=res.cuda().reshape(2, 3, 4, 48))
    assert y3.shape == (2, 3, 4, 48)
    ref.close(y3.reshape(24, 48), want["y"][0], want["y"][1], "y3")
    one = ops.gated_mlp(sx[5:6], si, so, b_in.cuda(), b_out.cuda(), residual=sr[5:6])
    ref.close(one, want["y"][0][5:6], want["y"][1][5:6], "one row")


def test_no_rows_and_partial_gradients():
    x, w_in, w_out, b_in, b_out, dy = (t.cuda() for t in _inputs(6, 16, 24, 8, torch.float32))
    y, saved = ops.gated_mlp(x[:0], w_in, w_out, b_in, b_out, save=True)
    grads = ops.gated_mlp_bwd(dy[:0], x[:0], w_in, w_out, saved, bias=True)
    assert y.shape == (0, 8) and grads[0].shape == (0, 16) and all(float(g.abs().sum()) == 0 for g in grads[1:])
    y, saved = ops.gated_mlp(x, w_in, w_out, b_in, b_out, save=True)
    full = ops.gated_mlp_bwd(dy, x, w_in, w_out, saved, bias=True)
    part = ops.gated_mlp_bwd(dy, x, w_in, w_out, saved, need=(False, False, True))
    assert part[0] is None and part[1] is None and part[3] is None and torch.equal(part[2], full[2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_bad_row_stays_its_own(dtype):
    x, w_in, w_out, b_in, b_out, dy = (t.cuda() for t in _inputs(70, 40, 48, 40, dtype))
    y0 = ops.gated_mlp(x, w_in, w_out, b_in, b_out)
    x[13, 5] = float("nan")
    x[50, 1] = float("inf")
    y1 = ops.gated_mlp(x, w_in, w_out, b_in, b_out)
    keep = [i for i in range(70) if i not in (13, 50)]
    assert torch.equal(y0[keep], y1[keep]) and bool(torch.isnan(y1[13]).all()) and not bool(torch.isfinite(y1[50]).all())


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_saturated_gates(act):
    # pre-activations of +-300: the gate is the identity or zero, its derivative one or zero, nothing is NaN
    x = torch.tensor([[300.0], [-300.0], [0.0], [88.0], [-104.0]])
    w_in, w_out = torch.ones(2, 1), torch.ones(1, 1)
    _check(x, w_in, w_out, None, None, torch.ones(5, 1), act=act)


def test_repeats_bit_for_bit():
    x, w_in, w_out, b_in, b_out, dy = (t.cuda() for t in _inputs(1500, 48, 40, 48, torch.float32))
    first = None
    for _ in range(3):
        y, saved = ops.gated_mlp(x, w_in, w_out, b_in, b_out, save=True)
        now = (y, *ops.gated_mlp_bwd(dy, x, w_in, w_out, saved, bias=True))
        assert first is None or all(torch.equal(p, q) for p, q in zip(first, now))
        first = now


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [True, False])
def test_blocks_too_large_for_a_second_plane(dtype, bias):
    # rows * hidden * (width + out) >= 2^28: h and [dg | du] in the tensors' type; no extent a multiple of a tile
    _check(*_inputs(700, 633, 611, 592, dtype, bias=bias), act="gelu" if bias else "silu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_rows_of_unaligned_widths(dtype):
    # from 2048 rows on 16-bit operands whose rows do not start on cache lines are packed, and the hidden axis is padded to 64
    _check(*_inputs(2050, 200, 1032, 136, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_dot_products_and_tiles_for_a_few_rows(dtype):
    # both sides of the rows where the tile products take over, for small and for large weights
    for rows in (3, 4, 5, 8, 9):
        x, w_in, w_out, b_in, b_out, _ = _inputs(rows, 72, 100, 64, dtype, seed=rows)
        want, _ = ref.gated_mlp(x, w_in, w_out, b_in, b_out, torch.zeros(rows, 64, dtype=dtype), "silu", None)
        y = ops.gated_mlp(x.cuda(), w_in.cuda(), w_out.cuda(), b_in.cuda(), b_out.cuda())
        ref.close(y, want["y"][0], want["y"][1], f"{rows} rows")
    x, w_in, w_out, b_in, b_out, _ = _inputs(5, 2048, 2816, 2048, dtype)  # 2816 x 6144 >= 2^24 weights
    want, _ = ref.gated_mlp(x, w_in, w_out, b_in, b_out, torch.zeros(5, 2048, dtype=dtype), "silu", None)
    for rows in (4, 5):
        y = ops.gated_mlp(x[:rows].cuda(), w_in.cuda(), w_out.cuda(), b_in.cuda(), b_out.cuda())
        ref.close(y, want["y"][0][:rows], want["y"][1][:rows], f"{rows} rows, large weights")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_weight_gradient_alone(dtype):
    # a weight gradient of large tiles and nothing beside it: dy's column sums have no other launch to go along with
    x, w_in, w_out, b_in, b_out, dy = _inputs(70, 4096, 2048, 40, dtype)
    want, _ = ref.gated_mlp(x, w_in, w_out, b_in, b_out, dy, "silu", None)
    gx, gi, go = x.cuda(), w_in.cuda(), w_out.cuda()
    _, saved = ops.gated_mlp(gx, gi, go, b_in.cuda(), b_out.cuda(), save=True)
    grads = ops.gated_mlp_bwd(dy.cuda(), gx, gi, go, saved, bias=True, need=(False, True, False))
    assert grads[0] is None and grads[2] is None
    for i in (1, 3, 4):
        ref.close(grads[i], want[NAMES[i]][0], want[NAMES[i]][1], NAMES[i])

"""The gated feed-forward block where its operands are staged in unusual ways: views inside wider buffers at sizes that
pad the hidden axis, long row strides, and the fp32 products' planes."""
import math

import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref
from tests.test_gated_mlp_gpu import DTYPES, NAMES, _inputs

pytestmark = pytest.mark.gpu


def _in_nan(t, cols):
    """t as the leading columns of a buffer of NaN rows of ``cols`` numbers."""
    buf = torch.full((t.shape[0], cols), float("nan"), dtype=t.dtype, device="cuda")
    view = buf[:, :t.shape[1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weights_inside_wider_buffers_with_a_padded_hidden_axis(dtype):
    # 2048 rows pad 1032 hidden units to 1088, and w_out's rows of 1088 numbers are staged as they lie: what is beside
    # its 1032 columns belongs to nobody
    x, w_in, w_out, b_in, b_out, dy = _inputs(2048, 128, 1032, 64, dtype)
    want, _ = ref.gated_mlp(x, w_in, w_out, b_in, b_out, dy, "silu")
    gx, gi, go = _in_nan(x, 192), _in_nan(w_in, 192), _in_nan(w_out, 1088)
    gb, gc = b_in.cuda(), b_out.cuda()
    y0 = ops.gated_mlp(gx, gi, go, gb, gc)
    y, saved = ops.gated_mlp(gx, gi, go, gb, gc, save=True)
    assert torch.equal(y0, y) and torch.equal(y, ops.gated_mlp(x.cuda(), w_in.cuda(), w_out.cuda(), gb, gc))
    ref.close(y, want["y"][0], want["y"][1], "y")
    for name, got in zip(NAMES, ops.gated_mlp_bwd(_in_nan(dy, 128), gx, gi, go, saved, bias=True)):
        ref.close(got, want[name][0], want[name][1], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 2, 20])
def test_rows_far_apart(rows, dtype):
    # row strides of 2^22 + 8 numbers (one row: its parent's, which nobody uses); weights that span 2^30 numbers
    x, w_in, w_out, b_in, b_out, dy = _inputs(rows, 40, 24, 16, dtype)
    want, _ = ref.gated_mlp(x, w_in, w_out, b_in, b_out, dy, "silu")
    far = (1 << 22) + 8

    def apart(t, ld):
        buf = torch.empty(t.shape[0] * ld, dtype=dtype, device="cuda")
        view = buf.as_strided(t.shape, (ld, 1))
        view.copy_(t)
        return view

    gx, gd, gi, go = apart(x, far), apart(dy, far), apart(w_in, 1 << 21 if dtype == torch.bfloat16 else 48), w_out.cuda()
    b = b_in.cuda(), b_out.cuda()
    ref.close(ops.gated_mlp(gx, gi, go, *b), want["y"][0], want["y"][1], "y (inference)")
    y, saved = ops.gated_mlp(gx, gi, go, *b, save=True)
    ref.close(y, want["y"][0], want["y"][1], "y")
    for name, got in zip(NAMES, ops.gated_mlp_bwd(gd, gx, gi, go, saved, bias=True)):
        ref.close(got, want[name][0], want[name][1], name)
    mean, rstd = ops.layer_norm(gx)[1:]
    assert torch.equal(ops.layer_norm_bwd(gx, gx, None, mean, rstd)[0], ops.layer_norm_bwd(x.cuda(), x.cuda(), None, mean, rstd)[0])


def _gate_alone(act, g):
    """act(g) and act'(g) as the block's output and input gradient in fp32: one hidden unit whose up projection is 1, so that
    nothing else is rounded (its one product is by 1)."""
    x = g.reshape(-1, 1).cuda()
    w_in, w_out, b_in = torch.tensor([[1.0], [0.0]]).cuda(), torch.ones(1, 1).cuda(), torch.tensor([0.0, 1.0]).cuda()
    y, saved = ops.gated_mlp(x, w_in, w_out, b_in, None, act=act, save=True)
    dx = ops.gated_mlp_bwd(torch.ones_like(y), x, w_in, w_out, saved, act=act)[0]
    few = torch.cat([ops.gated_mlp(part, w_in, w_out, b_in, None, act=act) for part in x[:400].split(8)])
    return (t.double().cpu().reshape(-1) for t in (y, dx, few))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_the_gate_in_fp32(act):
    g = torch.cat([8 * torch.rand(200, generator=torch.Generator().manual_seed(0)) - 8, torch.linspace(-8, 8, 3801)]).float()
    y, dx, few = _gate_alone(act, g)
    d, U = g.double(), ref.U
    if act == "silu":
        # the exponent's argument: two roundings of up to 1.45 |g|, the hardware's exp2 and reciprocal one step each
        s = torch.sigmoid(d)
        want, dwant = d * s, s * (1 + d * (1 - s))
        e_s = s * ((1 - s) * (1.5 * d.abs() + 3) + 3) * U
        e_d = e_s * (1 + d.abs() * (1 - s)) + s * d.abs() * (e_s + U) + 4 * U * s * (1 + d.abs() * (1 - s))
    else:
        # erfc within four steps, its argument rounded twice: a relative error of its argument's square
        s = 0.5 * torch.erfc(-d / math.sqrt(2))
        pdf = torch.exp(-0.5 * d * d) / math.sqrt(2 * math.pi)
        want, dwant = d * s, s + d * pdf
        e_s = s * 8 * U + 1.5 * d.abs() * pdf * U
        e_d = e_s + d.abs() * pdf * (2 * d * d + 8) * U + 2 * U * (s + d.abs() * pdf)
    bound = d.abs() * e_s + 2 * U * want.abs()
    assert bool(((y - want).abs() <= bound).all()), float(((y - want).abs() / bound.clamp_min(1e-300)).max())
    assert bool(((few - want[:400]).abs() <= bound[:400]).all())
    assert bool(((dx - dwant).abs() <= e_d + 2 * U * dwant.abs()).all()), float(((dx - dwant).abs() / (e_d + 2 * U * dwant.abs())).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_the_range_of_the_hidden_units(rows, dtype):
    # h = 300 * 300 beside a weight of 2^-10: y is an ordinary number of each type, but fp16's tile products hold h as fp16
    x = torch.full((rows, 1), 300.0, dtype=dtype).cuda()
    w_in, w_out = torch.ones(2, 1, dtype=dtype).cuda(), torch.full((1, 1), 2.0 ** -10, dtype=dtype).cuda()
    y = ops.gated_mlp(x, w_in, w_out)
    if dtype == torch.float16 and rows > 8:
        assert bool(torch.isinf(y).all())
    else:  # (h in fp32, or two roundings)
        assert bool(((y.double() - 90000.0 / 1024).abs() <= 2.1 * ref.HALF[dtype] * 88).all())


def test_fp16_gradients_that_vanish():
    # du = 2^-8 * 2^-10 * act(2^-7) = 2^-26 in each of 4096 rows, x = 2^-7 beside a second input of 1: the weights'
    # gradient would be 2^-14
    x = torch.tensor([[2.0 ** -7, 1.0]], dtype=torch.float16).repeat(4096, 1).cuda()
    w_in = torch.tensor([[1.0, 0.0], [1.0, 0.0]], dtype=torch.float16).cuda()
    w_out = torch.full((1, 1), 2.0 ** -10, dtype=torch.float16).cuda()
    dy = torch.full((4096, 1), 2.0 ** -8, dtype=torch.float16).cuda()
    _, saved = ops.gated_mlp(x, w_in, w_out, save=True)
    assert float(ops.gated_mlp_bwd(dy, x, w_in, w_out, saved)[1][1, 1]) == 0
    _, saved = ops.gated_mlp(x, w_in, w_out, save=True)
    scaled = ops.gated_mlp_bwd(dy * 2.0 ** 10, x, w_in, w_out, saved)[1][1, 1]  # a scaled loss brings it back
    # act(2^-7) = 2^-8 (1 + 2^-8): one rounding of the sum of equal terms to fp16
    assert abs(float(scaled) - 2.0 ** -4) <= 2.0 ** -4 * (2.0 ** -8 + 2 * ref.HALF[torch.float16])

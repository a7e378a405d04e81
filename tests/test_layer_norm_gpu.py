"""Layer norm forward / backward against the 64-bit definition."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(rows, width, dtype, seed=0, w_dtype=None):
    gen = torch.Generator().manual_seed(seed)
    scale = torch.exp(0.5 * torch.randn(rows, 1, generator=gen))
    x = ((torch.randn(rows, width, generator=gen) + 0.5) * scale).to(dtype)
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(w_dtype or dtype)
    b = (0.1 * torch.randn(width, generator=gen)).to(w_dtype or dtype)
    return x, w, b, torch.randn(rows, width, generator=gen).to(dtype)


def _check(x, w, b, dy, eps=1e-5):
    want = ref.layer_norm(x, w, b, dy, eps)
    gx, gw, gb, gdy = (None if t is None else t.cuda() for t in (x, w, b, dy))
    y, mean, rstd = ops.layer_norm(gx, gw, gb, eps=eps)
    dx, dw, db = ops.layer_norm_bwd(gdy, gx, gw, mean, rstd)
    for name, got in (("y", y), ("mean", mean), ("rstd", rstd), ("dx", dx), ("dw", dw), ("db", db)):
        ref.close(got, want[name][0], want[name][1], name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 512), (3, 7), (5, 64), (33, 400), (257, 513), (64, 1000), (19, 1024), (7, 1032),
                                        (11, 2048), (9, 3000), (6, 4096), (5, 5001), (4, 8192), (3, 12296), (3, 16384), (2, 32767),
                                        (2, 32768), (4099, 24)])
def test_against_definition(rows, width, dtype):
    _check(*_inputs(rows, width, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fp32_parameters_beside_16_bit_rows(dtype):
    _check(*_inputs(40, 264, dtype, w_dtype=torch.float32))


def test_without_parameters_and_a_row_far_from_zero():
    x, _, _, dy = _inputs(12, 300, torch.float32)
    x[3] += 1.0e4  # E[x^2] - mean^2 would lose this row's variance
    x[4] = 2.5     # a constant row: variance zero
    _check(x, None, None, dy)


def test_strided_rows_and_leading_axes():
    x, w, b, dy = _inputs(24, 200, torch.bfloat16)
    want = ref.layer_norm(x, w, b, dy)
    buf = torch.full((24, 333), float("nan"), dtype=torch.bfloat16, device="cuda")
    buf[:, 100:300] = x.cuda()  # rows 200 bytes off a 16-byte boundary's multiple, NaN on both sides
    y, mean, rstd = ops.layer_norm(buf[:, 100:300], w.cuda(), b.cuda())
    ref.close(y, want["y"][0], want["y"][1])
    y3, mean3, _ = ops.layer_norm(x.cuda().reshape(2, 3, 4, 200), w.cuda(), b.cuda())
    assert y3.shape == (2, 3, 4, 200) and mean3.shape == (2, 3, 4) and torch.equal(y3.reshape(24, 200), y)
    dyt = dy.cuda().t().contiguous().t()  # columns contiguous: no row view
    dx, dw, db = ops.layer_norm_bwd(dyt, buf[:, 100:300], w.cuda(), mean, rstd)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        ref.close(got, want[name][0], want[name][1], name)


def test_no_rows():
    w = torch.ones(16, device="cuda")
    x = torch.empty(0, 16, device="cuda")
    y, mean, rstd = ops.layer_norm(x, w, w)
    dx, dw, db = ops.layer_norm_bwd(x, x, w, mean, rstd)
    assert y.shape == (0, 16) and dx.shape == (0, 16) and mean.numel() == 0
    assert float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0


def test_a_bad_row_stays_its_own():
    x, w, b, dy = (t.cuda() for t in _inputs(9, 130, torch.float32))
    y0, *_ = ops.layer_norm(x, w, b)
    x[4, 7] = float("inf")
    y1, *_ = ops.layer_norm(x, w, b)
    keep = [i for i in range(9) if i != 4]
    assert torch.equal(y0[keep], y1[keep]) and bool(torch.isnan(y1[4]).any())


def test_gradients_repeat_bit_for_bit():
    x, w, b, dy = (t.cuda() for t in _inputs(3000, 400, torch.float32))
    _, mean, rstd = ops.layer_norm(x, w, b)
    first = ops.layer_norm_bwd(dy, x, w, mean, rstd)
    for _ in range(3):
        again = ops.layer_norm_bwd(dy, x, w, mean, rstd)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_backward_against_differences():
    x, w, b, dy = _inputs(4, 48, torch.float32, seed=3)
    want = ref.layer_norm(x, w, b, dy)
    d = torch.randn(4, 48, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    step = 1e-6
    f = lambda z: (ref.layer_norm(z, w, b, dy)["y"][0] * dy.double()).sum()
    slope = (f(x.double() + step * d) - f(x.double() - step * d)) / (2 * step)
    assert abs(float(slope) - float((want["dx"][0] * d).sum())) <= 1e-6 * float(want["dx"][0].abs().sum())

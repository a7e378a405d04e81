"""The orthogonalised update against its 64-bit definition."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _matrix(B, m, n, dtype, seed=0, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    r = max(1, min(m, n) // 8)
    g = torch.randn(B, m, n, generator=gen) + torch.randn(B, m, r, generator=gen) @ torch.randn(B, r, n, generator=gen)
    return (g * scale).to(dtype)


def _check(g, steps=5, coeffs=ops.NS_COEFFS):
    want = ref.orthogonalize(g, steps, coeffs)
    plain = ref.orthogonalize(g.float(), steps, coeffs, dtype=torch.float32).double()
    got = ops.orthogonalize(g.cuda(), steps=steps, coeffs=coeffs).double().cpu()
    assert bool(torch.isfinite(got).all())
    # 22-bit operands against fp32's 24: four times fp32's own error, and one rounding to the type
    err, own = float((got - want).norm() / want.norm()), float((plain - want).norm() / want.norm())
    assert err <= 4 * own + 4 * ref.U + ref.HALF[g.dtype], (err, own)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,m,n", [(1, 1, 1), (1, 1, 9), (2, 5, 3), (1, 64, 64), (3, 65, 64), (2, 100, 130), (1, 128, 128), (1, 400, 200),
                                   (2, 129, 257), (1, 40, 2100), (1, 1100, 300)])
def test_against_definition(B, m, n, dtype):
    _check(_matrix(B, m, n, dtype))


def test_sizes_of_every_tile():
    _check(_matrix(1, 2200, 2304, torch.float32))  # 128-wide tiles
    _check(_matrix(14, 600, 640, torch.float32))


def test_largest_tiles():
    g = _matrix(3, 4104, 4200, torch.bfloat16).cuda()
    got = ops.orthogonalize(g)
    for k in range(3):
        want = ref.orthogonalize(g[k].double(), 5, ops.NS_COEFFS)
        plain = ref.orthogonalize(g[k].float(), 5, ops.NS_COEFFS, dtype=torch.float32).double()
        err, own = float((got[k].double() - want).norm() / want.norm()), float((plain - want).norm() / want.norm())
        assert err <= 4 * own + 4 * ref.U + ref.HALF[g.dtype], (err, own)


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_steps_and_other_coefficients(steps):
    g = _matrix(2, 72, 96, torch.float32)
    _check(g, steps=steps)
    _check(g, steps=steps, coeffs=(2.0, -1.5, 0.5))


def test_singular_values_go_to_one():
    g = torch.randn(200, 320, generator=torch.Generator().manual_seed(1)).cuda()
    s = torch.linalg.svdvals(ops.orthogonalize(g, steps=12, coeffs=(2.0, -1.5, 0.5)).double().cpu())
    assert float((s - 1).abs().max()) < 1e-5  # (the cubic-order iteration has converged: sums of 320 terms of 2^-24 remain)


def test_strides_and_in_place():
    g = _matrix(2, 48, 72, torch.float32)
    want = ops.orthogonalize(g.cuda())
    buf = torch.full((2, 50, 101), float("nan"), device="cuda")
    buf[:, 1:49, 9:81] = g.cuda()
    assert torch.equal(ops.orthogonalize(buf[:, 1:49, 9:81]), want)
    assert torch.equal(ops.orthogonalize(g.cuda().transpose(1, 2).contiguous().transpose(1, 2)), want)
    x = g.cuda()
    assert ops.orthogonalize(x, out=x) is x and torch.equal(x, want)
    assert torch.equal(ops.orthogonalize(g.cuda().reshape(1, 2, 48, 72))[0], want)
    assert torch.equal(ops.orthogonalize(g[1].cuda()), want[1])
    assert torch.equal(ops.orthogonalize(g[:1].expand(3, 48, 72).cuda())[2], want[0])


def test_scales_zeros_and_what_is_not_finite():
    g = _matrix(1, 40, 56, torch.float32)
    base = ops.orthogonalize(g.cuda())
    for scale in (2.0 ** 60, 2.0 ** -8):  # squares of the first leave fp32's range
        got = ops.orthogonalize(g.cuda() * scale)
        assert float((got - base).norm() / base.norm()) < 1e-4  # (eps = 1e-7 beside a norm of 1e-2 in the second)
    assert float(ops.orthogonalize(torch.zeros(2, 24, 40, device="cuda")).abs().max()) == 0
    two = torch.cat([g, g]).cuda()
    two[0, 3, 5] = float("nan")
    got = ops.orthogonalize(two)
    assert bool(torch.isnan(got[0]).any()) and torch.equal(got[1], base[0])
    assert ops.orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert ops.orthogonalize(torch.empty(3, 0, 5, device="cuda")).shape == (3, 0, 5)


@pytest.mark.parametrize("m,n", [(48, 72), (200, 144)])
def test_result_over_a_part_of_the_input(m, n):
    # out starts one matrix further on in the same buffer (small matrices: one workgroup each; larger ones: several launches)
    g = _matrix(4, m, n, torch.float32)
    want = ops.orthogonalize(g[:3].cuda())
    buf = g.cuda()
    assert torch.equal(ops.orthogonalize(buf[:3], out=buf[1:]), want)
    buf = g.cuda()
    rows = buf.reshape(4 * m, n)[::2].reshape(2, m, n)  # every second row of what out begins with
    want = ops.orthogonalize(rows.clone())
    view = buf.reshape(4 * m, n).as_strided((2, m, n), (2 * m * n, 2 * n, 1))
    assert torch.equal(ops.orthogonalize(view, out=buf[:2]), want)

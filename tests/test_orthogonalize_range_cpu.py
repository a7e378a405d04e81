"""Which coefficients of the orthogonalised update the fp16 planes can hold, worked out on the host."""
import pytest
import torch

from cradle_vae_amd import hip, ops

# accepted by a bound on s and b s^2 + c s^4 alone, though S = s^2 leaves fp16's range on its way
OUTGROW = [((4.5, -0.25, 0.0), 2), ((1.5, 0.0, 0.0), 5), ((5.0, -0.3, 0.0), 2)]


def _planes(s, coeffs, steps):
    """The iteration on a 1 x 1 matrix with everything held times 2^12 as a sum of two fp16 numbers."""
    def hold(v):
        v = torch.tensor(v * 4096.0, dtype=torch.float32)
        hi = v.half()
        return float(hi.float() + (v - hi.float()).half().float()) / 4096.0 if bool(torch.isfinite(hi)) else float("inf")

    a, b, c = coeffs
    x = hold(s)
    for _ in range(steps):
        S = hold(x * x)
        B = hold(b * S + c * S * S)
        x = a * x + B * x
        if _ + 1 < steps:
            x = hold(x)
    return x


@pytest.mark.parametrize("coeffs,steps", OUTGROW)
def test_products_that_leave_the_planes_range_are_refused(coeffs, steps):
    exact = 1.0
    for _ in range(steps):
        exact = coeffs[0] * exact + coeffs[1] * exact ** 3 + coeffs[2] * exact ** 5
    held = _planes(1.0, coeffs, steps)
    assert abs(exact) < 8 and ops._ns_bound(coeffs, steps) < 8
    assert not abs(held - exact) < 1e-2  # infinity or NaN where the result is an ordinary number
    assert not ops._ns_holds(coeffs, steps)


def test_ordinary_coefficients_are_accepted():
    for coeffs, steps in ((ops.NS_COEFFS, 5), (ops.NS_COEFFS, 64), ((2.0, -1.5, 0.5), 64), ((1.5, -0.5, 0.0), 64), ((4.5, -0.25, 0.0), 1),
                          ((1.9, 0.0, 0.0), 3)):
        assert ops._ns_holds(coeffs, steps)


def test_what_the_bound_lets_through_stays_in_the_planes():
    gen = torch.Generator().manual_seed(0)
    seen = 0
    for _ in range(400):
        coeffs = tuple((torch.randn(3, generator=gen) * torch.tensor([3.0, 3.0, 1.5])).tolist())
        steps = int(torch.randint(1, 5, (1,), generator=gen))
        if not ops._ns_holds(coeffs, steps):
            continue
        seen += 1
        for s in torch.linspace(0, 1, 17).tolist():
            want = s
            for _k in range(steps):
                want = coeffs[0] * want + coeffs[1] * want ** 3 + coeffs[2] * want ** 5
            # each step holds three numbers to 2^-22 of at most 16 (2^-36 below) and multiplies what it got by at most
            # |a| + 3 |b| s^2 + 5 |c| s^4 <= 400: far below the size of an overflow, which is what is looked for
            assert abs(_planes(s, coeffs, steps) - want) < 1.0, (coeffs, steps, s)
    assert seen > 20


def test_the_call_is_refused_before_anything_runs(monkeypatch):
    class OnGpu:  # the checks come first: nothing of the tensor but its description is looked at
        is_cuda, dtype, device, shape = True, torch.float32, "cuda:0", (3, 4)

        def dim(self):
            return 2

    for coeffs, steps in OUTGROW:
        with pytest.raises(hip.CradleHipError, match="between steps"):
            ops.orthogonalize(OnGpu(), steps=steps, coeffs=coeffs)

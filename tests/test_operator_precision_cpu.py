"""What the number formats of the hidden-layer operators cost, emulated in 64 bits: the limits of the GPU tests tell the
formats that are used from ones that are a plane short."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref

FP32_NORMWISE = 16 * ref.U      # a product, a gate and a product of fp32 tensors, beside the norm of the result
ORTH_ROUNDINGS = {torch.bfloat16: 1.1, torch.float16: 1.05, torch.float32: 1.0}  # errors beside the final rounding's alone


def planes(t, dtype, n):
    """t as the first n planes of dtype numbers."""
    out, rest = [], t.clone()
    for _ in range(n):
        p = rest.to(dtype).to(t.dtype)
        out.append(p)
        rest = rest - p
    return out


def split_product(a, b, n):
    """a b^T from n bf16 planes of each: the products of order below n."""
    pa, pb = planes(a, torch.bfloat16, n), planes(b, torch.bfloat16, n)
    return sum(pa[i] @ pb[j].t() for i in range(n) for j in range(n - i))


@pytest.mark.parametrize("M,K,N", [(257, 200, 600), (96, 3001, 80), (40, 33, 64)])
def test_a_lost_plane_of_an_fp32_product_is_beyond_the_limit(M, K, N):
    gen = torch.Generator().manual_seed(K)
    a, b = torch.randn(M, K, generator=gen).double(), torch.randn(N, K, generator=gen).double() * K ** -0.5
    want = a @ b.t()
    err = [float((split_product(a, b, n) - want).norm() / want.norm()) for n in (2, 3)]
    assert err[0] > 2 * FP32_NORMWISE and err[1] < FP32_NORMWISE / 8, err


def orth_matrices(m, n, dtype):
    """Full rank, all singular values equal, a few directions that stand out, decaying spectra, low rank, few equal values."""
    gen = torch.Generator().manual_seed(m)
    r = lambda *s: torch.randn(*s, generator=gen)
    k = min(m, n)
    u, v = torch.linalg.qr(r(m, k))[0], torch.linalg.qr(r(n, k))[0]
    few = torch.full((k,), 1e-6)
    few[:max(1, k // 16)] = 1.0
    yield "full", (r(m, n) * 1e-2).to(dtype)
    yield "equal", (u @ v.t()).to(dtype)
    yield "spiked", ((r(m, n) + 4 * r(m, 4) @ r(4, n)) * 1e-2).to(dtype)
    yield "decaying", (u * torch.logspace(0, -3, k) @ v.t()).to(dtype)
    yield "decaying a little", (u * torch.logspace(0, -1, k) @ v.t()).to(dtype)
    yield "low rank", (r(m, max(1, k // 8)) @ r(max(1, k // 8), n) * 1e-2).to(dtype)
    yield "rank one", (r(m, 1) @ r(1, n)).to(dtype)
    yield "few equal", (u * few @ v.t()).to(dtype)


def orth_limit(g, want, own):
    """-> what the result in g's type may be off by, beside the norm; own: a plain fp32 evaluation's error."""
    rounding = float((want.to(g.dtype).double() - want).norm() / want.norm())
    return ORTH_ROUNDINGS[g.dtype] * rounding + 4 * own + 4 * ref.U


def _held(t, n):  # times 2^12 in n fp16 planes
    return sum(planes(t * 4096.0, torch.float16, n)) / 4096.0


def one_plane(k, m, n, steps):
    """The steps of a bf16 update whose products take one plane."""
    return k < 2 and k + 3 < steps <= 8 and min(m, n) >= 128


def _iterate(g, rule, steps):
    a, b, c = ops.NS_COEFFS
    x = g.double()
    flip = x.shape[0] > x.shape[1]
    x = (x.t() if flip else x) / (x.norm() + 1e-7)
    x = _held(x, 2)
    for k in range(steps):
        n = 1 if rule(k, *g.shape, steps) else 2
        xn = planes(x * 4096.0, torch.float16, 1)[0] / 4096.0 if n == 1 else x
        s = _held(xn @ xn.t(), n)
        q = _held(b * s + c * s @ s, n)
        x = a * x + q @ xn
        if k + 1 < steps:
            x = _held(x, 2)
    return x.t() if flip else x


# one plane in all but the last two steps: where every singular value is large early on (few of them, or all equal), or the
# iteration is long, its 11 bits show
@pytest.mark.parametrize("m,n,steps,short", [(769, 4, 5, True), (400, 32, 5, True), (150, 420, 5, False), (320, 900, 5, True), (256, 256, 8, True),
                                             (320, 200, 12, True), (140, 140, 4, False)])
def test_planes_of_the_orthogonalised_update(m, n, steps, short):
    worst = 0.0
    for kind, g in orth_matrices(m, n, torch.bfloat16):
        want = ref.orthogonalize(g, steps, ops.NS_COEFFS)
        plain = ref.orthogonalize(g.float(), steps, ops.NS_COEFFS, dtype=torch.float32).double()
        own = float((plain - want).norm() / want.norm())
        off = lambda x: float((x.to(g.dtype).double() - want).norm() / want.norm())
        limit = orth_limit(g, want, own)
        assert off(_iterate(g, one_plane, steps)) <= limit, kind
        worst = max(worst, off(_iterate(g, lambda k, m, n, steps: k + 2 < steps, steps)) / limit)
    assert not short or worst > 1.15, worst  # told apart

"""What the number formats of the hidden-layer operators cost, emulated in 64 bits: the limits of the GPU tests tell the
formats that are used from ones that are a plane short."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref

FP32_NORMWISE = 16 * ref.U      # a product, a gate and a product of fp32 tensors, beside the norm of the result
ORTH_ROUNDINGS = {torch.bfloat16: 1.3, torch.float16: 1.05, torch.float32: 1.0}  # errors beside the final rounding's alone


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
    """Full rank, a few directions that stand out, a decaying spectrum, low rank."""
    gen = torch.Generator().manual_seed(m)
    r = lambda *s: torch.randn(*s, generator=gen)
    k = min(m, n)
    u, v = torch.linalg.qr(r(m, k))[0], torch.linalg.qr(r(n, k))[0]
    yield "full", (r(m, n) * 1e-2).to(dtype)
    yield "spiked", ((r(m, n) + 4 * r(m, 4) @ r(4, n)) * 1e-2).to(dtype)
    yield "decaying", (u * torch.logspace(0, -3, k) @ v.t()).to(dtype)
    yield "low rank", (r(m, k // 8) @ r(k // 8, n) * 1e-2).to(dtype)


def orth_limit(g, want, own):
    """-> what the result in g's type may be off by, beside the norm; own: a plain fp32 evaluation's error."""
    rounding = float((want.to(g.dtype).double() - want).norm() / want.norm())
    return ORTH_ROUNDINGS[g.dtype] * rounding + 4 * own + 4 * ref.U


def _held(t, n):  # times 2^12 in n fp16 planes
    return sum(planes(t * 4096.0, torch.float16, n)) / 4096.0


def _iterate(g, one_plane_steps, steps=5):
    a, b, c = ops.NS_COEFFS
    x = g.double()
    flip = x.shape[0] > x.shape[1]
    x = (x.t() if flip else x) / (x.norm() + 1e-7)
    x = _held(x, 2)
    for k in range(steps):
        n = 1 if k < one_plane_steps else 2
        xn = planes(x * 4096.0, torch.float16, 1)[0] / 4096.0 if n == 1 else x
        s = _held(xn @ xn.t(), n)
        q = _held(b * s + c * s @ s, n)
        x = a * x + q @ xn
        if k + 1 < steps:
            x = _held(x, 2)
    return x.t() if flip else x


@pytest.mark.parametrize("m,n", [(150, 420), (320, 200)])
def test_planes_of_the_orthogonalised_update(m, n):
    worst = {}
    for kind, g in orth_matrices(m, n, torch.bfloat16):
        want = ref.orthogonalize(g, 5, ops.NS_COEFFS)
        plain = ref.orthogonalize(g.float(), 5, ops.NS_COEFFS, dtype=torch.float32).double()
        own = float((plain - want).norm() / want.norm())
        rounding = float((want.to(g.dtype).double() - want).norm() / want.norm())
        off = lambda x: float((x.to(g.dtype).double() - want).norm() / want.norm())
        used, short = off(_iterate(g, 3)), off(_iterate(g, 5))
        worst[kind] = (round(used / rounding, 3), round(short / rounding, 3))
        assert used <= orth_limit(g, want, own), (kind, used / rounding)
    assert max(s for _, s in worst.values()) > ORTH_ROUNDINGS[torch.bfloat16], worst  # one plane throughout is told apart

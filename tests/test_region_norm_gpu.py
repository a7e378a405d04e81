"""The squared gradient norm over the regions of the arena: the same for every cut of it."""
import ctypes
import math

import pytest
import torch

from cradle_vae_amd import hip

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _arr(vals):
    return (ctypes.c_int64 * len(vals))(*vals)


def _sums(g, cuts, pairs):
    lib, n = hip.load(), len(cuts) - 1
    ws = torch.zeros(lib.cradle_adam_regions_workspace_floats(), device=DEV)
    out = torch.full((2 * n + 1 if pairs else n + 1,), -7.0, device=DEV)
    f = lib.cradle_grad_region_sumsq_pairs if pairs else lib.cradle_grad_region_sumsq
    off, ln = _arr(cuts[:-1]), _arr([b - a for a, b in zip(cuts[:-1], cuts[1:])])
    hip.check(f(g.data_ptr(), off, ln, n, n, out.data_ptr(), ws.data_ptr(), hip.stream()), "region_sumsq")
    torch.cuda.synchronize()
    assert float(out[-1]) == -7.0  # nothing behind the last region's
    return out[:-1]


N = 35136
CUTS = [[0, N], [0, 64, N], [0, 8000, 8004, 20000, N], list(range(0, N, 1024)) + [N], [0] + [4 * k * k for k in range(1, 63)] + [N]]


@pytest.mark.parametrize("seed", range(4))
def test_the_norm_does_not_depend_on_the_cut(seed):
    gen = torch.Generator().manual_seed(seed)
    g = (torch.randn(N, generator=gen) * torch.exp(3 * torch.randn(N, generator=gen))).to(DEV)
    want = float((g.double() ** 2).sum())
    lib, norms = hip.load(), []
    for cuts in CUTS:
        one, two = _sums(g, cuts, False), _sums(g, cuts, True)
        assert torch.equal(one, two[0::2])
        tot = float(two.double().sum())
        # a pair is off by at most half a step of its lo number, 2^-48 of the sum; fp64's own sums by far less
        assert abs(tot - want) <= 2.0 ** -46 * want
        # what the update makes of it
        p, m, v = (torch.zeros(N, device=DEV) for _ in range(3))
        norm_out = torch.zeros(2, device=DEV)
        hip.check(lib.cradle_adam_step_regions(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), _arr([0]), _arr([N]), 1, two.data_ptr(),
                                               two.numel(), 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, 1.0, norm_out.data_ptr(), None,
                                               hip.stream()), "adam_step_regions")
        torch.cuda.synchronize()
        assert float(norm_out[1]) == 0
        norms.append((float(norm_out[0]), p))
    for norm, p in norms:
        assert norm == norms[0][0] and torch.equal(p, norms[0][1])
    assert abs(norms[0][0] - math.sqrt(want)) <= 2.0 ** -23 * math.sqrt(want)


def test_what_is_not_finite_and_bad_counts():
    g = torch.ones(256, device=DEV)
    lib = hip.load()
    for bad in (float("nan"), float("inf"), 1e30):  # (the square of the last is beyond fp32)
        g[100] = bad
        two = _sums(g, [0, 128, 256], True)
        p, m, v, norm_out = torch.zeros(256, device=DEV), torch.zeros(256, device=DEV), torch.zeros(256, device=DEV), torch.zeros(2, device=DEV)
        call = lambda n: lib.cradle_adam_step_regions(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), _arr([0]), _arr([256]), 1,
                                                      two.data_ptr(), n, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, 1.0, norm_out.data_ptr(), None,
                                                      hip.stream())
        hip.check(call(4), "adam_step_regions")
        torch.cuda.synchronize()
        assert float(norm_out[1]) == 1 and not bool(p.any()) and not bool(m.any())
        assert call(0) == 1 and call(129) == 1

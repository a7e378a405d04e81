"""The orthogonalised update at the edges of its range and precision."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref
from tests.test_orthogonalize_gpu import DTYPES, _matrix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(1, 1), (48, 72), (200, 144)])
@pytest.mark.parametrize("coeffs,steps", [((4.3, -0.4, 0.0), 2), ((7.9, 0.0, 0.0), 1), ((1.98, 0.0, 0.0), 3)])
def test_coefficients_just_inside_the_range(m, n, coeffs, steps):
    # S reaches 15.2 in the second step of the first, X 7.9 and 7.8 at the end of the others
    assert ops._ns_holds(coeffs, steps)
    g = torch.ones(2, m, n) + 1e-3 * _matrix(2, m, n, torch.float32)  # one singular value near the norm
    want = ref.orthogonalize(g, steps, coeffs)
    got = ops.orthogonalize(g.cuda(), steps=steps, coeffs=coeffs).double().cpu()
    # X, S and B are off by 2^-21 of themselves (22 bits, products without lo lo).  At s = 3.9 the last step of the first is
    # 16.8 - 23.7 = -7.0: B X is off by 2 * 23.7, a X by 16.8, and the step before by 3.9 times the slope 13.9, all 2^-21 and
    # beside 7.0: 17 of them; twice that
    assert float((got - want).norm() / want.norm()) <= 34 * 2.0 ** -21

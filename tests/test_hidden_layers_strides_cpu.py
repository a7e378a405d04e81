"""Leading dimensions that the hidden layers' wrappers hand to the kernels."""
import torch

from cradle_vae_amd import ops


def test_a_single_row_has_its_own_length():
    t = torch.zeros(3, 50)
    assert ops._ld(t[:, :8]) == 50 and ops._ld(t[1:2, :8]) == 8 and ops._ld(t[:0, :8]) == 8
    wide = torch.zeros(1).as_strided((1, 1), (1 << 23, 1))
    assert ops._ld(wide) == 1

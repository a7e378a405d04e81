"""Leading dimensions that the hidden layers' wrappers hand to the kernels."""
import ctypes

import torch

from cradle_vae_amd import hip, ops
from tests.test_hidden_layers_cpu import _desc, _refused


def test_a_single_row_has_its_own_length():
    t = torch.zeros(3, 50)
    assert ops._ld(t[:, :8]) == 50 and ops._ld(t[1:2, :8]) == 8 and ops._ld(t[:0, :8]) == 8
    wide = torch.zeros(1).as_strided((1, 1), (1 << 23, 1))
    assert ops._ld(wide) == 1


def test_misaligned_saved_buffers_are_refused_by_both_passes():
    lib = hip.load()
    for run in (lib.cradle_gated_mlp_fwd, lib.cradle_gated_mlp_bwd):
        for kw in (dict(saved_gu=4100, saved_h=8192), dict(saved_gu=4096, saved_h=8194)):
            _refused(run(ctypes.byref(_desc(**kw)), None), "16-byte")

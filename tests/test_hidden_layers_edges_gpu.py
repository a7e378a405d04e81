"""Calls of the hidden layers' functions and the optimiser that their documentation allows, beside the ordinary ones."""
import pytest
import torch
from torch.autograd import forward_ad

from cradle_vae_amd import functional as F_hip
from tests.test_hidden_layers_gpu import DEV, _params

pytestmark = pytest.mark.gpu


def test_forward_mode_is_refused():
    p = {k: v.to(DEV) for k, v in _params().items()}
    with forward_ad.dual_level():
        x = forward_ad.make_dual(p["x"], torch.ones_like(p["x"]))
        w = forward_ad.make_dual(p["w_out"], torch.ones_like(p["w_out"]))
        for call in (lambda: F_hip.layer_norm(x, p["w"], p["b"]), lambda: F_hip.gated_mlp(x, p["w_in"], p["w_out"]),
                     lambda: F_hip.gated_mlp(p["x"], p["w_in"], w)):
            with pytest.raises(NotImplementedError):
                call()
        assert bool(torch.isfinite(F_hip.layer_norm(p["x"], p["w"], p["b"])).all())

"""Calls of the hidden layers' functions and the optimiser that their documentation allows, beside the ordinary ones."""
import pytest
import torch
from torch.autograd import forward_ad

from cradle_vae_amd import functional as F_hip
from cradle_vae_amd.mlp import GaussianLikelihoodResidualMLP
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


@pytest.mark.parametrize("block", ["residual", "gated"])
def test_the_rest_of_a_head_from_its_first_layers_output(block):
    torch.manual_seed(0)
    m = GaussianLikelihoodResidualMLP(16, 6, 3, 16, block=block).to(DEV)
    h = torch.randn(2, 5, 16, device=DEV)
    lin = m.mlp.linears()[0]
    first = F_hip.linear(h.reshape(-1, 16), lin.weight, lin.bias, act=True)
    want = m(h)
    for got in (m.forward_from_hidden(first.reshape(2, 5, 16)), m.forward_from_hidden(first.reshape(2, 5, 16), True)):
        assert torch.equal(got.mean, want.mean) and torch.equal(got.stddev, want.stddev)
    got = m.forward_from_hidden(h, first_layer_done=False)
    again = m.forward_from_hidden(F_hip.linear(h, lin.weight, lin.bias, act=True, residual=h))
    assert torch.equal(got.mean, again.mean) and torch.equal(got.stddev, again.stddev)

"""Dual numbers (forward-mode differentiation) through the hidden layers' functions: refused, never read without their
tangent.  The kernels' wrappers are stood in for: only the way to them is looked at."""
import pytest
import torch
from torch.autograd import forward_ad

from cradle_vae_amd import functional as F_hip
from cradle_vae_amd import ops


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    monkeypatch.setattr(ops, "layer_norm", lambda x, w=None, b=None, eps=1e-5: (torch.zeros_like(x), x.sum(-1), x.sum(-1)))

    def gated(x, w_in, w_out, b_in=None, b_out=None, act="silu", residual=None, save=False):
        y = torch.zeros(x.shape[0], w_out.shape[0])
        return (y, (torch.zeros(1), torch.zeros(1))) if save else y

    monkeypatch.setattr(ops, "gated_mlp", gated)


LN = [torch.ones(3, 4), torch.ones(4), torch.ones(4)]
GATED = [torch.ones(3, 4), torch.ones(10, 4), torch.ones(4, 5), torch.ones(10), torch.ones(4), torch.ones(3, 4)]


def _gated(x, w_in, w_out, b_in, b_out, residual):
    return F_hip.gated_mlp(x, w_in, w_out, b_in, b_out, residual=residual)


@pytest.mark.parametrize("call,args", [(F_hip.layer_norm, LN), (_gated, GATED)])
def test_a_tangent_is_refused_in_every_place(call, args):
    with forward_ad.dual_level():
        call(*args)  # nothing to differentiate: an ordinary call
        for i, t in enumerate(args):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if k == i else a for k, a in enumerate(args)]
            with pytest.raises(NotImplementedError):
                call(*dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call(*dual)


@pytest.mark.parametrize("call,args", [(F_hip.layer_norm, LN), (_gated, GATED)])
def test_what_ran_before_takes_its_way(call, args):
    assert call(*args).grad_fn is None
    leaf = args[1].clone().requires_grad_()
    assert call(args[0], leaf, *args[2:]).grad_fn is not None
    with torch.no_grad():
        assert call(args[0], leaf, *args[2:]).grad_fn is None

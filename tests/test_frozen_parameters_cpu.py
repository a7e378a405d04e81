"""Parameters that do not train stay where they are, whichever optimiser runs."""
import torch

from cradle_vae_amd.optim import split_parameters
from cradle_vae_amd.trainer import TrainStep


class _Loss(torch.nn.Module):
    """As much of a loss module as a modular training step asks for."""

    def __init__(self):
        super().__init__()
        self.guide = torch.nn.Module()
        self.trained = torch.nn.Parameter(torch.ones(3))
        self.frozen = torch.nn.Parameter(torch.ones(3), requires_grad=False)

    def _use_fused(self, _):
        return False

    def loss(self, **kw):
        return (self.trained ** 2).sum(), {}


def test_a_frozen_parameter_with_an_old_gradient(monkeypatch):
    lm = _Loss()
    lm.frozen.grad = torch.ones(3)  # from before it was frozen
    st = TrainStep(lm, lr=0.1, weight_decay=0.5)
    monkeypatch.setattr(st, "draw_noise", lambda *a: (None, None))
    batch = dict.fromkeys(("X", "D", "D_obs_counts", "qc", "qc_obs_counts", "cfX", "library_size"), torch.zeros(1))
    st(batch, n_particles=1)
    assert torch.equal(lm.frozen, torch.ones(3)) and not torch.equal(lm.trained, torch.ones(3))
    assert sum(len(g["params"]) for g in st.optimizer.param_groups) == 1
    hidden, rest = split_parameters(lm)
    assert len(hidden) + len(rest) == 1

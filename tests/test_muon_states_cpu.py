"""The optimiser's states beside 16-bit parameters, in the group that needs no kernel."""
import copy

import pytest
import torch

from cradle_vae_amd.optim import Muon


def _run(dtype, grads, opt_kw, reload_at=None):
    p = torch.nn.Parameter(torch.full((4,), 0.5, dtype=dtype))
    opt = Muon([], [p], **opt_kw)
    for k, g in enumerate(grads):
        if k == reload_at:
            saved = copy.deepcopy(opt.state_dict())
            opt = Muon([], [p], **opt_kw)
            opt.load_state_dict(saved)
        p.grad = g.to(dtype)
        opt.step()
    return p, opt


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_gradient_of_zero_moves_nothing(dtype):
    p, _ = _run(dtype, [torch.zeros(4)] * 3, dict(lr=1e-2, weight_decay=0.0))
    assert torch.equal(p, torch.full((4,), 0.5, dtype=dtype))  # (eps = 1e-8 is zero in fp16: 0 / 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_second_moments_decay(dtype):
    # one gradient of 1, then 600 of 2^-12: the second moment follows 0.999^n (0.999 x rounds back to x in bf16; 2^-24 is
    # lost in fp16)
    grads = [torch.ones(4)] + [torch.full((4,), 2.0 ** -12)] * 600
    _, opt = _run(dtype, grads, dict(lr=1e-4, weight_decay=0.0))
    (st,) = opt.state.values()
    want = 0.001 * 0.999 ** 600 + 2.0 ** -24 * (1 - 0.999 ** 600)
    assert st["exp_avg_sq"].dtype == torch.float32 and st["exp_avg"].dtype == torch.float32
    # 600 steps of two roundings
    assert bool(((st["exp_avg_sq"].double() - want).abs() <= want * 1200 * 2.0 ** -24).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_survive_a_checkpoint(dtype):
    grads = [torch.randn(4, generator=torch.Generator().manual_seed(k)) for k in range(6)]
    a, oa = _run(dtype, grads, dict(lr=1e-2))
    b, ob = _run(dtype, grads, dict(lr=1e-2), reload_at=3)
    assert torch.equal(a, b)
    for x, y in zip(oa.state.values(), ob.state.values()):
        assert x["step"] == y["step"] and torch.equal(x["exp_avg"], y["exp_avg"]) and torch.equal(x["exp_avg_sq"], y["exp_avg_sq"])


def test_fp32_parameters_keep_their_results():
    # the update of the fp32 group, step by step as it was
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(7))
    opt = Muon([], [p], lr=1e-2, weight_decay=1e-3)
    want, m, v = p.detach().clone(), torch.zeros(7), torch.zeros(7)
    for k in range(1, 5):
        p.grad = torch.randn(7)
        g = p.grad.add(want, alpha=1e-3)
        m.lerp_(g, 1 - 0.9)
        v.mul_(0.999).addcmul_(g, g, value=1 - 0.999)
        want.addcdiv_(m, (v.sqrt() / (1 - 0.999 ** k) ** 0.5).add_(1e-8), value=-1e-2 / (1 - 0.9 ** k))
        opt.step()
        assert torch.equal(p, want)

"""Calls of the hidden layers' functions and the optimiser that their documentation allows, beside the ordinary ones."""
import pytest
import torch
from torch.autograd import forward_ad

from cradle_vae_amd import functional as F_hip
from cradle_vae_amd import hip, ops
from cradle_vae_amd.mlp import GaussianLikelihoodResidualMLP
from cradle_vae_amd.optim import Muon
from tests import operator_reference as ref
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_hidden_matrices_of_every_type(dtype):
    gen = torch.Generator().manual_seed(0)
    ps = [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(DEV, dtype)) for s in ((32, 48), (32, 48), (150, 130))]
    opt = Muon(ps, lr=0.02, momentum=0.9, weight_decay=0.01)
    want, buf = [p.detach().double().cpu() for p in ps], [torch.zeros(p.shape).double() for p in ps]
    for _ in range(3):
        for i, p in enumerate(ps):
            p.grad = torch.randn(p.shape, generator=gen).to(DEV, dtype)
            g = p.grad.double().cpu()
            buf[i] = 0.9 * buf[i] + g
            want[i] = want[i] * (1 - 0.02 * 0.01) - 0.02 * 0.2 * max(p.shape) ** 0.5 * ref.orthogonalize(g + 0.9 * buf[i], 5, ops.NS_COEFFS)
        opt.step()
    for i, p in enumerate(ps):
        st = opt.state[p]["momentum"]
        # three roundings of sums of two terms; per step an update of rms 0.2 off by at most 2e-5 of its norm, and one
        # rounding of the parameter
        assert st.dtype == torch.float32 and float((st.double().cpu() - buf[i]).norm()) <= 6 * ref.U * float(buf[i].norm()) * 2
        off = 3 * 2e-5 * 0.02 * 0.2 * p.numel() ** 0.5 * 2 + 8 * ref.U * float(want[i].norm())
        off += 3 * ref.HALF[dtype] * float(want[i].norm()) * 1.1
        assert p.dtype == dtype and float((p.detach().double().cpu() - want[i]).norm()) <= off


def test_saved_buffers_that_are_not_what_the_forward_pass_made():
    p = {k: v.to(DEV) for k, v in _params().items()}
    x, w_in, w_out, dy = p["x"], p["w_in"], p["w_out"], p["dy"]
    _, (gu, h) = ops.gated_mlp(x, w_in, w_out, save=True)
    want = ops.gated_mlp_bwd(dy, x, w_in, w_out, (gu, h))
    # the right count of numbers in too small a memory, or of another type
    for bad in ((gu[:1].expand(gu.shape), h), (gu, h[:1].expand(h.shape)), (gu.half(), h), (gu.int(), h), (gu, h.char()),
                (torch.stack([gu, gu], 1)[:, 0], h), (gu[:-1], h), (gu, h[:-1]), (gu.cpu(), h)):
        with pytest.raises(hip.CradleHipError):
            ops.gated_mlp_bwd(dy, x, w_in, w_out, bad)
    assert all(torch.equal(a, b) for a, b in zip(want[:3], ops.gated_mlp_bwd(dy, x, w_in, w_out, (gu, h))[:3]))

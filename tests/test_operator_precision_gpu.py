"""Errors of the hidden-layer operators beside the norm of the result, at limits that a lost operand plane would pass
(test_operator_precision_cpu)."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref
from tests.test_gated_mlp_gpu import NAMES, _inputs
from tests.test_operator_precision_cpu import FP32_NORMWISE, orth_limit, orth_matrices

pytestmark = pytest.mark.gpu

# small tiles, alone and sharing a launch; sums split along K in the forward pass (2100), of the weights' gradients (3001), of both;
# a training step's rows at the widths of the demo and of the Norman configuration; extents that fill no tile; large tiles
SIZES = [(33, 100, 51, 100), (257, 200, 300, 96), (20, 48, 2100, 40), (3001, 40, 24, 48), (512, 512, 1024, 512), (1280, 128, 256, 128),
         (2560, 400, 800, 400), (700, 633, 611, 592), (4100, 264, 4104, 264)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,K,F,O", SIZES)
def test_fp32_block_beside_its_norm(M, K, F, O, act):
    # every sum is a random walk of one rounding per 16 terms (U / sqrt(3) of the partial sum): for 4104 terms 9 U, for the
    # products of a chain together under 16; the operands' planes and the gate add half a U each
    x, w_in, w_out, b_in, b_out, dy = (t.cuda() for t in _inputs(M, K, F, O, torch.float32, seed=M))
    d = [t.double().requires_grad_() for t in (x, w_in, w_out, b_in, b_out)]
    g, u = (d[0] @ d[1].t() + d[3]).chunk(2, 1)
    a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
    want = (a * u) @ d[2].t() + d[4]
    wants = torch.autograd.grad(want, d, dy.double())
    y, saved = ops.gated_mlp(x, w_in, w_out, b_in, b_out, act=act, save=True)
    got = dict(zip(NAMES, ops.gated_mlp_bwd(dy, x, w_in, w_out, saved, act=act, bias=True)), y=y,
               **{"y (inference)": ops.gated_mlp(x, w_in, w_out, b_in, b_out, act=act)},
               **{"y (a few rows)": ops.gated_mlp(x[:3], w_in, w_out, b_in, b_out, act=act)})
    want = want.detach()
    for name, w in (("y", want), ("y (inference)", want), ("y (a few rows)", want[:3]), *zip(NAMES, wants)):
        err = float((got[name].double() - w).norm() / w.norm())
        assert err <= FP32_NORMWISE, (name, err / ref.U)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,steps", [(40, 56, 5), (128, 128, 5), (150, 420, 5), (320, 200, 5), (300, 1100, 5), (513, 1001, 5), (1500, 400, 5),
                                       (769, 4, 5), (400, 32, 5), (5, 700, 5), (320, 900, 5), (140, 140, 4), (256, 256, 8), (320, 200, 12)])
def test_orthogonalised_update_beside_its_rounding(m, n, steps, dtype):
    for kind, g in orth_matrices(m, n, dtype):
        g = g.cuda()
        want = ref.orthogonalize(g, steps, ops.NS_COEFFS)
        plain = ref.orthogonalize(g.float(), steps, ops.NS_COEFFS, dtype=torch.float32).double()
        own = float((plain - want).norm() / want.norm())
        err = float((ops.orthogonalize(g, steps=steps).double() - want).norm() / want.norm())
        limit = orth_limit(g, want, own)
        assert err <= limit, (kind, err, limit, own)

"""The gated feed-forward block where its operands are staged in unusual ways: views inside wider buffers at sizes that
pad the hidden axis, long row strides, and the fp32 products' planes."""
import pytest
import torch

from cradle_vae_amd import ops
from tests import operator_reference as ref
from tests.test_gated_mlp_gpu import NAMES, _inputs

pytestmark = pytest.mark.gpu


def _in_nan(t, cols):
    """t as the leading columns of a buffer of NaN rows of ``cols`` numbers."""
    buf = torch.full((t.shape[0], cols), float("nan"), dtype=t.dtype, device="cuda")
    view = buf[:, :t.shape[1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weights_inside_wider_buffers_with_a_padded_hidden_axis(dtype):
    # 2048 rows pad 1032 hidden units to 1088, and w_out's rows of 1088 numbers are staged as they lie: what is beside
    # its 1032 columns belongs to nobody
    x, w_in, w_out, b_in, b_out, dy = _inputs(2048, 128, 1032, 64, dtype)
    want, _ = ref.gated_mlp(x, w_in, w_out, b_in, b_out, dy, "silu")
    gx, gi, go = _in_nan(x, 192), _in_nan(w_in, 192), _in_nan(w_out, 1088)
    gb, gc = b_in.cuda(), b_out.cuda()
    y0 = ops.gated_mlp(gx, gi, go, gb, gc)
    y, saved = ops.gated_mlp(gx, gi, go, gb, gc, save=True)
    assert torch.equal(y0, y) and torch.equal(y, ops.gated_mlp(x.cuda(), w_in.cuda(), w_out.cuda(), gb, gc))
    ref.close(y, want["y"][0], want["y"][1], "y")
    for name, got in zip(NAMES, ops.gated_mlp_bwd(_in_nan(dy, 128), gx, gi, go, saved, bias=True)):
        ref.close(got, want[name][0], want[name][1], name)

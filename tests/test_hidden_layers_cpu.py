"""Hidden-layer operators and the orthogonalising optimiser without a GPU: refusals at the C boundary, argument checks,
parameter split, configuration."""
import ctypes

import pytest
import torch

from cradle_vae_amd import functional as F_hip
from cradle_vae_amd import hip, ops
from cradle_vae_amd.mlp import GatedResidualMLP, get_likelihood_mlp
from cradle_vae_amd.optim import Muon, make_optimizer, split_parameters

F32, BF16, F16 = 0, 1, 2


def _refused(rc, text):
    assert rc == 1
    assert text in hip.load().cradle_last_error().decode(), hip.load().cradle_last_error().decode()


def test_layer_norm_refusals():
    lib = hip.load()
    x = 4096  # any non-null address: every call below is refused before it is looked at
    fwd = lambda dtype=F32, w=F32, rows=4, width=8, ld=8, px=x, py=x: lib.cradle_layer_norm_fwd(
        px, ld, None, None, dtype, w, 1e-5, py, ld, None, None, rows, width, None)
    _refused(fwd(dtype=3), "dtype 3")
    _refused(fwd(dtype=F32, w=BF16), "weights must be")
    _refused(fwd(dtype=F16, w=BF16), "weights must be")
    _refused(fwd(rows=-1), "rows=-1")
    _refused(fwd(width=0), "width=0")
    _refused(fwd(width=32769, ld=32769), "width=32769")
    _refused(fwd(ld=7), "leading dimension")
    _refused(fwd(px=None), "null pointer")
    assert fwd(rows=0, px=None, py=None) == 0  # nothing to do
    bwd = lambda rows=4, ws=None, n=0, dw=x, mean=x: lib.cradle_layer_norm_bwd(
        x, 8, x, 8, None, mean, x, F32, F32, x, 8, dw, None, ws, n, rows, 8, None)
    _refused(bwd(rows=0), "no rows")
    _refused(bwd(mean=None), "null pointer")
    _refused(bwd(), "workspace of")
    need = lib.cradle_layer_norm_workspace_floats(4, 8)
    _refused(bwd(ws=x, n=need - 1), "workspace of")
    _refused(bwd(ws=x + 4, n=need), "workspace of")
    assert lib.cradle_layer_norm_workspace_floats(0, 8) == 0 and lib.cradle_layer_norm_workspace_floats(4, 40000) == 0


def _desc(**kw):
    d = hip.GatedMlpDesc()
    d.rows, d.width, d.hidden, d.out_width, d.dtype, d.act = 300, 64, 96, 64, BF16, 0
    d.x = d.w_in = d.w_out = d.y = d.dy = 4096
    d.ld_x = d.ld_w_in = d.ld_y = d.ld_dy = d.ld_dx = d.ld_residual = 64
    d.ld_w_out = 96
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_gated_mlp_refusals():
    lib = hip.load()
    fwd = lambda **kw: lib.cradle_gated_mlp_fwd(ctypes.byref(_desc(**kw)), None)
    bwd = lambda **kw: lib.cradle_gated_mlp_bwd(ctypes.byref(_desc(**kw)), None)
    assert lib.cradle_gated_mlp_fwd(None, None) == 1
    for kw, text in ((dict(dtype=5), "dtype 5"), (dict(act=2), "activation 2"), (dict(rows=-1), "rows=-1"), (dict(width=0), "width=0"),
                     (dict(hidden=0), "hidden=0"), (dict(ld_x=63), "leading dimension"), (dict(ld_w_in=63), "leading dimension"),
                     (dict(ld_w_out=95), "leading dimension"), (dict(ld_x=1 << 22), "2^22"),
                     (dict(hidden=1 << 19, ld_w_out=1 << 19, ld_w_in=1 << 12), "2^30"), (dict(width=(1 << 20) + 1), "2^20"),
                     (dict(saved_gu=4096), "go together"), (dict(x=None), "null pointer"), (dict(y=None), "null pointer"),
                     (dict(ld_y=63), "leading dimension"), (dict(residual=4096, ld_residual=63), "leading dimension"), ({}, "workspace of")):
        _refused(fwd(**kw), text)
    saved = dict(saved_gu=4096, saved_h=8192)
    for kw, text in ((dict(rows=0, **saved), "rows=0"), ({}, "null pointer"), (dict(dy=None, **saved), "null pointer"),
                     (dict(saved_gu=4100, saved_h=8192), "16-byte"), (dict(ld_dy=63, **saved), "leading dimension"),
                     (dict(dx=4096, ld_dx=63, **saved), "leading dimension"), (saved, "workspace of")):
        _refused(bwd(**kw), text)
    assert fwd(rows=0) == 0
    d = _desc()
    need = lib.cradle_gated_mlp_workspace_bytes(ctypes.byref(d), 0)
    assert need > 0
    _refused(fwd(workspace=4096, workspace_bytes=need - 1), "workspace of")
    _refused(fwd(workspace=4104, workspace_bytes=need), "workspace of")
    assert lib.cradle_gated_mlp_workspace_bytes(ctypes.byref(_desc(act=9)), 0) == -1


def test_orthogonalize_refusals():
    lib = hip.load()
    call = lambda g=4096, ld=40, dtype=F32, batch=1, m=300, n=40, steps=5, ws=None, nb=0: lib.cradle_orthogonalize(
        g, ld, 0, 4096, ld, 0, dtype, batch, m, n, steps, 2.0, -1.5, 0.5, 1e-7, ws, nb, None)
    for kw, text in ((dict(batch=0), "batch=0"), (dict(batch=65536), "65535"), (dict(m=0), "m=0"), (dict(n=(1 << 17) + 1, ld=1 << 18), "2^17"),
                     (dict(dtype=7), "dtype 7"), (dict(g=None), "null pointer"), (dict(ld=39), "leading dimension"), (dict(steps=0), "steps=0"),
                     (dict(steps=65), "steps=65"), ({}, "workspace of")):
        _refused(call(**kw), text)
    need = lib.cradle_orthogonalize_workspace_bytes(1, 300, 40)
    assert need > 0 and lib.cradle_orthogonalize_workspace_bytes(0, 3, 3) == -1
    _refused(call(ws=4096, nb=need - 1), "workspace of")
    _refused(call(ws=4104, nb=need), "workspace of")
    assert lib.cradle_orthogonalize_workspace_bytes(3, 100, 128) == 0  # (lives in LDS)


def test_descriptor_layout_matches_the_library():
    lib = hip.load()
    assert hip.struct_layout(hip.GatedMlpDesc) == hip.library_struct_layout(lib, "cradle_gated_mlp_desc")


def test_cpu_tensors_are_refused():
    x, w = torch.ones(3, 4), torch.ones(4)
    for call in (lambda: ops.layer_norm(x, w, w), lambda: F_hip.layer_norm(x, w, w), lambda: ops.orthogonalize(x),
                 lambda: ops.gated_mlp(x, torch.ones(6, 4), torch.ones(4, 3)), lambda: ops.layer_norm_bwd(x, x, w, w[:3], w[:3])):
        with pytest.raises(hip.CradleHipError):
            call()


def test_iterations_that_leave_the_range_are_bounded_on_the_host():
    assert ops._ns_bound(ops.NS_COEFFS, 5) < 3
    assert ops._ns_bound((2.0, -1.5, 0.5), 20) < 1.1
    assert ops._ns_bound((3.0, 0.0, 0.0), 3) == pytest.approx(27.0)  # grows without end
    assert ops._ns_bound((9.0, 0.0, 5.0), 30) == float("inf")
    assert not ops._ns_bound((float("nan"), 0.0, 0.0), 2) < 8


def test_parameter_split_and_constructor_checks():
    m = get_likelihood_mlp("normal", 12, 4, 3, 8, block="gated")
    hidden, rest = split_parameters(m)
    names = {id(p): n for n, p in m.named_parameters()}
    assert sorted(names[id(p)] for p in hidden) == ["mlp.layers.1.w_in", "mlp.layers.1.w_out", "mlp.layers.2.w_in", "mlp.layers.2.w_out"]
    assert len(hidden) + len(rest) == len(list(m.parameters()))
    plain = get_likelihood_mlp("normal", 12, 4, 3, 8)
    hidden, _ = split_parameters(plain)
    names = {id(p): n for n, p in plain.named_parameters()}
    assert sorted(names[id(p)] for p in hidden) == ["mlp.layers.1.0.weight", "mlp.layers.2.0.weight"]
    with pytest.raises(ValueError, match="only matrices"):
        Muon([torch.nn.Parameter(torch.ones(3))])
    for bad in (dict(momentum=1.0), dict(lr=-1.0), dict(steps=0)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(torch.ones(3, 3))], **bad)
    with pytest.raises(ValueError, match="optimizer="):
        make_optimizer("sgd", plain, 1e-3, 0.0)
    with pytest.raises(ValueError, match="mlp_block"):
        get_likelihood_mlp("normal", 12, 4, 3, 8, block="swish")
    assert isinstance(get_likelihood_mlp("library_nb", 6, 20, 2, 8, block="gated").mlp, GatedResidualMLP)


def test_default_configuration_is_untouched():
    from tests import golden_io as gio
    from tests.test_host_logic_cpu import _module

    mod = _module(gio.load_elbo("tiny"))
    assert type(mod.configure_optimizers()) is torch.optim.Adam and mod.optimizer_name == "adam"
    assert not any("w_in" in k or "norm." in k for k in mod.state_dict())


def test_an_optimizer_that_a_scheduler_would_replace_is_refused():
    from cradle_vae_amd.lightning_module import PerturbationLightningModule

    kwargs = dict(loss_module=torch.nn.Linear(2, 2), lr=1e-3, n_treatments=2, n_qc=2)
    with pytest.raises(ValueError, match="use_scheduler"):
        PerturbationLightningModule(**kwargs, optimizer="muon", use_scheduler=True)
    assert PerturbationLightningModule(**kwargs, optimizer="muon").optimizer_name == "muon"
    assert PerturbationLightningModule(**kwargs, use_scheduler=True).use_scheduler


def test_the_bound_on_the_coefficients_stays_on_the_host():
    ops._ns_bound.cache_clear()
    with torch.device("meta"):  # (a default device: no kernel may be needed to check the arguments)
        assert 1 < ops._ns_bound(ops.NS_COEFFS, 5) < 8

"""Layer norm, the gated block and the orthogonalising optimiser used together: autograd, streams, captured graphs, the
gated MLP trunk and training steps with it."""
import copy
import dataclasses

import pytest
import torch

from cradle_vae_amd import functional as F_hip
from cradle_vae_amd import hip, ops
from cradle_vae_amd.mlp import GatedBlock, GatedResidualMLP
from cradle_vae_amd.optim import Muon
from tests import golden_io as gio
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _params(K=40, F=56, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=gen) * scale).to(dtype)
    return dict(x=n(33, K), w=(1 + 0.2 * n(K)).to(dtype), b=n(K, scale=0.1), w_in=n(2 * F, K, scale=K ** -0.5),
                w_out=n(K, F, scale=F ** -0.5), b_in=n(2 * F, scale=0.2), b_out=n(K, scale=0.2), dy=n(33, K))


def _block64(p, act="silu"):
    """The pre-norm gated residual block in 64 bits with autograd; -> y and the gradients of x and the parameters."""
    t = {k: v.detach().double().cpu().requires_grad_(k != "dy") for k, v in p.items()}
    xh = torch.nn.functional.layer_norm(t["x"], t["x"].shape[-1:], t["w"], t["b"])
    g, u = (xh @ t["w_in"].t() + t["b_in"]).chunk(2, -1)
    a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g)
    y = t["x"] + (a * u) @ t["w_out"].t() + t["b_out"]
    keys = [k for k in t if k != "dy"]
    return y.detach(), dict(zip(keys, torch.autograd.grad(y, [t[k] for k in keys], t["dy"])))


def _block(p, act="silu"):
    h = F_hip.layer_norm(p["x"], p["w"], p["b"])
    return F_hip.gated_mlp(h, p["w_in"], p["w_out"], p["b_in"], p["b_out"], act=act, residual=p["x"])


def _rel(got, want):
    return float((got.detach().double().cpu() - want).norm() / want.norm())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_block_and_its_gradients(dtype, act):
    p = _params(dtype=dtype)
    want, grads = _block64(p, act)
    g = {k: v.to(DEV).requires_grad_(k != "dy") for k, v in p.items()}
    y = _block(g, act)
    y.backward(g["dy"])
    # the norm's output and its gradient are rounded to the type on their way, a value and each gradient once more, and every
    # rounding is at most half a step: six of them in the longest chain; fp32: sums of 56..112 terms in each of five stages
    tol = 6 * ref.HALF[dtype] if dtype != torch.float32 else 5 * 112 * ref.U
    assert _rel(y, want) <= tol
    for k, v in grads.items():
        assert g[k].grad.dtype == dtype and _rel(g[k].grad, v) <= tol, k


def test_only_what_needs_a_gradient_gets_one():
    p = {k: v.to(DEV) for k, v in _params().items()}
    p["w_out"].requires_grad_()
    y = F_hip.gated_mlp(p["x"], p["w_in"], p["w_out"], p["b_in"], p["b_out"])
    y.backward(p["dy"])
    assert p["w_out"].grad is not None and p["w_in"].grad is None
    p["b"].requires_grad_()
    F_hip.layer_norm(p["x"], p["w"], p["b"]).backward(p["dy"])
    assert torch.allclose(p["b"].grad, p["dy"].sum(0), rtol=1e-5, atol=1e-5) and p["w"].grad is None
    with torch.no_grad():
        assert F_hip.layer_norm(p["x"], p["w"], p["b"]).grad_fn is None
    x = p["x"].clone().requires_grad_()
    gx, = torch.autograd.grad(F_hip.layer_norm(x, None, None).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative, and it says so
        gx.sum().backward()


def test_a_weight_used_twice_and_an_expanded_input():
    p = {k: v.to(DEV) for k, v in _params().items()}
    w_in = p["w_in"].clone().requires_grad_()
    f = lambda t: F_hip.gated_mlp(t, w_in, p["w_out"], p["b_in"], p["b_out"])
    (f(p["x"]) + f(2 * p["x"])).backward(p["dy"])
    twice = w_in.grad.clone()
    w_in.grad = None
    f(p["x"]).backward(p["dy"])
    one = w_in.grad.clone()
    w_in.grad = None
    f(2 * p["x"]).backward(p["dy"])
    assert torch.allclose(twice, one + w_in.grad, rtol=1e-5, atol=1e-5)
    row = p["x"][:1].clone().requires_grad_()  # one row broadcast to 33: its gradient is the sum over them
    f(row.expand(33, -1)).backward(p["dy"])
    whole = p["x"][:1].repeat(33, 1).requires_grad_()
    f(whole).backward(p["dy"])
    assert torch.allclose(row.grad, whole.grad.sum(0, keepdim=True), rtol=1e-4, atol=1e-5)


def test_refusals():
    p = {k: v.to(DEV) for k, v in _params().items()}
    x, w, b = p["x"], p["w"], p["b"]
    for call in (lambda: ops.layer_norm(x, w[:-1], b), lambda: ops.layer_norm(x, w.bfloat16(), b.bfloat16()),
                 lambda: ops.layer_norm(x.bfloat16(), w, b.bfloat16()), lambda: ops.layer_norm(x.double(), w, b),
                 lambda: ops.layer_norm(x, w.cpu(), b), lambda: ops.layer_norm(torch.ones(2, 40000, device=DEV)),
                 lambda: ops.layer_norm(torch.ones(3, 0, device=DEV)),
                 lambda: ops.layer_norm_bwd(p["dy"].half(), x, w, w[:33], w[:33]), lambda: ops.layer_norm_bwd(p["dy"], x, w, w[:30], w[:33]),
                 lambda: ops.gated_mlp(x, p["w_in"][:-1], p["w_out"]), lambda: ops.gated_mlp(x, p["w_in"].half(), p["w_out"]),
                 lambda: ops.gated_mlp(x, p["w_in"], p["w_out"], act="relu"), lambda: ops.gated_mlp(x, p["w_in"], p["w_out"], b, None),
                 lambda: ops.gated_mlp(x, p["w_in"], p["w_out"], residual=x[:-1]), lambda: ops.gated_mlp(x[:, :-1], p["w_in"], p["w_out"]),
                 lambda: ops.orthogonalize(x.double()), lambda: ops.orthogonalize(x[0]), lambda: ops.orthogonalize(x, steps=0),
                 lambda: ops.orthogonalize(x, coeffs=(3.0, 0.0, 0.0)), lambda: ops.orthogonalize(x, out=x[:, :-1]),
                 lambda: ops.orthogonalize(x, coeffs=(1.0, 2.0))):
        with pytest.raises(hip.CradleHipError):
            call()
    _, saved = ops.gated_mlp(x, p["w_in"], p["w_out"], save=True)
    with pytest.raises(hip.CradleHipError):
        ops.gated_mlp_bwd(p["dy"][:-1], x[:-1], p["w_in"], p["w_out"], saved)  # saved buffers of another call


def test_on_a_side_stream():
    p = {k: v.to(DEV) for k, v in _params().items()}
    want, og = _block(p), ops.orthogonalize(p["w_in"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, oh = _block(p), ops.orthogonalize(p["w_in"])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(oh, og)


@pytest.mark.parametrize("dtype,M,K,F", [(torch.float32, 300, 40, 56), (torch.bfloat16, 300, 40, 56), (torch.bfloat16, 700, 640, 720)])
def test_captured_graphs_replay(dtype, M, K, F):
    """Forward, backward and the orthogonalisation captured once, replayed on new inputs between eager work."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    n = lambda *s: torch.randn(*s, device=DEV, generator=gen).to(dtype)
    x, dy, w_in, w_out, b_in, b_out, w = n(M, K), n(M, K), n(2 * F, K), n(K, F), n(2 * F), n(K), n(K)

    def work():
        h, mean, rstd = ops.layer_norm(x, w, b_out)
        y, saved = ops.gated_mlp(h, w_in, w_out, b_in, b_out, save=True, residual=x)
        dh, dw_in, dw_out, db_in, db_out = ops.gated_mlp_bwd(dy, h, w_in, w_out, saved, bias=True)
        dx, dw, db = ops.layer_norm_bwd(dh, x, w, mean, rstd)
        return [y, dx, dw, db, dw_in, dw_out, db_in, db_out, ops.orthogonalize(dw_in), ops.gated_mlp(x[:1], w_in, w_out)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of the same work, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work()
        graphs.append((g, out))
    for k in range(4):
        x.copy_(n(M, K))
        dy.copy_(n(M, K))
        g, out = graphs[k % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, work()):
            assert torch.equal(a, b), k


def test_gated_trunk_against_64_bits():
    torch.manual_seed(0)
    m = GatedResidualMLP(24, 32, 3, 32).to(DEV)
    x, dy = torch.randn(50, 24, device=DEV), torch.randn(50, 32, device=DEV)
    y = m(x)
    y.backward(dy)
    d = copy.deepcopy(m).double().cpu()
    lin = d.linears()[0]
    h = torch.nn.functional.leaky_relu(lin(x.double().cpu()), 0.01)
    for blk in d.layers[1:]:
        g, u = (blk.norm(h) @ blk.w_in.t() + blk.b_in).chunk(2, -1)
        h = h + (torch.nn.functional.silu(g) * u) @ blk.w_out.t() + blk.b_out
    d.zero_grad()
    h.backward(dy.double().cpu())
    # three blocks of five stages of sums of at most 128 terms
    tol = 15 * 128 * ref.U
    assert _rel(y, h.detach()) <= tol
    for (k, a), b in zip(m.named_parameters(), d.parameters()):
        assert _rel(a.grad, b.grad) <= tol, k
    with torch.no_grad():
        assert torch.allclose(m.tail(F_hip.linear(x, m.linears()[0].weight, m.linears()[0].bias, act=True)), y, rtol=1e-5, atol=1e-5)


def test_muon_against_a_plain_evaluation():
    torch.manual_seed(0)
    hidden = [torch.nn.Parameter(torch.randn(s, device=DEV) * 0.1) for s in ((32, 48), (32, 48), (200, 130))]
    rest = [torch.nn.Parameter(torch.randn(17, device=DEV))]
    want = [p.detach().double().cpu() for p in hidden]
    twin = [torch.nn.Parameter(p.detach().clone()) for p in rest]
    opt = Muon(hidden, rest, lr=0.02, momentum=0.9, weight_decay=0.01)
    adam = torch.optim.Adam(twin, lr=0.02, weight_decay=0.01)
    buf = [torch.zeros_like(w) for w in want]
    for k in range(3):
        for p in hidden + rest:
            p.grad = torch.randn(p.shape, device=DEV)
        twin[0].grad = rest[0].grad.clone()
        for i, p in enumerate(hidden):
            g = p.grad.double().cpu()
            buf[i] = 0.9 * buf[i] + g
            o = ref.orthogonalize(g + 0.9 * buf[i], 5, ops.NS_COEFFS)
            want[i] = want[i] * (1 - 0.02 * 0.01) - 0.02 * 0.2 * max(p.shape) ** 0.5 * o
        opt.step()
        adam.step()
    for p, w in zip(hidden, want):
        # per step an orthogonalised update of rms 0.2, off by at most 2e-5 of its norm (fp32 steps amplified by 3.44 each)
        assert float((p.detach().double().cpu() - w).norm()) <= 3 * 2e-5 * 0.02 * 0.2 * p.numel() ** 0.5 * 2 + 8 * ref.U * float(w.norm())
    assert torch.allclose(rest[0], twin[0], rtol=1e-5, atol=1e-6)
    opt.zero_grad(set_to_none=True)
    before = [p.detach().clone() for p in hidden]
    opt.step()  # nothing has a gradient: nothing moves
    assert all(torch.equal(a, b) for a, b in zip(before, hidden))
    state = opt.state_dict()
    opt.load_state_dict(state)
    assert torch.equal(opt.state[hidden[0]]["momentum"].double().cpu().float(), buf[0].float()) or _rel(opt.state[hidden[0]]["momentum"], buf[0]) < 1e-5


def _loss_module(block):
    from cradle_vae_amd import synthetic as syn
    from cradle_vae_amd.guide import ObservationNormalizationStatistics, cradle_vae_CorrelatedNormalGuide
    from cradle_vae_amd.loss_module import cradle_vae_ELBOLossModule
    from cradle_vae_amd.model import cradle_vae_Model

    shape = syn.MID
    batch = syn.make_batch(shape, seed=3, device=DEV)
    torch.manual_seed(0)
    model = cradle_vae_Model(n_latent=shape.n_latent, n_treatments=shape.n_treatments, n_phenos=shape.n_phenos, n_qc=shape.n_qc,
                             mask_prior_prob=0.05, embedding_prior_scale=1.0, likelihood_key="library_nb", decoder_n_layers=2,
                             decoder_n_hidden=32, sum_mode=False, mlp_block=block)
    stats = ObservationNormalizationStatistics(log_x_mean=batch["log_x_mean"].cpu(), log_x_std=batch["log_x_std"].cpu())
    guide = cradle_vae_CorrelatedNormalGuide(
        n_latent=shape.n_latent, n_treatments=shape.n_treatments, n_phenos=shape.n_phenos, n_qc=shape.n_qc, basal_encoder_n_layers=2,
        basal_encoder_n_hidden=32, basal_encoder_input_normalization="log_standardize", embedding_encoder_n_layers=2,
        embedding_encoder_n_hidden=32, x_normalization_stats=stats, mlp_block=block)
    return cradle_vae_ELBOLossModule(model=model, guide=guide, beta=0.5).to(DEV), batch, shape


@pytest.mark.filterwarnings("ignore:loss_module.step")
@pytest.mark.parametrize("block,impl", [("gated", "modular"), ("residual", "fused+muon")])
def test_training_steps_with_muon(block, impl):
    from cradle_vae_amd.trainer import TrainStep

    lm, batch, shape = _loss_module(block)
    lm.max_dosages_per_cell = 3
    st = TrainStep(lm, lr=1e-3, optimizer="muon", seed=5)
    assert st.impl == impl and isinstance(st.optimizer, Muon) and st.optimizer.param_groups[0]["orthogonal"]
    before = {k: p.detach().clone() for k, p in lm.named_parameters()}
    losses = [float(st(batch, n_particles=3)) for _ in range(3)]
    assert all(torch.isfinite(torch.tensor(losses)))
    moved = {k for k, p in lm.named_parameters() if not torch.equal(p, before[k])}
    assert any("layers.1" in k for k in moved) and any("normalized_mean_decoder" in k for k in moved)
    assert all(bool(torch.isfinite(p).all()) for p in lm.parameters())
    if impl == "fused+muon":  # a rejected batch never reaches the parameters
        bad = dict(batch, D=batch["D"].clone())
        bad["D"][0] = 0
        bad["D"][0, :5] = 1.0
        before = [p.detach().clone() for p in lm.parameters()]
        with pytest.raises(hip.CradleHipError, match="kmax"):
            st(bad, n_particles=3)
        assert all(torch.equal(a, b) for a, b in zip(before, lm.parameters()))
        st(batch, n_particles=3)


@pytest.mark.filterwarnings("ignore:loss_module.step")
def test_gated_inference_draws_equal_the_module_form():
    """The no-gradient forms (shared input product, first layer by lookup) and the differentiable ones agree."""
    lm, batch, shape = _loss_module("gated")
    g = lm.guide
    enc = g.z_basal_encoder
    x, tail = torch.randn(20, shape.n_phenos, device=DEV), torch.randn(3, 20, 2 * shape.n_latent, device=DEV)
    with torch.no_grad():
        a = enc.forward_shared(enc.shared_input_part(x), tail)
    b = enc(torch.cat([x.unsqueeze(0).expand(3, -1, -1), tail], dim=-1))
    assert torch.allclose(a.mean, b.mean, rtol=1e-4, atol=1e-4) and torch.allclose(a.stddev, b.stddev, rtol=1e-4, atol=1e-4)


@pytest.mark.filterwarnings("ignore:loss_module.step")
def test_configured_training_run(tmp_path):
    """mlp_block and optimizer through a yaml, train.py and eval.py."""
    import csv
    import os

    import numpy as np
    import yaml

    import eval as eval_entry
    import train as train_entry

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    cfg = yaml.safe_load(open(os.path.join(root, "demo", "cradle_vae_synthetic_gated.yaml")))
    assert cfg["lightning_module_kwargs.optimizer"] == "muon" and cfg["model_kwargs.mlp_block--guide_kwargs.mlp_block"] == "gated"
    cfg.update({"max_epochs": 1, "data_module_kwargs.n_cells": 700, "data_module_kwargs.n_genes": 64, "data_module_kwargs.n_guides": 5,
                "data_module_kwargs.batch_size": 128, "n_latent": 8, "model_kwargs.decoder_n_hidden": 32,
                "guide_kwargs.basal_encoder_n_hidden": 32, "guide_kwargs.embedding_encoder_n_hidden": 32})
    path = tmp_path / "cfg.yaml"
    path.write_text(yaml.safe_dump(cfg))
    train_entry.main(["--config", str(path), "--results-dir", str(tmp_path / "results")])
    rdir = tmp_path / "results" / cfg["name"]
    assert np.isfinite(float(list(csv.DictReader(open(rdir / "metrics.csv")))[-1]["train/loss"]))
    m = eval_entry.main(["--experiment_path", str(rdir), "--batch_size", "64", "--ate_n_particles", "32", "--qc_pass", "false"])
    assert np.isfinite(m["test/IWELBO"])


def test_two_calls_at_once():
    """Independent calls on two streams, each with its own workspace, against the same calls one after the other."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    n = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    x, dy, w_in, w_out, b_in, b_out = n(2, 600, 72), n(2, 600, 72), n(304, 72), n(72, 152), n(304), n(72)

    def work(i):
        h, mean, rstd = ops.layer_norm(x[i], b_out, b_out)
        y, saved = ops.gated_mlp(h, w_in, w_out, b_in, b_out, save=True)
        grads = ops.gated_mlp_bwd(dy[i], h, w_in, w_out, saved, bias=True)
        return [y, *grads, *ops.layer_norm_bwd(grads[0], x[i], b_out, mean, rstd), ops.orthogonalize(grads[1])]

    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for a, b in zip(got[0] + got[1], want[0] + want[1]):
            assert torch.equal(a, b)


def test_a_captured_backward_pass():
    """The autograd forms in a captured graph, no eager graph of the same leaves alive at the capture."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    n = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    x, dy = n(90, 40), n(90, 40)
    leaves = [p.requires_grad_() for p in (n(40), n(40), n(112, 40), n(40, 56), n(112), n(40))]

    def work():
        w, b, w_in, w_out, b_in, b_out = leaves
        y = F_hip.gated_mlp(F_hip.layer_norm(x, w, b), w_in, w_out, b_in, b_out, residual=x)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = work()
    for _ in range(3):
        x.copy_(n(90, 40))
        dy.copy_(n(90, 40))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, work()):
            assert torch.equal(a, b)

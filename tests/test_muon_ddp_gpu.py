"""Orthogonalised momentum on two ranks (gloo on one GPU): every rank applies the same update of the averaged gradients, and a
batch that one rank rejects reaches no rank's parameters."""
import os

import pytest
import torch
import torch.multiprocessing as mp

from tests.test_ddp_gpu import WORLD, _free_port

pytestmark = pytest.mark.gpu


def _worker(rank, port, block, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), GLOO_SOCKET_IFNAME="lo")
    import torch.distributed as dist

    dist.init_process_group("gloo", rank=rank, world_size=WORLD)
    try:
        from cradle_vae_amd import hip
        from cradle_vae_amd import synthetic as syn
        from cradle_vae_amd.trainer import TrainStep
        from tests.test_hidden_layers_gpu import _loss_module

        torch.cuda.set_device(0)
        lm, _, shape = _loss_module(block)
        lm.max_dosages_per_cell = 3
        st = TrainStep(lm, lr=1e-3, weight_decay=1e-3, world_size=WORLD, seed=5, optimizer="muon")
        copy = lambda: {k: p.detach().cpu().clone() for k, p in lm.named_parameters() if p.requires_grad}
        good = syn.make_batch(shape, seed=50 + rank, device="cuda:0")
        start, grads, losses = copy(), [], []
        for _ in range(3):
            losses.append(float(st(good, n_particles=3)))
            grads.append({k: p.grad.detach().cpu().clone() for k, p in lm.named_parameters() if p.requires_grad})
        st.check_flags()
        after = copy()
        msg = None
        if st.impl == "fused+muon":
            bad = dict(good)
            if rank == 1:  # a cell with five dosages where the step plans for three
                bad["D"] = good["D"].clone()
                bad["D"][0] = 0.0
                bad["D"][0, :5] = 1.0
            try:
                st(bad, n_particles=3)
            except hip.CradleHipError as e:
                msg = str(e)
        kept = copy()
        st(good, n_particles=3)
        st.check_flags()  # reported once; the valid step leaves nothing behind
        out[rank] = dict(impl=st.impl, start=start, grads=grads, losses=losses, after=after, msg=msg, kept=kept, end=copy())
    finally:
        dist.destroy_process_group()


@pytest.mark.filterwarnings("ignore:loss_module.step")
@pytest.mark.parametrize("block,impl", [("residual", "fused+muon"), ("gated", "modular")])
def test_two_ranks(block, impl):
    ctx = mp.get_context("spawn")
    with ctx.Manager() as mgr:
        out, port = mgr.dict(), _free_port()
        procs = [ctx.Process(target=_worker, args=(r, port, block, out)) for r in range(WORLD)]
        for p in procs:
            p.start()
        for p in procs:
            p.join(timeout=100)
        for p in procs:
            if p.is_alive():
                p.kill()
        assert sorted(out.keys()) == [0, 1], "a rank failed or hung"
        a, b = out[0], out[1]
    same = lambda x, y: x.keys() == y.keys() and all(torch.equal(x[k], y[k]) for k in x)
    assert a["impl"] == b["impl"] == impl and a["losses"] != b["losses"]  # each rank its own cells
    assert same(a["start"], b["start"]) and not same(a["start"], a["after"])
    for ga, gb in zip(a["grads"], b["grads"]):
        assert same(ga, gb)  # the averaged, clipped gradients
    assert same(a["after"], b["after"]) and same(a["end"], b["end"]) and not same(a["after"], a["end"])
    if impl == "fused+muon":
        assert "kmax" in b["msg"] and "another rank" in a["msg"]
        assert same(a["after"], a["kept"]) and same(b["after"], b["kept"])
    # one process that is given the same gradients arrives at the same parameters
    from cradle_vae_amd.optim import make_optimizer
    from tests.test_hidden_layers_gpu import _loss_module

    lm, _, _ = _loss_module(block)
    opt = make_optimizer("muon", lm, 1e-3, 1e-3)
    assert same(a["start"], {k: p.detach().cpu() for k, p in lm.named_parameters() if p.requires_grad})
    for g in a["grads"]:
        for k, p in lm.named_parameters():
            if p.requires_grad:
                p.grad = g[k].to(p.device)
        opt.step()
    assert same(a["after"], {k: p.detach().cpu() for k, p in lm.named_parameters() if p.requires_grad})

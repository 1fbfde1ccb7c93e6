"""ExpertFFN.forward / backward: the router, the weighted combine and their
gradients around the expert GEMMs, on one rank, and a training step with AdamW.

A token with k choices is the same work as k tokens with one choice each, in
the same send order, so ``step`` on such a batch gives every expected result
bit for bit."""
import multiprocessing as mp
import os

import numpy as np
import pytest
import torch

from ep_support import free_port
from oracle import router_oracle as ro

pytestmark = pytest.mark.gpu


def _layer(mxg, E, H, I, dev, seed=0, **kw):
    g = torch.Generator(device=dev).manual_seed(seed)
    wgu = (torch.randn(E, 2 * I, H, generator=g, device=dev) * 0.05).to(torch.bfloat16)
    wd = (torch.randn(E, H, I, generator=g, device=dev) * 0.05).to(torch.bfloat16)
    return wgu, wd, mxg.moe.ExpertFFN(mxg.ExpertParallel(E), wgu, wd, **kw)


def _batch(n, E, H, dev, seed=1):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(n, H, generator=g, device=dev).to(torch.bfloat16)
    logits = torch.randn(n, E, generator=g, device=dev) * 1.5
    dout = torch.randn(n, H, generator=g, device=dev).to(torch.bfloat16)
    return x, logits, dout


@pytest.mark.parametrize("comm", [False, True])
@pytest.mark.parametrize("k,score,kw", [(1, "softmax", {}), (2, "softmax", {}),
                                        (4, "sigmoid", dict(groups=4, topk_groups=2, group_score="top2", scale=2.5))])
def test_against_one_choice_a_token(mxg, cuda_dev, k, score, kw, comm):
    E, H, I, n = 16, 256, 128, 200
    stream = torch.cuda.Stream() if comm else None
    wgu, wd, layer = _layer(mxg, E, H, I, cuda_dev, comm_stream=stream)
    x, logits, dout = _batch(n, E, H, cuda_dev)
    bias = torch.randn(E, device=cuda_dev) * 0.02 if score == "sigmoid" else None
    router = mxg.moe.Router(k, score=score, bias=bias, **kw)
    fwd = layer.forward(x, logits, router)
    got = layer.backward(fwd, dout)
    w, ids = router(logits)
    assert torch.equal(fwd.weights, w) and torch.equal(fwd.ids, ids)

    # the same rows as n * k tokens of one choice
    one = torch.ones(n * k, 1, device=cuda_dev)
    rows_dy = (w[:, :, None] * dout[:, None, :].float()).to(torch.bfloat16).view(n * k, H)
    flat = layer.step(x.repeat_interleave(k, 0), ids.view(-1, 1), one, rows_dy)
    assert mxg.device_error() == 0
    assert torch.equal(got.dw_gate_up, flat.dw_gate_up) and torch.equal(got.dw_down, flat.dw_down)
    acc = torch.zeros(n, H, device=cuda_dev)
    for j in range(k):
        acc += flat.dx.view(n, k, H)[:, j].float()
    assert torch.equal(got.dx, acc.to(torch.bfloat16))
    y = flat.out.view(n, k, H)
    acc.zero_()
    for j in range(k):
        acc = torch.addcmul(acc, w[:, j:j + 1].expand(n, H), y[:, j].float())
    assert torch.all((fwd.out.float() - acc).abs() <= 2.0 ** -8 * acc.abs() + k * 2.0 ** -22 * y.float().abs().amax(1))
    # router: <dout, y> and the logits' gradient, from the definitions in 64 bits
    products = (dout.double()[:, None] * y.double()).cpu().numpy()
    dw = products.sum(2)
    ref = ro.router_bwd(logits.cpu().numpy(), ids.cpu().numpy(), dw, score=score, scale=kw.get("scale", 1.0))
    size = (np.abs(w.cpu().numpy()) * np.abs(products).sum(2)).sum(1)
    # dw: H / 8 + 13 roundings of its terms' size; the gradient's own 1e-5
    assert np.all(np.abs(got.dlogits.cpu().numpy() - ref) <= ((H / 8 + 13) * 2.0 ** -23 + 1e-5) * size[:, None])


def test_training_step_with_adamw(mxg, cuda_dev):
    """logits -> forward -> backward -> AdamW on the router and the experts ->
    reencode: the layer then multiplies by the new weights."""
    E, H, I, n = 8, 128, 64, 96
    wgu, wd, layer = _layer(mxg, E, H, I, cuda_dev, seed=3)
    gate = torch.randn(E, H, device=cuda_dev) * 0.1
    x, _, dout = _batch(n, E, H, cuda_dev, seed=4)
    router = mxg.moe.Router(2)
    for bits in (32, 8):
        opt = mxg.optim.AdamW([wgu, wd, gate], lr=1e-2, state_bits=bits)
        before = [p.clone() for p in opt.params]
        for _ in range(2):
            fwd = layer.forward(x, x.float() @ gate.t(), router)
            grads = layer.backward(fwd, dout)
            opt.step([grads.dw_gate_up, grads.dw_down, grads.dlogits.t() @ x.float()])
            layer.reencode(wgu, wd)
        assert all(not torch.equal(p, b) for p, b in zip(opt.params, before))
        fresh = mxg.moe.ExpertFFN(mxg.ExpertParallel(E), wgu, wd)
        for a, b in ((layer.wgu, fresh.wgu), (layer.wd, fresh.wd), (layer.wdt, fresh.wdt), (layer.wgut, fresh.wgut)):
            assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
        logits = x.float() @ gate.t()
        assert torch.equal(layer.forward(x, logits, router).out, fresh.forward(x, logits, router).out)
    assert mxg.device_error() == 0


def test_two_layers_share_one_expert_parallel(mxg, cuda_dev):
    """Both forwards run before either backward: nothing of the first is lost."""
    E, H, I = 8, 128, 64
    wgu, wd, a = _layer(mxg, E, H, I, cuda_dev, seed=5)
    b = mxg.moe.ExpertFFN(a.ep, wgu, wd)
    router = mxg.moe.Router(2, score="sigmoid")
    big, small = _batch(150, E, H, cuda_dev, 6), _batch(3, E, H, cuda_dev, 7)
    alone = [a.backward(a.forward(x, z, router), d) for x, z, d in (big, small)]
    fa, fb = a.forward(*big[:2], router), b.forward(*small[:2], router)
    gb, ga = b.backward(fb, small[2]), a.backward(fa, big[2])
    for got, want in ((ga, alone[0]), (gb, alone[1])):
        for p, q in zip(got, want):
            assert torch.equal(p, q)


def test_refusals(mxg, cuda_dev):
    wgu, wd, layer = _layer(mxg, 8, 128, 64, cuda_dev)
    x, z, d = _batch(4, 8, 128, cuda_dev)
    with pytest.raises(ValueError, match="logits"):
        layer.forward(x, z[:, :7], mxg.moe.Router(2))
    with pytest.raises(ValueError, match="topk"):
        layer.forward(x, z, mxg.moe.Router(9))
    with pytest.raises(ValueError, match="weights"):
        layer.reencode(wd, wgu)
    fwd = layer.forward(x, z, mxg.moe.Router(2))
    with pytest.raises(ValueError, match="dout"):
        layer.backward(fwd, d.float())


def _two_rank_worker(rank, world, port, q):
    try:
        import datetime

        import torch.distributed as dist
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        torch.cuda.set_device(rank)
        dist.init_process_group("nccl", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
        from conftest import load_pkg
        mxg = load_pkg()
        dev = torch.device("cuda", rank)
        E, H, I = 8, 256, 128
        El = E // world
        g = torch.Generator(device=dev).manual_seed(9)
        wgu = (torch.randn(E, 2 * I, H, generator=g, device=dev) * 0.05).to(torch.bfloat16)
        wd = (torch.randn(E, H, I, generator=g, device=dev) * 0.05).to(torch.bfloat16)
        mine = slice(rank * El, (rank + 1) * El)
        router = mxg.moe.Router(2, score="sigmoid")
        big, small = (_batch(n, E, H, dev, 20 + 2 * i + rank) for i, n in enumerate(([300, 217][rank], [7, 0][rank])))
        res = {}
        for dx in (True, False):
            for name, transport, comm, ce in (("nccl", "nccl", False, False), ("p2p", "p2p", False, False),
                                              ("p2p_side", "p2p", True, False), ("p2p_ce", "p2p", True, True)):
                ep = mxg.ExpertParallel(E, transport=transport)
                a, b = (mxg.moe.ExpertFFN(ep, wgu[mine], wd[mine], compute_dx=dx, copy_engines=ce,
                                          comm_stream=torch.cuda.Stream() if comm else None) for _ in range(2))
                got = []
                for _ in range(2):       # both forwards before both backwards
                    fa, fb = a.forward(*big[:2], router), b.forward(*small[:2], router)
                    gb, ga = b.backward(fb, small[2]), a.backward(fa, big[2])
                    got += [fa.out, fb.out, *ga, *gb]
                torch.cuda.synchronize()
                assert mxg.device_error() == 0
                res[dx, name] = [t.float().cpu().numpy() for t in got if t is not None]
                ep.close()
        dist.barrier()
        dist.destroy_process_group()
        q.put((rank, res))
    except Exception:
        import traceback
        q.put((rank, traceback.format_exc()))


def test_two_layers_over_two_ranks():
    """Layers of different batches share one ExpertParallel over two GPUs: every
    exchange gives the bytes of the all-to-all transport."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), free_port()
    procs = [ctx.Process(target=_two_rank_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = dict(q.get(timeout=600) for _ in procs)
    for p in procs:
        p.join(timeout=60)
    for r in range(2):
        assert isinstance(res[r], dict), res[r]
        for (dx, name), got in res[r].items():
            for i, (a, b) in enumerate(zip(got, res[r][dx, "nccl"])):
                assert np.array_equal(a, b), (r, dx, name, i)


@pytest.mark.parametrize("dx", [True, False])
def test_no_rows(mxg, cuda_dev, dx):
    """A rank without tokens whose experts nobody chose (small batches over many
    ranks): empty outputs, weight gradients of zero."""
    E, H, I = 8, 128, 64
    wgu, wd, layer = _layer(mxg, E, H, I, cuda_dev, compute_dx=dx)
    x, z, d = (t[:0] for t in _batch(4, E, H, cuda_dev))
    fwd = layer.forward(x, z, mxg.moe.Router(2))
    got = layer.backward(fwd, d)
    assert fwd.out.shape == (0, H) and got.dlogits.shape == (0, E) and fwd.weights.shape == (0, 2)
    assert got.dx is None if not dx else got.dx.shape == (0, H)
    one = layer.step(x, fwd.ids, fwd.weights, d)
    for dw, w in ((got.dw_gate_up, wgu), (got.dw_down, wd), (one.dw_gate_up, wgu), (one.dw_down, wd)):
        assert dw.shape == w.shape and torch.all(dw == 0)
    assert one.out.shape == (0, H) and mxg.device_error() == 0
    # the update of such a step: the weights only decay
    opt = mxg.optim.AdamW([wgu, wd], lr=0.0)
    keep = wgu.clone()
    opt.step([got.dw_gate_up, got.dw_down])
    assert torch.equal(wgu, keep)

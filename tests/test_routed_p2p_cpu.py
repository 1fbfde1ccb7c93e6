"""The peer-memory transport's orchestration over a world-size-2 ``gloo`` group:
receive buffers are files that both processes map, and the exchange kernels
plain loops over the oracle's tables.  A rank that is slow to read its buffer
stands for one whose kernels still read it."""
import multiprocessing as mp
import os
import time

import numpy as np
import pytest
import torch

from ep_support import free_port, make_rank_inputs
from oracle import ep_oracle
from test_routed_ep_cpu import Ops

E, K, H = 8, 3, 16


def _rows(raw, n, like):
    return raw[:n * like[0].numel() * like.element_size()].view(like.dtype).view((n,) + tuple(like.shape[1:]))


class Buffer:
    """``ep.PeerBuffer`` in mapped files."""
    made = 0

    def __init__(self, nbytes, group, world, rank, device):
        import torch.distributed as dist
        Buffer.made += 1
        name = lambda r: os.path.join(os.environ["PEER_FILES"], f"{Buffer.made}_{r}")
        torch.from_file(name(rank), shared=True, size=nbytes, dtype=torch.uint8).fill_(255)
        dist.barrier(group=group)
        self.ptrs = self.ptrs_host = [torch.from_file(name(r), shared=True, size=nbytes, dtype=torch.uint8)
                                      for r in range(world)]
        self.local = self.ptrs[rank]

    def view(self, rows, like):
        n = rows * int(np.prod(like.shape[1:])) * like.element_size()
        return self.local[:n].view(like.dtype).view((rows,) + tuple(like.shape[1:]))

    def close_peers(self):
        pass

    free = close_peers


class P2P:
    """``ep.CudaP2POps`` on mapped files."""

    def plan(self, counts, me, pad, m_pad, n_recv):
        got = ep_oracle.p2p_plan(counts.numpy(), me, pad)
        return tuple(torch.from_numpy(np.ascontiguousarray(a)) for a in got)

    def zero_pad_rows(self, local, back_rank):
        local[back_rank < 0] = 0

    def dispatch(self, src, send_rows, slot_start, dest_base, e_local, me, peers, capacity, max_blocks=0):
        for p, r in enumerate(send_rows.tolist()):
            s = int(np.searchsorted(slot_start.numpy(), p, side="right") - 1)
            _rows(peers[s // e_local], capacity, src)[int(dest_base[s]) + p] = src[r]

    def copy_runs(self, src, runs, peers, capacity):
        for a, b, n, d in zip(*(t.tolist() for t in runs)):
            _rows(peers[d], capacity, src)[b:b + n] = src[a:a + n]

    def ret(self, src, order, back_rank, back_row, peers, capacity, max_blocks=0):
        for q in order.tolist():
            _rows(peers[int(back_rank[q])], capacity, src)[int(back_row[q])] = src[q]


def _parallel(p2p):
    from conftest import load_pkg
    ep = load_pkg().ep
    ep.PeerBuffer = Buffer
    torch.cuda.synchronize = lambda *a: None
    par = ep.ExpertParallel(E, ops=Ops())
    if p2p:
        par.transport, par.p2p = "p2p", P2P()
    return par


def _inputs(rank, n, seed, width=H):
    ids, x, w = make_rank_inputs(rank, n, K, E, width, seed=seed)
    g = np.random.default_rng(seed + 77 + rank)
    dout = g.standard_normal((n, width)).astype(np.float32)
    return (torch.from_numpy(x).to(torch.bfloat16), torch.from_numpy(ids), torch.from_numpy(w),
            torch.from_numpy(dout).to(torch.bfloat16))


def _forward(par, x, ids, w, ce):
    """The exchanges of ExpertFFN.forward around an expert that doubles its rows."""
    local, plan = par.dispatch(x, ids)
    kept = local.clone()
    ret = par.combine_send(kept * 2, plan, copy_engines=ce).clone()
    return kept, plan, ret, par.combine_finish(ret, plan, w)


def _backward(par, fwd, w, dout, ce, dx, wait):
    """Those of ExpertFFN.backward; `wait` before the received rows are read."""
    _, plan, ret, _ = fwd
    dsent, dw = par.combine_grad(dout, ret, plan, w)
    local = par.dispatch_sent(dsent, plan, copy_engines=ce)
    time.sleep(wait)
    dy = local.clone()
    out = [dw, dy]
    if dx:
        out.append(par.combine_finish(par.combine_send(dy * 4, plan, buffer="ret_dx", copy_engines=ce), plan, None))
    return out


def _both_layers(rank, dx):
    """Two layers of different batches share one ExpertParallel: both forwards,
    then both backwards, twice; rank 1 reads its dy rows late.  Over the
    all-to-all transport, peer memory, and peer memory with copy engines."""
    big, small = _inputs(rank, [41, 23][rank], 1), _inputs(rank, [5, 0][rank], 2)
    every = []
    for p2p, ce in ((False, False), (True, False), (True, True)):
        par, got = _parallel(p2p), []
        for _ in range(2):
            fb, fs = _forward(par, *big[:3], ce), _forward(par, *small[:3], ce)
            got += [fb[0], fb[3], fs[0], fs[3]]
            wait = 0.5 if p2p and rank == 1 else 0.0
            got += _backward(par, fs, small[2], small[3], ce, dx, wait)
            got += _backward(par, fb, big[2], big[3], ce, dx, wait)
        if p2p:
            par.close()
        every.append([t.float().numpy() for t in got])
    return every


def _worker(rank, port, files, job, args, q):
    try:
        import datetime

        import torch.distributed as dist
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), PEER_FILES=files)
        dist.init_process_group("gloo", rank=rank, world_size=2, timeout=datetime.timedelta(seconds=60))
        got = job(rank, *args)
        dist.barrier()
        dist.destroy_process_group()
        q.put((rank, got))
    except Exception:
        import traceback
        q.put((rank, traceback.format_exc()))


def _run(job, args, files):
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), free_port()
    procs = [ctx.Process(target=_worker, args=(r, port, str(files), job, args, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=180) for _ in procs)
    for p in procs:
        p.join(60)
    assert all(not isinstance(g, str) for g in got.values()), got
    return got


@pytest.mark.parametrize("dx", [False, True])
def test_two_layers_over_peer_memory(tmp_path, dx):
    """The same rows as the all-to-all transport's, bit for bit: nothing is
    written to a receive buffer while a rank still reads it."""
    got = _run(_both_layers, (dx,), tmp_path)
    for r in range(2):
        want = got[r][0]
        for mode, rows in zip(("kernels", "copy engines"), got[r][1:]):
            assert len(rows) == len(want)
            for i, (a, b) in enumerate(zip(rows, want)):
                assert np.array_equal(a, b), (r, mode, i)


def _laid_out_again(rank):
    par, said = _parallel(True), []
    # 164 tokens' 492 rows: 246 at least on one rank; two a rank need 2 * 2 * 3 rows and 4 * 31 of padding, 136
    big, wide, small = _inputs(rank, [91, 73][rank], 1), _inputs(rank, 4, 2, 2 * H), _inputs(rank, 2, 3)
    first = _forward(par, *big[:3], False)
    _forward(par, *wide[:3], False)
    last = _forward(par, *small[:3], False)
    dsent, _ = par.combine_grad(big[3], first[2], first[1], big[2])
    for call in (lambda: par.dispatch_sent(dsent, first[1]), lambda: par.dispatch_like(big[3], first[1]),
                 lambda: par.combine_send(first[0], first[1]), lambda: par.return_target(first[1], first[0])):
        try:
            call()
            said.append("no error")
        except ValueError as e:
            said.append("refused" if "laid out again" in str(e) else str(e))
    got = _backward(par, last, small[2], small[3], False, True, 0.0)       # the latest plan goes on
    par.close()
    ref = _parallel(False)
    want = _backward(ref, _forward(ref, *small[:3], False), small[2], small[3], False, True, 0.0)
    return said, all(torch.equal(a, b) for a, b in zip(got, want))


def test_plans_of_buffers_laid_out_again_are_refused(tmp_path):
    """Rows of another size, then a small batch of the first size, leave smaller
    buffers than the first plan's: every rank refuses it, and nobody waits."""
    got = _run(_laid_out_again, (), tmp_path)
    assert got == {r: (["refused"] * 4, True) for r in range(2)}

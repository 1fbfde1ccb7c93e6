"""The combine's gradient and its way back to the experts over a world-size-2
``gloo`` group, with the oracle's pieces as the device work."""
import multiprocessing as mp
import os

import numpy as np
import torch

from ep_support import OracleEpOps, free_port, make_rank_inputs
from oracle import ep_oracle, router_oracle


class Ops(OracleEpOps):
    def combine_bwd(self, dout, rows, slot_pos, weights, n, k):
        w = None if weights is None else weights.numpy()
        drows, dw = router_oracle.combine_bwd(dout.float().numpy(), rows.float().numpy(),
                                              slot_pos.numpy().reshape(n, k), w)
        return torch.from_numpy(drows).to(torch.bfloat16), torch.from_numpy(dw)


def _bf16(a):
    return torch.from_numpy(a).to(torch.bfloat16)


def _rank(rank, world, port, q):
    import torch.distributed as dist

    from conftest import load_pkg
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    E, k, H, n = 8, 3, 16, [21, 34][rank]
    ids, x, w = make_rank_inputs(rank, n, k, E, H)
    ep = load_pkg().ExpertParallel(E, ops=Ops())
    _, plan = ep.dispatch(_bf16(x), torch.from_numpy(ids))
    g = np.random.default_rng(50 + rank)
    ret, dout = _bf16(g.standard_normal((n * k, H))), _bf16(g.standard_normal((n, H)))
    dsent, dw = ep.combine_grad(dout, ret, plan, torch.from_numpy(w))
    local = ep.dispatch_sent(dsent, plan)
    q.put((rank, plan.slot_pos.numpy().reshape(n, k), ret.float().numpy(), dout.float().numpy(), dsent.float().numpy(),
           dw.numpy(), local.float().numpy()))
    dist.barrier()
    dist.destroy_process_group()


def test_gradient_reaches_the_experts_of_both_ranks():
    ctx = mp.get_context("spawn")
    q, port, world = ctx.Queue(), free_port(), 2
    procs = [ctx.Process(target=_rank, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = dict((r[0], r[1:]) for r in (q.get(timeout=120) for _ in range(world)))
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    E, k, H = 8, 3, 16
    ids, ws, ns = [], [], [21, 34]
    for r in range(world):
        i, _, w = make_rank_inputs(r, ns[r], k, E, H)
        ids.append(i), ws.append(w)
    for r in range(world):
        slot_pos, ret, dout, dsent, dw, _ = got[r]
        for t in range(ns[r]):
            for j in range(k):
                p = slot_pos[t, j]
                want = torch.from_numpy(np.float64(ws[r][t, j]) * dout[t].astype(np.float64)).to(torch.bfloat16)
                assert np.array_equal(dsent[p], want.float().numpy())
                # H = 16 products in 64 bits
                assert abs(dw[t, j] - (dout[t].astype(np.float64) * ret[p]).sum()) < 1e-12
    # each expert's padded rows: every source rank's choices of it, in send order
    for d in range(world):
        row, local = 0, got[d][5]
        for e in range(d * 4, d * 4 + 4):
            rows = [got[r][3][got[r][0][t, j]] for r in range(world) for t in range(ns[r]) for j in range(k)
                    if ids[r][t, j] == e]
            assert np.array_equal(local[row:row + len(rows)], np.array(rows).reshape(-1, H))
            end = row + -(-len(rows) // 32) * 32
            assert np.all(local[row + len(rows):end] == 0)
            row = end
        assert row == local.shape[0]
    assert ep_oracle.route(ids[0], E)[0].sum() == ids[0].size

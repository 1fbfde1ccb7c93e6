"""Timed cases of the operators that train a mixture-of-experts layer around its grouped GEMMs.

Three operators, each with a plain form in torch and the library's own call:

``router``       scores of every expert, the top-k experts of each token (expert groups, a bias that only
                 selects, ties to the lowest index) and their weights; and the gradient of the logits.
``combine_bwd``  gradient of the weighted sum over each token's expert rows: the rows' gradient in send order
                 and the gradient of the router weights.
``adamw``        one AdamW step over a list of tensors, with moments in 32 bits or in 8 bits (blocks of 256
                 values, stochastic rounding from a counter-based hash).
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
BLOCK = 256                        # values that share one scale of the 8-bit moments
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # four tokens of a decode batch through a 256-expert gate with 8 groups: latency
        router("router_decode", "fwd", 4, 256, 8, groups=8, topk_groups=4, group_score="top2", score="sigmoid",
               bias=True, dtype="fp32", scale=2.5),
        # one GPU's tokens of the 256-expert expert-parallel layer
        router("router_train", "fwd", 16384, 256, 8, groups=8, topk_groups=4, group_score="top2", score="sigmoid",
               bias=True, dtype="fp32", scale=2.5),
        # 32768 tokens over 8 experts, top 2, renormalised softmax
        router("router_8_experts", "fwd", 32768, 8, 2, dtype="bf16"),
        # odd sizes: 160 experts, groups by their best expert, four experts switched off, weights not renormalised
        router("router_ragged", "fwd", 5003, 160, 6, groups=8, topk_groups=3, dtype="bf16", renormalize=False,
               masked=4, scale=16.0),
        # dense softmax gradient of a long batch
        router("router_grad_softmax", "bwd", 65536, 256, 8, dtype="bf16", renormalize=False),
        # sparse gradient of renormalised sigmoid weights, an odd number of experts
        router("router_grad_sigmoid", "bwd", 16384, 137, 6, score="sigmoid", dtype="fp32", scale=2.5),
        # a handful of tokens of the small configuration
        combine("combine_grad_small", 96, 2, 512, 4),
        # one GPU's tokens of the 256-expert layer
        combine("combine_grad_256_experts", 16384, 8, 7168, 256),
        # 14336-wide rows, an odd number of tokens
        combine("combine_grad_wide", 5001, 2, 14336, 8),
        # many small tensors: twelve small layers, everything in 32 bits
        adamw("adamw_small_tensors", 12, 4, 96, 40, 13, "fp32", "fp32", False, 32),
        # eight experts of a 7168 x 2048 layer: bf16 weights with a 32-bit copy, bf16 gradients, moments in 32 bits
        adamw("adamw_32bit", 1, 8, 7168, 2048, 256, "bf16", "bf16", True, 32),
        # the same with fp32 gradients, moments in 8 bits and no 32-bit copy of the weights
        adamw("adamw_8bit", 1, 8, 7168, 2048, 256, "bf16", "fp32", False, 8),
    ]


def router(name, way, n, experts, topk, groups=1, topk_groups=1, group_score="max", score="softmax", bias=False,
           dtype="bf16", renormalize=True, masked=0, scale=1.0):
    return {"name": name, "op": "router", "way": way, "n": n, "experts": experts, "topk": topk, "groups": groups,
            "topk_groups": topk_groups, "group_score": group_score, "score": score, "bias": bias, "dtype": dtype,
            "renormalize": renormalize, "masked": masked, "scale": scale}


def combine(name, n, topk, hidden, experts):
    return {"name": name, "op": "combine_bwd", "n": n, "topk": topk, "hidden": hidden, "experts": experts}


def adamw(name, layers, experts, hidden, inter, routed, param, grad, master, bits):
    return {"name": name, "op": "adamw", "layers": layers, "experts": experts, "hidden": hidden, "inter": inter,
            "routed": routed, "param": param, "grad": grad, "master": master, "bits": bits}


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["router", "router", "combine_bwd", "adamw"])
    if op == "router":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * log_int(rng, 3, 384 // groups)
        kept = rng.randint(1, groups)
        topk = rng.randint(1, min(10, kept * (experts // groups)))
        case = router("", rng.choice(["fwd", "fwd", "bwd"]), log_int(rng, 1, 65536), experts, topk, groups, kept,
                      rng.choice(["max", "top2"]), rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5,
                      rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.6,
                      rng.choice([0, 0, 1]) if experts > topk + 1 else 0, rng.choice([1.0, 2.5]))
    elif op == "combine_bwd":
        topk = rng.randint(1, 8)
        hidden = 8 * log_int(rng, 4, 1792)
        most = 16384 * 8 * 7168 // (topk * hidden)
        case = combine("", log_int(rng, 1, min(16384, most)), topk, hidden, topk + rng.randint(0, 60))
    else:
        layers = rng.randint(1, 12)
        hidden, inter = log_int(rng, 17, 4096), log_int(rng, 9, 2048)
        experts = log_int(rng, 1, max(1, min(16, 300_000_000 // (layers * 3 * hidden * inter))))
        param = rng.choice(["bf16", "bf16", "fp32"])
        case = adamw("", layers, experts, hidden, inter, log_int(rng, 2, 256), param, rng.choice(["bf16", "fp32"]),
                     param == "bf16" and rng.random() < 0.5, rng.choice([8, 32]))
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs
def package():
    import importlib
    return importlib.import_module("mxfp8-grouped-gemm_b200")


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = {"router": router_inputs, "combine_bwd": combine_inputs, "adamw": adamw_inputs}[case["op"]](case, gen)
    state["case"] = case
    if own:
        state["mxg"] = package()
        if case["op"] == "adamw":
            state["opt"] = optimizer(state)
    return state


def normal(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device=DEV).mul_(std).to(dtype)


def router_inputs(case, gen):
    n, E = case["n"], case["experts"]
    logits = normal(gen, n, E, std=1.5)
    if case["masked"]:                                   # experts that are switched off
        off = torch.randperm(E, generator=gen, device=DEV)[:case["masked"]]
        logits[:, off] = -math.inf
    state = {"logits": logits.to(DTYPES[case["dtype"]]),
             "bias": normal(gen, E, std=0.05) if case["bias"] else None}
    if case["way"] == "bwd":
        state["weights"], state["ids"] = router_plain(case, state["logits"], state["bias"])
        state["dweights"] = normal(gen, n, case["topk"])
    return state


def combine_inputs(case, gen):
    n, k, H = case["n"], case["topk"], case["hidden"]
    ids = torch.rand(n, case["experts"], generator=gen, device=DEV).argsort(dim=1)[:, :k]
    order = ids.reshape(-1).sort(stable=True).indices    # send order: by expert, tokens in order
    slot_pos = torch.empty(n * k, dtype=torch.int32, device=DEV)
    slot_pos[order] = torch.arange(n * k, dtype=torch.int32, device=DEV)
    weights = torch.rand(n, k, generator=gen, device=DEV) + 0.05
    return {"dout": normal(gen, n, H, dtype=torch.bfloat16), "rows": normal(gen, n * k, H, dtype=torch.bfloat16),
            "slot_pos": slot_pos.view(n, k), "weights": weights / weights.sum(1, keepdim=True)}


def tensors_of(case):
    """(shape, weight dtype, gradient dtype, has a 32-bit copy, weight decay) of every tensor, in order."""
    E, H, I = case["experts"], case["hidden"], case["inter"]
    p, g, f = DTYPES[case["param"]], DTYPES[case["grad"]], torch.float32
    layer = [((E, 2 * I, H), p, g, case["master"], 0.1), ((E, H, I), p, g, case["master"], 0.1),
             ((case["routed"], H), f, f, False, 0.1), ((H,), f, f, False, 0.0)]
    return layer * case["layers"]


def padded(shape):
    return -(-math.prod(shape) // BLOCK) * BLOCK


def adamw_inputs(case, gen):
    """Weights, gradients and the moments some steps into a run.  The moments are flat: every tensor starts at a
    multiple of 256 values, and zeros fill the gaps."""
    table = tensors_of(case)
    params = [normal(gen, *shape, std=0.02, dtype=p) for shape, p, _, _, _ in table]
    grads = [normal(gen, *shape, std=1e-3, dtype=g) for shape, _, g, _, _ in table]
    real = torch.cat([x for shape, *_ in table for x in
                      (torch.ones(math.prod(shape), dtype=torch.bool, device=DEV),
                       torch.zeros(padded(shape) - math.prod(shape), dtype=torch.bool, device=DEV))])
    state = {"params": params, "grads": grads, "table": table, "step": 40, "seed": 1234,
             "lr": 3e-4, "betas": (0.9, 0.95), "eps": 1e-8, "master": None}
    avg = normal(gen, real.numel(), std=3e-4).mul_(real)
    sq = normal(gen, real.numel(), std=1e-3).square_().add_(1e-8).mul_(real)
    if case["bits"] == 8:
        state["exp_avg"], state["exp_avg_scale"] = encode(avg, 112, None)
        state["exp_avg_sq"], state["exp_avg_sq_scale"] = encode(sq, 96, None)
    else:
        state["exp_avg"], state["exp_avg_sq"] = avg, sq
    if case["master"]:                                   # the 32-bit copies round to the bf16 weights
        kept = [pad(p.float() * (1 + 2.0 ** -11), padded(p.shape)) for p, t in zip(params, table) if t[3]]
        state["master"] = torch.cat(kept)
    return state


def optimizer(state):
    opt = state["mxg"].optim.AdamW(
        state["params"], lr=state["lr"], betas=state["betas"], eps=state["eps"],
        weight_decay=[t[4] for t in state["table"]], state_bits=state["case"]["bits"],
        master_weights=state["case"]["master"], seed=state["seed"])
    opt.load_state_dict({"step": state["step"], "exp_avg": state["exp_avg"], "exp_avg_sq": state["exp_avg_sq"],
                         "exp_avg_scale": state.get("exp_avg_scale"),
                         "exp_avg_sq_scale": state.get("exp_avg_sq_scale"), "master": state["master"]})
    return opt


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "router":
        return run_router(case, state)
    if case["op"] == "combine_bwd":
        if own:
            rows, weights = state["mxg"].ops.combine_bwd(state["dout"], state["rows"], state["slot_pos"],
                                                         state["weights"])
        else:
            rows, weights = combine_bwd_plain(state["dout"], state["rows"], state["slot_pos"], state["weights"])
        return {"rows": rows, "weights": weights}
    if own:
        opt = state["opt"]
        opt.step(state["grads"])
        avg, sq = opt.moments()
        return {"params": state["params"], "exp_avg": avg, "exp_avg_sq": sq, "master": opt.master}
    return adamw_plain(case, state)


def run_router(case, state):
    if case["way"] == "fwd":
        if own:
            weights, ids = state["mxg"].ops.router_topk(
                state["logits"], case["topk"], score=case["score"], bias=state["bias"], groups=case["groups"],
                topk_groups=case["topk_groups"], group_score=case["group_score"], renormalize=case["renormalize"],
                scale=case["scale"])
        else:
            weights, ids = router_plain(case, state["logits"], state["bias"])
        return {"weights": weights, "ids": ids}
    if own:
        return state["mxg"].ops.router_topk_bwd(
            state["logits"], state["weights"], state["ids"], state["dweights"], score=case["score"],
            renormalize=case["renormalize"], scale=case["scale"])
    return router_bwd_plain(case, state["logits"], state["weights"], state["ids"], state["dweights"])


def softmax(z):
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - torch.where(torch.isinf(top) & (top < 0), 0, top))
    total = e.sum(1, keepdim=True)
    return torch.where(total == 0, 0, e / total)         # nothing left in the row: no weight


def sigmoid(z):
    return 1 / (1 + torch.exp(-z))


def router_plain(case, logits, bias):
    """Experts in order of score (+ bias), each tie to the lowest index, from the groups that are kept."""
    n, E = logits.shape
    z = logits.float()
    score = softmax if case["score"] == "softmax" else sigmoid
    # the order is settled in 64 bits: the scores rise with the logits, so without a bias the logits give it
    choice = z if bias is None else score(z.double()) + bias.double()
    G = case["groups"]
    if G > 1:
        per = (choice if bias is not None or case["group_score"] == "max" else score(z.double())).view(n, G, E // G)
        best = per.sort(dim=2, descending=True).values
        group = best[:, :, 0] if case["group_score"] == "max" else best[:, :, :2].sum(2)
        kept = torch.zeros(n, G, dtype=torch.bool, device=logits.device)
        kept.scatter_(1, group.sort(dim=1, descending=True, stable=True).indices[:, :case["topk_groups"]], True)
        kept = kept.repeat_interleave(E // G, dim=1)
        order = choice.sort(dim=1, descending=True, stable=True).indices
        last = (~kept.gather(1, order)).to(torch.int8).sort(dim=1, stable=True).indices
        ids = order.gather(1, last)[:, :case["topk"]]
    else:
        ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :case["topk"]]
    picked = z.gather(1, ids)
    if case["score"] == "softmax":
        weights = softmax(picked) if case["renormalize"] else softmax(z).gather(1, ids)
    else:
        weights = sigmoid(picked)
        if case["renormalize"]:
            weights = weights / weights.sum(1, keepdim=True)
    return weights * case["scale"], ids.to(torch.int32)


def router_bwd_plain(case, logits, weights, ids, dweights):
    at = ids.long()
    z = logits.float()
    if case["score"] == "softmax" and not case["renormalize"]:
        pull = (weights * dweights).sum(1, keepdim=True)
        grad = (-softmax(z) * pull).scatter_add(1, at, weights * dweights)
        return grad.to(logits.dtype)
    if case["renormalize"]:
        share = weights / case["scale"]
        value = weights * (dweights - (share * dweights).sum(1, keepdim=True))
        if case["score"] == "sigmoid":
            value = value * sigmoid(-z.gather(1, at))
    else:
        s = z.gather(1, at)
        value = case["scale"] * dweights * sigmoid(s) * sigmoid(-s)
    return torch.zeros_like(z).scatter_add(1, at, value).to(logits.dtype)


def combine_bwd_plain(dout, rows, slot_pos, weights):
    at = slot_pos.reshape(-1).long()
    n, k = slot_pos.shape
    d = dout.float()
    grad = torch.zeros(rows.shape, dtype=torch.float32, device=rows.device)
    grad[at] = (weights[:, :, None] * d[:, None, :]).view(n * k, -1)
    dw = (rows.float()[at].view(n, k, -1) * d[:, None, :]).sum(2)
    return grad.to(rows.dtype), dw


# ---------------------------------------------------------------- AdamW
def pad(x, size):
    x = x.reshape(-1)
    return torch.cat([x, x.new_zeros(size - x.numel())])


def decode(codes, scale, lift):
    """Values of 8-bit codes.  112: sign, 4 exponent and 3 mantissa bits; 96: no sign, 5 and 3."""
    c = codes.to(torch.int32)
    size = (c & 127) if lift == 112 else c
    v = (size << 20).view(torch.float32) * 2.0 ** lift
    v = (v.view(-1, BLOCK) * scale[:, None]).view(-1)
    return torch.where(c > 127, -v, v) if lift == 112 else v


def encode(x, lift, noise):
    """8-bit codes and scales of x in blocks of 256: the size relative to the block's largest, its lowest 20 bits
    rounded by 20 random bits (to nearest where noise is None); what is above zero in the second moment stays so."""
    scale = x.view(-1, BLOCK).abs().amax(1).clamp_min(2.0 ** -100)
    ratio = (x.abs().view(-1, BLOCK) * (1 / scale)[:, None]).view(-1) * 2.0 ** -lift
    bits = ratio.view(torch.int32)
    code = (bits + (2 ** 19 if noise is None else noise)) >> 20
    if lift == 112:
        code = code.clamp_max(127) | ((x < 0).to(torch.int32) << 7)
    else:
        code = code.clamp_max(255).maximum((x > 0).to(torch.int32))
    return code.to(torch.uint8), scale


def mix(x, by):
    p = x * by
    return (p >> 32) ^ (p & 0xFFFFFFFF)


M1, M2, STEP, ADD, ALL = 0x6A09C55D, 0x5D1B8E63, 0x9E2F4D8B, 0x3C7A15E9, 0xFFFFFFFF


def random_words(seed, step, size):
    """Two 32-bit words for each value of a flat state, from the seed, the step and the value's place."""
    i = torch.arange(size, dtype=torch.int64, device=DEV)
    k = mix(((seed & ALL) + ADD) & ALL, M1)
    k = mix(k ^ (seed >> 32) ^ ADD, M2)
    k = mix((k + step + STEP) & ALL, M1)
    block = torch.arange(size // BLOCK, dtype=torch.int64, device=DEV)
    kb = mix((k + (block & ALL) + ADD) & ALL, M1)
    kb = mix(((kb ^ (block >> 32)) + STEP) & ALL, M2)
    x = (kb[:, None] ^ ((i.view(-1, BLOCK) & 255) * STEP & ALL)).view(-1)
    h = mix(mix((x + ADD) & ALL, M1) ^ STEP, M2)
    return h, mix((h ^ ADD) & ALL, M1)


def adamw_plain(case, state):
    """Every tensor laid flat (padded as the moments are), one update in 32 bits, and the weights written back."""
    state["step"] += 1
    step, table = state["step"], state["table"]
    lr, (b1, b2), eps = state["lr"], state["betas"], state["eps"]
    sizes = [padded(t[0]) for t in table]
    g = torch.cat([pad(x.float(), s) for x, s in zip(state["grads"], sizes)])
    copies = iter([] if state["master"] is None else state["master"].split([s for s, t in zip(sizes, table) if t[3]]))
    copies = [next(copies) if t[3] else None for t in table]
    p = torch.cat([pad(x.float(), s) if c is None else c for x, s, c in zip(state["params"], sizes, copies)])
    decay = torch.cat([torch.full((s,), t[4], device=DEV) for s, t in zip(sizes, table)])
    if case["bits"] == 8:
        avg = decode(state["exp_avg"], state["exp_avg_scale"], 112)
        sq = decode(state["exp_avg_sq"], state["exp_avg_sq_scale"], 96)
        words, more = random_words(state["seed"], step, g.numel())
    else:
        avg, sq = state["exp_avg"], state["exp_avg_sq"]
        more = random_words(state["seed"], step, g.numel())[1] if rounded(case) else None
    avg = avg * b1 + g * (1 - b1)
    sq = sq * b2 + (g * g) * (1 - b2)
    down = (sq / (1 - b2 ** step)).sqrt() + eps
    p = p * (1 - lr * decay) - (lr / (1 - b1 ** step)) * (avg / down)
    parts = p.split(sizes)
    whole = [q[:x.numel()].view(x.shape) for q, x in zip(parts, state["params"])]
    if rounded(case):                                    # bf16 without a 32-bit copy: 16 random bits decide
        up = ((p.view(torch.int32) + (more & 0xFFFF).to(torch.int32)) & -65536).view(torch.float32)
        up = [q[:x.numel()].view(x.shape) for q, x in zip(up.split(sizes), state["params"])]
        whole = [u if x.dtype == torch.bfloat16 else q for u, q, x in zip(up, whole, state["params"])]
    torch._foreach_copy_(state["params"], whole)
    if state["master"] is not None:
        state["master"] = torch.cat([q for q, t in zip(parts, table) if t[3]])
    if case["bits"] == 8:
        state["exp_avg"], state["exp_avg_scale"] = encode(avg, 112, ((words >> 16) << 4 | 8).to(torch.int32))
        state["exp_avg_sq"], state["exp_avg_sq_scale"] = encode(sq, 96, ((words & 0xFFFF) << 4 | 8).to(torch.int32))
        avg = decode(state["exp_avg"], state["exp_avg_scale"], 112)
        sq = decode(state["exp_avg_sq"], state["exp_avg_sq_scale"], 96)
    else:
        state["exp_avg"], state["exp_avg_sq"] = avg, sq
    return {"params": state["params"], "exp_avg": avg, "exp_avg_sq": sq, "master": state["master"]}


def rounded(case):
    return case["param"] == "bf16" and not case["master"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "router":
        n, E, k = case["n"], case["experts"], case["topk"]
        size = DTYPES[case["dtype"]].itemsize
        if case["way"] == "fwd":
            return {"bytes": n * E * size + 4 * E * case["bias"] + 8 * n * k, "flops": 8 * n * E}
        reads = 12 * n * k
        if case["score"] == "softmax" and not case["renormalize"]:
            reads += n * E * size
        elif case["score"] == "sigmoid":
            reads += n * k * size
        return {"bytes": reads + n * E * size, "flops": 4 * n * E}
    if case["op"] == "combine_bwd":
        n, k, H = case["n"], case["topk"], case["hidden"]
        return {"bytes": 2 * n * H + 4 * n * k * H + 12 * n * k, "flops": 3 * n * k * H}
    total = flops = 0
    for shape, p, g, master, _ in tensors_of(case):
        size = math.prod(shape)
        weights = 8 + p.itemsize if master else 2 * p.itemsize
        # 8 bits: codes and scales in and out, and the values that they stand for as the pass returns them
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
        total += size * (weights + g.itemsize + moments)
        flops += size * 18
    return {"bytes": int(total), "flops": flops}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "router":
        return router_exact(case, router_inputs(case, gen))
    if case["op"] == "combine_bwd":
        s = combine_inputs(case, gen)
        rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device=DEV)
        weights = torch.empty(s["weights"].shape, dtype=torch.float64, device=DEV)
        for j in range(case["topk"]):
            at = s["slot_pos"][:, j].long()
            rows[at] = s["weights"][:, j:j + 1].double() * s["dout"].double()
            weights[:, j] = torch.einsum("nh,nh->n", s["rows"][at].double(), s["dout"].double())
        return {"rows": rows, "weights": weights}
    return adamw_exact(case, adamw_inputs(case, gen))


def scores_exact(case, z):
    if case["score"] == "sigmoid":
        return torch.sigmoid(z)
    return torch.nan_to_num(torch.softmax(z, 1), nan=0.0)


def router_exact(case, s):
    z = s["logits"].double().cpu().numpy()
    n, E = z.shape
    score = scores_exact(case, s["logits"].double()).cpu().numpy()
    if case["way"] == "fwd":
        choice = z if s["bias"] is None else score + s["bias"].double().cpu().numpy()
        allowed = np.ones((n, E), dtype=bool)
        if case["groups"] > 1:
            G = case["groups"]
            by = choice if s["bias"] is not None else score
            best = -np.sort(-by.reshape(n, G, E // G), axis=2)
            total = best[:, :, 0] if case["group_score"] == "max" else best[:, :, :2].sum(2)
            rank = np.argsort(np.argsort(-total, axis=1, kind="stable"), axis=1, kind="stable")
            allowed = np.repeat(rank < case["topk_groups"], E // G, axis=1)
        place = np.broadcast_to(np.arange(E), (n, E))
        ids = np.lexsort((place, -choice, ~allowed), axis=1)[:, :case["topk"]]
        w = np.take_along_axis(score, ids, 1)
        if case["renormalize"]:
            w = w / w.sum(1, keepdims=True)
        return {"weights": w * case["scale"], "ids": ids.astype(np.int32)}
    # the gradient by the chain rule from the scores, weights = scale * s / (sum of the chosen s, or 1)
    ids = s["ids"].long().cpu().numpy()
    dw = s["dweights"].double().cpu().numpy() * case["scale"]
    picked = np.take_along_axis(score, ids, 1)
    if case["renormalize"]:
        total = picked.sum(1, keepdims=True)
        dpick = dw / total - (dw * picked).sum(1, keepdims=True) / total ** 2
    else:
        dpick = dw
    ds = np.zeros((n, E))
    np.put_along_axis(ds, ids, dpick, 1)
    if case["score"] == "sigmoid":
        return ds * score * (1 - score)
    return score * (ds - (score * ds).sum(1, keepdims=True))


def adamw_exact(case, s):
    step = s["step"] + 1
    lr, (b1, b2), eps = s["lr"], s["betas"], s["eps"]
    out = {"params": [], "exp_avg": [], "exp_avg_sq": [], "master": []}
    total = s["exp_avg"].numel()
    more = random_words(s["seed"], step, total)[1] if rounded(case) else None
    at = kept = 0
    for p, g, (shape, _, _, master, decay) in zip(s["params"], s["grads"], s["table"]):
        size, room = p.numel(), padded(shape)
        if case["bits"] == 8:
            b = slice(at // BLOCK, (at + room) // BLOCK)
            m = small_float(s["exp_avg"][at:at + room], s["exp_avg_scale"][b], True)
            v = small_float(s["exp_avg_sq"][at:at + room], s["exp_avg_sq_scale"][b], False)
        else:
            m, v = s["exp_avg"][at:at + room].double(), s["exp_avg_sq"][at:at + room].double()
        grad = pad(g.double(), room)
        m = b1 * m + (1 - b1) * grad
        v = b2 * v + (1 - b2) * grad ** 2
        w = s["master"][kept:kept + size].double() if master else p.double().reshape(-1)
        step_by = (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + eps)
        w = w - lr * decay * w - lr * step_by[:size]
        if master:
            out["master"].append(pad(w, room))
            kept += room
        elif p.dtype == torch.bfloat16:                  # which neighbour is drawn goes by the random bits
            gap = 2.0 ** (torch.frexp(w.abs())[1].double() - 8)
            w = torch.sign(w) * gap * torch.floor(w.abs() / gap + (more[at:at + size] & 0xFFFF).double() / 65536)
        out["params"].append(w.view(shape))
        out["exp_avg"].append(m)
        out["exp_avg_sq"].append(v)
        at += room
    if case["bits"] == 8:      # which code is drawn goes by the last bit of the 32-bit moment: no value in 64 bits
        out["exp_avg"] = out["exp_avg_sq"] = None
    else:
        out["exp_avg"], out["exp_avg_sq"] = torch.cat(out["exp_avg"]), torch.cat(out["exp_avg_sq"])
    return dict(out, master=torch.cat(out["master"]) if out["master"] else None)


def small_float(codes, scale, signed):
    """mantissa * 2^exponent of a code, 3 mantissa bits, the lowest exponent without the leading one."""
    c = codes.double()
    sign = torch.where(c >= 128, -1.0, 1.0) if signed else torch.ones_like(c)
    c = torch.where(c >= 128, c - 128, c) if signed else c
    e, f = torch.floor(c / 8), torch.remainder(c, 8) / 8
    top = 15 if signed else 31
    value = torch.where(e == 0, f * 2.0 ** (1 - top), (1 + f) * 2.0 ** (e - top))
    return (sign * value).view(-1, BLOCK).mul(scale.double()[:, None]).view(-1)

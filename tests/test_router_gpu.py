"""Expert routing (choice, weights, gradient) and the combine's gradient
against the definitions in 64 bits.

Tolerances.  A weight is a quotient of sums of exp(x) with |x| <= 16 here.
exp(x) through 2^(x log2 e): the product's rounding and the constant's give
1.5 |x| 2^-24 <= 1.5e-6, the instruction 2^-22; a sum of up to 384 of them
adds 13 roundings in a tree (8e-7 at most); numerator, sum, quotient and
scale together stay below 2 (1.5e-6 + 2.4e-7) + 8e-7 + 1.2e-7 < 5e-6.
A gradient is a product of such weights and differences of terms of the size
of sum |w dw|: 1e-5 of that sum, and half a step of the logits' type."""
import numpy as np
import pytest
import torch

from oracle import router_oracle as ro

pytestmark = pytest.mark.gpu

W_TOL, G_TOL = 5e-6, 1e-5
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _logits(n, E, dtype, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(n, E, generator=g, device=dev).mul_(1.5).clamp_(-8, 8).to(DT[dtype])


def _np(t):
    return t.detach().float().cpu().numpy()


def _check(mxg, z, k, bias=None, **how):
    w, ids = mxg.ops.router_topk(z, k, bias=bias, **how)
    assert mxg.device_error() == 0
    ref_w, ref_ids = ro.router(_np(z), k, bias=None if bias is None else _np(bias), **how)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and ids.shape == (z.shape[0], k)
    assert np.array_equal(ids.cpu().numpy(), ref_ids)
    got = w.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref_w))
    ok = ~np.isnan(ref_w)
    assert np.all(np.abs(got[ok] - ref_w[ok]) <= W_TOL * np.abs(ref_w[ok]) + 1e-37)
    return w, ids


# E covers every lane layout, whole and ragged
@pytest.mark.parametrize("E,k", [(1, 1), (3, 2), (8, 2), (8, 8), (13, 5), (16, 4), (31, 8), (32, 32), (60, 4), (64, 6),
                                 (100, 3), (128, 8), (137, 7), (160, 6), (255, 9), (256, 8), (257, 1), (384, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_choice_and_weights(mxg, cuda_dev, E, k, dtype, score):
    for n in (1, 3, 517):
        z = _logits(n, E, dtype, E * n, cuda_dev)
        bias = torch.randn(E, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(E)) * 0.05
        _check(mxg, z, k, score=score, renormalize=True, scale=2.5)
        _check(mxg, z, k, score=score, renormalize=False)
        _check(mxg, z, k, score=score, bias=bias, renormalize=True)


@pytest.mark.parametrize("E,groups,kept,k", [(8, 4, 2, 4), (8, 8, 3, 3), (16, 4, 3, 6), (48, 3, 2, 5), (64, 8, 4, 6),
                                             (96, 32, 7, 8), (160, 8, 3, 6), (256, 8, 4, 8), (256, 8, 1, 32),
                                             (384, 12, 5, 9), (384, 2, 1, 8)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_groups(mxg, cuda_dev, E, groups, kept, k, group_score, dtype):
    z = _logits(301, E, dtype, E + groups, cuda_dev)
    bias = torch.randn(E, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(E)) * 0.05
    how = dict(groups=groups, topk_groups=kept, group_score=group_score)
    for score in ("softmax", "sigmoid"):
        _check(mxg, z, k, score=score, **how)
        _check(mxg, z, k, score=score, bias=bias, renormalize=False, **how)


@pytest.mark.parametrize("E,groups,kept", [(137, 1, 1), (160, 5, 2), (192, 3, 2), (256, 1, 1), (256, 8, 4), (256, 2, 1),
                                           (257, 1, 1), (384, 1, 1), (384, 12, 4)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_long_batches(mxg, cuda_dev, E, groups, kept, dtype):
    """Enough tokens for the layout of several tokens a warp at every E."""
    z = _logits(8203, E, dtype, E + groups, cuda_dev)
    z[17] = -float("inf")
    z[18, 3:] = -float("inf")
    z[:, E // 2] = -float("inf")
    bias = torch.randn(E, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(E)) * 0.05
    how = dict(groups=groups, topk_groups=kept)
    for score in ("softmax", "sigmoid"):
        _check(mxg, z, 8, score=score, **how)
        _check(mxg, z, 5, score=score, renormalize=False, group_score="top2", **how)
        _check(mxg, z, 8, score=score, bias=bias, group_score="top2", renormalize=False, **how)
        _check(mxg, z, 7, score=score, bias=bias * 40, **how)
    _check(mxg, torch.zeros_like(z), 8, score="sigmoid", bias=bias * 0, **how)


@pytest.mark.parametrize("n", [64, 4200])
@pytest.mark.parametrize("many", [12, 200])
def test_long_rows_of_near_ties(mxg, cuda_dev, n, many):
    """s + bias of `many` of 256 experts meets at 1 to the last places of fp32."""
    g = torch.Generator(device=cuda_dev).manual_seed(many)
    bias = torch.rand(256, generator=g, device=cuda_dev) * 0.5 + 0.2
    s = 1 - bias.double() + torch.randn(n, 256, generator=g, device=cuda_dev, dtype=torch.float64) * 4e-8
    s[:, torch.randperm(256, generator=g, device=cuda_dev)[many:]] *= 0.5
    z = torch.log(s / (1 - s)).float()
    _check(mxg, z, 8, score="sigmoid", bias=bias)
    _check(mxg, z, 3, score="sigmoid", bias=bias, groups=8, topk_groups=4, group_score="top2")
    _check(mxg, z, 3, score="sigmoid", bias=bias, groups=8, topk_groups=4)


def test_ties_go_to_the_lowest_index(mxg, cuda_dev):
    z = torch.zeros(5, 256, device=cuda_dev)
    z[1, 200:] = 1.0
    z[2, ::2] = -0.0
    z[3] = torch.arange(256, device=cuda_dev) // 64
    z[4, 7] = z[4, 250] = 3.0
    zero = torch.zeros(256, device=cuda_dev)
    for score in ("softmax", "sigmoid"):
        for bias in (None, zero, zero + 0.25):
            for how in ({}, dict(groups=8, topk_groups=3), dict(groups=8, topk_groups=3, group_score="top2")):
                _check(mxg, z, 8, score=score, bias=bias, **how)
    assert mxg.ops.router_topk(z, 8)[1][0].tolist() == list(range(8))


def test_choices_that_32_bits_cannot_tell_apart(mxg, cuda_dev):
    """s + bias of many experts within a few units of the last place."""
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    z = _logits(400, 256, "fp32", 9, cuda_dev)
    s = 1 / (1 + torch.exp(-z.double()))
    jitter = torch.randn(256, generator=g, device=cuda_dev) * 3e-8
    for t in range(0, 400, 40):                 # this row's scores plus the bias almost meet at 1
        bias = (1 - s[t]).float() + jitter
        _check(mxg, z[t:t + 4].contiguous(), 8, score="sigmoid", bias=bias)
        _check(mxg, z[t:t + 4].contiguous(), 8, score="sigmoid", bias=bias, groups=8, topk_groups=4,
               group_score="top2")


@pytest.mark.parametrize("E", [64, 256, 384])
@pytest.mark.parametrize("n", [40, 8200])
def test_equal_experts_at_the_last_choice(mxg, cuda_dev, E, n):
    """Two equal experts stand on either side of the last choice, and a later
    one is larger by the last place of fp32: it comes before both."""
    g = torch.Generator(device=cuda_dev).manual_seed(E + n)
    z = torch.rand(n, E, generator=g, device=cuda_dev)
    for k, equal in ((1, 2), (3, 2), (3, 4), (8, 2), (8, 3), (8, 12)):
        # `equal` experts at 1.5, the last of them one place higher, and k - 1 above
        at = torch.rand(n, E, generator=g, device=cuda_dev).argsort(1)
        ties = at[:, :equal + 1].sort(1).values
        near = z.scatter(1, ties, 1.5)
        near.scatter_(1, ties[:, -1:], 1.5 + 2.0 ** -23)
        near.scatter_(1, at[:, equal + 1:equal + k], 2.0 + z[:, :k - 1])
        bias = torch.full((E,), 0.25, device=cuda_dev)
        _check(mxg, near, k)
        for score in ("softmax", "sigmoid"):
            _check(mxg, near, k, score=score, bias=bias)
        if E == 256:
            _check(mxg, near, k, score="sigmoid", bias=bias, groups=8, topk_groups=8)


@pytest.mark.parametrize("E", [40, 256, 384])
@pytest.mark.parametrize("n", [70, 8203])
def test_many_ties(mxg, cuda_dev, E, n):
    """Logits of few digits in every type, and a bias of zero."""
    zero = torch.zeros(E, device=cuda_dev)
    for dtype in DT.values():
        z = _logits(n, E, "bf16", E, cuda_dev).to(dtype)
        _check(mxg, z, 8)
        _check(mxg, z, 3, groups=2, topk_groups=1)
        for score in ("softmax", "sigmoid"):
            _check(mxg, z, 8, score=score, bias=zero)


@pytest.mark.parametrize("E", [16, 40, 256, 384])
@pytest.mark.parametrize("n", [20, 8200])
def test_logits_and_biases_far_from_zero(mxg, cuda_dev, E, n):
    """Softmax does not change with an offset, the choice does not with either."""
    g = torch.Generator(device=cuda_dev).manual_seed(E)
    z = torch.randn(n, E, generator=g, device=cuda_dev).mul_(1.5)
    b = torch.randn(E, generator=g, device=cuda_dev)
    for off in (-1e4, -300.0, -61.7, 61.7, 5e3, 1e30):
        _check(mxg, z + off, 4)
        _check(mxg, z + off, 8, renormalize=False)
    for score in ("softmax", "sigmoid"):
        for by in (3.0, 12.0, 1e3, 1e6):
            _check(mxg, z, 4, score=score, bias=b * by)
            _check(mxg, z, 8, score=score, bias=b + by)


@pytest.mark.parametrize("E", [8, 64, 160, 256])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_experts_and_rows(mxg, cuda_dev, E, score):
    inf = float("inf")
    z = _logits(9, E, "fp32", 5, cuda_dev)
    z[0] = -inf                                  # nothing left
    z[1, 1:] = -inf                              # one expert left
    z[2, ::2] = -inf
    z[3] = torch.finfo(torch.float32).min        # the type's lowest value
    z[4, 3] = torch.finfo(torch.float32).min
    z[5] = -200.0                                # scores that vanish in fp32
    z[5, 2] = -201.0
    z[6, :4] = 100.0
    for renorm in (True, False):
        w, ids = mxg.ops.router_topk(z, 4, score=score, renormalize=renorm)
        ref_w, ref_ids = ro.router(_np(z), 4, score=score, renormalize=renorm)
        assert np.array_equal(ids.cpu().numpy(), ref_ids)
        assert torch.all(w[0] == 0) if score == "softmax" or not renorm else True
        keep = np.isfinite(ref_w) & (np.abs(ref_w) > 1e-30)
        keep[3] &= score == "softmax"            # sigmoid's oracle has no share of scores of 0
        got = w.cpu().numpy()
        # |x| up to 201 in the exponent: 1.5 * 201 * 2^-24 * 2 more
        assert np.all(np.abs(got[keep] - ref_w[keep]) <= 4.5e-5 * np.abs(ref_w[keep]))
        assert np.all(np.isfinite(got))
    assert torch.all(mxg.ops.router_topk(z, 4, score=score)[0][0] == 0)
    dz = mxg.ops.router_topk_bwd(z, *mxg.ops.router_topk(z, 4, score=score), torch.ones(9, 4, device=cuda_dev),
                                 score=score)
    assert torch.isfinite(dz).all() and torch.all(dz[0] == 0)
    bias = torch.zeros(E, device=cuda_dev)
    bias[1:5] = -inf                             # switched off by the bias
    _, ids = mxg.ops.router_topk(_logits(64, E, "bf16", 1, cuda_dev), 3, score=score, bias=bias)
    assert not torch.isin(ids, torch.arange(1, 5, device=cuda_dev)).any()


@pytest.mark.parametrize("E", [17, 64, 256, 384])
@pytest.mark.parametrize("n", [3, 8200])
def test_rows_without_an_expert_go_by_the_bias(mxg, cuda_dev, E, n):
    """Every score is 0: the order is the bias's, however close its values are."""
    g = torch.Generator(device=cuda_dev).manual_seed(E)
    z = torch.randn(n, E, generator=g, device=cuda_dev)
    z[1::2] = -float("inf")
    bias = torch.randint(-2, 3, (E,), generator=g, device=cuda_dev).float() * 1e-7
    for score in ("softmax", "sigmoid"):
        for k in (1, 4, 8):
            _check(mxg, z, k, score=score, bias=bias)


@pytest.mark.parametrize("E", [7, 24, 64, 256])
@pytest.mark.parametrize("n", [40, 4200])
def test_scores_at_the_end_of_the_range_of_fp32(mxg, cuda_dev, E, n):
    """Scores and biases of about 1e-38 beside a larger one."""
    g = torch.Generator(device=cuda_dev).manual_seed(E)
    z = torch.rand(n, E, generator=g, device=cuda_dev) * 6 - 91
    z[:, E // 2] = -79.0
    bias = -torch.sigmoid(z[0].double()).float()
    for k in (1, 4, 7):
        _check(mxg, z, k, score="sigmoid", bias=bias)
        _check(mxg, z + 79, k, score="softmax", bias=bias)
        if E != 7:
            _check(mxg, z, k, score="sigmoid", bias=bias, groups=8, topk_groups=5, group_score="top2")


def test_nan_rows_have_ids_in_range(mxg, cuda_dev):
    z = _logits(6, 256, "fp32", 5, cuda_dev)
    z[0, 17] = z[1, :] = float("nan")
    z[2, 5] = float("inf")
    bias = torch.zeros(256, device=cuda_dev)
    for b in (None, bias):
        for how in ({}, dict(groups=8, topk_groups=2, group_score="top2")):
            w, ids = mxg.ops.router_topk(z, 8, bias=b, **how)
            assert torch.isnan(w[:3]).all() and torch.isfinite(w[3:]).all()
            assert ids.min() >= 0 and ids.max() < 256
            assert all(len(set(r)) == 8 for r in ids.tolist())
    w, ids = mxg.ops.router_topk(z, 8, score="sigmoid")
    assert torch.isfinite(w[0]).all() and 17 not in ids[0].tolist()
    bias[3] = float("nan")
    w, ids = mxg.ops.router_topk(z[3:], 8, score="sigmoid", bias=bias)
    assert torch.isfinite(w).all() and not (ids == 3).any()


def test_strided_and_misaligned_rows(mxg, cuda_dev):
    for dtype in DT:
        wide = _logits(70, 300, dtype, 8, cuda_dev)
        for view in (wide[:, 8:264], wide[:, 3:259], wide[::2, 40:168], wide[:, :256].t().contiguous().t(),
                     wide[:1].expand(5, 300)[:, :64], wide[5:6, 1:9]):
            w, ids = _check(mxg, view, 4, score="sigmoid")
            dw = torch.ones_like(w)
            a = mxg.ops.router_topk_bwd(view, w, ids, dw, score="sigmoid")
            b = mxg.ops.router_topk_bwd(view.contiguous(), w, ids, dw, score="sigmoid")
            assert torch.equal(a, b)


def test_no_tokens(mxg, cuda_dev):
    z = torch.empty(0, 64, device=cuda_dev)
    w, ids = mxg.ops.router_topk(z, 4)
    assert w.shape == ids.shape == (0, 4)
    assert mxg.ops.router_topk_bwd(z, w, ids, w).shape == (0, 64)


@pytest.mark.parametrize("E,k", [(1, 1), (5, 3), (8, 2), (24, 24), (64, 6), (137, 6), (256, 8), (384, 10)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_gradient(mxg, cuda_dev, E, k, score, renorm, dtype):
    z = _logits(203, E, dtype, E + k, cuda_dev)
    how = dict(score=score, renormalize=renorm, scale=2.5)
    w, ids = mxg.ops.router_topk(z, k, **how)
    dw = torch.randn(203, k, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(1))
    dz = mxg.ops.router_topk_bwd(z, w, ids, dw, **how)
    assert dz.dtype == z.dtype and dz.shape == z.shape
    ref = ro.router_bwd(_np(z), ids.cpu().numpy(), _np(dw), **how)
    size = np.abs(_np(w) * _np(dw)).sum(1, keepdims=True)
    half = 0.0 if dtype == "fp32" else torch.finfo(DT[dtype]).eps / 2
    tiny = torch.finfo(DT[dtype]).smallest_normal * torch.finfo(DT[dtype]).eps
    assert np.all(np.abs(_np(dz) - ref) <= G_TOL * size + half * np.abs(ref) + tiny)


def test_gradient_against_differences(mxg, cuda_dev):
    """Central differences of the oracle's weights at the kernel's choice."""
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            z = _logits(4, 24, "fp32", 2, cuda_dev)
            leaf = z.clone().requires_grad_(True)
            w, ids = mxg.router_topk(leaf, 3, score=score, renormalize=renorm, scale=1.5)
            up = torch.randn(4, 3, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(7))
            (w * up).sum().backward()
            zz, at = _np(z).astype(np.float64), ids.cpu().numpy().astype(np.int64)

            def value(x):
                s = np.take_along_axis(ro.scores(x, score), at, 1)
                s = s / s.sum(1, keepdims=True) if renorm else s
                return (1.5 * s * _np(up)).sum(1)
            for e in range(24):
                d = np.zeros((1, 24))
                d[0, e] = 1e-5
                slope = (value(zz + d) - value(zz - d)) / 2e-5     # error: h^2 f''' / 6 < 1e-9, 1e-16 / h
                assert np.all(np.abs(leaf.grad[:, e].cpu().numpy() - slope) < 1e-5)


def test_gradient_of_ids_named_twice_and_out_of_range(mxg, cuda_dev):
    z = _logits(3, 64, "fp32", 4, cuda_dev)
    ids = torch.tensor([[5, 5, 9], [1, 2, 1], [0, 63, 7]], dtype=torch.int32, device=cuda_dev)
    w = torch.rand(3, 3, device=cuda_dev)
    dw = torch.randn(3, 3, device=cuda_dev)
    dz = mxg.ops.router_topk_bwd(z, w, ids, dw, score="sigmoid", renormalize=False)
    ref = ro.router_bwd(_np(z), ids.cpu().numpy(), _np(dw), score="sigmoid", renormalize=False)
    assert np.all(np.abs(_np(dz) - ref) <= G_TOL * np.abs(_np(dw)).sum())
    ids[0, 1], ids[2, 2] = -1, 64
    dz = mxg.ops.router_topk_bwd(z, w, ids, dw, score="sigmoid", renormalize=False)
    assert mxg.device_error() == mxg._lib.MXG_ERR_INVALID_ARGUMENT
    assert torch.isfinite(dz).all() and int((dz != 0).sum()) == 2 + 2 + 2
    assert mxg.device_error() == 0


def test_long_batch_passes_32_bit_offsets(mxg, cuda_dev):
    n, E = 5_700_000, 384                        # n * E > 2^31
    z = torch.zeros(n, E, dtype=torch.bfloat16, device=cuda_dev)
    z[-300:] = _logits(300, E, "bf16", 6, cuda_dev)
    w, ids = mxg.ops.router_topk(z, 6, renormalize=False)
    ref_w, ref_ids = ro.router(_np(z[-300:]), 6, renormalize=False)
    assert np.array_equal(ids[-300:].cpu().numpy(), ref_ids)
    assert np.all(np.abs(_np(w[-300:]) - ref_w) <= W_TOL * ref_w)
    dw = torch.ones_like(w)
    dz = mxg.ops.router_topk_bwd(z, w, ids, dw, renormalize=False)
    small = mxg.ops.router_topk_bwd(z[-300:], w[-300:], ids[-300:], dw[-300:], renormalize=False)
    assert torch.equal(dz[-300:], small)
    del z, dz, w, ids, dw, small
    torch.cuda.empty_cache()


def test_captured_and_on_another_stream(mxg, cuda_dev):
    z = _logits(64, 256, "fp32", 1, cuda_dev)
    bias = torch.randn(256, device=cuda_dev) * 0.05
    how = dict(score="sigmoid", bias=bias, groups=8, topk_groups=4, group_score="top2")
    want = mxg.ops.router_topk(z, 8, **how)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mxg.ops.router_topk(z, 8, **how)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids = mxg.ops.router_topk(z, 8, **how)
        dz = mxg.ops.router_topk_bwd(z, w, ids, torch.ones_like(w), score="sigmoid")
    z.copy_(_logits(64, 256, "fp32", 2, cuda_dev))
    graph.replay()
    want = mxg.ops.router_topk(z, 8, **how)
    assert torch.equal(w, want[0]) and torch.equal(ids, want[1])
    assert torch.equal(dz, mxg.ops.router_topk_bwd(z, w, ids, torch.ones_like(w), score="sigmoid"))


# ---------------------------------------------------------------- the combine's gradient
def _combine_inputs(n, k, H, P, seed, dev, missing=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    dout = torch.randn(n, H, generator=g, device=dev).to(torch.bfloat16)
    rows = torch.randn(P, H, generator=g, device=dev).to(torch.bfloat16)
    pos = torch.randperm(P, generator=g, device=dev)[:n * k].to(torch.int32).view(n, k)
    if missing:
        pos.view(-1)[torch.randperm(n * k, generator=g, device=dev)[:missing]] = -1
    return dout, rows, pos, torch.rand(n, k, generator=g, device=dev) + 0.1


@pytest.mark.parametrize("n,k,H,extra,missing", [(1, 1, 8, 0, 0), (1, 8, 512, 0, 0), (33, 2, 520, 0, 3), (7, 3, 2048, 5, 0),
                                                 (96, 2, 512, 0, 0), (5, 6, 4104, 0, 2), (3, 8, 7168, 1, 1),
                                                 (2, 32, 14336, 0, 0), (4, 5, 8200, 300, 4)])
def test_combine_gradient(mxg, cuda_dev, n, k, H, extra, missing):
    """A dot product of H terms: its fp32 sum runs over at most H / 8 + 13
    roundings of partial sums, each below sum |x y|."""
    dout, rows, pos, w = _combine_inputs(n, k, H, n * k + extra, n + H, cuda_dev, missing)
    for weights in (w, None):
        drows, dw = mxg.ops.combine_bwd(dout, rows, pos, weights)
        ref_rows, ref_dw = ro.combine_bwd(_np(dout), _np(rows), pos.cpu().numpy(), None if weights is None else _np(w))
        assert mxg.device_error() == 0
        assert np.all(np.abs(_np(drows) - ref_rows) <= (2.0 ** -8 + 2.0 ** -23) * np.abs(ref_rows))
        size = ro.combine_bwd(np.abs(_np(dout)), np.abs(_np(rows)), pos.cpu().numpy(), None)[1]
        assert np.all(np.abs(_np(dw) - ref_dw) <= (H / 8 + 13) * 2.0 ** -24 * size)
        assert torch.equal(mxg.ops.combine_bwd(dout, rows, pos, weights, need_weights=False)[0], drows)
        assert torch.equal(mxg.ops.combine_bwd(dout, rows, pos, weights, need_rows=False)[1], dw)


def test_combine_gradient_of_rows_that_nothing_names(mxg, cuda_dev):
    """More rows than one block looks after, most of them named by nothing."""
    for n, k, P, missing in ((40, 2, 100_003, 5), (16_500, 2, 33_000, 7), (9000, 8, 72_001, 0)):
        dout, rows, pos, w = _combine_inputs(n, k, 64, P, n, cuda_dev, missing)
        drows, dw = mxg.ops.combine_bwd(dout, rows, pos, w)
        want = torch.zeros_like(rows)
        ok = pos >= 0
        t = torch.arange(n, device=cuda_dev)[:, None].expand(n, k)[ok]
        want[pos[ok].long()] = (w[ok][:, None] * dout[t].float()).to(torch.bfloat16)
        assert torch.equal(drows, want) and torch.all(dw[~ok] == 0)


def test_combine_gradient_skips_positions_beyond_the_rows(mxg, cuda_dev):
    dout, rows, pos, w = _combine_inputs(16, 2, 64, 32, 1, cuda_dev)
    lost = int(pos[3, 1])
    pos[3, 1] = 32
    drows, dw = mxg.ops.combine_bwd(dout, rows, pos, w)
    assert mxg.device_error() == mxg._lib.MXG_ERR_INVALID_ARGUMENT
    assert dw[3, 1] == 0 and torch.all(drows[lost] == 0)
    mxg.ops.combine(rows, pos, w)
    assert mxg.device_error() == mxg._lib.MXG_ERR_INVALID_ARGUMENT


def test_combine_gradient_reports_a_row_named_twice(mxg, cuda_dev):
    dout, rows, pos, w = _combine_inputs(40, 2, 64, 80, 2, cuda_dev)
    pos[7, 0] = pos[30, 1]
    drows, dw = mxg.ops.combine_bwd(dout, rows, pos, w)
    assert mxg.device_error() == mxg._lib.MXG_ERR_INVALID_ARGUMENT
    at = int(pos[7, 0])
    either = [(w[t, j] * dout[t].float()).to(torch.bfloat16) for t, j in ((7, 0), (30, 1))]
    assert torch.all((drows[at] == either[0]) | (drows[at] == either[1])) and torch.isfinite(dw).all()


def test_combine_gradient_without_tokens(mxg, cuda_dev):
    rows = torch.ones(3, 16, dtype=torch.bfloat16, device=cuda_dev)
    drows, dw = mxg.ops.combine_bwd(rows[:0], rows, torch.empty(0, 2, dtype=torch.int32, device=cuda_dev))
    assert torch.all(drows == 0) and dw.shape == (0, 2)


def test_combine_gradient_passes_32_bit_offsets(mxg, cuda_dev):
    n, k, H = 37_500, 8, 7168                    # n * k * H > 2^31
    dout, rows, pos, w = _combine_inputs(n, k, H, n * k, 3, cuda_dev)
    drows, dw = mxg.ops.combine_bwd(dout, rows, pos, w)
    for t in (0, n // 2, n - 1):
        at = pos[t].long()
        assert torch.equal(drows[at], (w[t][:, None] * dout[t].float()).to(torch.bfloat16))
        want = (dout[t].double() * rows[at].double()).sum(1)
        size = (dout[t].double() * rows[at].double()).abs().sum(1)
        assert torch.all((dw[t].double() - want).abs() <= (H / 8 + 13) * 2.0 ** -24 * size)
    del dout, rows, pos, w, drows, dw
    torch.cuda.empty_cache()


def test_router_and_combine_through_autograd(mxg, cuda_dev):
    """Logits -> weights -> combine: both gradients in one backward pass."""
    n, E, k, H = 50, 16, 4, 64
    z = _logits(n, E, "fp32", 3, cuda_dev).requires_grad_(True)
    w, ids = mxg.router_topk(z, k, score="sigmoid", scale=2.0)
    counts, send_rows, slot_pos = mxg.ep.CudaEpOps().route(ids, E)
    slot_pos = slot_pos.view(n, k)
    rows = torch.randn(n * k, H, device=cuda_dev).to(torch.bfloat16).requires_grad_(True)
    out = mxg.combine(rows, slot_pos, w)
    up = torch.randn(n, H, device=cuda_dev).to(torch.bfloat16)
    out.backward(up)
    ref_rows, ref_dw = ro.combine_bwd(_np(up), _np(rows), slot_pos.cpu().numpy(), _np(w))
    ref_z = ro.router_bwd(_np(z), ids.cpu().numpy(), ref_dw, score="sigmoid", scale=2.0)
    assert np.all(np.abs(_np(rows.grad) - ref_rows) <= (2.0 ** -8 + 2.0 ** -23) * np.abs(ref_rows))
    size = np.abs(ref_dw).max(1, keepdims=True)
    assert np.all(np.abs(_np(z.grad) - ref_z) <= 4 * G_TOL * size)
    assert mxg.device_error() == 0


def test_captured_backward_pass(mxg, cuda_dev):
    """Forward and backward through autograd in one graph, replayed on new inputs."""
    n, E, k, H = 40, 64, 4, 64
    z = _logits(n, E, "fp32", 3, cuda_dev).requires_grad_(True)
    rows = torch.randn(n * k, H, device=cuda_dev).to(torch.bfloat16).requires_grad_(True)
    pos = torch.randperm(n * k, device=cuda_dev).to(torch.int32).view(n, k)
    up = torch.randn(n, H, device=cuda_dev).to(torch.bfloat16)

    def both():
        w, _ = mxg.router_topk(z, k, score="sigmoid")
        return torch.autograd.grad(mxg.combine(rows, pos, w), (z, rows), up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    with torch.no_grad():
        z.copy_(_logits(n, E, "fp32", 4, cuda_dev))
        rows.mul_(2)
    graph.replay()
    want = both()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert mxg.device_error() == 0


@pytest.mark.parametrize("E,k", [(8, 2), (16, 16), (64, 4), (256, 8), (384, 12)])
@pytest.mark.parametrize("n", [5, 8200])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_sigmoid_of_infinite_logits(mxg, cuda_dev, E, k, n, dtype):
    """sigmoid(inf) is 1, in a share too: weights and gradients are finite."""
    inf = float("inf")
    z = _logits(n, E, dtype, 7, cuda_dev)
    z[0, E // 2] = inf
    z[1, ::2] = inf
    z[2] = inf
    z[3] = -inf
    z[3, 1] = inf
    bias = torch.randn(E, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(E)) * 0.05
    for renorm in (True, False):
        for b in (None, bias):
            w, ids = _check(mxg, z, k, score="sigmoid", bias=b, renormalize=renorm, scale=2.5)
            assert torch.isfinite(w).all()
        dw = torch.randn(n, k, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(8))
        dz = mxg.ops.router_topk_bwd(z, w, ids, dw, score="sigmoid", renormalize=renorm, scale=2.5)
        assert torch.isfinite(dz).all() and torch.all(dz[z == inf] == 0)


@pytest.mark.parametrize("E", [8, 30, 64, 137, 256, 384])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_dense_gradient_of_logits_far_from_zero(mxg, cuda_dev, E, dtype):
    """Softmax, not renormalised, at offsets up to the end of the type's range
    (the logits that are left of them, the oracle takes as they are)."""
    top = torch.finfo(DT[dtype]).max
    z = _logits(14, E, "fp32", 11, cuda_dev)
    for r, off in enumerate((-1e4, 300.0, 5e5, -7.3e5, 1e6, -3e6, 3e9, 1e30, -1e30, 3e38, -3e38)):
        z[r] += off
    z[11] = -top                                 # the lowest value throughout
    z[12] = top
    z[13] = -top
    z[13, 3] = -float("inf")
    z[13, 5] = top
    z[0, 1] = z[7, 2] = -float("inf")
    z = z.clamp(-top, top).where(z != -float("inf"), z).to(DT[dtype])
    k = min(E, 6)
    w, ids = mxg.ops.router_topk(z, k, renormalize=False, scale=2.5)
    dw = torch.randn(14, k, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(1))
    dz = mxg.ops.router_topk_bwd(z, w, ids, dw, renormalize=False, scale=2.5)
    ref = ro.router_bwd(_np(z), ids.cpu().numpy(), _np(dw), renormalize=False, scale=2.5)
    size = np.abs(_np(w) * _np(dw)).sum(1, keepdims=True)
    half = 0.0 if dtype == "fp32" else torch.finfo(DT[dtype]).eps / 2
    assert np.all(np.abs(_np(dz) - ref) <= G_TOL * size + half * np.abs(ref) + 1e-37)
    assert mxg.device_error() == 0


@pytest.mark.filterwarnings("ignore:invalid value")     # the oracle's inf - inf
@pytest.mark.parametrize("n", [3, 8200])
@pytest.mark.parametrize("E,groups", [(64, 4), (256, 8)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_infinite_biases_in_groups(mxg, cuda_dev, n, E, groups, score):
    """A bias of +inf takes its expert always.  In a group whose others are
    switched off by -inf the sum of the two best has no value and counts as
    -inf: the best of the other groups are kept, as many as asked for."""
    inf, per = float("inf"), E // groups
    z = _logits(n, E, "fp32", 12, cuda_dev)
    bias = torch.randn(E, device=cuda_dev, generator=torch.Generator(cuda_dev).manual_seed(E)) * 0.05
    bias[2 * per:3 * per] = -inf
    bias[2 * per + 1] = inf
    for kept in (1, 2, groups - 1):
        _check(mxg, z, 3, score=score, bias=bias, groups=groups, topk_groups=kept, group_score="top2")
        w, ids = _check(mxg, z, 3, score=score, bias=bias, groups=groups, topk_groups=kept)
        assert torch.all(ids[:, 0] == 2 * per + 1)
    bias[2 * per:3 * per] = 0.0
    bias[2 * per + 1] = bias[5] = inf
    for how in (dict(), dict(groups=groups, topk_groups=2, group_score="top2"), dict(groups=groups, topk_groups=2)):
        w, ids = _check(mxg, z, 3, score=score, bias=bias, **how)
        assert torch.all(ids[:, 0] == 5) and torch.all(ids[:, 1] == 2 * per + 1)


@pytest.mark.parametrize("E,groups", [(16, 8), (64, 32), (96, 6), (256, 8)])
def test_nan_in_sums_of_groups(mxg, cuda_dev, E, groups):
    """Sigmoid scores without a bias, groups by the sum of their two best: a NaN
    is ordered as -inf there too, while a logit of -inf has the score 0."""
    z = _logits(60, E, "fp32", 13, cuda_dev)
    u = torch.rand(60, E, generator=torch.Generator(cuda_dev).manual_seed(2), device=cuda_dev)
    z[u < 0.2] = -float("inf")
    z[20:][u[20:] > 0.8] = float("nan")
    per = E // groups
    z[40:, :per] = float("nan")                  # a group whose one expert is far ahead, beside NaN alone
    z[40:, 0] = 9.0
    for kept in (1, groups // 2):
        for k in (1, min(per, 4)):
            w, ids = mxg.ops.router_topk(z, k, score="sigmoid", groups=groups, topk_groups=kept, group_score="top2")
            ref = ro.router(_np(z), k, score="sigmoid", groups=groups, topk_groups=kept, group_score="top2")
            full = np.isfinite(np.take_along_axis(_np(z), ref[1].astype(np.int64), 1)).all(1)
            assert np.array_equal(ids.cpu().numpy()[full], ref[1][full]) and full[:20].any() and full[20:].any()
            assert np.all(np.abs(w.cpu().numpy()[full] - ref[0][full]) <= W_TOL * ref[0][full])

"""Argument checks of the router, the combine's gradient and AdamW, and the
8-bit codes, on a machine without a GPU."""
import os
import subprocess

import numpy as np
import pytest
import torch

from oracle import adamw_oracle as ao


def test_router_refuses_bad_arguments(mxg):
    R = mxg.ops.router_topk
    z = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        R(z, 4)
    with pytest.raises(ValueError, match="score"):
        R(z, 4, score="relu")
    with pytest.raises(ValueError, match="scale"):
        R(z, 4, scale=0.0)
    with pytest.raises(ValueError, match="group_score"):
        R(z, 4, group_score="sum")
    with pytest.raises(TypeError):
        R(z.double(), 4)
    with pytest.raises(TypeError):
        R(z[0], 4)
    with pytest.raises(ValueError, match="experts"):
        R(torch.zeros(2, 385), 4)
    with pytest.raises(ValueError, match="CUDA"):
        mxg.ops.router_topk_bwd(z, z[:, :2], z[:, :2].int(), z[:, :2])
    with pytest.raises(ValueError, match="scale"):
        mxg.ops.router_topk_bwd(z, z[:, :2], z[:, :2].int(), z[:, :2], scale=float("inf"))


def test_router_abi_refuses_bad_shapes(mxg):
    L, pack = mxg._lib.load(), mxg._lib.router_args

    def call(ld=64, dtype=1, n=4, E=64, k=4, score=0, groups=1, kept=1, gs=0, scale=1.0, z=16):
        return L.mxg_router_topk(pack(z, 0, 16, 16, 0, 0, n, ld, E, dtype, E, k, score, groups, kept, gs, 1, scale, 0),
                                 None)
    assert call(n=0) == 0
    assert call(n=-1) == 1 and call(E=0) == 1 and call(k=0) == 1 and call(dtype=3) == 1 and call(score=2) == 1
    assert call(E=385, ld=385) == 2 and call(k=65) == 2 and call(k=33) == 2 and call(ld=63) == 2
    assert call(groups=0) == 1 and call(groups=4, kept=5) == 1 and call(gs=2) == 1 and call(scale=-1.0) == 1
    assert call(scale=float("nan")) == 1 and call(z=0) == 1
    assert call(groups=5) == 2 and call(groups=64, kept=64) == 2
    assert call(groups=16, kept=1, k=5) == 2                   # four experts are left
    assert L.mxg_router_topk(None, None) == 1 and L.mxg_router_topk_bwd(None, None) == 1

    def bwd(ld=64, n=4, E=64, k=4, ld_out=64, scale=1.0, w=16):
        return L.mxg_router_topk_bwd(pack(16, 0, w, 16, 16, 16, n, ld, ld_out, 1, E, k, 0, 0, 0, 0, 1, scale, 0), None)
    assert bwd(n=0) == 0 and bwd(ld_out=60) == 2 and bwd(scale=0.0) == 1 and bwd(w=0) == 1 and bwd(k=65) == 2


def test_combine_gradient_refuses_bad_arguments(mxg):
    rows = torch.zeros(4, 16, dtype=torch.bfloat16)
    pos = torch.zeros(2, 2, dtype=torch.int32)
    for fn in (lambda: mxg.ops.combine_bwd(rows[:2], rows, pos), lambda: mxg.ops.combine(rows, pos)):
        with pytest.raises(ValueError, match="CUDA"):
            fn()
    with pytest.raises(TypeError):
        mxg.ops.combine_bwd(rows[:2], rows[:, :12], pos)
    with pytest.raises(TypeError):
        mxg.ops.combine_bwd(rows[:2], rows, pos.long())
    L = mxg._lib.load()
    call = lambda n=2, k=2, H=16, P=4, dout=16, rows=16, pos=16: L.mxg_ep_combine_bwd(
        dout, rows, pos, None, n, k, H, P, 16, 16, None)
    assert call(n=-1) == 1 and call(k=0) == 1 and call(H=12) == 2 and call(k=400) == 2 and call(P=-1) == 1
    assert call(dout=None) == 1 and call(pos=None) == 1 and call(rows=24) == 3
    assert L.mxg_ep_combine_bwd(16, 16, 16, None, 2, 2, 16, 4, None, None, None) == 0


def test_adamw_refuses_bad_arguments(mxg):
    A = mxg.optim.AdamW
    p = torch.zeros(8)
    with pytest.raises(ValueError, match="CUDA"):
        A([p])
    with pytest.raises(ValueError, match="at least one"):
        A([])
    with pytest.raises(ValueError, match="state_bits"):
        A([p], state_bits=16)
    with pytest.raises(ValueError, match="betas"):
        A([p], betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="eps"):
        A([p], eps=-1.0)
    with pytest.raises(ValueError, match="decay"):
        A([p], weight_decay=[0.1, 0.1])
    with pytest.raises(ValueError, match="decay"):
        A([p], weight_decay=-0.1)
    with pytest.raises(TypeError):
        A([p.half()])
    with pytest.raises(ValueError, match="contiguous"):
        A([torch.zeros(4, 4).t()])


def test_adamw_abi_refuses_bad_arguments(mxg):
    L = mxg._lib.load()
    begin, grads, kinds = np.zeros(2, np.int64), np.array([16], np.uint64), np.array([1], np.int32)

    def call(n=1, bits=32, m=16, ms=0, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, grads=grads, kinds=kinds, begin=begin,
             step=16, chunk=4096):
        return L.mxg_adamw_step(mxg._lib.adamw_args(
            16, 16, begin.ctypes.data, grads.ctypes.data, kinds.ctypes.data, m, 16, ms, ms, 0, step, 16, 0, lr, b1, b2,
            eps, 0, n, chunk, bits, 0), None)
    assert L.mxg_adamw_step(None, None) == 1
    assert call(n=0) == 1 and call(bits=16) == 1 and call(m=0) == 1 and call(step=0) == 1
    assert call(bits=8) == 1                                     # no scales
    assert call(chunk=0) == 1 and call(chunk=4000) == 1
    assert call(lr=-1.0) == 1 and call(b1=1.0) == 1 and call(b2=-0.1) == 1 and call(eps=float("nan")) == 1
    assert call(kinds=np.array([2], np.int32)) == 1
    assert call(grads=np.array([18], np.uint64)) == 3 and call(m=24) == 3
    assert call(begin=np.array([3, 1], np.int64)) == 1
    assert L.mxg_adamw_moments(16, 16, 16, 16, 100, 16, 16, None) == 2
    assert L.mxg_adamw_moments(16, 16, 16, 16, 0, 16, 16, None) == 0
    assert L.mxg_adamw_moments(16, None, 16, 16, 256, 16, 16, None) == 1


def test_argument_layouts_match_the_header(mxg, tmp_path):
    """Sizes and field offsets as the C compiler lays the structs out."""
    assert len(mxg._lib.router_args(*[0] * 17, 1.0, 0)) == 6 * 8 + 3 * 8 + 8 * 4 + 8
    assert len(mxg._lib.adamw_args(*[0] * 13, *[0.0] * 4, *[0] * 5)) == 13 * 8 + 4 * 8 + 8 + 4 * 4
    e = mxg.optim._ENTRY
    assert e.itemsize == 48
    assert [e.fields[n][1] for n in ("param", "numel", "offset", "master", "decay", "kind", "first_chunk")] == \
        [0, 8, 16, 24, 32, 36, 40]
    source = tmp_path / "sizes.c"
    source.write_text('#include <stdio.h>\n#include "mxg.h"\nint main(void) { printf("%zu %zu %zu %zu %zu %zu", '
                      'sizeof(mxg_router_args), offsetof(mxg_router_args, scale), sizeof(mxg_adamw_args), '
                      'offsetof(mxg_adamw_args, seed), sizeof(mxg_adamw_tensor), '
                      'offsetof(mxg_adamw_tensor, first_chunk)); return 0; }')
    subprocess.run(["gcc", "-I", os.path.dirname(mxg._lib.HEADER_PATH), str(source), "-o", str(tmp_path / "sizes")],
                   check=True)
    sizes = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout
    assert sizes.split() == ["112", "104", "160", "136", "48", "40"]
    text = open(mxg._lib.HEADER_PATH).read()
    for name, value in (("MXG_ADAMW_BLOCK", 256), ("MXG_ROUTER_MAX_TOPK", 32),
                        ("MXG_ROUTER_MAX_GROUPS", 32), ("MXG_EP_MAX_EXPERTS", 384)):
        assert f"#define {name} {value}" in text
        assert getattr(mxg._lib, name[4:]) == value


@pytest.mark.parametrize("first", [True, False])
def test_codes_round_without_bias(first):
    """Mean of the decoded codes over many steps: within 5 standard errors."""
    g = np.random.default_rng(0)
    x = (g.standard_normal(256) * np.exp(g.uniform(-8, 0, 256))).astype(np.float32)
    x = x if first else x * x
    total, count = np.zeros(256), 3000
    for t in range(count):
        h, _ = ao.words(3, t, 512, 256)
        codes, scale = ao.encode(x, ao.noise(h, first), first)
        total += ao.decode(codes, scale, first)
    gap = np.maximum(np.abs(x), scale[0] * 2.0 ** (-14 if first else -30)) / 8   # at most a code's step
    # a second moment under the lowest code, 2^-33, is held at that code: up to one code above its mean
    held = 0.0 if first else np.where(x < scale[0] * 2.0 ** -33, gap, 0.0)
    assert np.all(np.abs(total / count - x) <= 5 * gap / 2 / np.sqrt(count) + 2.0 ** -16 * gap + held)


def test_every_code_is_kept_by_a_round_trip():
    codes = np.arange(256, dtype=np.uint8)
    scale = np.ones(1, np.float32)
    for first, top in ((True, 0x78), (False, 0xF8)):
        kept = codes[(codes & (127 if first else 255)) <= top]
        x = np.zeros(256, np.float32)
        x[:kept.size] = ao.decode(np.resize(kept, 256), scale, first)[:kept.size]
        again, s = ao.encode(x, np.zeros(256, np.uint64), first)
        assert s[0] == 1.0 and np.array_equal(ao.decode(again, s, first)[:kept.size], x[:kept.size])


def test_adamw_refuses_settings_beyond_fp32(mxg):
    """An eps that fp32 holds as 0 or as a subnormal (0 / eps has no value
    there), an lr or a decay that it holds as infinity."""
    A, p, inf = mxg.optim.AdamW, torch.zeros(8), float("inf")
    for eps in (1e-50, 1e-39, inf, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            A([p], eps=eps)
    for decay in (inf, 1e39, [1e39], float("nan")):
        with pytest.raises(ValueError, match="decay"):
            A([p], weight_decay=decay)
    begin, grads, kinds = np.zeros(2, np.int64), np.array([16], np.uint64), np.array([1], np.int32)
    for lr, eps in ((1e39, 1e-8), (inf, 1e-8), (1e-3, 1e-50), (1e-3, 1e-39), (1e-3, inf)):
        assert mxg._lib.load().mxg_adamw_step(mxg._lib.adamw_args(
            16, 16, begin.ctypes.data, grads.ctypes.data, kinds.ctypes.data, 16, 16, 0, 0, 0, 16, 16, 0, lr, 0.9,
            0.99, eps, 0, 1, 4096, 32, 0), None) == 1


def test_random_words_pass_for_independent_uniform_draws():
    """Means, spreads and single bits of both words' halves, and correlations
    between the halves, neighbours, blocks, steps and seeds, over 2^18 draws.
    A mean of n uniform draws is off by sqrt(1 / 12 n), a mean square by
    sqrt(4 / 45 n), a bit's by 1 / 2 sqrt(n), a correlation by 1 / sqrt(n): 5.5
    of each, which one of these 500 figures passes by chance once in 5 * 10^4."""
    n, off = 1 << 18, 5.5

    def halves(seed, step, first):
        h, more = ao.words(seed, step, first, n)
        return [x.astype(np.float64) / 65536 + 2.0 ** -17
                for w in (h, more) for x in (w >> ao.U(16), w & ao.U(0xFFFF))]

    def apart(x, y):
        x, y = x - 0.5, y - 0.5
        assert abs(12 * np.mean(x * y)) <= off / np.sqrt(x.size)

    for seed, step, first in ((0, 1, 0), (1234, 41, 256 * 7), (2 ** 63 + 5, 100_000, 2 ** 33), (1, 2, 0)):
        here = halves(seed, step, first)
        for x in here:
            assert abs(np.mean(x) - 0.5) <= off * np.sqrt(1 / 12 / n)
            assert abs(np.mean(x * x) - 1 / 3) <= off * np.sqrt(4 / 45 / n)
            word = (x * 65536).astype(np.int64)
            for bit in range(16):
                assert abs(np.mean(word >> bit & 1) - 0.5) <= off / 2 / np.sqrt(n)
            for gap in (1, 2, 4, 32, 128, 256, 512, 4096):     # neighbours, lanes, blocks, chunks
                apart(x[:-gap], x[gap:])
        others = [halves(seed, step + 1, first), halves(seed + 1, step, first), halves(seed ^ 1 << 40, step, first),
                  halves(seed, step, first + n)]
        for i, x in enumerate(here):
            for y in here[i + 1:]:
                apart(x, y)
            for other in others:
                apart(x, other[i])

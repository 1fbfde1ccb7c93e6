"""AdamW: moments bit for bit (32-bit values and 8-bit codes), weights against
64 bits.

Tolerance of a weight: p (1 - lr wd) rounds its factor twice and the sum once,
3 * 2^-24 |p| and a step of the result; the update's lr, corrections, root,
quotients and products are 14 roundings of at most 2^-24 each: 2^-20 of it."""
import numpy as np
import pytest
import torch

from oracle import adamw_oracle as ao

pytestmark = pytest.mark.gpu

SHAPES = [(1,), (255,), (256,), (257,), (3, 1000), (0,), (4096,), (4097,), (16, 33, 29)]
BF, F32 = torch.bfloat16, torch.float32


def _np(t):
    return t.detach().float().cpu().numpy()


def _make(shapes, dtypes, seed, dev, std=0.02):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(*s, generator=g, device=dev).mul_(std).to(d) for s, d in zip(shapes, dtypes)]


def _weights_close(got, p, m, v, k):
    """got fp32 against the update of p in 64 bits."""
    ref = ao.weights(p, m, v, **k)
    moved = np.abs(ref - (1 - k["lr"] * k["decay"]) * p.astype(np.float64))
    assert np.all(np.abs(got - ref) <= 2.0 ** -22 * np.abs(p) + 2.0 ** -20 * moved + 1e-38)
    return ref


class Mirror:
    """The oracle's state beside an optimiser's."""

    def __init__(self, opt):
        self.opt = opt
        n = opt.exp_avg.numel()
        self.m, self.v = np.zeros(n, np.float32), np.zeros(n, np.float32)
        self.t = 0

    def step(self, grads):
        opt, bits = self.opt, self.opt.state_bits
        before = [p.detach().clone() for p in opt.params]
        copies = None if opt.master is None else opt.master.cpu().numpy().copy()
        opt.step(grads)
        self.t += 1
        b1, b2 = opt.betas
        avg, sq = (x.cpu().numpy() for x in opt.moments())
        for i, (p, g) in enumerate(zip(opt.params, grads)):
            at, size, n = opt.offsets[i], opt.offsets[i + 1] - opt.offsets[i], p.numel()
            if g is None or n == 0:
                assert torch.equal(p, before[i])
                assert np.array_equal(avg[at:at + size], self.m[at:at + size])
                continue
            gp = np.zeros(size, np.float32)
            gp[:n] = _np(g).reshape(-1)
            m, v = ao.moments(self.m[at:at + size], self.v[at:at + size], gp, b1, b2)
            h, more = ao.words(opt.seed, self.t, at, size)
            k = dict(step=self.t, lr=float(opt.lr), b1=b1, b2=b2, eps=opt.eps, decay=opt.weight_decay[i])
            got = _np(p).reshape(-1)
            if p.dtype == F32:
                _weights_close(got, _np(before[i]).reshape(-1), m[:n], v[:n], k)
            elif opt.master is not None:
                c = opt._copies[i]
                now = opt.master[c:c + size].cpu().numpy()
                _weights_close(now[:n], copies[c:c + n], m[:n], v[:n], k)
                assert np.all(now[n:] == 0)
                assert torch.equal(p.reshape(-1), opt.master[c:c + n].to(BF))
            else:
                ref = ao.weights(_np(before[i]).reshape(-1), m[:n], v[:n], **k)
                gap = 2.0 ** (np.frexp(np.abs(ref))[1] - 8.0)
                low = np.floor(np.abs(ref) / gap)
                up = np.abs(ref) / gap - low + (more[:n] & ao.U(0xFFFF)).astype(np.float64) / 65536
                want = np.sign(ref) * gap * (low + (up >= 1))
                # a border closer than the fp32 result's error may go either way: the head's tolerance in bf16
                # steps, which are small where the update has all but cancelled the weight
                old = np.abs(_np(before[i]).reshape(-1))
                near = (2.0 ** -22 * old + 2.0 ** -20 * (np.abs(ref) + old)) / gap
                sure = np.abs(up - 1) > near
                assert np.array_equal(got[sure], want[sure].astype(np.float32))
                assert np.all(np.abs(got - ref) <= gap * (1 + near)) and np.mean(sure) > 0.95
            if bits == 8:
                cm, sm = ao.encode(m, ao.noise(h, True), True)
                cv, sv = ao.encode(v, ao.noise(h, False), False)
                b = slice(at // 256, (at + size) // 256)
                assert np.array_equal(opt.exp_avg[at:at + size].cpu().numpy(), cm)
                assert np.array_equal(opt.exp_avg_sq[at:at + size].cpu().numpy(), cv)
                assert np.array_equal(opt.exp_avg_scale[b].cpu().numpy(), sm)
                assert np.array_equal(opt.exp_avg_sq_scale[b].cpu().numpy(), sv)
                m, v = ao.decode(cm, sm, True), ao.decode(cv, sv, False)
            assert np.array_equal(avg[at:at + size], m) and np.array_equal(sq[at:at + size], v)
            self.m[at:at + size], self.v[at:at + size] = m, v


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [True, False])
@pytest.mark.parametrize("grad", [BF, F32])
def test_steps_against_the_oracle(mxg, cuda_dev, bits, master, grad):
    dtypes = [BF, F32, BF, BF, BF, F32, BF, F32, BF]
    params = _make(SHAPES, dtypes, 1, cuda_dev)
    opt = mxg.optim.AdamW(params, lr=1e-3, betas=(0.9, 0.95), weight_decay=[0.1 * (i % 2) for i in range(9)],
                          state_bits=bits, master_weights=master, seed=2 ** 40 + 17)
    mirror = Mirror(opt)
    for t in range(4):
        grads = _make(SHAPES, [grad if t != 2 else F32] * 9, 10 + t, cuda_dev, std=10.0 ** (t - 3))
        mirror.step([None if (t == 1 and i == 4) else g for i, g in enumerate(grads)])
    assert mxg.device_error() == 0 and opt.state_dict()["step"] == 4
    assert int(opt._done.item()) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_misaligned_tensors(mxg, cuda_dev, bits):
    base, gbase = _make([(9000,), (9000,)], [BF, BF], 3, cuda_dev)
    params = [base[1:5001], base[5003:5004], base[5008:]]
    grads = [gbase[3:5003], gbase[0:1], gbase[5009:].float()[:0].new_zeros(1)]
    grads[2] = torch.cat([gbase.float(), gbase.float()])[1:1 + params[2].numel()]
    mirror = Mirror(mxg.optim.AdamW(params, state_bits=bits, master_weights=False))
    edge = base[5001:5003].clone()
    for _ in range(2):
        mirror.step(grads)
    assert torch.equal(base[5001:5003], edge)     # what lies between the tensors stays


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(mxg, cuda_dev, bits):
    shapes = [(1 + 7 * (i % 90),) for i in range(1100)]      # more than one launch carries
    params = _make(shapes, [F32] * 1100, 4, cuda_dev)
    mirror = Mirror(mxg.optim.AdamW(params, state_bits=bits, weight_decay=0.0))
    for t in range(2):
        mirror.step(_make(shapes, [BF] * 1100, 5 + t, cuda_dev, std=1e-3))
    assert mirror.opt.state_dict()["step"] == 2


def test_scattered_sizes_of_gradients(mxg, cuda_dev):
    """Blocks of zeros, of tiny and of huge gradients, and gradients in strides."""
    p = _make([(2048,)], [F32], 6, cuda_dev)
    g = _make([(2048,)], [F32], 7, cuda_dev)[0]
    g[:256] = 0
    g[256:512] *= 1e-36
    g[512:768] *= 1e15
    g[800] = 1e12
    mirror = Mirror(mxg.optim.AdamW(p, state_bits=8, eps=1e-8))
    for _ in range(3):
        mirror.step([g])
    wide = torch.randn(64, 32, device=cuda_dev)
    q = _make([(32, 64)], [F32], 8, cuda_dev)
    mirror = Mirror(mxg.optim.AdamW(q))
    mirror.step([wide.t()])


def test_second_moment_above_zero_stays_above_zero(mxg, cuda_dev):
    p = [torch.zeros(256, device=cuda_dev)]
    opt = mxg.optim.AdamW(p, state_bits=8)
    g = torch.full((256,), 1e-9, device=cuda_dev)
    g[0] = 1.0
    for _ in range(3):
        opt.step([g])
    assert torch.all(opt.moments()[1] > 0)
    assert torch.all(p[0].abs() <= 3 * 1e-3 * 8)     # no update runs away: |m| / sqrt(v) < 8 here


def test_non_finite_gradient_stays_in_its_block(mxg, cuda_dev):
    p = _make([(1024,)], [BF], 9, cuda_dev)
    opt = mxg.optim.AdamW(p, state_bits=8, master_weights=False)
    g = _make([(1024,)], [F32], 10, cuda_dev)
    g[0][300] = float("nan")
    g[0][600] = float("inf")
    opt.step(g)
    opt.step(g)
    bad = ~torch.isfinite(p[0])
    assert bad[300] and bad[600] and not bad[:256].any() and not bad[768:].any()


def test_captured_steps_count_on(mxg, cuda_dev):
    make = lambda: _make([(5000,), (77, 3)], [BF, F32], 11, cuda_dev)
    a, b = make(), make()
    grads = _make([(5000,), (77, 3)], [F32, F32], 12, cuda_dev, std=1e-3)
    lr = torch.full((1,), 1e-3, device=cuda_dev)
    for bits in (32, 8):
        eager = mxg.optim.AdamW(a, lr=1e-3, state_bits=bits)
        other = mxg.optim.AdamW(b, lr=lr, state_bits=bits)
        lr.fill_(1e-3)
        eager.step(grads), other.step(grads)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            other.step(grads)
        for t in range(3):
            eager.lr = 1e-3 / (t + 1)
            lr.fill_(1e-3 / (t + 1))
            grads[0].mul_(1.5)
            eager.step(grads)
            graph.replay()
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        assert torch.equal(eager.exp_avg, other.exp_avg) and torch.equal(eager.exp_avg_sq, other.exp_avg_sq)
        assert eager.state_dict()["step"] == other.state_dict()["step"] == 4


def test_state_dict_carries_a_run_on(mxg, cuda_dev):
    shapes, dtypes = [(700,), (40, 9)], [BF, F32]
    grads = [_make(shapes, [F32, BF], 20 + t, cuda_dev, std=1e-3) for t in range(4)]
    for bits, master in ((32, True), (8, True), (8, False)):
        kw = dict(state_bits=bits, master_weights=master, seed=5)
        a = _make(shapes, dtypes, 13, cuda_dev)
        one = mxg.optim.AdamW(a, **kw)
        one.step(grads[0]), one.step(grads[1])
        saved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in one.state_dict().items()}
        b = [x.clone() for x in a]
        two = mxg.optim.AdamW(b, **kw)
        two.load_state_dict(saved)
        for g in grads[2:]:
            one.step(g), two.step(g)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(one.exp_avg, two.exp_avg)
        with pytest.raises(ValueError):
            mxg.optim.AdamW(b, state_bits=40 - bits, master_weights=master).load_state_dict(saved)


def test_moved_weights_and_grad_attribute(mxg, cuda_dev):
    p = [torch.nn.Parameter(x) for x in _make([(300,)], [F32], 14, cuda_dev)]
    opt = mxg.optim.AdamW(p)
    p[0].grad = torch.ones_like(p[0])
    version = p[0]._version
    opt.step()
    assert p[0]._version > version
    old = p[0].data
    p[0].data = old.clone()
    keep = old.clone()
    opt.step()
    assert torch.equal(old, keep) and not torch.equal(p[0].data, keep)
    for bad in ([torch.ones(301, device=cuda_dev)], [torch.ones(300, device=cuda_dev).half()], [], [torch.ones(300)]):
        with pytest.raises((ValueError, TypeError)):
            opt.step(bad)


def test_settings_changed_between_steps(mxg, cuda_dev):
    p = _make([(300,), (4097,)], [F32, BF], 24, cuda_dev)
    mirror = Mirror(mxg.optim.AdamW(p))
    opt = mirror.opt
    for t, (lr, decay, betas) in enumerate([(1e-3, 0.1, (0.9, 0.999)), (0.0, [0.0, 0.5], (0.9, 0.999)),
                                            (3e-2, 0.0, (0.0, 0.5)), (1e-4, 0.2, (0.5, 0.0))]):
        opt.lr, opt.weight_decay, opt.betas = lr, decay, betas
        if not isinstance(decay, list):
            opt.weight_decay = [decay, decay] if t % 2 else decay
        k = opt.weight_decay
        opt.weight_decay = k
        grads = _make([(300,), (4097,)], [F32, BF], 30 + t, cuda_dev, std=1e-2)
        if not isinstance(k, list):
            opt._lay_out()                        # what the step does: one number for every tensor
        mirror.step(grads)
    opt.weight_decay = [0.1]
    with pytest.raises(ValueError, match="decay"):
        opt.step(grads)
    opt.weight_decay, opt.eps = 0.1, 0.0
    with pytest.raises(mxg.MxgError):
        opt.step(grads)


def test_nothing_to_do(mxg, cuda_dev):
    p = [torch.empty(0, device=cuda_dev), torch.empty(0, 7, device=cuda_dev)]
    opt = mxg.optim.AdamW(p)
    opt.step([torch.empty(0, device=cuda_dev), None])
    assert opt.state_dict()["step"] == 1
    q = _make([(40,)], [BF], 25, cuda_dev)
    keep = q[0].clone()
    opt = mxg.optim.AdamW(q, state_bits=8)
    opt.step([None])
    assert torch.equal(q[0], keep) and opt.state_dict()["step"] == 1


def test_another_stream(mxg, cuda_dev):
    a, b = _make([(5000,)], [BF], 15, cuda_dev), _make([(5000,)], [BF], 15, cuda_dev)
    g = _make([(5000,)], [BF], 16, cuda_dev)
    one, two = mxg.optim.AdamW(a), mxg.optim.AdamW(b)
    side = torch.cuda.Stream()
    one.step(g)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two.step(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[0], b[0])


def test_elements_past_32_bits(mxg, cuda_dev):
    n = 2 ** 31 + 4500
    p = torch.full((n,), 0.5, dtype=BF, device=cuda_dev)
    g = torch.full((n,), 1e-3, dtype=BF, device=cuda_dev)
    g[-1000:] = _make([(1000,)], [BF], 17, cuda_dev)[0]
    opt = mxg.optim.AdamW([p], lr=1e-3, state_bits=8, master_weights=False, weight_decay=0.0)
    opt.step([g])
    at = (n - 2000) // 256 * 256
    size = opt.offsets[1] - at
    gp = np.zeros(size, np.float32)
    gp[:n - at] = _np(g[at:])
    m, v = ao.moments(np.zeros(size, np.float32), np.zeros(size, np.float32), gp, 0.9, 0.999)
    h, more = ao.words(0, 1, at, size)
    assert np.array_equal(opt.exp_avg[at:].cpu().numpy(), ao.encode(m, ao.noise(h, True), True)[0])
    assert np.array_equal(opt.exp_avg_sq[at:].cpu().numpy(), ao.encode(v, ao.noise(h, False), False)[0])
    assert 0 < float((p != 0.5).float().mean()) and torch.all((p - 0.5).abs() <= 2.0 ** -8)
    del p, g, opt
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [True, False])
@pytest.mark.parametrize("lr", [0.0, 1e-42])
def test_lr_zero_leaves_every_weight(mxg, cuda_dev, bits, master, lr):
    """A warm-up's first step, with second moments of 0 and under fp32's normal
    range among others.  1e-42: an update of at most 10 * lr, under half a
    step of any weight here."""
    shapes, dtypes = [(700,), (513,), (300,)], [BF, F32, BF]
    for as_tensor in (False, True):
        params = [p.add_(1.0) for p in _make(shapes, dtypes, 40, cuda_dev)]
        before = [p.clone() for p in params]
        opt = mxg.optim.AdamW(params, state_bits=bits, master_weights=master, weight_decay=0.1,
                              lr=torch.full((1,), lr, device=cuda_dev) if as_tensor else lr)
        grads = _make(shapes, [F32, BF, BF], 41, cuda_dev)
        grads[0][::2] = 0
        grads[0][1::4] = 1e-25
        grads[1].zero_()
        grads[2][:256] = 1e-25
        for _ in range(2):
            opt.step(grads)
        assert all(torch.equal(p, b) for p, b in zip(params, before))
        if opt.master is not None:
            assert torch.equal(opt.master[:700], before[0].float())
        # and the run goes on from there
        if as_tensor:
            opt.lr.fill_(1e-3)
        else:
            opt.lr = 1e-3
        opt.step(grads)
        assert all(torch.isfinite(p).all() for p in params)
        decayed = before[1].double() * (1 - 1e-4)
        assert torch.all((params[1].double() - decayed).abs() <= 2.0 ** -22 * decayed)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-8, 1e-12, 1e-18, 1e-30])
def test_second_moments_under_the_normal_range(mxg, cuda_dev, bits, eps):
    """Gradients whose squares are subnormal or vanish beside an eps of any
    size: the head's tolerance holds (the root has 2 units of the last place
    there too)."""
    params = [p.mul_(50) for p in _make([(1024,), (700,)], [F32, BF], 42, cuda_dev)]
    mirror = Mirror(mxg.optim.AdamW(params, state_bits=bits, eps=eps, betas=(0.9, 0.999)))
    for t in range(2):
        grads = _make([(1024,), (700,)], [F32, BF], 43 + t, cuda_dev)
        for g in grads:
            g[:256] *= 1e-16                     # g^2 (1 - b2) of about 1e-38
            g[256:512] *= 1e-18
            g[512:600] *= 1e-21                  # vanishes
            g[600:] *= 1e-17
        mirror.step(grads)
    assert all(torch.isfinite(p).all() for p in params)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_outlives_a_new_layout(mxg, cuda_dev, bits):
    """A graph's table of tensors is the optimiser's: an eager step with another
    weight decay, or after a tensor has moved, changes it in place."""
    shapes, dtypes = [(5000,), (77, 3)], [BF, F32]
    make = lambda: _make(shapes, dtypes, 50, cuda_dev)
    a, b = make(), make()
    grads = _make(shapes, [F32, F32], 51, cuda_dev, std=1e-3)
    eager = mxg.optim.AdamW(a, state_bits=bits, weight_decay=0.1)
    other = mxg.optim.AdamW(b, state_bits=bits, weight_decay=0.1)
    table = other._table.data_ptr()
    eager.step(grads), other.step(grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.step(grads)
    graph.replay(), eager.step(grads)
    for opt in (eager, other):
        opt.weight_decay = 0.5
        opt.step(grads)
    assert other._table.data_ptr() == table
    held = [torch.full((64,), 255, dtype=torch.uint8, device=cuda_dev) for _ in range(64)]   # what is freed, is reused
    graph.replay(), eager.step(grads)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    old = b[0].data
    b[0].data = old.clone()
    keep = old.clone()
    eager.step(grads), other.step(grads)
    assert other._table.data_ptr() == table
    graph.replay(), eager.step(grads)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(old, keep)
    assert torch.equal(eager.exp_avg, other.exp_avg) and torch.equal(eager.exp_avg_sq, other.exp_avg_sq)
    assert eager.state_dict()["step"] == other.state_dict()["step"] == 6     # step, replay, step, replay, step, replay
    del held


def test_tensors_without_memory_are_refused(mxg, cuda_dev):
    """A weight or gradient whose storage was given back (sharded training does
    that): no step, and the optimiser goes on once it is there again."""
    p, g = _make([(300,), (40,)], [F32, BF], 60, cuda_dev), _make([(300,), (40,)], [F32, BF], 61, cuda_dev)
    opt = mxg.optim.AdamW(p)
    for t, name in ((g[1], "grads"), (p[0], "params")):
        keep = t.clone()
        t.untyped_storage().resize_(0)
        with pytest.raises(ValueError, match=rf"{name}\[\d\] has no memory"):
            opt.step(g)
        t.untyped_storage().resize_(keep.numel() * keep.element_size())
        t.copy_(keep)
    assert opt.state_dict()["step"] == 0
    opt.step(g)
    assert opt.state_dict()["step"] == 1 and mxg.device_error() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_made_in_inference_mode(mxg, cuda_dev, bits):
    """The state is changed in place outside that mode too."""
    a = _make([(300,), (77,)], [BF, F32], 70, cuda_dev)
    b = [x.clone() for x in a]
    g = _make([(300,), (77,)], [F32, F32], 71, cuda_dev)
    one = mxg.optim.AdamW(a, state_bits=bits)
    with torch.inference_mode():
        two = mxg.optim.AdamW(b, state_bits=bits)
        two.step(g)
    one.step(g)
    one.weight_decay = two.weight_decay = 0.5
    one.step(g), two.step(g)
    two.load_state_dict({k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in one.state_dict().items()})
    with torch.inference_mode():
        two.step(g)
    one.step(g)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(one.exp_avg, two.exp_avg)

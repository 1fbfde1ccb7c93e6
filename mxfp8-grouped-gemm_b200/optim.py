"""AdamW over many tensors in one kernel launch, with moments in 32 or in 8 bits.

The step that follows the weight gradients (``moe.LayerStep.dw_gate_up`` and
``dw_down``, or those of ``autograd.grouped_mm``): the reference trains with
its trainer's AdamW (``port_mxfp8.py:175-194`` swaps only the grouped GEMMs).
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib

_GRAD = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_F32 = torch.finfo(torch.float32)
_ENTRY = np.dtype([("param", "<u8"), ("numel", "<i8"), ("offset", "<i8"), ("master", "<i8"), ("decay", "<f4"),
                   ("kind", "<i4"), ("first_chunk", "<i8")])     # mxg_adamw_tensor


_data_ptr, _get_device, _is_contiguous = torch.Tensor.data_ptr, torch.Tensor.get_device, torch.Tensor.is_contiguous


def _padded(n: int) -> int:
    return -(-n // _lib.ADAMW_BLOCK) * _lib.ADAMW_BLOCK


class AdamW:
    """AdamW (decoupled weight decay) over ``params``, bf16 or fp32 CUDA tensors
    of one device, updated in place by ``step``:

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

    in fp32 whatever the types of weights and gradients.

    state_bits      32: fp32 moments.  8: a byte a value in blocks of 256 that
                    share an fp32 scale, rounded stochastically (a rounding to
                    nearest would hold an average still whose steps are
                    smaller than half a code); ``mxg.h`` gives the codes.
    master_weights  keep an fp32 copy of every bf16 weight, which takes the
                    updates and is rounded to the weight.  Without it the bf16
                    weight itself is rounded stochastically.
    weight_decay    one number, or one for each tensor.
    seed            of the random bits; (seed, step, element) fix each of them.

    The moments are flat arrays: tensor i starts at element ``offsets[i]``, a
    multiple of 256, and zeros fill the gaps.  The step count lives on the
    device, so a captured ``step`` counts on at every replay; ``lr`` may be a
    number (fixed at capture) or a one-element fp32 CUDA tensor that is read
    at every step.  ``lr``, ``betas``, ``eps`` and ``weight_decay`` may be set
    between steps; a graph captured before keeps its ``betas``, ``eps``, number
    ``lr`` and gradients' addresses, and from the next ``step`` call on takes
    over a new ``weight_decay`` and the addresses of tensors that have moved.
    One optimiser's steps run one after the other: do not issue them on several
    streams at once."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01, *,
                 state_bits: int = 32, master_weights: bool = True, seed: int = 0):
        params = list(params)
        if not params:
            raise ValueError("AdamW needs at least one tensor")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if not _F32.tiny <= eps <= _F32.max:
            raise ValueError(f"eps must be positive and a normal fp32 number, got {eps}")
        decay = self._decays(weight_decay, len(params))
        for i, p in enumerate(params):
            if p.dtype not in _GRAD:
                raise TypeError(f"params[{i}] must be bf16 or fp32, got {p.dtype}")
            if not p.is_contiguous():
                raise ValueError(f"params[{i}] must be contiguous")
            if not p.is_cuda:
                raise ValueError(f"params[{i}] must be a CUDA tensor")
            if p.device != params[0].device:
                raise ValueError(f"params[{i}] is on {p.device}, params[0] on {params[0].device}")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("two of the params share memory")
        self.params, self.device = params, params[0].device
        self._shapes, self._dtypes = [p.shape for p in params], [p.dtype for p in params]
        self._on = {self.device.index}
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, decay
        self.state_bits, self.master_weights, self.seed = state_bits, bool(master_weights), int(seed) & (2 ** 64 - 1)
        sizes = [_padded(p.numel()) for p in params]
        self.offsets = np.concatenate([[0], np.cumsum(sizes)]).tolist()
        copied = [self.master_weights and p.dtype == torch.bfloat16 for p in params]
        self._copies, total = [], 0
        for c, s in zip(copied, sizes):
            self._copies.append(total if c else -1)
            total += s if c else 0
        dev, n = self.device, max(self.offsets[-1], _lib.ADAMW_BLOCK)
        with torch.inference_mode(False), torch.no_grad():      # state that any mode may change in place
            self.exp_avg_scale = self.exp_avg_sq_scale = self.master = None
            if state_bits == 8:
                self.exp_avg = torch.zeros(n, dtype=torch.uint8, device=dev)
                self.exp_avg_sq = torch.zeros(n, dtype=torch.uint8, device=dev)
                self.exp_avg_scale = torch.zeros(n // _lib.ADAMW_BLOCK, device=dev)
                self.exp_avg_sq_scale = torch.zeros(n // _lib.ADAMW_BLOCK, device=dev)
            else:
                self.exp_avg, self.exp_avg_sq = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
            if total:
                self.master = torch.zeros(total, device=dev)
                for p, at in zip(params, self._copies):
                    if at >= 0:
                        self.master[at:at + p.numel()].copy_(p.detach().reshape(-1))
            self._table = torch.empty(len(params) * _ENTRY.itemsize, dtype=torch.uint8, device=dev)
            self._step = torch.zeros(1, dtype=torch.int64, device=dev)
            self._done = torch.zeros(1, dtype=torch.int32, device=dev)
        # What a thread block takes at a time: about 128 shares, long runs where there is much.  us of a bf16 step
        # with 32 / 8 bits at 4096, 8192, 32768: 1 M values 6.7 / 8.6, 6.7 / 7.9, 13.8 / 15.7; 64 M 330 / 289,
        # 339 / 219, 337 / 185.
        self._chunk = min(32768, max(4096, 1 << max(0, (self.offsets[-1] // 128).bit_length() - 1)))
        chunks = [-(-p.numel() // self._chunk) for p in params]
        self._chunk_begin = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int64)
        table = np.repeat(np.arange(len(params), dtype=np.int32), chunks)
        self._chunks = torch.from_numpy(table if table.size else np.zeros(1, np.int32)).to(dev)
        self._lay_out()

    @staticmethod
    def _decays(weight_decay, count):
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * count
        if len(decay) != count:
            raise ValueError(f"{len(decay)} weight decays for {count} tensors")
        if not all(0.0 <= d <= _F32.max for d in decay):
            raise ValueError("weight_decay must not be negative, nor beyond fp32's range")
        return decay

    def _lay_out(self):
        """The device table of the tensors (again when one has moved, or a weight decay changed).  It stays where
        it is: a captured step reads it at every replay."""
        self.weight_decay = self._decays(self.weight_decay, len(self.params))
        for i, (p, shape) in enumerate(zip(self.params, self._shapes)):
            if p.shape != shape or p.dtype != self._dtypes[i] or p.device != self.device or not p.is_contiguous():
                raise ValueError(f"params[{i}] is no longer a contiguous {tuple(shape)} {self._dtypes[i]} tensor on "
                                 f"{self.device}")
            if p.numel() and p.data_ptr() == 0:
                raise ValueError(f"params[{i}] has no memory")
        self._at = [p.data_ptr() for p in self.params]
        t = np.zeros(len(self.params), _ENTRY)
        t["param"], t["numel"] = self._at, [p.numel() for p in self.params]
        t["offset"], t["master"] = self.offsets[:-1], self._copies
        t["decay"], t["first_chunk"] = self.weight_decay, self._chunk_begin[:-1]
        t["kind"] = [_lib.ADAMW_F32 if p.dtype == torch.float32 else
                     _lib.ADAMW_BF16_MASTER if c >= 0 else _lib.ADAMW_BF16 for p, c in zip(self.params, self._copies)]
        self._table.copy_(torch.from_numpy(t.view(np.uint8)))
        self._laid_out = list(self.weight_decay)

    def step(self, grads=None) -> None:
        """One update.  ``grads``: a gradient for each tensor (bf16 or fp32; None
        leaves the tensor and its moments as they are); without ``grads`` the
        tensors' ``.grad``."""
        params = self.params
        if grads is None:
            grads = [p.grad for p in params]
        elif len(grads) != len(params):
            raise ValueError(f"{len(grads)} gradients for {len(params)} tensors")
        lr, lr_ptr = self.lr, 0
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != self.device:
                raise ValueError(f"lr must be a number or a one-element fp32 tensor on {self.device}")
            lr, lr_ptr = 0.0, lr.data_ptr()
        elif not 0.0 <= lr <= _F32.max:
            raise ValueError(f"lr must not be negative, nor beyond fp32's range, got {lr}")
        held = None                                # contiguous copies, until the launch
        # all at once where every gradient is as it should be
        types, ptrs = self._types(grads), None
        if (None not in types and [g.shape for g in grads] == self._shapes
                and set(map(_get_device, grads)) == self._on and all(map(_is_contiguous, grads))):
            ptrs = list(map(_data_ptr, grads))
        if ptrs is None or 0 in ptrs:
            grads = held = self._checked(grads)
            types = [t or 0 for t in self._types(grads)]
            ptrs = [0 if g is None else g.data_ptr() for g in grads]
        kinds, ptrs = np.array(types, np.int32), np.array(ptrs, np.uint64)
        if list(map(_data_ptr, params)) != self._at or self.weight_decay != self._laid_out:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a tensor moved, or a weight decay changed, since the last step: take one step "
                                   "before the capture")
            self._lay_out()
        at = lambda t: 0 if t is None else t.data_ptr()
        _lib.launch("mxg_adamw_step", self.device, _lib.adamw_args(
            at(self._table), at(self._chunks), self._chunk_begin.ctypes.data, ptrs.ctypes.data, kinds.ctypes.data,
            at(self.exp_avg), at(self.exp_avg_sq), at(self.exp_avg_scale), at(self.exp_avg_sq_scale), at(self.master),
            at(self._step), at(self._done), lr_ptr, lr, *self.betas, self.eps, self.seed, len(params), self._chunk,
            self.state_bits, 0))
        del held
        tracked = [p for p in params if p.requires_grad]
        if tracked:                                # autograd sees the change in place
            torch.autograd.graph.increment_version(tracked)

    @staticmethod
    def _types(grads):
        return [None if g is None else _GRAD.get(g.dtype) for g in grads]

    def _checked(self, grads):
        """The gradients one by one: refusals, and contiguous copies where needed."""
        out = []
        for i, (g, shape) in enumerate(zip(grads, self._shapes)):
            if g is not None:
                if g.dtype not in _GRAD:
                    raise TypeError(f"grads[{i}] must be bf16 or fp32, got {g.dtype}")
                if g.shape != shape or g.device != self.device:
                    raise ValueError(f"grads[{i}] is {tuple(g.shape)} on {g.device}, expected {tuple(shape)} on "
                                     f"{self.device}")
                if g.numel() and g.data_ptr() == 0:
                    raise ValueError(f"grads[{i}] has no memory")
                g = g.contiguous()
            out.append(g)
        return out

    def moments(self):
        """(exp_avg, exp_avg_sq) as flat fp32 arrays: the state itself with 32
        bits, the values that the codes stand for with 8."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        n, dev = self.exp_avg.numel(), self.device
        avg, sq = torch.empty(n, device=dev), torch.empty(n, device=dev)
        _lib.launch("mxg_adamw_moments", dev, self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(),
                    self.exp_avg_scale.data_ptr(), self.exp_avg_sq_scale.data_ptr(), n, avg.data_ptr(), sq.data_ptr())
        return avg, sq

    def view(self, flat: torch.Tensor, i: int) -> torch.Tensor:
        """Tensor i's part of a flat moment, in its shape."""
        p, at = self.params[i], self.offsets[i]
        return flat[at:at + p.numel()].view(p.shape)

    def state_dict(self) -> dict:
        """Step count and state tensors (not copies)."""
        return {"step": int(self._step.item()), "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq,
                "exp_avg_scale": self.exp_avg_scale, "exp_avg_sq_scale": self.exp_avg_sq_scale, "master": self.master}

    def load_state_dict(self, state: dict) -> None:
        """Copy the values of a ``state_dict`` of the same tensors and options in."""
        names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")
        for name in names:
            mine, its = getattr(self, name), state[name]
            if (mine is None) != (its is None) or (mine is not None and (
                    mine.shape != its.shape or mine.dtype != its.dtype)):
                raise ValueError(f"{name} does not fit this optimiser's state")
        if state["step"] < 0:
            raise ValueError("step must not be negative")
        for name in names:
            if state[name] is not None:
                getattr(self, name).copy_(state[name])
        self._step.fill_(int(state["step"]))

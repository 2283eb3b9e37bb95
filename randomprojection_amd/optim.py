"""AdamW over many tensors at once, its states in 32 or in 8 bits.

One launch updates every tensor of the list (the adapters of many tenants, say), each with a step count of its
own, and writes the rounded bfloat16 operands the next projection reads (csrc/rp_optim.hip, which also has the
format of the states in 8 bits; no reference counterpart).
"""
from __future__ import annotations

import ctypes
import weakref

import torch

from . import _native as nat
from .adapters import raw_stream
from .gaussian import stream_of

__all__ = ["AdamW", "BLOCK"]

BLOCK = 256  # elements of a tensor that share one scale of a state in 8 bits; states are padded to whole blocks
_STATES = {32: ("steps", "exp_avg", "exp_avg_sq"),
           8: ("steps", "exp_avg", "exp_avg_root", "exp_avg_scale", "exp_avg_root_scale")}


def _overlap(written, read):
    """Whether a written tensor shares memory with any other."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w) for ts, w in ((written, True), (read, False))
                   for t in ts if t.numel())
    end = end_written = 0
    for start, stop, w in spans:
        if start < (end if w else end_written):
            return True
        end = max(end, stop)
        end_written = max(end_written, stop) if w else end_written
    return False


class AdamW:
    """``AdamW(params, grads)``: params float32, grads (all float32 or all bfloat16) of the same sizes, read at every
    ``step``; copies: bfloat16 tensors of the same sizes that receive the rounded parameters, or None. The tensors are
    contiguous, on one GPU, and are used in place: their memory must not be exchanged while the optimizer lives, and the optimizer
    must outlive the graphs that hold its steps.

    Per tensor, with t its own step count:
        m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
        w = w (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    state_bits 32 holds m and v in float32; state_bits 8 holds m and sqrt(v) in a byte each, in blocks of 256 elements
    with one power-of-two scale, rounded at random by ``seed`` (hashed with the step, the tensor and the element: the same
    seed gives the same bits). An m under the least of its block's codes, 2^-17 to 2^-16 of the largest m, is held as 0 where that code is
    more than its root allows: elements whose gradients are under some 2^-19 of their block's largest move by their current
    gradient alone, slower by 1 - b1. A gradient that is not finite makes its element's state NaN, with 8 bits its block's."""

    def __init__(self, params, grads, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=32,
                 copies=None, seed=0):
        params, grads = list(params), list(grads)
        copies = None if copies is None else list(copies)
        if not params or len(grads) != len(params) or (copies is not None and len(copies) != len(params)):
            raise ValueError("params, grads and copies must be lists of the same, positive, length")
        if state_bits not in _STATES:
            raise ValueError("state_bits must be 32 or 8")
        if not isinstance(seed, int) or not 0 <= seed < 1 << 64:
            raise ValueError("seed must be a whole number in [0, 2^64)")
        self.lr, self.betas, self.eps, self.weight_decay = lr, tuple(betas), eps, weight_decay
        self._check_numbers(lr)
        gdt = grads[0].dtype
        if gdt not in (torch.float32, torch.bfloat16):
            raise ValueError(f"grads must be float32 or bfloat16, got {gdt}")
        dev = params[0].device
        for name, ts, dt in (("params", params, torch.float32), ("grads", grads, gdt), ("copies", copies or [], torch.bfloat16)):
            for i, t in enumerate(ts):
                if t.dtype != dt or t.numel() != params[i].numel() or not t.is_contiguous() or t.device != dev:
                    raise ValueError(f"{name}[{i}] must be a contiguous {dt} tensor of {params[i].numel()} elements on {dev}, "
                                     f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        if _overlap(params + (copies or []), grads):
            raise ValueError("params and copies must not share memory, nor with a gradient")
        if dev.type != "cuda":
            raise RuntimeError("AdamW needs an MI355X (no CPU fallback)")
        self.params, self.grads, self.copies, self.state_bits, self.seed, self.device = params, grads, copies, state_bits, seed, dev
        sizes = [t.numel() for t in params]
        blocks = max(1, sum(-(-s // BLOCK) for s in sizes))
        zeros = lambda k, dt: torch.zeros(k, dtype=dt, device=dev)  # noqa: E731
        self.state = {"steps": zeros(len(params), torch.int32)}
        if state_bits == 32:
            self.state |= {k: zeros(blocks * BLOCK, torch.float32) for k in ("exp_avg", "exp_avg_sq")}
        else:
            self.state |= {"exp_avg": zeros(blocks * BLOCK, torch.float8_e4m3fn), "exp_avg_root": zeros(blocks * BLOCK, torch.uint8),
                           "exp_avg_scale": zeros(blocks, torch.uint8), "exp_avg_root_scale": zeros(blocks, torch.uint8)}
        s, T = self.state, len(params)
        array = lambda ts: (ctypes.c_void_p * T)(*(t.data_ptr() for t in ts))  # noqa: E731
        second = s["exp_avg_sq" if state_bits == 32 else "exp_avg_root"]
        h, lib = ctypes.c_void_p(), nat.load()
        nat.check(lib.rp_adamw_create(
            dev.index, T, (ctypes.c_int64 * T)(*sizes), array(params), array(grads),
            nat.RP_BF16 if gdt == torch.bfloat16 else nat.RP_F32, None if copies is None else array(copies), state_bits,
            s["exp_avg"].data_ptr(), second.data_ptr(), *(s[k].data_ptr() if k in s else None for k in
                                                          ("exp_avg_scale", "exp_avg_root_scale")),
            s["steps"].data_ptr(), ctypes.byref(h)))
        self._h = h
        self._close = weakref.finalize(self, lib.rp_adamw_destroy, h)

    def _check_numbers(self, lr):
        b1, b2 = self.betas
        if not (0 <= lr < float("inf")) or not 0 <= b1 < 1 or not 0 <= b2 < 1 or not self.eps >= 0 or not self.weight_decay >= 0:
            raise ValueError("lr, eps and weight_decay must not be negative, the betas lie in [0, 1)")

    def _stream(self, stream, *tensors):
        now = raw_stream(self.device.index)
        if stream is None or stream == now:
            return now
        cur = torch.cuda.current_stream(self.device)
        ext = stream_of(stream, self.device)
        ext.wait_stream(cur)
        for t in tensors:
            if t is not None:
                t.record_stream(ext)
        return stream

    def step(self, active=None, *, lr=None, stream=None):
        """One step of every tensor, or of those whose entry of ``active`` (a uint8 or bool device tensor, one for each
        tensor) is not zero: the others keep their values, states and step counts. lr: for this step only. Asynchronous on
        ``stream`` (default: torch's current one); can be captured into a graph, with the numbers of the call. Steps of one
        optimizer follow each other: two streams need an event between theirs."""
        lr = self.lr if lr is None else lr
        self._check_numbers(lr)
        if active is not None and (active.dtype not in (torch.uint8, torch.bool) or tuple(active.shape) != (len(self.params),)
                                   or active.device != self.device or not active.is_contiguous()):
            raise ValueError(f"active must be a contiguous uint8 or bool tensor of {len(self.params)} entries on {self.device}")
        nat.check(nat.load().rp_adamw_step(
            self._h, lr, *self.betas, self.eps, self.weight_decay, self.seed, None if active is None else active.data_ptr(),
            self._stream(stream, active)))

    def state_values(self, *, stream=None):
        """(m, sqrt(v)) of all blocks in float32: 256 elements a block, the last block of a tensor padded with zeros."""
        m, root = (torch.empty(self.state["exp_avg"].numel(), dtype=torch.float32, device=self.device) for _ in range(2))
        now, on = raw_stream(self.device.index), self._stream(stream, m, root)
        if self.state_bits == 8:
            nat.check(nat.load().rp_adamw_values(self._h, m.data_ptr(), root.data_ptr(), on))
            return m, root
        with torch.cuda.stream(None if on == now else stream_of(on, self.device)):  # None: the current one stays
            m.copy_(self.state["exp_avg"])
            torch.sqrt(self.state["exp_avg_sq"], out=root)
        return m, root

    def state_dict(self):
        """The states as they are held (the buffers themselves): ``steps`` and, with 32 bits, ``exp_avg`` and ``exp_avg_sq``;
        with 8, codes and scales. Tensor i's begin at 256 times the number of blocks of the tensors before it."""
        return dict(self.state)

    def load_state_dict(self, state):
        """Copies states of the same list of sizes and the same ``state_bits`` in."""
        if set(state) != set(_STATES[self.state_bits]):
            raise ValueError(f"states held in {self.state_bits} bits are {_STATES[self.state_bits]}, got {tuple(state)}")
        for k, t in state.items():
            if t.shape != self.state[k].shape or t.dtype != self.state[k].dtype:
                raise ValueError(f"{k} must be {self.state[k].dtype} {tuple(self.state[k].shape)}, got {t.dtype} {tuple(t.shape)}")
        for k, t in state.items():
            self.state[k].copy_(t)

"""Helpers of the tests of the linear recurrence and the page cache: device tensors of 16-bit types, the
definitions in 64 bits on the host, and the error that arithmetic in 32 bits may leave.

In an emulated session (tests/conftest.py) the package's own device checks are relaxed here, as conftest
does for thrust_amd.api, and every allocation of the package ends at a guard page where the session asks
for that."""
import contextlib
import ctypes
import os

import torch

import gpu_util
from conftest import EMULATED
from thrust_amd import api, device

if EMULATED:
    def _cpu(*tensors):
        return torch.device("cpu")

    def _empty(like, shape, dtype):
        if os.environ.get("THRUST_CDNA4_EMULATED_GUARD") != "1":
            return torch.empty(shape, dtype=dtype)
        two = dtype in (torch.float16, torch.bfloat16)
        return api.torch.empty(shape, torch.int16 if two else dtype).view(dtype)

    device.need_device = _cpu
    device.empty_like = lambda t: _empty(t, t.shape, t.dtype)
    device.current = lambda d: contextlib.nullcontext()
    device.is_current = lambda d: True
    device.stream = lambda d: ctypes.c_void_p(0)
    device.empty = _empty


def put(t):
    """A host tensor's copy on the device."""
    if t is None:
        return None
    t = t.contiguous()
    if t.dtype in (torch.float16, torch.bfloat16):
        return gpu_util.dev(t.view(torch.int16).numpy()).view(t.dtype).view(t.shape)
    return gpu_util.dev(t.numpy()).view(t.shape)


def get(t):
    return t.detach().cpu()


U32 = 2.0 ** -24  # half a step of float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half a step of the smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def spans_of(shape, offsets):
    """(batch, sequence, first row, last row + 1) of [batch, rows, channels]."""
    if offsets is None:
        return [(b, b, 0, shape[1]) for b in range(shape[0])]
    at = offsets.tolist()
    return [(0, s, at[s], at[s + 1]) for s in range(len(at) - 1)]


class Recurrence:
    """The definitions, in 64 bits.  gate, x [batch, rows, channels] or packed; `size_*` are the same sums of absolute values and
    `error_*` bounds what 32-bit arithmetic may be off: every row adds two roundings to each term of the sum (product and sum; in
    whatever order the maps of rows are composed, a term meets each row once, and at most as many folds of maps again), and a gate
    that is computed by exp adds that function's error of at most one unit in the last place, two half steps."""

    def __init__(self, gate, x, init, offsets, log):
        shape = x.shape if offsets is None else (1,) + tuple(x.shape)
        self.wide, self.shape = x.shape, shape
        a = gate.double().reshape(shape)
        self.log = log
        self.a = a.exp() if log else a
        self.x = x.double().reshape(shape)
        self.spans = spans_of(shape, offsets)
        sequences = len(self.spans)
        self.init = torch.zeros(sequences, shape[2], dtype=torch.float64) if init is None else init.double()
        self.roundings = U32 * (4 + (2 if log else 0))
        self.inside = torch.zeros(shape[:2], dtype=torch.bool)
        self.before, self.out = torch.zeros_like(self.x), torch.zeros_like(self.x)
        self.error_before, self.error_out = torch.zeros_like(self.x), torch.zeros_like(self.x)
        self.final, self.error_final = self.init.clone(), torch.zeros_like(self.init)
        for b, s, begin, end in self.spans:
            h = self.init[s]
            size, error = h.abs(), torch.zeros_like(h)
            for t in range(begin, end):
                self.inside[b, t] = True
                self.before[b, t], self.error_before[b, t] = h, error
                at = self.a[b, t]
                h = at * h + self.x[b, t]
                size = at.abs() * size + self.x[b, t].abs()
                error = at.abs() * error + self.roundings * size
                self.out[b, t], self.error_out[b, t] = h, error
            self.final[s], self.error_final[s] = h, error

    def gradient(self, grad_out, grad_final):
        d = grad_out.double().reshape(self.shape)
        self.grad_x, self.error_x = torch.zeros_like(d), torch.zeros_like(d)
        self.grad_init, self.error_init = torch.zeros_like(self.init), torch.zeros_like(self.init)
        for b, s, begin, end in self.spans:
            c = torch.zeros_like(self.init[s]) if grad_final is None else grad_final.double()[s]
            size, error = c.abs(), torch.zeros_like(c)
            for t in range(end - 1, begin - 1, -1):
                g = d[b, t] + c
                size = d[b, t].abs() + size
                error = error + self.roundings * size
                self.grad_x[b, t], self.error_x[b, t] = g, error
                at = self.a[b, t]
                c, size, error = at * g, at.abs() * size, at.abs() * error + self.roundings * (at * g).abs()
            self.grad_init[s], self.error_init[s] = c, error
        scale = self.a if self.log else torch.ones_like(self.a)
        self.grad_gate = self.grad_x * self.before * scale
        self.error_gate = (self.error_x * self.before.abs() + self.grad_x.abs() * self.error_before + self.error_x * self.error_before) * scale.abs() \
            + 2 * self.roundings * self.grad_gate.abs()
        return self


def check(got, want, error, what):
    """got, rounded once from a value that is `error` off `want` at most.  (Where one is not finite the other is the same.)"""
    g, w = got.double().reshape(want.shape), want
    fine = torch.isfinite(w)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    assert torch.equal(g[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)]), what
    bound = error + half_step(got.dtype) * (w.abs() + error) + smallest(got.dtype)
    off = (g - w).abs() - bound
    bad = (off > 0) & fine
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), bad.nonzero()[:4].tolist())

"""Gated linear recurrence: h[t] = a[t] * h[t-1] + x[t] for every channel, its gradient, and its step
for single tokens.  A scan, as thrust::inclusive_scan is, of affine maps along the rows.

Gates and inputs are [batch, rows, channels], or packed [rows, channels] with `offsets` [sequences + 1]
(int32 or int64, ascending; sequence s is the rows offsets[s] .. offsets[s + 1] - 1, which may be none).
Channels are next to each other; batches and rows may have any strides, as the halves of one projection
have.  x is float32, float16 or bfloat16, gates are of the same type or float32; with log_gate they are
logarithms of the factors.  States are float32 [sequences or batch, channels].  Sums are in 32 bits and
rounded once.
"""
import ctypes

import torch

from . import capi, device as dev

_DT = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}


def _types(gate, x):
    if x.dtype not in _DT or gate.dtype not in (x.dtype, torch.float32):
        raise ValueError("x must be float32, float16 or bfloat16, and the gates of its type or float32")


def _rows(t, shape, what):
    """(batch stride, row stride) of a tensor of this shape."""
    if t.shape != shape:
        raise ValueError(f"{what} must have the shape of x")
    if t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel():
        raise ValueError(f"{what}: channels must be next to each other")
    return (t.stride(0), t.stride(1)) if t.dim() == 3 else (0, t.stride(0))


def _distinct(t, what):
    """Refuses an output whose elements share memory."""
    need = t.shape[-1]
    for size, stride in sorted(((n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1), key=lambda v: v[1]):
        if stride < need:
            raise ValueError(f"{what}: rows overlap")
        need = stride * (size - 1) + need


def _span(t):
    """Bytes from the first element to behind the last one."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _rows_at(t):
    """The addresses at which the rows of t begin, ascending, and the bytes of one."""
    at = torch.tensor([t.data_ptr()], device="cpu")
    for n, s in zip(t.shape[:-1], t.stride()[:-1]):
        if n > 1 and s > 0:
            at = (at[:, None] + torch.arange(n, device="cpu") * (s * t.element_size())).flatten()
    return at.sort().values, t.shape[-1] * t.element_size()


def _layout(t):
    return [s * t.element_size() for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1]


def _meet(a, b):
    """Whether two tensors share memory.  (Channels are next to each other in both.)"""
    if not a.numel() or not b.numel() or a.data_ptr() >= b.data_ptr() + _span(b) or b.data_ptr() >= a.data_ptr() + _span(a):
        return False
    pitches, row = _layout(a), a.shape[-1] * a.element_size()
    if pitches and a.shape == b.shape and pitches == _layout(b) and min(pitches) > 0 and not any(s % min(pitches) for s in pitches):
        apart = (a.data_ptr() - b.data_ptr()) % min(pitches)  # columns of one array, as the parts of one projection are
        if apart >= b.shape[-1] * b.element_size() and min(pitches) - apart >= row:
            return False
    (rows_a, row_a), (rows_b, row_b) = _rows_at(a), _rows_at(b)
    return bool((torch.searchsorted(rows_a, rows_b + row_b) > torch.searchsorted(rows_a, rows_b - row_a, right=True)).any())


def _apart(out, tensors, inputs=()):
    """Refuses an output that shares memory with one of `tensors`, or of `inputs` without being it."""
    for t in inputs:
        if t.data_ptr() == out.data_ptr() and t.dtype == out.dtype and _layout(t) == _layout(out):
            continue
        if _meet(out, t):
            raise ValueError("an output shares memory with an input, and is not the same tensor")
    for t in tensors:
        if t is not None and _meet(out, t):
            raise ValueError("an output shares memory with an input")


def _state(t, sequences, channels, what):
    if t is None:
        return
    if t.dtype != torch.float32 or t.shape != (sequences, channels) or not t.is_contiguous():
        raise ValueError(f"{what} must be float32 [{sequences}, {channels}], contiguous")


def _shape(gate, x, offsets, log_gate, clear_outside):
    """The arguments that say what is computed, the number of sequences and the shape of the chunks' states."""
    _types(gate, x)
    shape = x.shape
    if offsets is None:
        if len(shape) != 3:
            raise ValueError("x must be [batch, rows, channels], or [rows, channels] with offsets")
        batch, rows, channels = shape
        sequences, size = batch, 0
    else:
        if len(shape) != 2:
            raise ValueError("x must be [rows, channels] where offsets are given")
        if offsets.dim() != 1 or offsets.dtype not in (torch.int32, torch.int64) or not offsets.is_contiguous() or offsets.numel() < 1:
            raise ValueError("offsets must be int32 or int64 [sequences + 1], contiguous")
        batch, (rows, channels) = 1, shape
        sequences, size = offsets.numel() - 1, offsets.element_size()
    fields = (_DT[gate.dtype], _DT[x.dtype], bool(log_gate), size, clear_outside, batch, rows, channels, sequences)
    return fields, sequences, (batch, -(-rows // capi.LINEAR_SCAN_CHUNK), channels)


def _strided(t, shape, what):
    return (t.data_ptr(), *_rows(t, shape, what))


_ONE_TILE = ctypes.c_size_t(256)
_UNUSED = 256  # an address that is never used


def _run(entry, args, rows, device, x, what):
    nbytes, where = ctypes.c_size_t(0), ctypes.byref(args)
    stream = dev.stream(device)
    with dev.current(device):
        if rows <= capi.LINEAR_SCAN_CHUNK:  # a single tile has nothing to store: no query, no allocation
            rc = entry(_UNUSED, ctypes.byref(_ONE_TILE), where, stream)
        elif (rc := entry(None, ctypes.byref(nbytes), where, stream)) == 0:
            temp = dev.empty(x, (nbytes.value,), torch.uint8)
            rc = entry(temp.data_ptr(), ctypes.byref(nbytes), where, stream)
    if rc:
        capi.check(rc, what)


def linear_scan(gate, x, init=None, offsets=None, log_gate=False, out=None, return_states=False):
    """h[t] = a[t] * h[t-1] + x[t]; returns (out, final): every h in the type of x, and the last one of
    each sequence in float32.  `init`: the states before the first rows (zero if None).  `out` may be x
    or gate; one that shares memory with them, or with init, in another way is refused.  return_states: also the state that enters each chunk of 64 rows, for linear_scan_backward.
    Packed rows that belong to no sequence are left as they were in a given `out`, and zero in a new one."""
    device = dev.need_device(gate, x, init, offsets, out)
    dev.no_autograd(gate, x, init, out)
    fields, sequences, chunks = _shape(gate, x, offsets, log_gate, out is None)
    given = out
    shape = x.shape
    state = (sequences, shape[-1])
    _state(init, *state, "init")
    gate_args, x_args = _strided(gate, shape, "gate"), _strided(x, shape, "x")
    if out is None:
        out = dev.empty_like(x)
    else:
        if out.dtype != x.dtype:
            raise ValueError("out must have the type of x")
        _distinct(out, "out")
        _rows(out, shape, "out")
        _apart(out, (init, offsets), (gate, x))
    out_args = _strided(out, shape, "out")
    final = dev.empty(x, state, torch.float32) if init is None else dev.empty_like(init)
    states = dev.empty(x, chunks, torch.float32) if return_states else None
    args = capi.LinearScanArgs(*fields, *gate_args, *x_args, *out_args, dev.pointer(offsets), dev.pointer(init), final.data_ptr(), dev.pointer(states))
    _run(capi.lib().thrust_cdna4_linear_scan, args, shape[-2], device, x, "linear_scan")
    if given is not None:
        dev.wrote((given,))
    return (out, final, states) if return_states else (out, final)


def linear_scan_backward(grad_out, gate, x, states, init=None, grad_final=None, offsets=None, log_gate=False):
    """The gradient of linear_scan for the gradients of its out and final (zero if None): returns
    (grad_gate, grad_x, grad_init), in the types of gate, x and init (None if there is no init).
    `states` are those that linear_scan returned."""
    device = dev.need_device(grad_out, gate, x, states, init, grad_final, offsets)
    dev.no_autograd(grad_out, gate, x, init, grad_final)
    fields, sequences, chunks = _shape(gate, x, offsets, log_gate, True)
    shape = x.shape
    state = (sequences, shape[-1])
    _state(init, *state, "init")
    _state(grad_final, *state, "grad_final")
    if states.dtype != torch.float32 or states.shape != chunks or not states.is_contiguous():
        raise ValueError("states must be what linear_scan returned for these shapes")
    if grad_out.dtype != x.dtype:
        raise ValueError("grad_out must have the type of x")
    inputs = (*_strided(gate, shape, "gate"), *_strided(x, shape, "x"), *_strided(grad_out, shape, "grad_out"))
    grad_gate, grad_x = dev.empty_like(gate), dev.empty_like(x)
    grad_init = None if init is None else dev.empty_like(init)
    args = capi.LinearScanBackwardArgs(*fields, *inputs, *_strided(grad_gate, shape, "grad_gate"), *_strided(grad_x, shape, "grad_x"),
                                       dev.pointer(offsets), dev.pointer(init), states.data_ptr(), dev.pointer(grad_final), dev.pointer(grad_init))
    _run(capi.lib().thrust_cdna4_linear_scan_backward, args, shape[-2], device, x, "linear_scan_backward")
    return grad_gate, grad_x, grad_init


def linear_scan_step(gate, x, state, slots=None, log_gate=False, out=None):
    """One row for each of a batch: state[slots[i]] = a[i] * state[slots[i]] + x[i], in place; returns the
    new states in the type of x.  gate and x are [batch, channels], state float32 [slots, channels],
    slots int32 [batch] (None: row i has slot i).  A slot outside the cache marks a padded row, whose out
    is zero.  Rows of one slot are taken in their order.  `out` may be x or gate;
    otherwise out and state share no memory with each other and the inputs."""
    device = dev.need_device(gate, x, state, slots, out)
    dev.no_autograd(gate, x, state, out)
    _types(gate, x)
    shape = x.shape
    if len(shape) != 2:
        raise ValueError("x must be [batch, channels]")
    batch, channels = shape
    if state.dim() != 2:
        raise ValueError("state must be [slots, channels]")
    num_slots = state.shape[0]
    _state(state, num_slots, channels, "state")
    if slots is None:
        if batch > num_slots:
            raise ValueError("more rows than slots")
    elif slots.dtype != torch.int32 or slots.shape != shape[:1] or not slots.is_contiguous():
        raise ValueError("slots must be int32 [batch], contiguous")
    written = (state,)
    if out is None:
        out, out_stride = dev.empty_like(x), channels
    else:
        written = (state, out)
        if out.dtype != x.dtype:
            raise ValueError("out must have the type of x")
        _distinct(out, "out")
        out_stride = _rows(out, shape, "out")[1]
        _apart(out, (state, slots), (gate, x))
    args = (_DT[gate.dtype], _DT[x.dtype], bool(log_gate), gate.data_ptr(), _rows(gate, shape, "gate")[1], x.data_ptr(), _rows(x, shape, "x")[1],
            out.data_ptr(), out_stride, state.data_ptr(), num_slots, dev.pointer(slots), batch, channels, dev.stream(device))
    entry = capi.lib().thrust_cdna4_linear_scan_step
    if dev.is_current(device):
        rc = entry(*args)
    else:
        with torch.cuda.device(device):
            rc = entry(*args)
    if rc:
        _apart(state, (gate, x))  # which the call refuses
        capi.check(rc, "linear_scan_step")
    dev.wrote(written)
    return out

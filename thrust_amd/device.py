"""Where the calls on torch tensors run: the tensors' device, torch's current stream on it.

A call's own time on the host is most of a small call's time: nothing here builds a Python object that
it can do without."""
import contextlib

import torch
from torch.autograd import forward_ad

_HERE = contextlib.nullcontext()


def need_device(*tensors):
    """The one device that all of the tensors (None: left out) are on."""
    first = None
    for t in tensors:
        if t is not None:
            if not t.is_cuda:
                raise ValueError("device tensors required: there is no CPU path")
            if first is None:
                first = t
            elif t.get_device() != first.get_device():
                raise ValueError("tensors on different devices")
    return None if first is None else first.device


def is_current(device):
    return device.index == torch.cuda.current_device()


def current(device):
    """A context in which `device` is the current one."""
    return _HERE if is_current(device) else torch.cuda.device(device)


def stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def empty(like, shape, dtype):
    """Uninitialised, on the device of `like`."""
    return like.new_empty(shape, dtype=dtype)


def empty_like(t):
    """Uninitialised and contiguous, of the shape and type of `t`, which costs less to say than a shape."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def capturing():
    return torch._C._cuda_isCurrentStreamCapturing()


_CAPTURED = []


class Outliving:
    """Private memory that calls read on the device: no other tensor gets it while work on any stream may
    still read it, also when its owner is gone.  Where a graph has captured such a call it is kept for good."""

    def __init__(self, tensor, device):
        self.tensor, self.device = tensor, device
        self._streams, self._captured = [stream(device)], False

    def used(self, s):
        """By a call on stream `s`, the current one of the device, which is the current one."""
        if self.device.type != "cuda" or s == 0 == self._streams[0]:  # its own; the default stream captures nothing
            return
        if capturing():
            if not self._captured:
                self._captured = True
                _CAPTURED.append(self.tensor)
        elif s not in self._streams:
            self.tensor.record_stream(torch.cuda.current_stream(self.device))
            self._streams.append(s)


def pointer(t):
    return None if t is None else t.data_ptr()


def no_autograd(*tensors):
    """These calls are no nodes of torch's graph: a tensor that wants its gradient, or brings a tangent, is not dropped in silence."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError("no automatic differentiation: call under torch.no_grad(), with linear_scan_backward as the gradient")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("no automatic differentiation in forward mode")


def wrote(tensors):
    """Tells torch that a call has written to these, as its own operations in place do."""
    torch._C._increment_version(tensors)

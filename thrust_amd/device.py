"""Where the calls on torch tensors run: the tensors' device, torch's current stream on it."""
import contextlib
import ctypes

import torch


def need_device(*tensors):
    """The one device that all of the tensors (None: left out) are on."""
    device = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("device tensors required: there is no CPU path")
        if device is not None and t.device != device:
            raise ValueError("tensors on different devices")
        device = t.device
    return device


def current(device):
    """A context in which `device` is the current one."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def empty(shape, dtype, device):
    return torch.empty(shape, dtype=dtype, device=device)


def pointer(t):
    return None if t is None else t.data_ptr()


def no_autograd(*tensors):
    """These calls are no nodes of torch's graph: a tensor that wants its gradient is not dropped in silence."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("no automatic differentiation: call under torch.no_grad(), with linear_scan_backward as the gradient")

"""Calls of the C entry points with little host work: a generated token or a short prompt is bound by the
host, so pointers go as plain integers, the device is switched only when it is another one, and the
stream handle is read without a stream object."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

_current_device = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream


def ptr(t):
    return None if t is None else t.data_ptr()


def invoke(fn, index, *args):
    """fn(*args, current stream of device ``index``) with that device current; raises on a status."""
    if _current_device() == index:
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _raw_stream(index))
    if st:
        _lib.check(st)


def cuda_index(*tensors):
    """The device index of the given tensors (None among them is skipped); raises unless all are on one."""
    index = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError('ccq_b200 operators run on CUDA tensors only (got a CPU tensor)')
        i = t.device.index
        if index is None:
            index = i
        elif i != index:
            raise RuntimeError(f'tensors on different devices: cuda:{index} and cuda:{i}')
    return index


def written(*tensors):
    """Tells autograd that a kernel wrote to these tensors (None among them is skipped): a backward that saved one of
    them raises, as after an in-place operation of torch, instead of reading the new values."""
    for t in tensors:
        if t is not None:
            torch.autograd.graph.increment_version(t)


def wants_grad(*tensors):
    """Whether a call goes through its autograd function: a gradient is asked for, or an input carries a forward-mode
    tangent, which the function refuses and a plain call would drop."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _FirstOnly(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, *grads):
        return grads

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError('the gated delta rule and the norms have no second derivative')


def first_derivative(backward):
    """For an autograd function's backward: gradients asked for with create_graph=True raise if they are differentiated
    again, as the kernels' outputs would otherwise count as constants."""
    def run(ctx, *seen):
        if not torch.is_grad_enabled():
            return backward(ctx, *seen)
        with torch.no_grad():
            grads = backward(ctx, *seen)
        real = [t for t in grads if t is not None]
        real = iter(_FirstOnly.apply(torch.zeros((), device=real[0].device, requires_grad=True), *real))
        return tuple(None if t is None else next(real) for t in grads)
    return run

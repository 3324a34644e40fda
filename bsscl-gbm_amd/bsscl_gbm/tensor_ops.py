"""Operators on device tensors: the softmax head over a large vocabulary with
its gradient, and the norm and clipping of many tensors' gradients.

They stand beside the estimator's softmax (which holds every score of up to 16
classes) for class counts where the scores are too many to keep.  Inputs and
outputs are torch tensors on one GPU; the kernels are libbsscl_hip.so's
(``bsscl_head_*``, ``bsscl_grad_norm``, ``bsscl_clip_grads`` in
include/bsscl_hip.h) and run on torch's current stream of that GPU.  Calls
return without waiting for the GPU and can be captured into a HIP graph.
Nothing is recorded for autograd: gradients are what the calls return.  A loss
of inputs that require gradients says so when backward reaches it.
"""
from __future__ import annotations

import ctypes
import math
from array import array
from collections import namedtuple
from operator import attrgetter

from . import _native

__all__ = ["linear_softmax_loss", "linear_softmax_grad", "grad_norm", "clip_grads"]

SoftmaxLoss = namedtuple("SoftmaxLoss", "loss row_loss lse")
SoftmaxGrad = namedtuple("SoftmaxGrad", "loss row_loss lse d_hidden d_weight")

_REDUCTIONS = {"sum": 0, "mean": 1}  # BSSCL_SUM, BSSCL_MEAN
_requires_grad = attrgetter("requires_grad")
_dtype_codes = None
_no_backward = None


def _torch():
    """torch, which only these operators need, and the C ABI's dtype codes."""
    global _dtype_codes
    import torch
    if _dtype_codes is None:
        _dtype_codes = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
    return torch


def _without_graph(torch, call, inputs):
    """call(), whose results raise an error in backward and forward mode if an
    input requires gradients or has a tangent: they would be missed silently."""
    global _no_backward
    forward_ad = torch.autograd.forward_ad
    inputs = [t for t in inputs if isinstance(t, torch.Tensor)]
    for t in inputs:
        if (t.requires_grad and torch.is_grad_enabled()
                or forward_ad.unpack_dual(t).tangent is not None):
            break
    else:
        return call()
    if _no_backward is None:
        class NoBackward(torch.autograd.Function):
            @staticmethod
            def forward(ctx, call, *inputs):
                return tuple(call())

            @staticmethod
            def backward(ctx, *grads):
                raise RuntimeError("linear_softmax_loss records nothing for autograd: "
                                   "linear_softmax_grad returns the gradient")

            @staticmethod
            def jvp(ctx, *tangents):
                raise RuntimeError("linear_softmax_loss has no forward mode")

        _no_backward = NoBackward
    return _no_backward.apply(call, *inputs)


def _stream(torch, device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _workspace(torch, device, fn, *args):
    size = ctypes.c_int64()
    _native.check(fn(*args, ctypes.byref(size)))
    return torch.empty(size.value, dtype=torch.uint8, device=device)


def _head(hidden, weight, labels, row_weight, reduction, softcap, z_loss, grad_scale):
    torch = _torch()
    if not (isinstance(hidden, torch.Tensor) and isinstance(weight, torch.Tensor)
            and isinstance(labels, torch.Tensor)):
        raise ValueError("hidden, weight and labels must be torch tensors")
    code = _dtype_codes.get(hidden.dtype)
    if code is None or weight.dtype != hidden.dtype:
        raise ValueError("hidden and weight must both be bfloat16, float16 or float32, got "
                         f"{hidden.dtype} and {weight.dtype}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden (..., width) and weight (vocab, width) do not fit: "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels {tuple(labels.shape)} must have the shape of hidden without its "
                         f"last axis, {tuple(hidden.shape[:-1])}")
    if labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"labels must be int64 or int32, got {labels.dtype}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean' or 'sum', got {reduction!r}")
    if row_weight is not None and (not isinstance(row_weight, torch.Tensor)
                                   or row_weight.dtype != torch.float32
                                   or row_weight.shape != labels.shape):
        raise ValueError("row_weight must be a float32 tensor of the labels' shape")
    for name, x in (("softcap", softcap), ("z_loss", z_loss)):
        if not 0.0 <= x < math.inf:
            raise ValueError(f"{name} must be finite and >= 0, got {x}")
    if 0.0 < softcap < 1e-6:
        raise ValueError(f"softcap must be 0 or at least 1e-6, got {softcap}")
    if grad_scale is not None and not math.isfinite(grad_scale):
        raise ValueError(f"grad_scale must be finite, got {grad_scale}")
    dev = hidden.device
    if dev.type != "cuda":
        raise ValueError("hidden must be on a GPU")
    for name, t in (("weight", weight), ("labels", labels), ("row_weight", row_weight)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, hidden on {dev}")
    vocab, width = weight.shape
    if vocab < 1 or width < 1:
        raise ValueError("vocab and width must be at least 1")
    rows = labels.numel()
    grad = grad_scale is not None
    f32 = dict(dtype=torch.float32, device=dev)
    out = [torch.empty((), **f32), torch.empty(labels.shape, **f32),
           torch.empty(labels.shape, **f32)]
    if grad:
        out += [torch.empty(hidden.shape, dtype=hidden.dtype, device=dev),
                torch.empty(weight.shape, dtype=weight.dtype, device=dev)]
    if rows == 0:
        out[0].zero_()
        if grad:
            out[4].zero_()
        return out
    hidden, weight = hidden.reshape(rows, width).resolve_neg(), weight.resolve_neg()
    if width > 1 and hidden.stride(1) != 1 or rows > 1 and hidden.stride(0) < width:
        hidden = hidden.contiguous()
    if width > 1 and weight.stride(1) != 1 or vocab > 1 and weight.stride(0) < width:
        weight = weight.contiguous()
    labels = labels.reshape(rows).resolve_neg().to(torch.int64).contiguous()
    if row_weight is not None:
        row_weight = row_weight.reshape(rows).resolve_neg().contiguous()
    h_stride = max(hidden.stride(0), width)  # a single row may have any stride
    w_stride = max(weight.stride(0), width)
    L = _native.lib()
    ws = _workspace(torch, dev, L.bsscl_head_workspace, code, rows, width, vocab,
                    weight.data_ptr(), w_stride, int(grad))
    args = [dev.index, _stream(torch, dev), code, hidden.data_ptr(), h_stride, weight.data_ptr(),
            w_stride, labels.data_ptr(), None if row_weight is None else row_weight.data_ptr(),
            rows, width, vocab, _REDUCTIONS[reduction], float(softcap), float(z_loss)]
    head = [t.data_ptr() for t in out[:3]]
    if grad:
        _native.check(L.bsscl_head_grad(*args, float(grad_scale), *head, out[3].data_ptr(), width,
                                        out[4].data_ptr(), width, ws.data_ptr(), ws.numel()))
    else:
        _native.check(L.bsscl_head_loss(*args, *head, ws.data_ptr(), ws.numel()))
    return out


def linear_softmax_loss(hidden, weight, labels, *, row_weight=None, reduction="mean", softcap=0.0,
                        z_loss=0.0):
    """Softmax cross entropy of the scores hidden @ weight.T, without keeping
    the scores: what a call takes besides its outputs is a copy of the rows with
    a label and 8 bytes a row and 128 or 256 classes (and a copy of a weight
    whose rows are not of 16-byte multiples).

    hidden (..., width) and weight (vocab, width) are bfloat16, float16 or
    float32; labels (...) int64 or int32.  A row whose label is outside
    [0, vocab), such as -1 or -100, is left out: its loss and lse are 0,
    whatever its hidden values are.  row_weight (...) float32 weighs the rows;
    reduction "mean" divides by the counting rows' sum of weights, "sum" does
    not.  softcap c >= 1e-6 puts c * tanh(s / c) in the place of each score, and
    z_loss zeta adds zeta * lse^2 to each row's loss.

    Returns (loss, row_loss, lse) in float32: the reduced loss, each row's
    unweighted loss (for z_loss=0 the negative log-probability of its label)
    and each row's log of the sum of exponentials.  Where an input requires
    gradients, backward through the results raises an error: take
    linear_softmax_grad.
    """
    return SoftmaxLoss(*_without_graph(
        _torch(),
        lambda: _head(hidden, weight, labels, row_weight, reduction, softcap, z_loss, None),
        (hidden, weight, row_weight)))


def linear_softmax_grad(hidden, weight, labels, *, row_weight=None, reduction="mean", softcap=0.0,
                        z_loss=0.0, grad_scale=1.0):
    """linear_softmax_loss with its gradient: (loss, row_loss, lse, d_hidden,
    d_weight).

    d_hidden and d_weight are the gradients of the reduced loss times
    grad_scale (the loss scale of a float16 run; clip_grads and grad_norm take
    its inverse), in the inputs' dtype; rows left out have zeros.  All results
    are values without a graph, also where inputs require gradients: hand
    d_hidden on with hidden.backward(r.d_hidden).

    While it runs, a call takes room for exponentials of the scores in the
    inputs' dtype: of all rows up to about 1 GiB + vocab * width * 4 bytes, of 1
    GiB of rows at a time beyond that, with float32 sums of d_weight then.
    """
    return SoftmaxGrad(*_head(hidden, weight, labels, row_weight, reduction, softcap, z_loss,
                              float(grad_scale)))


def _dense(t):
    """Whether t's values fill one block of memory, in whatever order."""
    size = 1
    for stride, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != size:
            return False
        size *= n
    return True


def _list(torch, tensors, what):
    """(addresses, lengths, dtype codes, GPU) of the tensors as arrays for the
    C ABI, and whether all are contiguous.  Lists are long and the kernels short:
    one pass of the tensors' methods each, and no loop of Python statements unless
    something is odd."""
    if not tensors:
        raise ValueError(f"{what} is empty")
    Tensor = torch.Tensor
    try:
        ptrs = array("Q", map(Tensor.data_ptr, tensors))
        lengths = array("q", map(Tensor.numel, tensors))
        devices = set(map(Tensor.get_device, tensors))
        dense = all(map(Tensor.is_contiguous, tensors))
        dtypes = [t.dtype for t in tensors]
    except (TypeError, RuntimeError):
        bad = [t for t in tensors if not isinstance(t, Tensor)]
        if not bad:
            raise
        raise ValueError(f"{what} must be torch tensors, got {type(bad[0]).__name__}") from None
    kinds = set(dtypes)
    if not kinds <= _dtype_codes.keys():
        raise ValueError(f"{what} must be bfloat16, float16 or float32, got "
                         f"{(kinds - _dtype_codes.keys()).pop()}")
    if len(devices) != 1 or min(devices) < 0:
        raise ValueError(f"{what} must all be on one GPU")
    if not dense:
        for t in tensors:
            if not t.is_contiguous() and not _dense(t):
                raise ValueError(f"{what} must be dense: a tensor of shape {tuple(t.shape)} has "
                                 f"strides {t.stride()}")
    if len(kinds) == 1:
        codes = array("i", [_dtype_codes[dtypes[0]]]) * len(tensors)
    else:
        codes = array("i", map(_dtype_codes.__getitem__, dtypes))
    return ptrs, lengths, codes, devices.pop(), dense


def _norm(tensors, inv_scale, max_norm, out):
    torch = _torch()
    tensors = list(tensors)
    ptrs, lengths, codes, index, dense = _list(torch, tensors, "tensors")
    n = len(tensors)
    outs = ptrs
    if out is not None:
        out = list(out)
        outs, _, out_codes, out_index, out_dense = _list(torch, out, "out")
        Tensor = torch.Tensor
        if (len(out) != n or out_codes != codes or out_index != index
                or not all(map(Tensor.is_same_size, out, tensors))
                or not (dense and out_dense)  # (contiguous values lie alike)
                and any(o.stride() != t.stride() for o, t in zip(out, tensors))
                or list(map(Tensor.is_neg, out)) != list(map(Tensor.is_neg, tensors))):
            raise ValueError("out must match tensors in number, shape, strides, dtype and GPU")

    def at(a):
        return a.buffer_info()[0]

    written = () if max_norm is None else tensors if out is None else out
    if torch.is_grad_enabled() and any(map(_requires_grad, written)):
        raise ValueError("clip_grads writes to tensors that require gradients (parameters in the "
                         "place of their gradients?): detach them or call it under no_grad")
    dev = torch.device("cuda", index)
    L = _native.lib()
    ws = _workspace(torch, dev, L.bsscl_grad_norm_workspace, n, at(lengths))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    args = (index, _stream(torch, dev), n, at(ptrs))
    if max_norm is None:
        _native.check(L.bsscl_grad_norm(*args, at(lengths), at(codes), float(inv_scale),
                                        norm.data_ptr(), ws.data_ptr(), ws.numel()))
    else:
        _native.check(L.bsscl_clip_grads(*args, at(outs), at(lengths), at(codes),
                                         float(inv_scale), max_norm, norm.data_ptr(),
                                         ws.data_ptr(), ws.numel()))
        # (So that a graph that saved one of them says so in backward.)
        torch.autograd.graph.increment_version(written)
    return norm


def grad_norm(tensors, *, inv_scale=1.0):
    """The 2-norm over all values of the tensors, times abs(inv_scale), as a
    float32 tensor.  tensors: dense (in any order of axes) bfloat16, float16
    or float32 tensors on one GPU, mixed and of any sizes."""
    return _norm(tensors, inv_scale, None, None)


def clip_grads(tensors, max_norm, *, inv_scale=1.0, out=None):
    """Scales the tensors by inv_scale * min(1, max_norm / norm), where norm
    is grad_norm(tensors, inv_scale=inv_scale), in place or into the tensors
    of `out` (same shapes, strides and dtypes), and returns norm.

    A norm that is NaN or infinite clips nothing (the factor is inv_scale):
    look at the returned norm and skip the step.  Tensors to be written may
    not overlap each other or another tensor, nor, while gradients are
    recorded, require gradients."""
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    return _norm(tensors, inv_scale, max_norm, out)

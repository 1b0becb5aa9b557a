"""The 2-norm over all gradients of a step and their clipping by it (muzero_amd/csrc/gradnorm_kernels.hip): what stands between
loss.backward() and optimizer.step() (main.py:266-267) when a step must not be allowed to run away.

A list of tensors is one operator: one launch per 128 tensors for the norm and one for the scaling, whatever their sizes; the flat
buffer of a ``train.FlatGradBucket`` is a list of one.  Nothing here waits for the GPU.  No CPU fallback: host tensors raise."""
import ctypes as C

import torch

from . import _lib as L

_DT = {torch.float32: L.MZ_F32, torch.bfloat16: L.MZ_BF16, torch.float16: L.MZ_F16}


def _dense(t):
    """its elements lie together, in any order of the axes (a channels_last gradient does)"""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _list(who, tensors):
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not tensors:
        raise L.MzError("%s: needs at least one tensor" % who)
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise L.MzError("%s: muzero_amd kernels need device tensors; got a %s tensor (no CPU fallback)" % (who, t.device))
        if t.dtype not in _DT:
            raise L.MzError("%s: float32, bfloat16 or float16 tensors, got %s" % (who, t.dtype))
        if not t.is_contiguous() and not _dense(t):
            raise L.MzError("%s: the elements of a tensor have to lie together, got shape %s with strides %s" % (who, tuple(t.shape), t.stride()))
    if len({t.get_device() for t in tensors}) != 1:
        raise L.MzError("%s: the tensors are on different devices" % who)
    return tensors, dev


def _call(name, tensors, outs, dev, *args):
    k = len(tensors)
    words = []
    for t, o in zip(tensors, outs):
        words += (t.data_ptr(), o.data_ptr(), t.numel(), _DT[t.dtype] | _DT[o.dtype] << 32)   # mz_grad_tensor
    table = (C.c_int64 * (4 * k))(*words)
    with torch.cuda.device(dev):
        nbytes = L.lib.mz_grad_workspace_bytes(k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        L.call(name, table, k, *args, C.c_void_p(ws.data_ptr()), nbytes, C.c_void_p(norm.data_ptr()), L.current_stream())
    return norm


@torch.no_grad()
def grad_norm(tensors):
    """sqrt of the sum of squares over all elements of `tensors` (a tensor or a list; float32 / bfloat16 / float16, mixed as they come,
    elements lying together in any order of the axes) as a 0-d float32 tensor.  The sums are held in 64 bits in a fixed order.
    inf or NaN among the elements gives inf or NaN."""
    tensors, dev = _list("grad_norm", tensors)
    return _call("mz_grad_norm", tensors, tensors, dev)


@torch.no_grad()
def clip_grad_norm(tensors, max_norm, out=None):
    """scale all of `tensors` by min(1, max_norm / (norm + 1e-6)) and return the norm they had (a 0-d float32 tensor, not waited for).
    out: None = in place; or a list of tensors of the same shapes and strides, of the gradients' dtypes or float32 (16-bit gradients
    into the ones that the optimiser reads), which get the scaled values while `tensors` stay as they are.  With an infinite norm the
    factor is 0, with a NaN it is NaN, as the formula has it: the returned norm says so, and the step can be left out."""
    tensors, dev = _list("clip_grad_norm", tensors)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise L.MzError("clip_grad_norm: max_norm has to be 0 or more, got %r" % max_norm)
    outs = tensors
    if out is not None:
        outs, odev = _list("clip_grad_norm out", out)
        if len(outs) != len(tensors) or odev != dev:
            raise L.MzError("clip_grad_norm: out needs one tensor per gradient, on their device")
        for t, o in zip(tensors, outs):
            if o.shape != t.shape or (o.stride() != t.stride() and not (o.is_contiguous() and t.is_contiguous())):
                raise L.MzError("clip_grad_norm: out has to have the gradients' shapes and strides, got %s %s for %s %s"
                                % (tuple(o.shape), o.stride(), tuple(t.shape), t.stride()))
            if o.dtype != t.dtype and o.dtype != torch.float32:
                raise L.MzError("clip_grad_norm: out has the gradients' dtype or float32, got %s for %s" % (o.dtype, t.dtype))
    return _call("mz_grad_clip", tensors, outs, dev, max_norm)

"""The 2-norm over all gradients of a step and their clipping by it (muzero_amd/csrc/gradnorm_kernels.hip): what stands between
loss.backward() and optimizer.step() (main.py:266-267) when a step must not be allowed to run away.

A list of tensors is one operator: one launch per 256 tensors for the norm and per 128 for the scaling, whatever their sizes; the flat
buffer of a ``train.FlatGradBucket`` is a list of one.  Nothing here waits for the GPU.  No CPU fallback: host tensors raise.

Neither has a derivative: where tensors carry a graph of their own and gradients are recorded, a backward pass that comes to the norm
or to what was scaled raises an error.  Not so under torch.no_grad(); and leaves are scaled as values, as an optimiser does."""
import operator
import struct

import torch

from . import _lib as L

_DT = {torch.float32: L.MZ_F32, torch.bfloat16: L.MZ_BF16, torch.float16: L.MZ_F16}
_T = torch.Tensor
_DTYPE_OF = operator.attrgetter("dtype")


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


def _columns(who, tensors):
    """-> pointers, sizes, dtype codes, GPU index of a list that the kernels can take, and whether all are contiguous.  (Most of a call's time on the host: each
    question goes over the whole list at once, and the checks over the answers.)"""
    if not tensors:
        raise L.MzError("%s: needs at least one tensor" % who)
    gpus = list(map(_T.get_device, tensors))
    index = gpus[0]
    if index < 0 or gpus.count(index) != len(gpus):
        raise L.MzError("%s: muzero_amd kernels need device tensors, all on one GPU; got %s (no CPU fallback)" % (who, sorted({str(t.device) for t in tensors})))
    dtypes = list(map(_DTYPE_OF, tensors))
    kinds = set(dtypes)
    if not kinds <= _DT.keys():
        raise L.MzError("%s: float32, bfloat16 or float16 tensors, got %s" % (who, kinds - _DT.keys()))
    together = all(map(_T.is_contiguous, tensors))
    if not together:
        for t in tensors:
            if not _dense(t):
                raise L.MzError("%s: the elements of a tensor have to lie together, got shape %s with strides %s" % (who, tuple(t.shape), t.stride()))
    codes = [_DT[dtypes[0]]] * len(dtypes) if len(kinds) == 1 else [_DT[d] for d in dtypes]
    return list(map(_T.data_ptr, tensors)), list(map(_T.numel, tensors)), codes, index, together


class _NoDerivative(torch.autograd.Function):
    """the norm as a function of the tensors"""

    @staticmethod
    def forward(ctx, norm, *tensors):
        return norm.view_as(norm)

    @staticmethod
    def backward(ctx, go):
        raise L.MzError("gradnorm: the norm and the clipping have no derivative (detach the tensors, or call under torch.no_grad())")


class _ScaledInPlace(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tensor):
        ctx.mark_dirty(tensor)
        return tensor

    backward = _NoDerivative.backward


def _recorded(tensors):
    """those that carry a graph, where gradients are recorded.  (One pass over the list in torch itself.)"""
    if torch.is_grad_enabled() and torch._C._any_requires_grad(*tensors):
        return [t for t in tensors if t.requires_grad]
    return []


def _call(name, dev, src, dst, sizes, types, index, *args):
    k = len(src)
    words = [0] * (4 * k)                      # mz_grad_tensor: src, dst, n, src_dtype | dst_dtype << 32
    words[::4] = src
    if dst is not None:
        words[1::4] = dst
    words[2::4] = sizes
    words[3::4] = types
    table = struct.pack("%dq" % (4 * k), *words)
    nbytes = L.lib.mz_grad_workspace_bytes(k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    L.call_on(index, name, table, k, *args, ws.data_ptr(), nbytes, norm.data_ptr())
    return norm


def grad_norm(tensors):
    """sqrt of the sum of squares over all elements of `tensors` (a tensor or a list; float32 / bfloat16 / float16, mixed as they come,
    elements lying together in any order of the axes) as a 0-d float32 tensor without a derivative.  The sums are held in 64 bits in a fixed order.
    inf or NaN among the elements gives inf or NaN."""
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    ptrs, sizes, codes, index, _ = _columns("grad_norm", tensors)
    norm = _call("mz_grad_norm", tensors[0].device, ptrs, None, sizes, codes, index)
    recorded = _recorded(tensors)
    return _NoDerivative.apply(norm, *recorded) if recorded else norm


def clip_grad_norm(tensors, max_norm, out=None):
    """scale all of `tensors` by min(1, max_norm / (norm + 1e-6)) and return the norm they had (a 0-d float32 tensor, not waited for).
    out: None = in place; or a list of tensors of the same shapes and strides, of the gradients' dtypes or float32 (16-bit gradients
    into the ones that the optimiser reads), which get the scaled values while `tensors` stay as they are.  With an infinite norm the
    factor is 0, with a NaN it is NaN, as the formula has it: the returned norm says so, and the step can be left out."""
    who = "clip_grad_norm"
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    ptrs, sizes, codes, index, together = _columns(who, tensors)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise L.MzError("%s: max_norm has to be 0 or more, got %r" % (who, max_norm))
    if out is None:
        outs, dst, dst_codes = tensors, ptrs, codes
    else:
        outs = [out] if torch.is_tensor(out) else list(out)
        dst, _, dst_codes, oindex, out_together = _columns(who + " out", outs)
        if len(outs) != len(tensors) or oindex != index:
            raise L.MzError("%s: out needs one tensor per gradient, on their GPU" % who)
        if [t.shape for t in tensors] != [o.shape for o in outs] or (not (together and out_together) and any(
                o.stride() != t.stride() and not (o.is_contiguous() and t.is_contiguous()) for t, o in zip(tensors, outs))):
            raise L.MzError("%s: out has to have the gradients' shapes and strides" % who)
        if dst_codes != codes and any(d != s and d != L.MZ_F32 for s, d in zip(codes, dst_codes)):
            raise L.MzError("%s: out has the gradients' dtype or float32" % who)
    recorded = _recorded(tensors)
    if recorded and out is not None:
        raise L.MzError("%s: out= takes no tensors that carry a graph (detach them, or call under torch.no_grad())" % who)
    inner = [t for t in (recorded if out is None else _recorded(outs)) if not t.is_leaf]
    for t in inner:
        _ScaledInPlace.apply(t)
    if out is None and codes.count(codes[0]) == len(codes):
        types = [codes[0] * (1 + (1 << 32))] * len(codes)
    else:
        types = [s | d << 32 for s, d in zip(codes, dst_codes)]
    norm = _call("mz_grad_clip", tensors[0].device, ptrs, dst, sizes, types, index, max_norm)
    torch.autograd.graph.increment_version(outs)      # autograd's check of tensors changed in place sees these too
    return _NoDerivative.apply(norm, *recorded) if recorded else norm

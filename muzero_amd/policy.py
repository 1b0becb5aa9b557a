"""What is done with a policy's logits: drawing an action (beside ``mcts.select_action`` and ``arena.softmax_sample``, which draw
from visit counts, main.py:128-140, test.py:228-243) and learning from target distributions (the cross-entropy of main.py:261 with the
gradient that main.py:266 asks autograd for), on the hand-written kernels of muzero_amd/csrc/policy_*.hip.

The network's ``Prediction`` returns softmaxed probabilities; these operators take what stands before that softmax (or the
logarithm of the probabilities, which differs from it by a constant per row).  Rows are games, positions or requests; the columns
are actions: this game's 65 or any other number.  ``legal`` says which of them may be played: a bool tensor of the logits' shape, or
for 65 actions the (n,) int64 bitboards that ``BatchedEnv.legal`` holds (the pass is legal where no square is).  No CPU fallback:
host tensors raise."""
import struct

import torch

from . import _lib as L

_DT = {torch.float32: L.MZ_F32, torch.bfloat16: L.MZ_BF16, torch.float16: L.MZ_F16}
# the argument structures of include/muzero_amd.h as bytes: a third of the time that filling a ctypes.Structure takes
_LOSS_ARGS = struct.Struct("9Q6qd4i").pack      # mz_policy_loss_args
_SAMPLE_ARGS = struct.Struct("9Q5q3di4x").pack  # mz_sample_args


def _rows(who, name, t, shape=None, dtypes=tuple(_DT)):
    """(n, v) on the GPU whose rows hold their elements together; returns the rows' stride"""
    if not t.is_cuda:
        raise L.MzError("%s: muzero_amd kernels need device tensors; got %s on %s (no CPU fallback)" % (who, name, t.device))
    if t.dim() != 2 or t.dtype not in dtypes:
        raise L.MzError("%s: %s has to be (n, actions) of %s, got %s %s" % (who, name, " / ".join(str(d) for d in dtypes), tuple(t.shape), t.dtype))
    if shape is not None and t.shape != shape:
        raise L.MzError("%s: %s has shape %s, the logits have %s" % (who, name, tuple(t.shape), tuple(shape)))
    if t.shape[1] < 1:
        raise L.MzError("%s: needs at least one action" % who)
    stride, step = t.stride()
    if step != 1 and t.shape[1] > 1:
        raise L.MzError("%s: the actions of a row of %s have to lie together, got strides %s" % (who, name, t.stride()))
    return stride


def _per_row(who, name, t, n, dtype, dev):
    if not t.is_cuda or t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous() or t.device != dev:
        raise L.MzError("%s: %s has to be a contiguous %s tensor of shape (%d,) on %s, got %s %s on %s"
                        % (who, name, dtype, n, dev, tuple(t.shape), t.dtype, t.device))
    return t.data_ptr()


def _legal(who, legal, logits):
    """-> (pointer of the bytes, their row stride, pointer of the bitboards); 0: none"""
    if legal is None:
        return 0, 0, 0
    if legal.device != logits.device:
        raise L.MzError("%s: legal has to be on the logits' device, got %s (no CPU fallback)" % (who, legal.device))
    if legal.dtype == torch.int64:
        if logits.shape[1] != 65:
            raise L.MzError("%s: bitboards go with 65 actions, the logits have %d" % (who, logits.shape[1]))
        return 0, 0, _per_row(who, "legal", legal, logits.shape[0], torch.int64, logits.device)
    return legal.data_ptr(), _rows(who, "legal", legal, logits.shape, (torch.bool,)), 0


def _places(who, logits, targets, weight, legal):
    """-> what a call of the loss reads: the addresses and the rows' strides"""
    stride = _rows(who, "logits", logits)
    targets_stride = _rows(who, "targets", targets, logits.shape, (logits.dtype, torch.float32))
    if targets.device != logits.device:
        raise L.MzError("%s: targets are on %s, the logits on %s" % (who, targets.device, logits.device))
    weight_ptr = 0 if weight is None else _per_row(who, "weight", weight, logits.shape[0], torch.float32, logits.device)
    allowed, allowed_stride, board = _legal(who, legal, logits)
    return (logits.data_ptr(), targets.data_ptr(), allowed, board, weight_ptr), (stride, targets_stride, allowed_stride)


class _CrossEntropy(torch.autograd.Function):
    """The gradient comes out of the forward pass over the rows, for a loss whose own gradient is 1 (what loss.backward() starts
    from).  backward launches the same kernel with the gradient it is given: where that is 1 the kernel leaves at once, otherwise it
    computes the rows again, so a scaled 16-bit gradient is rounded once, after the scale.  No gradient comes out of the forward pass where
    none is recorded, or where each row has a factor of its own ("none")."""

    @staticmethod
    def forward(ctx, logits, targets, weight, legal, reduction, head, sizes, strides, rest, need):
        n, v = logits.shape
        dev = logits.device
        out = torch.empty((n,) if reduction == "none" else (), dtype=torch.float32, device=dev)
        nbytes = L.lib.mz_policy_loss_workspace_bytes(n, v)
        if nbytes < 0:
            raise L.MzError("cross_entropy: (n, actions) = (%d, %d) is too large" % (n, v))
        grad = None
        if need:
            ctx.save_for_backward(logits, targets, weight, legal)
            ctx.call = head, sizes, strides, rest, nbytes
            if reduction != "none":
                grad = torch.empty((n, v), dtype=logits.dtype, device=dev)
                ctx.capture = L.capture_id(dev.index)
            ctx.ready = grad
        if n == 0:
            return out.fill_(float("nan") if reduction == "mean" else 0.0)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        to = out.data_ptr()
        rows, loss = (to, 0) if reduction == "none" else (0, to)
        L.call_on(dev.index, "mz_policy_loss", _LOSS_ARGS(*head, 0, rows, loss, 0 if grad is None else grad.data_ptr(), *sizes, *strides, *rest, 0, 0), ws.data_ptr(), nbytes)
        return out

    @staticmethod
    def backward(ctx, go):
        saved = ctx.saved_tensors              # also says if one of them was changed in place; asked for once, as recomputed ones have to be
        if torch.is_grad_enabled():            # create_graph: the gradient, and an error when its own is asked for
            with torch.no_grad():
                grad = _CrossEntropy.gradient(ctx, go, *saved)
            grad = _NoSecondDerivative.apply(grad, saved[0], go)
        else:
            grad = _CrossEntropy.gradient(ctx, go, *saved)
        return (grad,) + (None,) * 9

    @staticmethod
    def gradient(ctx, go, logits, targets, weight, legal):
        grad = ctx.ready
        ctx.ready = None                       # handed out once; a second backward pass gets memory of its own
        # ... and so does one in another capture than its forward pass: it may replay without that, and once another factor was there the memory holds
        # that one's gradient.
        skip = grad is not None and ctx.capture == L.capture_id(grad.get_device())
        if not skip:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if logits.shape[0]:
            head, sizes, strides, rest, nbytes = ctx.call
            # Where hooks pack saved tensors (kept on the host, or computed again) these are new ones with strides of their own.  (Asking for all
            # places anew takes 8 us of a pass's 90, the question whether it is needed 1.)
            if (logits.data_ptr() != head[0] or targets.data_ptr() != head[1] or logits.stride() != (strides[0], 1) or targets.stride() != (strides[1], 1)
                    or (weight is not None and weight.data_ptr() != head[4])
                    or (legal is not None and (legal.data_ptr() != (head[2] or head[3]) or (head[2] and legal.stride() != (strides[2], 1))))):
                head, strides = _places("cross_entropy", logits, targets, weight, legal)
            if not go.is_contiguous():
                go = go.contiguous()
            ws = torch.empty(nbytes, dtype=torch.uint8, device=grad.device)   # not the forward's: a captured backward keeps its own
            L.call_on(grad.get_device(), "mz_policy_loss", _LOSS_ARGS(*head, go.data_ptr(), 0, 0, grad.data_ptr(), *sizes, *strides, *rest, go.dim(), skip), ws.data_ptr(), nbytes)
        return grad


class _NoSecondDerivative(torch.autograd.Function):
    """The gradient as a function of the logits and of the loss's own gradient: whatever is asked for behind either of them, a backward pass
    that would need this one's derivative comes through here."""

    @staticmethod
    def forward(ctx, grad, logits, go):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, go):
        raise L.MzError("cross_entropy: there is no second derivative")


def cross_entropy(logits, targets, weight=None, legal=None, reduction="mean"):
    """-sum over the legal actions of targets * log softmax(logits), per row times `weight`: the mean over the n rows, their "sum", or
    "none" = the (n,) rows, in float32, differentiable in the logits (once).

    logits (n, v) float32 / bfloat16 / float16; targets (n, v) of the same dtype or float32, any non-negative shares (they need not add
    up to 1); rows may be strided, a row's elements lie together.  weight float32 (n,): a row of weight 0 (padding) counts in the mean's n
    but gives no loss and no gradient, whatever it holds.  legal: see the module; other places are never used, their gradient is 0,
    and a row without a legal action gives 0.  Targets of 0 count as 0 also against a logit of -inf."""
    who = "cross_entropy"
    if targets.requires_grad or (weight is not None and weight.requires_grad):
        raise L.MzError("%s: targets and weights carry no gradient (detach them)" % who)
    head, strides = _places(who, logits, targets, weight, legal)
    if reduction not in ("mean", "sum", "none"):
        raise L.MzError("%s: reduction is 'mean', 'sum' or 'none', got %r" % (who, reduction))
    n, v = logits.shape
    rest = v, 1.0 / n if reduction == "mean" and n else 1.0, _DT[logits.dtype], _DT[targets.dtype]
    need = logits.requires_grad and torch.is_grad_enabled()   # asked for here: inside forward, gradients are never recorded
    return _CrossEntropy.apply(logits, targets, weight, legal, reduction, head, (n, v), strides, rest, need)


def _setting(who, name, value, n, dtype, dev, low, high):
    """-> (pointer of one value per row or 0, the one value of all rows)"""
    if isinstance(value, torch.Tensor):
        return _per_row(who, name, value, n, dtype, dev), 0
    if not low <= value <= high:
        raise L.MzError("%s: %s = %r is out of its range" % (who, name, value))
    return 0, value


def sample_actions(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, legal=None, out=None):
    """One action per row of logits (n, actions), drawn with the given uniforms u (float64 (n,) in [0, 1)): int32 (n,).

    The draw is from softmax(logits / temperature) over the legal actions, cut to the top_k most likely (0 = all), of these to the
    fewest most likely that together reach the share top_p, of these to the ones at least min_p times as likely as the best; equal
    logits go to the lower index, the best action always stays, temperature 0 takes it.  The answer is the lowest index at which the
    kept mass, cumulated in the order of the indices, exceeds u times its total.  Every setting is a number, or a tensor with one value
    per row (float32; top_k int32).  Masses are held in 64 bits in a fixed order (a long row's total comes from masses of 128
    actions that are right to 2e-12): the same call gives the same actions.

    logits float32 / bfloat16 / float16, up to 2^19 actions, rows may be strided; legal: see the module.  A row without a legal action
    (all others -inf count as not legal), with NaN or +inf at a legal place, or with a temperature of NaN or +inf gives -1.  out: int32
    (n,) to write into."""
    who = "sample_actions"
    stride = _rows(who, "logits", logits)
    n, v = logits.shape
    dev = logits.device
    allowed, allowed_stride, board = _legal(who, legal, logits)
    temperature_of, temperature = _setting(who, "temperature", temperature, n, torch.float32, dev, 0.0, 1e30)
    top_k_of, top_k = _setting(who, "top_k", top_k, n, torch.int32, dev, 0, 1 << 62)
    top_p_of, top_p = _setting(who, "top_p", top_p, n, torch.float32, dev, 0.0, 1.0)
    min_p_of, min_p = _setting(who, "min_p", min_p, n, torch.float32, dev, 0.0, 1.0)
    if int(top_k) != top_k:
        raise L.MzError("%s: top_k = %r is no whole number" % (who, top_k))
    u_ptr = _per_row(who, "u", u, n, torch.float64, dev)
    nbytes = L.lib.mz_sample_actions_workspace_bytes(n, v)
    if nbytes < 0:
        raise L.MzError("%s: (n, actions) = (%d, %d) is too large" % (who, n, v))
    if out is None:
        out = torch.empty(n, dtype=torch.int32, device=dev)
    else:
        _per_row(who, "out", out, n, torch.int32, dev)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    args = _SAMPLE_ARGS(logits.data_ptr(), allowed, board, u_ptr, temperature_of, top_k_of, top_p_of, min_p_of, out.data_ptr(), n, v, stride,
                        allowed_stride, int(top_k), temperature, top_p, min_p, _DT[logits.dtype])
    L.call_on(dev.index, "mz_sample_actions", args, None if ws is None else ws.data_ptr(), nbytes)
    torch.autograd.graph.increment_version(out)
    return out

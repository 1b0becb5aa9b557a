"""Host side of muzero_amd/gradnorm.py without a GPU: what it refuses (no CPU fallback: host tensors raise), and the C entry points'
checks of their lists, which come before any launch."""
import ctypes as C

import pytest
import torch


def _table(L, rows):
    words = []
    for src, dst, n, sd, dd in rows:
        words += (src, dst, n, sd | dd << 32)
    return (C.c_int64 * max(1, len(words)))(*words)


def test_host_tensors_and_empty_lists_are_refused():
    from muzero_amd import _lib as L
    from muzero_amd import gradnorm as G
    with pytest.raises(L.MzError, match="no CPU fallback"):
        G.grad_norm([torch.zeros(4)])
    with pytest.raises(L.MzError, match="no CPU fallback"):
        G.clip_grad_norm(torch.zeros(4), 1.0)
    with pytest.raises(L.MzError, match="at least one"):
        G.grad_norm([])


def test_elements_that_lie_together():
    from muzero_amd.gradnorm import _dense
    t = torch.zeros(4, 6, 5, 3)
    assert _dense(t) and _dense(t.to(memory_format=torch.channels_last)) and _dense(t.permute(2, 0, 3, 1)) and _dense(torch.zeros(1, 5).t())
    assert _dense(torch.zeros(8, 4)[2:5])
    assert not _dense(t[:, 1:]) and not _dense(t[..., ::2]) and not _dense(torch.zeros(1, 3).expand(4, 3))


def test_lists_are_checked_before_any_launch():
    from muzero_amd import _lib as L
    P = 1 << 40                                  # never read: every call below is refused on the host
    nbytes = L.lib.mz_grad_workspace_bytes(1)
    assert nbytes > 0 and L.lib.mz_grad_workspace_bytes(257) == 2 * nbytes and L.lib.mz_grad_workspace_bytes(0) == -1

    def norm(rows, count=None, ws=P, wb=1 << 20, out=P):
        L.call("mz_grad_norm", _table(L, rows), len(rows) if count is None else count, ws, wb, out, None)

    def clip(rows, max_norm=1.0, ws=P, wb=1 << 20, out=P):
        L.call("mz_grad_clip", _table(L, rows), len(rows), max_norm, ws, wb, out, None)

    ok = (P + 4096, P + 4096, 16, 0, 0)
    for rows, why in (([], "at least one"), ([(P, P, -1, 0, 0)], "negative size"), ([(P, P, 4, 7, 0)], "unknown dtype"), ([(0, 0, 4, 0, 0)], "null"),
                      ([(P + 2, P, 4, 0, 0)], "misaligned"), ([(P + 1, P, 4, 1, 1)], "misaligned"), ([(P, P, (1 << 40) + 1, 0, 0)], "too large")):
        with pytest.raises(L.MzError, match=why):
            norm(rows)
        with pytest.raises(L.MzError, match=why):
            clip(rows)
    for kw, why in ((dict(ws=None), "workspace"), (dict(ws=P + 4), "misaligned"), (dict(wb=nbytes - 1), "needed"), (dict(out=None), "null")):
        with pytest.raises(L.MzError, match=why):
            norm([ok], **kw)
        with pytest.raises(L.MzError, match=why):
            clip([ok], **kw)
    for m in (-1.0, float("nan")):
        with pytest.raises(L.MzError, match="max_norm"):
            clip([ok], max_norm=m)
    for row, why in (((P, P, 4, 0, 1), "its dtype or is f32"), ((P, P, 4, 1, 2), "its dtype or is f32"), ((P, 0, 4, 0, 0), "output 0"), ((P, P + 2, 4, 1, 0), "output 0")):
        with pytest.raises(L.MzError, match=why):
            clip([row])


@pytest.mark.parametrize("rows", [
    [(0, 0, 8, 0, 0), (0, 0, 8, 0, 0)],          # the same tensor twice, in place
    [(0, 0, 8, 0, 0), (16, 16, 8, 0, 0)],        # two views that share elements
    [(0, 64, 8, 0, 0), (32, 80, 8, 0, 0)],       # outputs that share elements
    [(0, 32, 8, 0, 0), (32, 96, 8, 0, 0)],       # one's output on the other's gradient
    [(0, 16, 8, 0, 0)],                          # its own output in part
    [(0, 0, 8, 1, 0)],                           # f32 over bf16 in place
    [(64, 128, 8, 0, 0), (0, 0, 32, 0, 0)],      # a gradient inside another one that is written
])
def test_overlapping_outputs_are_refused(rows):
    from muzero_amd import _lib as L
    P = 1 << 40
    with pytest.raises(L.MzError, match="overlaps"):
        L.call("mz_grad_clip", _table(L, [(P + a, P + b, n, s, d) for a, b, n, s, d in rows]), len(rows), 1.0, P, 1 << 20, P, None)

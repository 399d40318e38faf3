"""CPU: what r3det.ops.log_probs refuses, at the Python boundary and at the C entries (which check before any launch)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from r3det import _C
from r3det.ops.log_probs import label_log_probs


def test_refusals_of_the_python_entry():
    x, y = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        label_log_probs(x, y)
    with pytest.raises(TypeError, match="tensor"):
        label_log_probs([1.0, 2.0])
    with pytest.raises(TypeError, match="dimension"):
        label_log_probs(torch.tensor(1.0))
    for bad in (x.double(), x.to(torch.int32)):
        with pytest.raises(RuntimeError, match="fp32, fp16 or bf16"):
            label_log_probs(bad, y)
    with pytest.raises(ValueError, match="classes"):
        label_log_probs(torch.zeros(3, 0))
    for k in (-1, 6, 1.5, True):
        with pytest.raises(ValueError, match="top_k"):
            label_log_probs(x, y, top_k=k)
    with pytest.raises(ValueError, match="top_k"):
        label_log_probs(torch.zeros(2, 100), top_k=65)
    with pytest.raises(RuntimeError, match="int64"):
        label_log_probs(x, y.int())
    with pytest.raises(ValueError, match="shape"):
        label_log_probs(x, y[:2])
    with pytest.raises(TypeError, match="ignore_index"):
        label_log_probs(x, y, ignore_index=1.0)
    with pytest.raises(TypeError, match="ignore_index"):
        label_log_probs(x, y, ignore_index=True)
    with pytest.raises(ValueError, match="64 bits"):
        label_log_probs(x, y, ignore_index=2 ** 63)


def test_refusals_of_the_c_entries():
    L = _C.lib()
    p = ctypes.c_void_p(1 << 20)  # (never followed: every call below ends at its checks)

    def forward(x=p, dtype=0, rows=4, classes=8, stride=8, labels=p, k=0, lp=p, top=p, ws=None, nbytes=0):
        return L.r3det_label_log_probs(x, dtype, rows, classes, stride, labels, 0, 0, k, lp, p, top, top, None, ws, nbytes, None)
    assert forward(rows=0) == 0
    for bad in (dict(x=None), dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(classes=0), dict(classes=1 << 31),
                dict(stride=-1), dict(k=-1), dict(k=9), dict(classes=100, k=65), dict(lp=None), dict(k=2, top=None)):
        assert forward(**bad) == -1, bad
    need = L.r3det_label_log_probs_workspace_bytes(1, 1 << 20, 4)
    assert need > 0
    assert forward(rows=1, classes=1 << 20, k=4) == -3
    assert forward(rows=1, classes=1 << 20, k=4, ws=p, nbytes=need - 1) == -3
    assert L.r3det_label_log_probs_workspace_bytes(1000, 1000, 4) == 0

    def backward(x=p, dtype=0, rows=4, classes=8, labels=p, k=0, stats=p, h=p, ix=p, dlp=p, dh=p, dtop=None, dx=p):
        return L.r3det_label_log_probs_backward(x, dtype, rows, classes, classes, labels, 0, 0, k, stats, h, ix, dlp, dh, dtop,
                                                dx, None)
    assert backward(rows=0) == 0
    for bad in (dict(x=None), dict(dtype=3), dict(rows=-1), dict(classes=0), dict(stats=None), dict(dx=None), dict(labels=None),
                dict(h=None), dict(dtop=p), dict(k=2, dtop=p, ix=None)):
        assert backward(**bad) == -1, bad


def test_dual_tensors_are_refused():
    """A dual tensor needs no gradient: computed all the same, its result would have no tangent, which reads as zero."""
    x, y = torch.randn(3, 5), torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert not dual.requires_grad
        with pytest.raises(RuntimeError, match="forward-mode"):
            label_log_probs(dual, y)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            label_log_probs(dual, y)
        with pytest.raises(RuntimeError, match="CUDA tensor"):  # (no tangent: the next check's)
            label_log_probs(x, y)

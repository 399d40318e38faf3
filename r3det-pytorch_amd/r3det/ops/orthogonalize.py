"""Orthogonalised updates of weight matrices by Newton-Schulz products (include/r3det_hip.h: r3det_orthogonalize,
r3det_orthogonal_update), for a ragged list of matrices in one chain of launches.

Not one of the reference's extension ops: it serves the training step's optimiser (``dist_train.Muon``).  A weight of more
than two dimensions is the matrix of its first dimension against all others, as for a convolution's (out, in * kh * kw).
"""
import bisect
import ctypes
import math

import torch

from .. import _C
from .log_probs import DTYPES

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
MOST_ROWS, MOST_COLUMNS, MOST_MATRICES = 32768, 65535 * 64, 65536  # (the C entries', too)


def _numbers(steps, coefficients, eps):
    if isinstance(steps, bool) or not isinstance(steps, int) or not 1 <= steps <= 64:
        raise ValueError(f"steps must be an integer between 1 and 64, got {steps!r}")
    a, b, c = (float(v) for v in coefficients)
    if not float(eps) >= 0:
        raise ValueError(f"eps must not be negative, got {eps!r}")
    return steps, a, b, c, float(eps)


def _check(t, name, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t)}")
    if t.dim() < 2:
        raise ValueError(f"{name} must have at least two dimensions, got {t.dim()}")
    if like is not None and (t.shape != like.shape or t.device != like.device):
        raise ValueError(f"{name} must match its weight: {tuple(t.shape)} on {t.device} against {tuple(like.shape)} on {like.device}")


def _same(ts, name):
    if ts and ts[0].dtype not in DTYPES:
        raise RuntimeError(f"{name} must be fp32, fp16 or bf16, got {ts[0].dtype}")
    for t in ts:
        if t.dtype != ts[0].dtype or t.device != ts[0].device:
            raise RuntimeError(f"{name} must be of one type and on one device")
        rows, cols = t.size(0), t.numel() // max(t.size(0), 1)
        if t.numel() >= 2 ** 31 or min(rows, cols) > MOST_ROWS or (t.numel() and max(rows, cols) > MOST_COLUMNS):
            raise ValueError(f"{name}: a matrix of {rows} x {cols} is not taken (at most 2^31 - 1 elements, {MOST_ROWS} on the "
                             f"smaller side, {MOST_COLUMNS} on the longer)")
    if len(ts) > MOST_MATRICES and sum(t.numel() > 0 for t in ts) > MOST_MATRICES:
        raise ValueError(f"{name}: at most {MOST_MATRICES} matrices are taken at once, got {len(ts)}")
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be CUDA tensors (HIP device tensors on ROCm)")


def _pointers(ts):
    return (ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts])


def _sizes(ts):
    rows = [t.size(0) for t in ts]
    make = ctypes.c_int * len(ts)
    return make(*rows), make(*[t.numel() // r for t, r in zip(ts, rows)])


def _workspace(count, rows, cols, device):
    n = _C.lib().r3det_orthogonalize_workspace_bytes(count, rows, cols)
    return torch.empty(n, dtype=torch.uint8, device=device), n


@torch.no_grad()
def orthogonalize(tensors, steps=STEPS, coefficients=COEFFICIENTS, eps=1e-7):
    """One matrix or a list of matrices (fp32, fp16 or bf16, all alike; more than two dimensions: (size(0), rest)) ->
    new, contiguous tensors of the same shapes and type: ``X = G / (|G| + eps)``, then ``steps`` times
    ``X = a X + (b A + c A A) X`` with ``A = X X^t`` (of the transpose where there are more rows than columns), which moves
    every singular value towards 1 and keeps the singular vectors.  Computed to fp32's accuracy whatever the type and
    whatever else is in the list, and rounded once: as far from 64 bits as the formula op by op in fp32 is, within a factor of
    three and 1e-6 of its norm (some 1e-6; more both ways where one singular value is far above the others).  What a norm far
    below ``eps`` leaves small is exact to 5e-9 an entry only (with the usual steps).  A zero matrix stays zero (with eps = 0:
    NaN); NaN or an infinity in a matrix makes that matrix NaN and no other.  The coefficients must keep the spectral norms of
    X, A and P A, with P = a + b A + c A A, and of P less its vertex a - b b / 4 c below 15 (RuntimeError otherwise).  No
    gradient flows through it.  Runs on the current stream of the tensors' device, without a host synchronisation.

    At most 65536 matrices at a time, of at most 2^31 - 1 elements, 32768 on the smaller side and 4194240 on the longer
    (ValueError otherwise).  The call takes a workspace: for a matrix of n x m, n the smaller, both rounded up to a multiple of
    128, 8 to 12 n m + 24 n n bytes and up to 4 n n more for every 512 of m (14 bytes an element for a detector's weights, 0.6 GB;
    a single row counts as 128: 1.06 GB for one of a million); nothing for matrices of at most 64 x 128."""
    one = isinstance(tensors, torch.Tensor)
    ts = [tensors] if one else list(tensors)
    steps, a, b, c, eps = _numbers(steps, coefficients, eps)
    for t in ts:
        _check(t, "tensors")
    _same(ts, "tensors")
    outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in ts]
    live = [(t.contiguous(), o) for t, o in zip(ts, outs) if t.numel()]
    if live:
        src, dst = [p[0] for p in live], [p[1] for p in live]
        rows, cols = _sizes(src)
        ws, n = _workspace(len(src), rows, cols, src[0].device)
        _C.run_on(src[0].device, "r3det_orthogonalize", _C.lib().r3det_orthogonalize, len(src), _pointers(src), _pointers(dst),
                  DTYPES[src[0].dtype], rows, cols, steps, a, b, c, eps, ws.data_ptr(), n)
    return outs[0] if one else outs


def alike(t, like):
    """Whether two tensors of one shape have the same strides, where those say something (a dimension of size one has any)."""
    return t.stride() == like.stride() or all(n < 2 or a == b for a, b, n in zip(t.stride(), like.stride(), t.shape))


def _dense(t):
    """Whether the tensor's memory, read in order, is (size(0), rest) in some order of the rest -- contiguous, or a
    channels_last convolution weight.  The order of the columns does not matter to the update as long as the weight,
    its gradient and its momentum have the same one."""
    if t.is_contiguous():
        return True
    return t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last)


def _apart(params, buffers, grads):
    """All matrices are updated at once: none may share memory with another, nor with a gradient."""
    def span(t):
        at = t.data_ptr()
        return at, at + t.numel() * t.element_size()

    spans = sorted(map(span, params + buffers))
    starts = [s[0] for s in spans]
    shared = any(a[1] > b for a, b in zip(spans, starts[1:]))
    for begin, end in () if shared else map(span, grads):
        i = bisect.bisect_right(starts, begin)
        shared = shared or (i > 0 and spans[i - 1][1] > begin) or (i < len(starts) and starts[i] < end)
    if shared:
        raise ValueError("the same weight or buffer comes twice, or shares memory with another one or with a gradient")


@torch.no_grad()
def orthogonal_update_(params, grads, buffers, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=STEPS,
                       coefficients=COEFFICIENTS, eps=1e-7, scale="rms"):
    """One optimiser step for a list of weights, in place, per weight W with gradient G and momentum M:

        M = momentum * M + G;   U = G + momentum * M (nesterov) or M
        W = (1 - lr * weight_decay) * W - lr * s * orthogonalize(U)

    with ``s = 0.2 sqrt(max(rows, cols))`` for ``scale="rms"`` (the update's entries are then of about the size of an adaptive
    optimiser's) or ``sqrt(max(1, rows / cols))`` for ``"spectral"``, or a number.  ``params`` and ``grads`` fp32, fp16 or bf16,
    all alike; ``buffers`` fp32.  A weight must be contiguous or channels_last, its momentum laid out alike; a gradient
    laid out otherwise is copied.  No weight or buffer may share memory with another or with a gradient.  ``lr`` and the
    other numbers are read when the call is made (a captured graph keeps them).  Sizes and workspace as for
    ``orthogonalize``."""
    params, grads, buffers = list(params), list(grads), list(buffers)
    if not len(params) == len(grads) == len(buffers):
        raise ValueError(f"{len(params)} params, {len(grads)} grads and {len(buffers)} buffers")
    steps, a, b, c, eps = _numbers(steps, coefficients, eps)
    lr, momentum, weight_decay = float(lr), float(momentum), float(weight_decay)
    if not (lr >= 0 and momentum >= 0 and weight_decay >= 0):
        raise ValueError("lr, momentum and weight_decay must not be negative")
    if not (scale in ("rms", "spectral") if isinstance(scale, str) else isinstance(scale, (int, float))):
        raise ValueError(f'scale must be "rms", "spectral" or a number, got {scale!r}')
    for p, g, m in zip(params, grads, buffers):
        _check(p, "params")
        _check(g, "grads", p)
        _check(m, "buffers", p)
        if g.dtype != p.dtype:
            raise RuntimeError(f"grads must be of their weight's type {p.dtype}, got {g.dtype}")
        if m.dtype != torch.float32:
            raise RuntimeError(f"buffers must be fp32, got {m.dtype}")
        if not _dense(p) or not (alike(m, p) or p.numel() == 0):
            raise RuntimeError("params must be contiguous or channels_last, and their buffers laid out alike")
    live = [(p, g, m, alike(g, p)) for p, g, m in zip(params, grads, buffers) if p.numel()]
    ps, ms = [t[0] for t in live], [t[2] for t in live]
    _apart(ps, ms, [g for _, g, _, alike in live if alike])
    _same(params, "params")
    if not live:
        return
    gs = [g if alike else torch.empty_like(p).copy_(g) for p, g, _, alike in live]
    rows, cols = _sizes(ps)
    if scale == "rms":
        s = [0.2 * math.sqrt(max(r, k)) for r, k in zip(rows, cols)]
    elif scale == "spectral":
        s = [math.sqrt(max(1.0, r / k)) for r, k in zip(rows, cols)]
    else:
        s = [float(scale)] * len(ps)
    rates = (ctypes.c_float * len(ps))(*[lr * v for v in s])
    ws, n = _workspace(len(ps), rows, cols, ps[0].device)
    _C.run_on(ps[0].device, "r3det_orthogonal_update", _C.lib().r3det_orthogonal_update, len(ps), _pointers(gs), _pointers(ps),
              _pointers(ms), DTYPES[ps[0].dtype], rows, cols, rates, 1.0 - lr * weight_decay, momentum, int(bool(nesterov)), steps,
              a, b, c, eps, ws.data_ptr(), n)
    torch.autograd.graph.increment_version(ps + ms)

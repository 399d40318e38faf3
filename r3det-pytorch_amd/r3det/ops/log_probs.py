"""Log probabilities of given labels with the entropy and the best alternatives of every row, and their gradient
(include/r3det_hip.h: r3det_label_log_probs).

Not one of the reference's extension ops: mmdet's softmax classification loss (``CrossEntropyLoss(use_sigmoid=False)``,
which the rotated heads' ``use_sigmoid_cls=False`` branch selects) and the ranking of softmax scores are made of it
(models/losses.py, models/heads.py).
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from .. import _C

TOP_MAX = 64
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class LabelLogProbs(NamedTuple):
    log_prob: Optional[torch.Tensor]      # (...) fp32; None without labels
    entropy: Optional[torch.Tensor]       # (...) fp32; None with entropy=False
    top_log_prob: Optional[torch.Tensor]  # (..., top_k) fp32, best first; None with top_k=0
    top_index: Optional[torch.Tensor]     # (..., top_k) int64


def _rows(logits):
    """(..., classes) -> a (rows, classes) view whose rows are contiguous; a copy only where there is no such view."""
    classes = logits.size(-1)
    if logits.stride(-1) != 1 and classes > 1:
        logits = logits.contiguous()
    try:
        return logits.view(-1, classes)
    except RuntimeError:
        return logits.reshape(-1, classes)


def _forward(logits, labels, top_k, want_entropy, ignore_index, want_stats):
    x = _rows(logits)
    rows, classes = x.shape
    lead, dev = logits.shape[:-1], logits.device
    f32 = torch.float32
    log_prob = torch.empty(lead, dtype=f32, device=dev) if labels is not None else None
    entropy = torch.empty(lead, dtype=f32, device=dev) if want_entropy else None
    top_lp = top_ix = stats = ws = None
    if top_k:
        top_lp = torch.empty((*lead, top_k), dtype=f32, device=dev)
        top_ix = torch.empty((*lead, top_k), dtype=torch.int64, device=dev)
    if want_stats:
        stats = torch.empty((rows, 2), dtype=f32, device=dev)
    if labels is not None:
        labels = labels.contiguous()
    if rows:
        L = _C.lib()
        nbytes = L.r3det_label_log_probs_workspace_bytes(rows, classes, top_k)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _C.run_on(dev, "r3det_label_log_probs", L.r3det_label_log_probs, x.data_ptr(), DTYPES[x.dtype], rows, classes, x.stride(0),
                  _at(labels), ignore_index or 0, int(ignore_index is not None), top_k, _at(log_prob), _at(entropy), _at(top_lp),
                  _at(top_ix), _at(stats), _at(ws), nbytes)
    return log_prob, entropy, top_lp, top_ix, labels, stats


def _at(t):
    return None if t is None else t.data_ptr()


class _LabelLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, top_k, want_entropy, ignore_index):
        log_prob, entropy, top_lp, top_ix, labels, stats = _forward(logits.detach(), labels, top_k, want_entropy, ignore_index,
                                                                    True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, labels, stats, entropy, top_ix)
        ctx.args = (top_k, ignore_index)
        if top_ix is not None:
            ctx.mark_non_differentiable(top_ix)
        return log_prob, entropy, top_lp, top_ix

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_lp, d_h, d_top, _):
        if d_lp is None and d_h is None and d_top is None:
            return None, None, None, None, None
        logits, labels, stats, entropy, top_ix = ctx.saved_tensors
        top_k, ignore_index = ctx.args
        x = _rows(logits)
        rows, classes = x.shape
        dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        d_lp, d_h, d_top = (None if d is None else d.contiguous() for d in (d_lp, d_h, d_top))  # (fp32, as the outputs are)
        if rows:
            _C.run_on(logits.device, "r3det_label_log_probs_backward", _C.lib().r3det_label_log_probs_backward, x.data_ptr(),
                      DTYPES[x.dtype], rows, classes, x.stride(0), _at(labels), ignore_index or 0, int(ignore_index is not None),
                      top_k, _at(stats), _at(entropy), _at(top_ix), _at(d_lp), _at(d_h), _at(d_top), dx.data_ptr())
        return dx, None, None, None, None


def label_log_probs(logits, labels=None, top_k=0, entropy=True, ignore_index=None):
    """``logits`` (..., classes) fp32 / fp16 / bf16 on the device, ``labels`` (...) int64 or None ->
    ``LabelLogProbs(log_prob, entropy, top_log_prob, top_index)``; everything in 32 bits whatever the logits' type.

    ``log_prob`` is the log softmax at the label (0, without a gradient, where the label is ``ignore_index``; NaN where a
    label is outside [0, classes) -- nothing here reads labels on the host), ``entropy`` the row's -sum p log p, the top
    ones its ``top_k`` <= min(classes, 64) best classes in order, ties to the lowest index.  Logits of -inf are classes
    that are not offered: a row with none left has log probabilities of -inf, the entropy 0 and no gradient.  NaN or +inf
    in a row makes its numbers NaN; NaN is ranked first.  Differentiable (once, backwards; dual tensors are refused) through all but
    ``top_index``; the logits must stay as they are until the backward pass.  Rows may be any distance apart; other strides are copied first.  Works on the current
    stream of the logits' device; nothing synchronises with the host."""
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        raise TypeError("logits must be a tensor of at least one dimension")
    if logits.dtype not in DTYPES:
        raise RuntimeError(f"logits must be fp32, fp16 or bf16, got {logits.dtype}")
    classes = logits.size(-1)
    if classes < 1 or classes >= 2 ** 31:
        raise ValueError(f"logits must have between 1 and 2^31 - 1 classes, got {classes}")
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k <= min(classes, TOP_MAX):
        raise ValueError(f"top_k must be an integer between 0 and min(classes, {TOP_MAX}), got {top_k!r} for {classes} classes")
    if ignore_index is not None and (isinstance(ignore_index, bool) or not isinstance(ignore_index, int)):
        raise TypeError("ignore_index must be an integer or None")
    if ignore_index is not None and not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must fit 64 bits")
    if labels is not None:
        if not isinstance(labels, torch.Tensor) or labels.dtype != torch.int64:
            raise RuntimeError("labels must be an int64 tensor")
        if labels.device != logits.device:
            raise RuntimeError(f"labels are on {labels.device}, logits on {logits.device}")
        if labels.shape != logits.shape[:-1]:
            raise ValueError(f"labels must have the shape {tuple(logits.shape[:-1])}, got {tuple(labels.shape)}")
    if forward_ad.unpack_dual(logits).tangent is not None:  # (requires_grad says nothing of these)
        raise RuntimeError("label_log_probs has no forward-mode derivative: its result would have no tangent")
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDA tensor (HIP device tensor on ROCm)")
    if logits.requires_grad and torch.is_grad_enabled():
        return LabelLogProbs(*_LabelLogProbs.apply(logits, labels, top_k, bool(entropy), ignore_index))
    return LabelLogProbs(*_forward(logits, labels, top_k, bool(entropy), ignore_index, False)[:4])

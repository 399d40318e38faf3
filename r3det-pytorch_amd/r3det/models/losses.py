"""The two losses the r3det configs select (configs/r3det/r3det_r50_fpn_1x_dota_v1.py:37-43,62-68):
``FocalLoss(use_sigmoid=True, gamma=2.0, alpha=0.25)`` and ``SmoothL1Loss(beta=0.11)``; beside them ``L1Loss`` and, for
heads with a softmax over the classes and the background, ``CrossEntropyLoss(use_sigmoid=False)``.

The classes are mmdet 2.19's (third-party, not under the reference tree); their rules are restated:
elementwise loss, times the per-sample weight, reduced as ``sum / avg_factor`` when ``avg_factor`` is
given with ``reduction='mean'`` (mmdet ``weight_reduce_loss``), times ``loss_weight``.  ``avg_factor``
may be a tensor (the positive count stays on the device: no host synchronisation in the step).
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops.log_probs import label_log_probs


def weight_reduce_loss(loss, weight=None, reduction='mean', avg_factor=None):
    if weight is not None:
        loss = loss * weight
    if avg_factor is None:
        return {'none': loss, 'mean': loss.mean(), 'sum': loss.sum()}[reduction]
    if reduction == 'mean':
        return loss.sum() / avg_factor
    if reduction == 'none':
        return loss
    raise ValueError('avg_factor can not be used with reduction="sum"')


def sigmoid_focal_loss(pred, target, weight=None, gamma=2.0, alpha=0.25, reduction='mean', avg_factor=None):
    """pred (n, C) logits, target (n,) class index with C = background.  Per element
    ``-alpha (1 - p)^gamma log p`` for the target class, ``-(1 - alpha) p^gamma log(1 - p)`` otherwise
    (the formula of mmcv's sigmoid_focal_loss op that mmdet calls on the device)."""
    C = pred.size(1)
    t = F.one_hot(target, num_classes=C + 1)[:, :C].to(pred.dtype)
    p = pred.sigmoid()
    pt = (1 - p) * t + p * (1 - t)
    focal = (alpha * t + (1 - alpha) * (1 - t)) * pt.pow(gamma)
    loss = F.binary_cross_entropy_with_logits(pred, t, reduction='none') * focal
    if weight is not None and weight.shape != loss.shape:
        weight = weight.view(-1, 1) if weight.size(0) == loss.size(0) else weight.view(loss.size(0), -1)
    return weight_reduce_loss(loss, weight, reduction, avg_factor)


def cross_entropy(pred, target, weight=None, class_weight=None, ignore_index=-100, reduction='mean', avg_factor=None):
    """pred (n, C) logits, target (n,) class index.  Per sample ``-class_weight[target] log softmax(pred)[target]``, 0
    where the target is ``ignore_index``.  On the device one pass over the logits and one in the backward pass
    (ops/log_probs.py; a target that is no class makes its loss NaN there); op by op on the host."""
    if pred.dim() != 2:
        raise ValueError(f'pred must be (n, C), got {tuple(pred.shape)}')
    if class_weight is not None and class_weight.numel() != pred.size(1):
        raise ValueError(f'class_weight has {class_weight.numel()} entries for {pred.size(1)} classes')
    if pred.is_cuda:
        loss = -label_log_probs(pred, target, entropy=False, ignore_index=ignore_index).log_prob
    else:
        loss = F.cross_entropy(pred if pred.dtype == torch.float64 else pred.float(), target, reduction='none',
                               ignore_index=ignore_index)
    if class_weight is not None:
        # (an ignored target's loss is 0 whatever it is multiplied with, that of one that is no class NaN)
        loss = loss * class_weight[target.clamp(0, pred.size(1) - 1)]
    return weight_reduce_loss(loss, weight, reduction, avg_factor)


class CrossEntropyLoss(nn.Module):
    """mmdet CrossEntropyLoss, its softmax form (``use_sigmoid=False, use_mask=False``).  A head with this loss has one
    class channel more, the background's, at the end."""

    def __init__(self, use_sigmoid=False, use_mask=False, reduction='mean', class_weight=None, ignore_index=None,
                 loss_weight=1.0):
        super().__init__()
        if use_sigmoid or use_mask:
            raise NotImplementedError('CrossEntropyLoss: only the softmax form (use_sigmoid=False, use_mask=False)')
        self.use_sigmoid = False
        self.reduction, self.loss_weight = reduction, loss_weight
        self.ignore_index = -100 if ignore_index is None else ignore_index
        if class_weight is not None:  # (moves with the module: no copy from the host in the step)
            class_weight = torch.tensor([float(w) for w in class_weight])
        self.register_buffer('class_weight', class_weight, persistent=False)

    def forward(self, pred, target, weight=None, avg_factor=None, reduction_override=None):
        return self.loss_weight * cross_entropy(pred, target, weight, self.class_weight, self.ignore_index,
                                                reduction_override or self.reduction, avg_factor)


class FocalLoss(nn.Module):
    def __init__(self, use_sigmoid=True, gamma=2.0, alpha=0.25, reduction='mean', loss_weight=1.0):
        super().__init__()
        assert use_sigmoid, 'only the sigmoid focal loss is used by the rotated heads'
        self.use_sigmoid, self.gamma, self.alpha = use_sigmoid, gamma, alpha
        self.reduction, self.loss_weight = reduction, loss_weight

    def forward(self, pred, target, weight=None, avg_factor=None, reduction_override=None):
        reduction = reduction_override or self.reduction
        return self.loss_weight * sigmoid_focal_loss(pred, target, weight, self.gamma, self.alpha, reduction,
                                                     avg_factor)


def smooth_l1_loss(pred, target, beta=1.0):
    assert beta > 0
    if target.numel() == 0:
        return pred.sum() * 0
    diff = (pred - target).abs()
    return torch.where(diff < beta, 0.5 * diff * diff / beta, diff - 0.5 * beta)


class SmoothL1Loss(nn.Module):
    def __init__(self, beta=1.0, reduction='mean', loss_weight=1.0):
        super().__init__()
        self.beta, self.reduction, self.loss_weight = beta, reduction, loss_weight

    def forward(self, pred, target, weight=None, avg_factor=None, reduction_override=None):
        reduction = reduction_override or self.reduction
        loss = smooth_l1_loss(pred, target, self.beta)
        return self.loss_weight * weight_reduce_loss(loss, weight, reduction, avg_factor)


class L1Loss(nn.Module):
    """mmdet L1Loss (configs/rretinanet/rretinanet_obb_r50_fpn_1x_dota_v1.py:49)."""

    def __init__(self, reduction='mean', loss_weight=1.0):
        super().__init__()
        self.reduction, self.loss_weight = reduction, loss_weight

    def forward(self, pred, target, weight=None, avg_factor=None, reduction_override=None):
        reduction = reduction_override or self.reduction
        return self.loss_weight * weight_reduce_loss((pred - target).abs(), weight, reduction, avg_factor)


from ..registry import LOSSES, build_from  # noqa: E402

for _c in (FocalLoss, CrossEntropyLoss, SmoothL1Loss, L1Loss):
    if _c.__name__ not in LOSSES:
        LOSSES.register_module(module=_c)


def build_loss(cfg):
    return build_from(LOSSES, cfg)

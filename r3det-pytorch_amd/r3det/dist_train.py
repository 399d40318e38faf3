"""Data-parallel training plumbing for BASELINE configs[4] (training): one process per
GPU, each rank assigns / refines its own images (the custom ops never communicate), and the ONLY
exchange is DistributedDataParallel's bucketed gradient all-reduce (backend 'nccl' = RCCL over xGMI
on ROCm, 'gloo' on CPU in the tests), overlapped with backward.

The reference reaches the same arrangement through mmcv's MMDistributedDataParallel around
``model.train_step`` (tools/train.py -> mmdet.apis.train_detector; third-party).  Loss normalisation is
per rank, as in the reference: every head divides by ITS OWN rank's positive count
(rotate_anchor_head.py:470-471; mmdet 2.19's anchor heads do not all-reduce ``num_total_samples``), so the
averaged gradient is the mean of the per-rank gradients, not the gradient of one big batch.
"""
import torch
import torch.distributed as dist
from torch.nn.parallel import DistributedDataParallel

from .models.detectors import parse_losses
from .ops.orthogonalize import COEFFICIENTS, DTYPES, STEPS, alike, orthogonal_update_

# xGMI is point to point (7 links x ~153 GB/s per GPU): a ring all-reduce is bound per link, and the
# 168 MB of fp32 gradients of R3Det-R50 go out in few, large buckets -- 4 x ~48 MB instead of torch's
# 25 MB default -- so that each collective is well past RCCL's latency-bound regime while three of the
# four still overlap with the backbone's backward.
BUCKET_CAP_MB = 48


def wrap_ddp(model, device=None, bucket_cap_mb=BUCKET_CAP_MB):
    """DistributedDataParallel around a detector whose ``forward(img, return_loss=True, ...)`` returns the
    loss dict.  Frozen parameters (stem + layer1) take no part; every trainable parameter receives a
    gradient each step (both heads and the FR module are always used), so unused-parameter detection stays
    off.  Single-process (no process group): the model itself."""
    from .dist_infer import force_group
    if not dist.is_initialized() or (dist.get_world_size() == 1 and not force_group()):
        return model
    ids = [device.index] if device is not None and device.type == 'cuda' else None
    return DistributedDataParallel(model, device_ids=ids, bucket_cap_mb=bucket_cap_mb, gradient_as_bucket_view=True,
                                   broadcast_buffers=False)  # BatchNorm runs in eval mode (norm_eval=True)


def train_step(model, optimizer, img, gt_bboxes, gt_labels, img_metas=None):
    """One optimisation step: losses -> total -> backward (gradient all-reduce inside) -> optimizer.
    Returns (loss, log_vars) as device tensors; nothing here synchronises with the host."""
    optimizer.zero_grad(set_to_none=True)
    losses = model(img, img_metas, return_loss=True, gt_bboxes=gt_bboxes, gt_labels=gt_labels)
    loss, log_vars = parse_losses(losses)
    loss.backward()
    optimizer.step()
    return loss.detach(), log_vars


class Muon(torch.optim.Optimizer):
    """Orthogonalised momentum for weights of two and more dimensions (ops/orthogonalize.py: all of a group's weights in
    one chain of launches), SGD with momentum for the groups with ``orthogonal=False`` (biases, norms).

        orthogonal:  M = momentum M + G;  U = G + momentum M (nesterov) or M
                     W = (1 - lr weight_decay) W - lr s orthogonalize(U)     (s: ``scale``)
        otherwise:   M = momentum M + G + weight_decay W;  U = G + weight_decay W + momentum M (nesterov) or M
                     W = W - lr U

    The momentum is fp32 whatever the weights' type and is laid out as its weight is.  The same gradients give the same
    bits on cards alike, so replicas that exchange gradients stay equal.  ``lr`` and the others are read from the group at every step
    (schedulers work; a captured step keeps them).  Device tensors only."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, orthogonal=True, scale='rms',
                 steps=STEPS, coefficients=COEFFICIENTS, eps=1e-7):
        if not (lr >= 0 and momentum >= 0 and weight_decay >= 0):
            raise ValueError('lr, momentum and weight_decay must not be negative')
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      orthogonal=orthogonal, scale=scale, steps=steps, coefficients=tuple(coefficients),
                                      eps=eps))

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        for p in group['params']:
            if p.dtype not in DTYPES or (group['orthogonal'] and p.dim() < 2):
                self.param_groups.pop()
                raise ValueError('Muon: weights are fp32, fp16 or bf16, and of two and more dimensions in an orthogonal '
                                 'group; put the others into a group with orthogonal=False')

    def _momentum(self, p, orthogonal):
        state = self.state[p]
        m = state.get('momentum_buffer')
        # (laid out as the weight is where both are one matrix; the others' may be any way)
        if m is not None and m.device == p.device and (not orthogonal or alike(m, p)):
            return m
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError('Muon: take one step before the capture (every replay would begin with the momentum as it is now)')
        m = torch.zeros_like(p, dtype=torch.float32) if m is None else torch.empty_like(p, dtype=torch.float32).copy_(m)
        state['momentum_buffer'] = m
        return m

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for g in self.param_groups:
            kinds = {}  # (one call takes weights of one type on one device)
            for p in g['params']:
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise RuntimeError('Muon: sparse gradients are not taken')
                    kinds.setdefault((p.device, p.dtype), []).append(p)
            for ps in kinds.values():
                grads, buffers = [p.grad for p in ps], [self._momentum(p, g['orthogonal']) for p in ps]
                if g['orthogonal']:
                    orthogonal_update_(ps, grads, buffers, g['lr'], g['momentum'], g['nesterov'], g['weight_decay'], g['steps'],
                                       g['coefficients'], g['eps'], g['scale'])
                else:
                    self._sgd(ps, grads, buffers, g)
        return loss

    @staticmethod
    def _sgd(ps, grads, buffers, g):
        wide = [p.float() for p in ps]  # (16-bit weights: every step rounds once; fp32 ones are themselves)
        grads = [d.float() for d in grads]
        if g['weight_decay']:
            grads = torch._foreach_add(grads, wide, alpha=g['weight_decay'])
        torch._foreach_mul_(buffers, g['momentum'])
        torch._foreach_add_(buffers, grads)
        update = torch._foreach_add(grads, buffers, alpha=g['momentum']) if g['nesterov'] else buffers
        torch._foreach_add_(wide, update, alpha=-g['lr'])
        if wide[0] is not ps[0]:
            torch._foreach_copy_(ps, wide)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # (the base class casts the state to the weights' type: the momentum stays 32 bits wide)
        saved = [i for group in state_dict['param_groups'] for i in group['params']]
        for i, p in zip(saved, (p for group in self.param_groups for p in group['params'])):
            m = state_dict['state'].get(i, {}).get('momentum_buffer')
            if m is not None:
                self.state[p]['momentum_buffer'] = torch.empty_like(p, dtype=torch.float32).copy_(m)


MUON_NUMBERS = {'lr', 'momentum', 'nesterov', 'weight_decay', 'scale', 'steps', 'coefficients', 'eps'}


def build_optimizer(model, lr=0.0025, momentum=0.9, weight_decay=0.0001, type='SGD', **matrices):
    """configs/_base_/schedules/schedule_1x.py: SGD(lr=0.0025, momentum=0.9, weight_decay=0.0001)
    over the trainable parameters (grad clipping max_norm=35 is applied by the caller if wanted).
    ``type='Muon'``: the weights of two and more dimensions take orthogonalised updates with ``matrices`` (``lr``,
    ``momentum``, ``scale``, ... of ``Muon``, spelt ``matrix_lr`` and so on; its defaults and the same weight decay
    otherwise), the rest the numbers above."""
    params = [p for p in model.parameters() if p.requires_grad]
    if type == 'SGD' and not matrices:
        return torch.optim.SGD(params, lr=lr, momentum=momentum, weight_decay=weight_decay)
    own = {k[len('matrix_'):]: v for k, v in matrices.items() if k.startswith('matrix_')}
    if type != 'Muon' or len(own) != len(matrices) or not set(own) <= MUON_NUMBERS:
        raise ValueError(f"type must be 'SGD', or 'Muon' with matrix_ numbers of it, got {type!r} with {sorted(matrices)}")
    groups = [dict(dict(weight_decay=weight_decay), params=[p for p in params if p.dim() >= 2], **own),
              dict(params=[p for p in params if p.dim() < 2], orthogonal=False, lr=lr, momentum=momentum, nesterov=False,
                   weight_decay=weight_decay)]
    return Muon([g for g in groups if g['params']])

"""Softmax classification heads, their loss and the choice of optimiser: shapes, formulas and refusals on the host."""
import copy
import json
import math
import pathlib

import pytest
import torch

CFG = json.loads((pathlib.Path(__file__).parent / "golden" / "configs.json").read_text())
R3 = "configs/r3det/r3det_r50_fpn_1x_dota_v1.py"
SOFTMAX = dict(type='CrossEntropyLoss', use_sigmoid=False, loss_weight=1.0)


def head(num_classes=5, cls=None, **kw):
    from r3det.models import RRetinaHead
    torch.manual_seed(4)
    return RRetinaHead(num_classes=num_classes, in_channels=8, feat_channels=8, stacked_convs=1, strides=(8, 16),
                       loss_cls=SOFTMAX, **kw)


def outputs(h, seed=0, n=2):
    g = torch.Generator().manual_seed(seed)
    sizes = [(4, 6), (2, 3)]
    A, C = h.num_anchors, h.cls_out_channels
    return ([torch.randn(n, A * C, *s, generator=g) * 2 for s in sizes], [torch.randn(n, A * 5, *s, generator=g) * 0.2 for s in sizes])


def test_config_with_a_softmax_loss_builds():
    from r3det.models import build_detector
    c = copy.deepcopy(CFG[R3])
    c['bbox_head']['loss_cls'] = dict(SOFTMAX)
    for r in c['refine_heads']:
        r['loss_cls'] = dict(SOFTMAX)
    m = build_detector(c)
    for h in [m.bbox_head] + list(m.refine_head):
        assert h.cls_out_channels == h.num_classes + 1 and not h.use_sigmoid_cls
        assert h.retina_cls.out_channels == h.num_anchors * (h.num_classes + 1)
    # the sigmoid heads are what they were
    m = build_detector(copy.deepcopy(CFG[R3]))
    assert m.bbox_head.cls_out_channels == m.bbox_head.num_classes and m.bbox_head.use_sigmoid_cls


def test_a_sampler_is_refused():
    from r3det.models.heads import S0_TRAIN_CFG
    with pytest.raises(NotImplementedError, match='sampler'):
        head(train_cfg=dict(S0_TRAIN_CFG, sampler=dict(type='RandomSampler')))


def test_a_sigmoid_loss_in_a_softmax_head_is_refused():
    from r3det.models import RRetinaHead
    with pytest.raises(NotImplementedError, match='use_sigmoid'):
        RRetinaHead(loss_cls=dict(type='FocalLoss'))
    with pytest.raises(NotImplementedError, match='softmax form'):
        RRetinaHead(loss_cls=dict(type='CrossEntropyLoss', use_sigmoid=True))


def test_calibration_refuses_softmax():
    from r3det.models import RRetinaNet
    from r3det.models.detectors import calibrate_score_bias
    m = RRetinaNet()
    m.bbox_head = head()
    with pytest.raises(NotImplementedError, match='softmax'):
        calibrate_score_bias(m, torch.zeros(1, 3, 32, 32))


@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
def test_cross_entropy_formula(reduction):
    from r3det.models.losses import CrossEntropyLoss
    g = torch.Generator().manual_seed(1)
    x = torch.randn(7, 4, generator=g, dtype=torch.float64).requires_grad_(True)
    y = torch.tensor([0, 3, 1, -100, 2, 3, 0])
    w, cw = torch.rand(7, generator=g, dtype=torch.float64), [0.5, 1.0, 2.0, 0.25]
    loss = CrossEntropyLoss(reduction=reduction, class_weight=cw, loss_weight=1.5)
    got = loss(x, y, w)
    lp = x.log_softmax(-1)
    each = torch.stack([-lp[i, y[i]] * cw[y[i]] * w[i] if y[i] >= 0 else lp[0, 0] * 0 for i in range(7)])
    want = 1.5 * dict(none=each, sum=each.sum(), mean=each.mean())[reduction]
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda t: loss(t, y, w), (x,))
    if reduction == 'mean':
        assert torch.allclose(loss(x, y, w, avg_factor=3.0), 1.5 * each.sum() / 3)
        assert torch.allclose(loss(x, y, w, reduction_override='sum'), 1.5 * each.sum())
    if reduction == 'sum':
        with pytest.raises(ValueError, match='avg_factor'):
            loss(x, y, w, avg_factor=3.0)


def test_cross_entropy_refusals_and_defaults():
    from r3det.models.losses import LOSSES, CrossEntropyLoss, build_loss
    assert 'CrossEntropyLoss' in LOSSES
    for kw in (dict(use_sigmoid=True), dict(use_mask=True)):
        with pytest.raises(NotImplementedError):
            CrossEntropyLoss(**kw)
    loss = build_loss(dict(SOFTMAX, ignore_index=2))
    assert float(loss(torch.zeros(1, 3), torch.tensor([2]))) == 0 and not loss.state_dict()
    assert not CrossEntropyLoss(class_weight=[1.0, 2.0]).state_dict()
    with pytest.raises(ValueError, match='class_weight'):
        CrossEntropyLoss(class_weight=[1.0, 2.0])(torch.zeros(1, 3), torch.tensor([0]))
    with pytest.raises(ValueError, match='pred'):
        loss(torch.zeros(1, 3, 2), torch.zeros(1, 2, dtype=torch.int64))
    assert abs(float(loss(torch.zeros(2, 4).half(), torch.tensor([0, 1]))) - math.log(4)) < 1e-6


def test_loss_is_averaged_over_all_samples():
    from r3det import synthetic as syn
    from cpu_standins import cpu_kernels
    h = head()
    cls, reg = outputs(h)
    gtb = [syn.dota_like_rboxes(3, 5 + i, size=48, wmax=30.0) for i in range(2)]
    gtl = [torch.tensor([0, 4, 2])] * 2
    metas = [dict(img_shape=(32, 48, 3), pad_shape=(32, 48, 3))] * 2
    with cpu_kernels():
        got = h.loss(cls, reg, gtb, gtl, metas)
        al, fl = h.get_anchors([c.shape[-2:] for c in cls], metas, 'cpu')
        labels, lw, bt, bw, pos = h.get_targets(al, fl, gtb, metas, gtl)
    sampled = torch.cat(lw, 1) > 0
    neg = (sampled & (torch.cat(labels, 1) == h.num_classes)).sum(1).clamp(min=1).sum()
    assert int(neg) > int(pos)
    for l in range(2):
        lp = cls[l].permute(0, 2, 3, 1).reshape(-1, 6).log_softmax(-1)
        y = labels[l].reshape(-1)
        want = (-lp[torch.arange(len(y)), y] * lw[l].reshape(-1)).sum() / (pos + neg)
        assert torch.allclose(got['loss_cls'][l], want, rtol=1e-5)


@pytest.mark.parametrize('nms_pre', [-1, 20])
def test_decode_keeps_the_best_foreground_rows(nms_pre):
    h = head()
    cls, reg = outputs(h)
    boxes, scores = h.decode_bboxes(cls, reg, (32, 48), dict(nms_pre=nms_pre))
    off = 0
    for c, a in zip(cls, h.anchors([t.shape[-2:] for t in cls], 'cpu')):
        p = c.permute(0, 2, 3, 1).reshape(2, -1, 6).softmax(-1)
        r = p.size(1) if nms_pre < 0 else min(nms_pre, p.size(1))
        if r < p.size(1):
            p = torch.stack([q[q[:, :5].max(1)[0].argsort(descending=True)[:r]] for q in p])
        assert torch.allclose(scores[:, off:off + r], p, rtol=1e-6, atol=1e-7)
        off += r
    assert scores.shape == (2, off, 6) and boxes.shape == (2, off, 5)
    assert torch.allclose(scores.sum(-1), torch.ones(2, off))


def test_filter_takes_the_anchor_whose_class_is_most_probable():
    h = head()
    cls, reg = outputs(h)
    cls[0][:, 5::6] += 3.0                # the background's logits decide nothing but through the softmax
    got = h.filter_bboxes(cls, reg)
    A = h.num_anchors
    for l, anchors in enumerate(h.anchors([t.shape[-2:] for t in cls], 'cpu')):
        p = cls[l].permute(0, 2, 3, 1).reshape(2, -1, A, 6).softmax(-1)
        best = p[..., :5].max(-1)[0].argmax(-1)
        from r3det.models.coder import delta2bbox_v1
        d = reg[l].permute(0, 2, 3, 1).reshape(2, -1, A, 5)
        for i in range(2):
            at = torch.arange(best.size(1))
            want = delta2bbox_v1(anchors.view(-1, A, 5)[at, best[i]][None], d[i][at, best[i]][None])[0]
            assert torch.equal(got[i][l], want)


def test_optimiser_choice():
    from r3det import dist_train as dt
    h = head()
    assert type(dt.build_optimizer(h)) is torch.optim.SGD
    opt = dt.build_optimizer(h, lr=0.01, type='Muon', matrix_lr=0.03, matrix_scale='spectral')
    mats, rest = opt.param_groups
    assert all(p.dim() >= 2 for p in mats['params']) and all(p.dim() < 2 for p in rest['params'])
    assert len(mats['params']) + len(rest['params']) == len(list(h.parameters()))
    assert (mats['lr'], mats['scale'], mats['momentum'], mats['weight_decay'], mats['orthogonal']) == (0.03, 'spectral', 0.95,
                                                                                                    0.0001, True)
    assert (rest['lr'], rest['momentum'], rest['nesterov'], rest['orthogonal']) == (0.01, 0.9, False, False)
    for kw in (dict(type='Adam'), dict(type='Muon', lr2=1), dict(type='Muon', matrix_beta=1), dict(matrix_lr=0.1)):
        with pytest.raises(ValueError, match='SGD'):
            dt.build_optimizer(h, **kw)
    only = torch.nn.Linear(3, 2, bias=False)
    assert len(dt.build_optimizer(only, type='Muon').param_groups) == 1


def test_muon_refusals():
    from r3det.dist_train import Muon
    w, b = torch.nn.Parameter(torch.ones(3, 4)), torch.nn.Parameter(torch.ones(3))
    for bad in (dict(lr=-1.0), dict(momentum=-1.0), dict(weight_decay=float('nan'))):
        with pytest.raises(ValueError, match='negative'):
            Muon([w], **bad)
    with pytest.raises(ValueError, match='orthogonal=False'):
        Muon([w, b])
    with pytest.raises(ValueError, match='bf16'):
        Muon([torch.nn.Parameter(torch.ones(3, 4, dtype=torch.float64))])
    opt = Muon([w])
    opt.step()                                        # (no gradients: nothing to do)
    with pytest.raises(ValueError, match='orthogonal=False'):
        opt.add_param_group(dict(params=[b]))
    assert len(opt.param_groups) == 1
    w.grad = torch.ones(3, 4)
    with pytest.raises(RuntimeError, match='CUDA tensor'):
        opt.step()
    w.grad = torch.ones(3, 4).to_sparse()
    with pytest.raises(RuntimeError, match='sparse'):
        opt.step()


def test_muon_sgd_groups_and_state_on_the_host():
    """The groups without orthogonal updates are SGD's; the momentum stays 32 bits wide through a saved state."""
    from r3det.dist_train import Muon
    g = torch.Generator().manual_seed(2)
    mine = [torch.nn.Parameter(torch.randn(5, generator=g)), torch.nn.Parameter(torch.randn(2, 3, generator=g))]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    for nesterov in (False, True):
        a = Muon([dict(params=mine, orthogonal=False, nesterov=nesterov)], lr=0.1, momentum=0.9, weight_decay=0.01)
        b = torch.optim.SGD(theirs, lr=0.1, momentum=0.9, weight_decay=0.01, nesterov=nesterov)
        for _ in range(3):
            for p, q in zip(mine, theirs):
                p.grad = torch.randn(p.shape, generator=g)
                q.grad = p.grad.clone()
            a.step()
            b.step()
            # about ten roundings a step, each of at most 2^-24 of values below 8
            for p, q in zip(mine, theirs):
                assert torch.allclose(p, q, rtol=0, atol=3 * 10 * 8 * 2 ** -24)
                q.data.copy_(p)
    p = torch.nn.Parameter(torch.randn(6, generator=g).bfloat16())
    a = Muon([dict(params=[p], orthogonal=False)])
    p.grad = torch.randn(6, generator=g).bfloat16()
    a.step()
    a.step()
    m = a.state[p]['momentum_buffer']
    assert m.dtype == torch.float32 and not torch.equal(m, m.bfloat16().float())
    c = Muon([dict(params=[p], orthogonal=False)])
    c.load_state_dict(a.state_dict())
    n = c.state[p]['momentum_buffer']
    assert n.dtype == torch.float32 and torch.equal(m, n) and n.data_ptr() != m.data_ptr()

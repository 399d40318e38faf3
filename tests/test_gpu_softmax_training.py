"""GPU: the softmax classification loss and heads against formulas in 64 bits, the optimiser with orthogonalised updates,
and both together in training steps of a detector."""
import copy
import json
import pathlib

import pytest
import torch

from test_gpu_train import batch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = 'cuda:0'
CFG = json.loads((pathlib.Path(__file__).parent / "golden" / "configs.json").read_text())
SOFTMAX = dict(type='CrossEntropyLoss', use_sigmoid=False, loss_weight=1.0)


def detector(name="configs/r3det/r3det_r50_fpn_1x_dota_v1.py", seed=7):
    from r3det.models import build_detector
    c = copy.deepcopy(CFG[name])
    c['bbox_head']['loss_cls'] = dict(SOFTMAX)
    for r in c.get('refine_heads', []):
        r['loss_cls'] = dict(SOFTMAX)
    torch.manual_seed(seed)
    return build_detector(c)


def head(num_classes=15):
    from r3det.models import RRetinaHead
    torch.manual_seed(4)
    return RRetinaHead(num_classes=num_classes, in_channels=8, feat_channels=8, stacked_convs=1, strides=(8, 16),
                       loss_cls=SOFTMAX).to(DEV)


# ------------------------------------------------------------------------------------------------ the loss
@pytest.mark.parametrize('n,classes', [(1, 2), (5, 16), (1000, 16), (37, 21), (300, 81), (3, 5000)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
def test_cross_entropy_and_its_gradient(n, classes, dtype):
    from r3det.models.losses import CrossEntropyLoss
    g = torch.Generator().manual_seed(n + classes)
    x = (torch.randn(n, classes, generator=g) * 3).to(dtype)
    y = torch.randint(0, classes, (n,), generator=g)
    y[::7] = -100
    w, cw = torch.rand(n, generator=g), (torch.rand(classes, generator=g) + 0.5).tolist()
    loss = CrossEntropyLoss(class_weight=cw, reduction='none').to(DEV)
    leaf = x.to(DEV).requires_grad_(True)
    each = loss(leaf, y.to(DEV), w.to(DEV))
    total = loss(leaf, y.to(DEV), w.to(DEV), avg_factor=torch.tensor(float(n), device=DEV), reduction_override='mean')
    dx, = torch.autograd.grad(total, leaf)
    lp = x.double().log_softmax(-1)
    at = y.clamp(min=0)
    f = torch.where(y >= 0, torch.tensor(cw).double()[at] * w.double(), 0.0)
    want = -lp.gather(1, at[:, None])[:, 0] * f
    # log p is off by (classes / 64 + 40 + |log S| + 2 |x - m| + |log p|) u (the sum's, the differences' and its own
    # roundings), with |x - m| <= 30 and log S <= 9; the two weights round the loss four times more
    off = (classes / 64 + 40 + 9 + 60 + lp.abs().max(1).values) * U
    assert each.dtype == torch.float32
    assert ((each.detach().cpu().double() - want).abs() <= off * f + 4 * U * want.abs()).all()
    # the mean: one rounding for each addition and for the quotient
    assert abs(float(total.detach()) - float(want.sum() / n)) <= float((off * f).sum() / n + (n + 6) * U * want.abs().sum() / n)
    p = lp.exp()
    p[torch.arange(n), at] -= 1
    ref = p * f[:, None] / n
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0          # (half of fp16's smallest step)
    # p is off by p times what log p is off by, the two factors by five roundings, the type by half a step
    assert ((dx.cpu().double() - ref).abs() <= (off + 8 * U)[:, None] * f[:, None] / n + half * ref.abs() * 1.01 + tiny).all()
    assert not dx[(y < 0).to(DEV)].any()


def test_gradient_against_differences():
    """The mean loss along a direction v: differences with h = 1/8 are off by at most h^2 / 6 times the third derivative, a
    row's third central moment of v, which R^3 / (6 sqrt 3) bounds for a spread of R; the loss itself by 150 u (see above)."""
    from r3det.models.losses import CrossEntropyLoss
    g = torch.Generator().manual_seed(3)
    x, v = torch.randn(64, 16, generator=g).to(DEV), torch.rand(64, 16, generator=g).to(DEV)
    y = torch.randint(0, 16, (64,), generator=g).to(DEV)
    loss, h = CrossEntropyLoss(), 0.125
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(loss(leaf, y), leaf)
    got = float((dx.double() * v.double()).sum())
    diff = (float(loss(x + h * v, y)) - float(loss(x - h * v, y))) / (2 * h)
    assert abs(got - diff) <= h * h / 6 / (6 * 3 ** 0.5) + 2 * 150 * U * 4 / (2 * h)


def test_labels_that_are_no_class_make_their_loss_nan():
    from r3det.models.losses import CrossEntropyLoss
    y = torch.tensor([0, 4, -1, 2], device=DEV)
    each = CrossEntropyLoss(reduction='none', class_weight=[1.0] * 4).to(DEV)(torch.zeros(4, 4, device=DEV), y)
    assert torch.isnan(each).tolist() == [False, True, True, False]


# ------------------------------------------------------------------------------------------------ the heads
def spaced(h, n=2, seed=0):
    """Outputs whose rows' best foreground probabilities lie far apart (0.01 in the logit), in a random order."""
    g = torch.Generator().manual_seed(seed)
    A, C = h.num_anchors, h.cls_out_channels
    cls, reg = [], []
    for H, W in ((8, 12), (4, 6)):
        L = H * W * A
        x = torch.full((n, L, C), -6.0)
        x[..., C - 1] = 2.0
        order = torch.stack([torch.randperm(L, generator=g) for _ in range(n)]).float()
        which = torch.randint(0, C - 1, (n, L), generator=g)
        x.scatter_(2, which[..., None], (order * 0.01 - 0.005 * L)[..., None])
        cls.append(x.view(n, H, W, A * C).permute(0, 3, 1, 2).contiguous().to(DEV))
        reg.append((torch.randn(n, A * 5, H, W, generator=g) * 0.2).to(DEV))
    return cls, reg


@pytest.mark.parametrize('layout', [torch.contiguous_format, torch.channels_last])
@pytest.mark.parametrize('classes', [1, 15, 80, 200])
def test_heads_equal_their_host_form(classes, layout):
    h = head(classes)
    cls, reg = spaced(h)
    cls, reg = [c.contiguous(memory_format=layout) for c in cls], [r.contiguous(memory_format=layout) for r in reg]
    host = copy.deepcopy(h).cpu()
    host._anchor_cache = {}
    cc, cr = [c.cpu().double() for c in cls], [r.cpu() for r in reg]
    for nms_pre in (-1, 100):
        boxes, scores = h.decode_bboxes(cls, reg, (64, 96), dict(nms_pre=nms_pre))
        b, s = host.decode_bboxes(cc, cr, (64, 96), dict(nms_pre=nms_pre))
        # (the same rows in the same order, or these would be far off; a probability is off by the softmax's roundings, a
        # box by those of sizes up to 96 through a dozen operations)
        assert torch.allclose(scores.cpu(), s, rtol=1e-5, atol=1e-7)
        assert torch.allclose(boxes.cpu(), b, rtol=1e-5, atol=1e-3)
    got, want = h.filter_bboxes(cls, reg), host.filter_bboxes(cc, cr)
    for i in range(2):
        for x, y in zip(got[i], want[i]):
            assert torch.allclose(x.cpu(), y, rtol=1e-5, atol=1e-3)


def test_best_foreground_class():
    h = head(3)
    inf = float('inf')
    rows = torch.tensor([[[1.0, 2.0, 0.0, 5.0], [9.0, 2.0, 0.0, 5.0], [1.0, 1.0, 1.0, 1.0], [-inf, -inf, -inf, 0.0],
                          [-inf, 3.0, -inf, -inf]]], device=DEV)
    got = h._foreground(rows).cpu()
    want = torch.log_softmax(rows.cpu().double(), -1)[..., :3].max(-1)[0].float()
    assert torch.allclose(got, want, rtol=1e-5)


def test_detection_from_a_softmax_head_and_captured():
    h = head(15)
    cls, reg = spaced(h)
    static_c, static_r = [c.clone() for c in cls], [r.clone() for r in reg]
    cfg = dict(nms_pre=100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h.decode_bboxes(static_c, static_r, (64, 96), cfg)
        h.filter_bboxes(static_c, static_r)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        boxes, scores = h.decode_bboxes(static_c, static_r, (64, 96), cfg)
        first = h.filter_bboxes(static_c, static_r)
    for seed in (1, 2, 1, 3, 2):
        cls, reg = spaced(h, seed=seed)
        for a, b in zip(static_c + static_r, cls + reg):
            a.copy_(b)
        graph.replay()
        b, s = h.decode_bboxes(cls, reg, (64, 96), cfg)
        f = h.filter_bboxes(cls, reg)
        torch.cuda.synchronize()
        assert torch.equal(boxes, b) and torch.equal(scores, s)
        assert all(torch.equal(x, y) for p, q in zip(first, f) for x, y in zip(p, q))
    dets = h.get_bboxes(cls, reg, (64, 96))
    assert len(dets) == 2 and all(d.size(1) == 6 and bool(((lab >= 0) & (lab < 15)).all()) and len(d) for d, lab in dets)


# ------------------------------------------------------------------------------------------------ the optimiser
def weights(dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    ws = [torch.randn(s, generator=g).to(DEV, dtype) for s in ((16, 8, 3, 3), (12, 40), (5,), (64, 3, 7, 7), (1, 9))]
    ws[3] = ws[3].contiguous(memory_format=torch.channels_last)
    return [torch.nn.Parameter(w) for w in ws]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_muon_is_the_update_of_its_weights(dtype):
    from r3det.dist_train import Muon
    from r3det.ops.orthogonalize import orthogonal_update_
    ps = weights(dtype)
    mats = [0, 1, 3, 4]
    opt = Muon([dict(params=[ps[i] for i in mats], lr=0.05, weight_decay=0.1),
                dict(params=[ps[2]], orthogonal=False, lr=0.01)])
    ws, ms = [p.detach().clone() for p in ps], [torch.zeros_like(p, dtype=torch.float32) for p in ps]
    for step in range(3):
        for p, q in zip(ps, weights(dtype, step + 1)):
            p.grad = q.detach()
        if step == 2:
            opt.param_groups[0]['lr'] = 0.02
        opt.step()
        gs = [p.grad for p in ps]
        orthogonal_update_([ws[i] for i in mats], [gs[i] for i in mats], [ms[i] for i in mats],
                           lr=0.02 if step == 2 else 0.05, weight_decay=0.1)
        for i in mats:
            assert torch.equal(ps[i], ws[i]) and torch.equal(opt.state[ps[i]]['momentum_buffer'], ms[i])
        assert opt.state[ps[2]]['momentum_buffer'].dtype == torch.float32 and not torch.equal(ps[2], ws[2])


def test_muon_goes_on_from_a_saved_state_and_another_layout():
    from r3det.dist_train import Muon
    a, b = weights(), weights()
    del a[2], b[2]
    oa, ob = Muon(a), Muon(b)
    for step in range(4):
        for p, q, r in zip(a, b, [w for i, w in enumerate(weights(seed=step + 1)) if i != 2]):
            p.grad = r.detach()
            q.grad = r.detach().clone()
        oa.step()
        ob.step()
        if step == 1:
            saved = copy.deepcopy(ob.state_dict())
            ob = Muon(b, lr=1.0)
            ob.load_state_dict(saved)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    # the weight is laid out anew: its momentum follows
    before = oa.state[a[0]]['momentum_buffer'].clone()
    a[0].data = a[0].data.contiguous(memory_format=torch.channels_last)
    a[0].grad = torch.zeros_like(a[0])
    oa.step()
    after = oa.state[a[0]]['momentum_buffer']
    assert after.stride() == a[0].stride() and torch.equal(after, 0.95 * before)


def test_a_first_step_inside_a_capture_is_refused():
    from r3det.dist_train import Muon
    w = torch.nn.Parameter(torch.randn(8, 8, device=DEV))
    w.grad = torch.randn(8, 8, device=DEV)
    opt = Muon([w])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='before the capture'):
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
    eager = torch.nn.Parameter(w.detach().clone())
    other = Muon([eager])
    other.load_state_dict(opt.state_dict())
    eager.grad = w.grad.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
        other.step()
        torch.cuda.synchronize()
        assert torch.equal(w, eager)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize('name', ["configs/r3det/r3det_r50_fpn_1x_dota_v1.py",
                                  "configs/rretinanet/rretinanet_obb_r50_fpn_1x_dota_v1.py"])
@pytest.mark.parametrize('channels_last', [False, True])
def test_training_steps_of_a_softmax_detector(name, channels_last):
    """Two steps: finite losses, every trainable weight moved by what the update of its gradient says."""
    from r3det import dist_train as dt
    from r3det.ops.orthogonalize import orthogonal_update_
    m = detector(name).train().to(DEV)
    if channels_last:
        m = m.to(memory_format=torch.channels_last)
    opt = dt.build_optimizer(m, type='Muon', matrix_lr=0.001)
    mats = opt.param_groups[0]['params']
    img, gtb, gtl = batch(2, 256, 20, 21, DEV)
    if channels_last:
        img = img.contiguous(memory_format=torch.channels_last)
    ws = [p.detach().clone() for p in mats]
    ms = [torch.zeros_like(p) for p in mats]
    for _ in range(2):
        loss, _ = dt.train_step(m, opt, img, gtb, gtl)
        assert bool(torch.isfinite(loss))
        grads = [p.grad for p in mats]
        assert all(bool(g.any()) for g in grads)
        orthogonal_update_(ws, grads, ms, lr=0.001, weight_decay=0.0001)
        for p, w in zip(mats, ws):
            assert torch.equal(p, w)


def test_gradient_of_the_class_biases_against_differences():
    """One bias of the class prediction: the loss of the other form, computed in 64 bits from the same logits and targets, at
    both sides (h = 1/8; the third derivative of a row's loss is at most 1 / (6 sqrt 3) for a shift of one class)."""
    m = detector("configs/rretinanet/rretinanet_obb_r50_fpn_1x_dota_v1.py").train().to(DEV)
    h, (img, gtb, gtl) = m.bbox_head, batch(2, 256, 20, 22, DEV)
    metas = [dict(img_shape=(256, 256, 3), pad_shape=(256, 256, 3)) for _ in range(2)]
    cls, reg = h(m.extract_feat(img))
    sum(h.loss(cls, reg, gtb, gtl, metas)['loss_cls']).backward()
    al, fl = h.get_anchors([c.shape[-2:] for c in cls], metas, torch.device(DEV))
    labels, lw, _, _, pos = h.get_targets(al, fl, gtb, metas, gtl)
    rows = torch.cat([h._rows(c.detach()) for c in cls], 1).cpu().double()
    y, w = torch.cat(labels, 1).cpu(), torch.cat(lw, 1).cpu().double()
    avg = float(pos) + float(((w > 0) & (y == h.num_classes)).sum(1).clamp(min=1).sum())
    A, C, step = h.num_anchors, h.cls_out_channels, 0.125
    for channel in (0, C - 1, (A - 1) * C + 3):
        a, c = divmod(channel, C)
        side = []
        for s in (step, -step):
            x = rows.clone()
            x[:, a::A, c] += s
            side.append(float(-(x.log_softmax(-1).gather(2, y[..., None])[..., 0] * w).sum() / avg))
        want = (side[0] - side[1]) / (2 * step)
        # (the differences' share, and n additions of gradients of at most 1 / avg by the convolution's backward pass)
        share = float(w[:, a::A].sum()) / avg
        assert abs(float(h.retina_cls.bias.grad[channel]) - want) <= step ** 2 / 6 / (6 * 3 ** 0.5) * share + 1e-5


def captured(opt):
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    return graph


def test_momentum_of_a_strided_weight_goes_on_through_replays():
    """A weight that no tensor is laid out like (every second element of another): its momentum stays where it is."""
    from r3det.dist_train import Muon
    g = torch.randn(12, device=DEV)
    pair = [torch.nn.Parameter(torch.arange(24.0, device=DEV)[::2]) for _ in range(2)]
    opts = [Muon([dict(params=[p], orthogonal=False)], lr=0.1) for p in pair]
    assert pair[0].stride() == (2,)
    for p, o in zip(pair, opts):
        p.grad = g.clone()
        o.step()
        at = o.state[p]['momentum_buffer']
        o.step()
        assert o.state[p]['momentum_buffer'] is at
    graph = captured(opts[0])
    for _ in range(4):
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        assert torch.equal(pair[0], pair[1])
        assert torch.equal(*(o.state[p]['momentum_buffer'] for p, o in zip(pair, opts)))


def test_a_layout_that_changed_before_a_capture_is_refused_inside_it():
    """The momentum would be copied out of its old place by every replay, and none would go on from the one before."""
    from r3det.dist_train import Muon
    w = torch.nn.Parameter(torch.randn(16, 8, 3, 3, device=DEV))
    opt = Muon([w])
    w.grad = torch.randn_like(w)
    opt.step()
    w.data = w.data.contiguous(memory_format=torch.channels_last)
    w.grad = torch.randn_like(w)
    before = w.detach().clone()
    with pytest.raises(RuntimeError, match='before the capture'):
        captured(opt)
    assert torch.equal(w, before)
    opt.step()
    other = torch.nn.Parameter(w.detach().clone())
    eager = Muon([other])
    eager.load_state_dict(opt.state_dict())
    other.grad = w.grad.clone()
    graph = captured(opt)
    for _ in range(3):
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(w, other)

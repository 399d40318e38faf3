"""r3det.ops.log_probs against the formulas in 64 bits, at the sizes, masks, layouts and labels where it can go wrong.

Tolerances, in units of u = 2^-24 (half a step of fp32, relative).  x - m, its product with log2 e and the exponential are
off by at most one unit each, so a term e^d of the sum is off by (|d| + 3) u relatively, and e^d |d| <= 1 / e bounds what
|d| does to the sum; a lane adds at most classes / 64 + 32 terms one after the other.  log S therefore is off by at most
(classes / 64 + 32 + 8) u absolutely, plus its own rounding |log S| u, and log p by |x - m| u and the last difference's
|log p| u more.  H has the same sum behind it twice.  A result of 16 bits adds half a step of its own."""
import math

import pytest
import torch

from r3det.ops.log_probs import label_log_probs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100


def reference(x, labels=None, k=0, ignore=None):
    """64-bit, on the CPU: log p of every class, entropy, order of the classes."""
    x = x.detach().cpu().double()
    classes = x.size(-1)
    empty = (x == -math.inf).all(-1)
    lp = torch.log_softmax(torch.where(empty[..., None], 0.0, x), -1)
    lp = torch.where(empty[..., None], -math.inf, lp)
    p = lp.exp()
    h = -torch.special.xlogy(p, p).sum(-1)
    out = dict(lp=lp, p=p, h=h, empty=empty)
    if labels is not None:
        y = labels.cpu()
        ignored = (y == ignore) if ignore is not None else torch.zeros_like(y, dtype=torch.bool)
        bad = ~ignored & ((y < 0) | (y >= classes))
        at = torch.where(ignored | bad, 0, y)
        picked = lp.gather(-1, at[..., None])[..., 0]
        out.update(ignored=ignored, bad=bad, at=at)
        out["log_prob"] = torch.where(bad, math.nan, torch.where(ignored, 0.0, picked))
    if k:
        order = x.sort(dim=-1, descending=True, stable=True).indices[..., :k]
        out.update(top_index=order, top_lp=lp.gather(-1, order))
    return out


def slack(ref, x):
    """(tolerance of log S, of log p) per row / per element."""
    x = x.detach().cpu().double()
    m = x.max(-1, keepdim=True).values
    d = torch.where(torch.isfinite(x - m), (x - m).abs(), 0.0)
    s = torch.where(ref["empty"][..., None], 0.0, (ref["lp"].max(-1, keepdim=True).values).abs())
    log_s = (x.size(-1) / 64 + 40 + s) * U
    lp = torch.where(torch.isfinite(ref["lp"]), ref["lp"].abs(), 0.0)
    return log_s[..., 0], log_s + (2 * d + lp) * U


def close(got, want, tol):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
    off = (got - want).abs()[fin]
    over = off > tol.expand(want.shape)[fin]
    assert not over.any(), (off[over].max().item(), tol.expand(want.shape)[fin][over].min().item())


def check(x, labels=None, k=0, ignore=None, grads=True):
    ref = reference(x, labels, k, ignore)
    ts, tl = slack(ref, x)
    got = label_log_probs(x, labels, top_k=k, ignore_index=ignore)
    close(got.entropy, ref["h"], 3 * ts + ref["h"] * 4 * U)
    if labels is not None:
        close(got.log_prob, ref["log_prob"], tl.gather(-1, ref["at"][..., None])[..., 0])
    else:
        assert got.log_prob is None
    if k:
        assert torch.equal(got.top_index.cpu(), ref["top_index"])
        close(got.top_log_prob, ref["top_lp"], tl.gather(-1, ref["top_index"]))
    else:
        assert got.top_index is None and got.top_log_prob is None
    if not grads:
        return got
    leaf = x.detach().as_strided(x.size(), x.stride(), x.storage_offset()).requires_grad_(True)
    got = label_log_probs(leaf, labels, top_k=k, ignore_index=ignore)
    g = torch.Generator().manual_seed(7)
    lead = x.shape[:-1]
    dl, dh = (torch.randn(lead, generator=g, dtype=torch.float64).float() for _ in range(2))
    dt = torch.randn(lead + (k,), generator=g, dtype=torch.float64).float()
    outs, ds = [got.entropy], [dh.to(DEV)]
    if labels is not None:
        outs.append(got.log_prob), ds.append(dl.to(DEV))
    if k:
        outs.append(got.top_log_prob), ds.append(dt.to(DEV))
    dx, = torch.autograd.grad(outs, [leaf], ds)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    hot = torch.zeros_like(ref["lp"])
    if labels is not None:
        use = torch.where(ref["ignored"], 0.0, torch.where(ref["bad"], math.nan, dl.double()))
        hot.scatter_add_(-1, ref["at"][..., None], torch.where(ref["bad"], 0.0, use)[..., None])
    else:
        use = torch.zeros(lead, dtype=torch.float64)
    mass = use.clone()
    size = use.abs()
    if k:
        hot.scatter_add_(-1, ref["top_index"], dt.double())
        mass += dt.double().sum(-1)
        size = size + dt.double().abs().sum(-1)
    lp0 = torch.where(ref["p"] > 0, torch.nan_to_num(ref["lp"], neginf=0.0), 0.0)
    factor = mass[..., None] + dh.double()[..., None] * (lp0 + ref["h"][..., None])
    want = hot - ref["p"] * factor
    want = torch.where(ref["empty"][..., None], 0.0, want)
    # p is off by tl relatively (and by the product with log2 e: |log p| u), its factor by the sums in it
    wide = size[..., None] + dh.double().abs()[..., None] * (lp0.abs() + ref["h"][..., None])
    tol = ref["p"] * (wide * (tl + (lp0.abs() + 8 + k) * U) + dh.double().abs()[..., None] * (tl + 3 * ts[..., None]))
    tol = tol + (hot.abs() + size[..., None] * (hot != 0)) * (2 + k) * U
    t = torch.finfo(x.dtype)
    tol = tol + (want.abs() + tol) * t.eps / 2 + t.smallest_normal * t.eps / 2 + 2.0 ** -126
    close(dx, want, tol)
    return got


def logits(rows, classes, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 131 + classes)
    x = scale * torch.randn(rows, classes, generator=g)
    y = torch.randint(0, classes, (rows,), generator=g)
    return x.to(TYPES[dtype]).to(DEV), y.to(DEV)


SIZES = [(1, 1), (3, 2), (257, 3), (5, 4), (1000, 16), (7, 17), (33, 31), (64, 64), (9, 65), (33, 100), (5, 128), (6, 129),
         (3, 1000), (5, 1031), (2, 4096), (3, 4097), (2, 8193), (300, 5000), (2, 50001)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,classes", SIZES)
def test_sizes(rows, classes, dtype):
    x, y = logits(rows, classes, dtype)
    check(x, y, k=min(classes, 5))
    check(x, y, ignore=int(y[0]))
    check(x, None, k=min(classes, 1), grads=rows < 100)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,classes,k", [(1, 140001, 20), (3, 131072, 64), (1, 1 << 20, 3), (40, 65536, 7)])
def test_few_long_rows_are_split(rows, classes, k, dtype):
    x, y = logits(rows, classes, dtype)
    check(x, y, k=k, grads=rows == 3)


@pytest.mark.parametrize("classes,k", [(20, 20), (64, 64), (100, 64), (1000, 64), (6000, 64), (5, 5)])
def test_many_alternatives_and_ties(classes, k):
    x, y = logits(11, classes, "fp32")
    check(x.round(), y, k=k)  # (whole numbers: ties everywhere)
    check(torch.zeros_like(x), y, k=k)
    check(-torch.zeros_like(x), y, k=k)


@pytest.mark.parametrize("classes", [2, 16, 17, 100, 1000, 5000, 70001])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_masks(classes, dtype):
    x, y = logits(12, classes, dtype)
    low = torch.finfo(x.dtype).min
    g = torch.Generator().manual_seed(3)
    x[torch.rand(12, classes, generator=g).to(DEV) < 0.5] = -math.inf
    x[2] = -math.inf                      # nothing left
    x[3] = -math.inf
    x[3, classes - 1] = 1.5               # one left
    x[4] = low                            # the type's lowest value everywhere: all alike
    x[5, : classes // 2] = low
    x[6] = low
    x[6, 0] = -math.inf
    x[7] = -math.inf
    x[7, 0] = low
    x[8] = torch.finfo(x.dtype).max if dtype != "fp16" else 60000.0
    check(x, y, k=min(classes, 4))


@pytest.mark.parametrize("classes", [3, 16, 33, 1000, 5000, 40000])
def test_nan_and_inf_stay_in_their_rows(classes):
    x, y = logits(6, classes, "fp32")
    x[1, classes // 2] = math.nan
    x[3, classes - 1] = math.inf
    x[4] = -math.inf
    x[4, 1] = math.nan
    leaf = x.clone().requires_grad_(True)
    got = label_log_probs(leaf, y, top_k=2)
    dx, = torch.autograd.grad((got.log_prob + got.entropy).sum(), leaf)
    clean = [0, 2, 5]
    want = reference(x[clean], y[clean])
    for r in (1, 3, 4):
        assert torch.isnan(got.log_prob[r]) and torch.isnan(got.entropy[r]) and torch.isnan(dx[r]).all()
        assert torch.isnan(got.top_log_prob[r]).all()
    assert ((got.top_index >= 0) & (got.top_index < classes)).all()
    close(got.log_prob[clean], want["log_prob"], slack(want, x[clean])[1].gather(-1, want["at"][:, None])[:, 0])
    assert torch.isfinite(dx[clean]).all()


@pytest.mark.parametrize("rows,classes", [(9, 4), (9, 5), (9, 15), (9, 32), (9, 33), (9, 64), (9, 65), (9, 128), (9, 129), (5, 1024),
                                          (5, 1025), (3, 2047), (300, 1500), (3, 4096), (2, 33000), (1, 66000)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_where_one_form_ends_and_the_next_begins(rows, classes, dtype):
    x, y = logits(rows, classes, dtype)
    check(x, y, k=min(classes, 9))


@pytest.mark.parametrize("rows,classes", [(5, 1000), (5, 70001), (300, 6000), (2, 300000)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_few_classes_left_for_the_best_ones(rows, classes, dtype):
    """The masked classes that fill up the list are the lowest; what is left lies in one lane's pack, or far apart."""
    x = torch.full((rows, classes), -math.inf, dtype=TYPES[dtype], device=DEV)
    x[0, classes - 3:] = torch.tensor([1.0, 3.0, 1.0], device=DEV).to(x.dtype)
    x[1, :3] = 2.0
    x[1, classes // 2] = 4.0
    if rows > 2:
        x[2, ::classes // 40] = 0.5
        x[3, 40:140] = torch.finfo(x.dtype).min
        x[4, 1::2] = -1.0
    for k in (1, 8, 64):
        check(x, k=k, grads=False)


@pytest.mark.parametrize("classes", [16, 100, 1000, 5000, 70001])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_nan_is_ranked_first_whatever_its_sign(classes, dtype):
    x, _ = logits(5, classes, dtype)
    x[0] = -torch.tensor(math.nan, dtype=x.dtype, device=DEV)
    x[1] = torch.tensor(math.nan, dtype=x.dtype, device=DEV)
    x[2, classes // 2] = -math.nan
    x[2, classes - 1] = math.inf
    x[3] = -math.inf
    x[3, 1::3] = math.nan
    x[4, classes - 2:] = -math.nan
    k = min(classes, 20)
    got = label_log_probs(x, top_k=k)
    want = x.cpu().float().sort(dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(got.top_index.cpu(), want)
    assert torch.isnan(got.top_log_prob).all()


def test_labels_ignored_and_out_of_range():
    for classes in (16, 300, 6000):
        x, y = logits(9, classes, "fp32")
        y[0], y[1], y[2], y[3], y[4] = IGNORE, classes, -1, 2 ** 40, -2 ** 60
        check(x, y, ignore=IGNORE)
        check(x, torch.full_like(y, IGNORE), ignore=IGNORE)
        got = label_log_probs(x, y)  # no index is ignored
        assert torch.isnan(got.log_prob[:5]).all() and torch.isfinite(got.log_prob[5:]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("classes", [1, 16, 21, 500, 4100])
def test_layouts(classes, dtype):
    t = TYPES[dtype]
    base = logits(40, classes + 9, dtype)[0]
    y = torch.arange(40, device=DEV) % classes
    check(base[:, 3:3 + classes], y)                                             # rows apart, not aligned
    check(base[:, :classes][::3], y[::3])
    check(logits(classes, 24, dtype)[0].t()[:24], y[:24], k=min(2, classes))     # columns contiguous
    check(base[:1, :classes].expand(8, classes), y[:8])                          # one row, eight times
    check(base[:, :classes].reshape(2, 5, 4, classes), y.reshape(2, 5, 4), k=1)
    check(base[0, :classes], y[0], k=1)                                          # one row without a leading dimension
    head = torch.randn(2, 3 * classes, 4, 5, device=DEV).to(t)                   # a head's output, as the losses take it
    check(head.permute(0, 2, 3, 1).reshape(-1, classes), torch.zeros(120, dtype=torch.int64, device=DEV))
    cl = head.contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    check(cl.view(2, 4, 5, 3, classes), torch.zeros(2, 4, 5, 3, dtype=torch.int64, device=DEV))


def test_no_rows():
    for shape in ((0, 7), (3, 0, 7)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        got = label_log_probs(x, torch.zeros(shape[:-1], dtype=torch.int64, device=DEV), top_k=2)
        assert got.log_prob.shape == shape[:-1] and got.top_index.shape == shape[:-1] + (2,)
        dx, = torch.autograd.grad(got.entropy.sum() + got.log_prob.sum(), x)
        assert dx.shape == shape


def test_offsets_beyond_32_bits():
    classes, stride = 4500, (1 << 30) + 24
    store = torch.empty(2 * stride + classes, dtype=torch.bfloat16, device=DEV)
    x = store.as_strided((3, classes), (stride, 1))
    x.copy_(logits(3, classes, "bf16")[0])
    y = torch.tensor([0, classes - 1, 17], device=DEV)
    check(x, y, k=3)
    check(x[:, :100], y.clamp(max=99), k=3)
    del store, x
    torch.cuda.empty_cache()


def test_gradient_against_differences():
    """Central differences of the 64-bit formula: the gradient's formula itself."""
    x, y = logits(5, 12, "fp32")
    w = torch.tensor([0.3, -1.0, 2.0, 0.5, 1.5], dtype=torch.float64)
    leaf = x.clone().requires_grad_(True)
    got = label_log_probs(leaf, y, top_k=2)
    loss = (got.log_prob * w.float().to(DEV)).sum() + 0.7 * got.entropy.sum() - 0.4 * got.top_log_prob[:, 1].sum()
    dx, = torch.autograd.grad(loss, leaf)
    second = got.top_index[:, 1].cpu()

    def f(z):
        lp = torch.log_softmax(z, -1)
        h = -(lp.exp() * lp).sum(-1)
        return ((lp.gather(1, y.cpu()[:, None])[:, 0] * w).sum() + 0.7 * h.sum() - 0.4 * lp.gather(1, second[:, None]).sum())
    z, step = x.cpu().double(), 1e-5
    num = torch.zeros_like(z)
    for i in range(5):
        for j in range(12):
            e = torch.zeros_like(z)
            e[i, j] = step
            num[i, j] = (f(z + e) - f(z - e)) / (2 * step)
    # differences of 64-bit values of size ~20: 20 * 2^-52 / 1e-5 and the third derivative's 1e-10; then fp32's own
    assert (dx.cpu().double() - num).abs().max() < 1e-8 + 64 * U


def test_parts_of_the_result():
    x, y = logits(50, 40, "fp32")
    got = label_log_probs(x, y, entropy=False)
    assert got.entropy is None and got.top_index is None
    leaf = x.clone().requires_grad_(True)
    got = label_log_probs(leaf, y, top_k=3)
    assert not got.top_index.requires_grad
    only, = torch.autograd.grad(got.log_prob.sum(), leaf, retain_graph=True)  # (an expanded gradient; the others None)
    p = torch.softmax(x.double(), -1)
    want = torch.nn.functional.one_hot(y, 40).double() - p
    assert (only.double() - want).abs().max() < 64 * U
    # the second time the same, bit by bit
    again, = torch.autograd.grad(got.log_prob.sum(), leaf)
    assert torch.equal(only, again)
    with torch.no_grad():
        assert not label_log_probs(leaf, y).log_prob.requires_grad


def test_streams_run_apart():
    """Two streams, each with its own workspace, many calls in flight."""
    cases = [logits(2, 140001, "fp32", seed=s) for s in range(4)]
    want = [label_log_probs(x, y, top_k=9) for x, y in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=DEV) for _ in range(2)]
    got = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 2]):
            x, y = cases[i % 4]
            got.append(label_log_probs(x, y, top_k=9))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for a, b in zip(g, want[i % 4]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,classes", [(500, 16), (70, 3000), (1, 140001)])
def test_captured_and_replayed(rows, classes):
    x, y = logits(rows, classes, "fp32")
    static = x.clone().requires_grad_(True)
    w = torch.ones(rows, device=DEV)

    def step():
        got = label_log_probs(static, y, top_k=2)
        dx, = torch.autograd.grad([got.log_prob, got.entropy], [static], [w, w])
        return got.log_prob, got.entropy, got.top_index, dx
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        new, _ = logits(rows, classes, "fp32", seed=10 + i)
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def test_forward_mode_is_refused_and_not_lost():
    from torch.autograd import forward_ad

    from r3det.models.losses import CrossEntropyLoss
    x, y = torch.randn(6, 9, device=DEV), torch.arange(6, device=DEV)
    want = label_log_probs(x, y)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: label_log_probs(dual, y), lambda: CrossEntropyLoss()(dual, y)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        got = label_log_probs(x, y)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: label_log_probs(t, y).log_prob, (x,), (torch.ones_like(x),))
    assert torch.equal(got.log_prob, want.log_prob) and torch.equal(got.entropy, want.entropy)


@pytest.mark.parametrize("k", [1, 2, 3, 20])
@pytest.mark.parametrize("rows,classes", [(9, 40), (9, 100), (9, 900), (9, 1025), (9, 4000), (9, 70000), (300, 4000)])
def test_infinities_are_ranked_as_values(rows, classes, k):
    """One, two and many of +inf at a row's beginning, in its middle and at its end: their places come first, in order."""
    x = torch.randn(rows, classes, generator=torch.Generator().manual_seed(3)).to(DEV)
    x[0, 5] = math.inf
    x[1, classes // 2] = math.inf
    x[2, classes - 1] = math.inf
    x[3, 7] = x[3, 30] = math.inf
    x[4, ::3] = math.inf
    x[5] = math.inf
    x[6] = -math.inf
    x[6, 11] = math.inf
    x[7, 8:] = -math.inf
    x[7, 3] = math.inf
    for t in (torch.float32, torch.bfloat16):
        got = label_log_probs(x.to(t), top_k=k)
        want = reference(x.to(t), k=k)["top_index"]
        assert torch.equal(got.top_index.cpu(), want)
        assert got.top_log_prob[:6].isnan().all() and got.entropy[:8].isnan().all()
        assert torch.equal(got.top_index[5].cpu(), torch.arange(k))


@pytest.mark.parametrize("k", [1, 3, 20])
@pytest.mark.parametrize("rows,classes", [(3, 100), (3, 900), (3, 4000), (3, 70000), (300, 4000)])
def test_smallest_negative_numbers_are_ranked_as_values(rows, classes, k):
    """Subnormal logits below zero, next to -0 in the order."""
    step = torch.randint(1, 30000, (rows, classes), generator=torch.Generator().manual_seed(4))
    x = -(step * 2.0 ** -149).to(torch.float32).to(DEV)
    assert (x < 0).all()
    got = label_log_probs(x, top_k=k)
    assert torch.equal(got.top_index.cpu(), reference(x, k=k)["top_index"])
    assert (got.top_log_prob + math.log(classes)).abs().max() <= (classes / 64 + 60) * U + 2e-6


@pytest.mark.parametrize("rows,classes", [((1 << 22) + 3, 5), ((1 << 22) + 3, 1030), ((1 << 26) + 5, 129)])
def test_more_rows_than_a_launch_takes(rows, classes):
    """Rows are independent: those at the ends and around every border are what they are by themselves, and none is left out."""
    x = torch.empty(rows, classes, dtype=torch.bfloat16, device=DEV).normal_()
    y = torch.arange(rows, device=DEV) % classes
    y[-2] = IGNORE
    leaf = x.requires_grad_(True)
    got = label_log_probs(leaf, y, top_k=2, ignore_index=IGNORE)
    weight = torch.linspace(-1, 1, rows, device=DEV)
    d, = torch.autograd.grad([got.log_prob, got.top_log_prob], [leaf], [weight, weight[:, None].expand(rows, 2)])
    assert got.log_prob.max() <= 0 and (got.top_index >= 0).all() and (got.top_index < classes).all()
    at = sorted({r for b in range(0, rows, 1 << 22) for r in (b - 1, b, b + 1) if 0 <= r < rows} | set(range(rows - 5, rows)))
    at = torch.tensor(at, device=DEV)
    few = x.detach()[at].clone().requires_grad_(True)
    want = label_log_probs(few, y[at], top_k=2, ignore_index=IGNORE)
    dw, = torch.autograd.grad([want.log_prob, want.top_log_prob], [few], [weight[at], weight[at][:, None].expand(len(at), 2)])
    for a, b in zip(got, want):
        assert torch.equal(a[at], b)
    assert torch.equal(d[at], dw)
    # the gradient of a row sums to nothing, whatever its place
    sums = torch.cat([part.float().sum(1) for part in d.split(1 << 22)])
    assert sums.abs().max() <= 3 * 2.0 ** -8 * 2
    del x, leaf, d, got, sums
    torch.cuda.empty_cache()


def test_the_most_classes():
    """2^31 - 1 of them in one row, zeros but for a peak at the last and a masked one: log S is known.  256 workgroups of sixteen
    wavefronts add at most 8192 terms a lane, so S is off by 8300 u relatively."""
    n = 2 ** 31 - 1
    x = torch.zeros(1, n, dtype=torch.bfloat16, device=DEV)
    x[0, -1] = 5
    x[0, 7] = -math.inf
    leaf = x.requires_grad_(True)
    got = label_log_probs(leaf, torch.tensor([n - 1], device=DEV), top_k=9)
    total = n - 2 + math.exp(5)
    lp = 5 - math.log(total)
    assert abs(got.log_prob.item() - lp) <= (8300 + 2 * abs(lp)) * U
    assert abs(got.entropy.item() - (math.log(total) - 5 * math.exp(5) / total)) <= (2 * 8300 + 3 * abs(lp)) * U
    assert got.top_index.tolist() == [[n - 1, 0, 1, 2, 3, 4, 5, 6, 8]]
    d, = torch.autograd.grad(got.log_prob.sum(), leaf)
    some = d[0, [0, 6, 7, 8, n // 2, n - 2, n - 1]].double().cpu()
    want = torch.tensor([-1 / total] * 7, dtype=torch.float64)
    want[2], want[6] = 0, 1 - math.exp(lp)
    assert ((some - want).abs() <= want.abs() * (2.0 ** -8 + 9000 * U)).all()
    assert bool((d[0, 8:-1].view(torch.int16).split(1 << 28)[3] == d[0, 8].view(torch.int16)).all())
    del x, leaf, d
    torch.cuda.empty_cache()


def test_two_threads_at_once():
    """Calls on two streams from two threads, long rows with workspaces among them."""
    import threading
    cases = [logits(r, c, t) for r, c, t in ((3, 70000, "fp32"), (300, 4000, "bf16"), (5000, 16, "fp32"), (67, 33000, "fp16"))]
    want = [label_log_probs(x, y, top_k=8) for x, y in cases]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        stream = torch.cuda.Stream(device=DEV)
        with torch.cuda.stream(stream):
            for i in range(40):
                x, y = cases[(i + k) % 4]
                got = label_log_probs(x, y, top_k=8)
                bad.extend([(k, i)] * (not all(torch.equal(a, b) for a, b in zip(got, want[(i + k) % 4]))))
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad

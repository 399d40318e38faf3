"""r3det.ops.orthogonalize against the formulas in 64 bits, over shapes, types, layouts, spectra and lists.

Tolerance of the iteration, in u = 2^-24, in the Frobenius norm.  An iterate held as hi + lo is off by u relatively, a
product of two by 3 u more (the part left out among it), and its sum over K terms in fp32 by the roundings of its partial
sums: K / 16 additions of random sign, sqrt(K) u at the most.  The step's polynomial has |a| + |b| + |c| = 10.3 of such
products in it, so a step adds e = (32 + 10 sqrt(K)) u |X| (K the longer side).  What is there already is multiplied by the
step's largest slope: the slopes a + 3 b s^2 + 5 c s^4, the quotients p(s) / s and the divided differences of the
polynomial lie below 4 on [0, 1.21] for the usual coefficients, so the error of `steps` steps is at most
sum_k 4^(steps - k) e_k.  That holds for every spectrum; for the ones here the op-by-op form in fp32 says much more, so
the result must also be no further from 64 bits than three times that form is (their roundings have like sizes and
different signs).  A result of 16 bits adds half a step of its own.

The second bound says nothing for a matrix of equal rows (``alike``).  The op-by-op form rounds equal rows equally, so its
error stays in the one direction the matrix has, where the slope is small; any form that sums an entry's terms in an order
of its own (in blocks, or with the diagonal apart) has errors in the directions the matrix does not have, where a step
multiplies them by a = 3.4445 exactly.  There the first bound holds alone, with the slope a."""
import math

import pytest
import torch

from r3det.ops.orthogonalize import COEFFICIENTS, orthogonal_update_, orthogonalize

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def iterate(g, steps=5, co=COEFFICIENTS, eps=1e-7, dtype=torch.float64):
    """(result, norms of the iterates) in `dtype`."""
    x = g.to(dtype).reshape(g.size(0), -1)
    tall = x.size(0) > x.size(1)
    x = (x.t() if tall else x).contiguous()
    x = x / (x.double().norm() + eps).to(dtype)
    norms = [x.double().norm().item()]
    a, b, c = co
    for _ in range(steps):
        p = x @ x.t()
        p = b * p + c * (p @ p)
        x = a * x + p @ x
        norms.append(x.double().norm().item())
    return (x.t() if tall else x).reshape(g.shape), norms


def tolerances(g, norms, plain_error, steps, dtype, slope=4.0, alike=False):
    k = max(g.size(0), g.numel() // g.size(0))
    e = (32 + 10 * math.sqrt(k)) * U
    proven = sum(slope ** (steps - i) * e * norms[i] for i in range(steps)) + e * norms[-1]
    yard = math.inf if alike else 3 * plain_error + 16 * U * norms[-1]
    t = torch.finfo(dtype)
    own = 0.0 if dtype == torch.float32 else t.eps / 2 * norms[-1] + t.smallest_normal * t.eps / 2 * math.sqrt(g.numel())
    return min(proven, yard) + own


def check(tensors, steps=5, co=COEFFICIENTS, eps=1e-7, slope=4.0, alike=False):
    got = orthogonalize(tensors, steps=steps, coefficients=co, eps=eps)
    for g, o in zip(tensors, got):
        assert o.shape == g.shape and o.dtype == g.dtype and o.is_contiguous()
        want, norms = iterate(g, steps, co, eps)
        plain = iterate(g, steps, co, eps, torch.float32)[0]
        tol = tolerances(g, norms, (plain.double() - want).norm().item(), steps, o.dtype, slope, alike)
        off = (o.double() - want).norm().item()
        assert off <= tol, (tuple(g.shape), off, tol, norms[-1])
    return got


def matrix(n, m, kind="noise", dtype="fp32", seed=0):
    gen = torch.Generator().manual_seed(seed * 7919 + n * 101 + m)
    g = torch.randn(n, m, generator=gen)
    if kind == "low":  # a few directions over noise: small singular values among large ones
        r = min(n, m, 8)
        g = torch.randn(n, r, generator=gen) @ torch.randn(r, m, generator=gen) + 0.02 * g
    if kind == "rank1":
        g = torch.randn(n, 1, generator=gen) @ torch.randn(1, m, generator=gen)
    if kind == "ones":
        g = torch.ones(n, m)
    if kind == "eye":
        g = torch.eye(n, m)
    return g.to(TYPES[dtype]).to(DEV)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (5, 3), (63, 64), (64, 64), (65, 64), (64, 129), (127, 65), (1, 4097), (4097, 1),
          (5, 2304), (15, 2304), (256, 256), (257, 300), (300, 257), (256, 2304), (777, 1000), (1000, 777), (130, 9000)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, dtype):
    check([matrix(*shape, dtype=dtype)])


@pytest.mark.parametrize("kind", ["low", "rank1", "ones", "eye"])
@pytest.mark.parametrize("shape", [(64, 64), (200, 130), (256, 1280), (512, 600)], ids=str)
def test_spectra(shape, kind):
    if kind == "ones":
        check([matrix(*shape, kind=kind)], slope=COEFFICIENTS[0], alike=True)
    else:
        check([matrix(*shape, kind=kind)])


def test_a_ragged_list_of_many():
    shapes = [(1 + (37 * i) % 200, 1 + (91 * i) % 300) for i in range(110)]  # (more than one table's worth)
    check([matrix(*s, seed=i) for i, s in enumerate(shapes)])


@pytest.mark.parametrize("count", [170, 171, 172, 213, 214])
def test_lists_that_just_fill_the_card(count):
    """Three 128 x 128 tiles a symmetric matrix, 512 of which the card takes at a time: none, one, four, 127 and 130 are left."""
    shapes = [(200, 300), (256, 129), (130, 140)]
    check([matrix(*shapes[i % 3], seed=i) for i in range(count)])


@pytest.mark.parametrize("kind", ["noise", "low"])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("shape", [(300, 500), (300, 1025), (300, 5000), (940, 1000), (1100, 1300), (2100, 1200)], ids=str)
def test_steps_one_by_one_and_in_groups(shape, steps, kind):
    """21 tiles of 64: single steps without parts of X X^t, groups of them otherwise, the n x n products two to a launch
    where they can; those of 136, 171 and 210 where they must."""
    check([matrix(*shape, kind=kind)], steps=steps)


@pytest.mark.parametrize("steps", [3, 4, 5, 6])
@pytest.mark.parametrize("rows", [2, 3, 5, 9])
def test_a_large_singular_value_beside_small_ones(rows, steps):
    """What a step rounds in the large one's direction is carried over into the others', which grow: few rows show it, as the
    op-by-op form is off by little there."""
    for cols in (60, 200, 700):
        for large in (3.0, 12.0, 40.0):
            g = matrix(rows, cols, seed=rows)
            u, _, v = torch.linalg.svd(g.double().cpu(), full_matrices=False)
            s = torch.ones(rows, dtype=torch.float64)
            s[0] = large
            check([((u * s) @ v).float().to(DEV)], steps=steps)


@pytest.mark.parametrize("shape", [(4100, 4300), (8200, 4097)], ids=str)
def test_large(shape):
    check([matrix(*shape, kind="low"), matrix(64, 64)])


@pytest.mark.parametrize("steps,co,slope", [(1, COEFFICIENTS, 4.0), (2, COEFFICIENTS, 4.0), (10, COEFFICIENTS, 4.0),
                                            (12, (1.5, -0.5, 0.0), 1.5), (6, (15 / 8, -10 / 8, 3 / 8), 1.9)])
def test_steps_and_coefficients(steps, co, slope):
    check([matrix(100, 170), matrix(70, 30)], steps=steps, co=co, slope=slope)


def test_converges_to_the_polar_factor():
    """With the cubic coefficients (slope 0 at 1) the result is U V^t, whatever the formula's rounding."""
    g = matrix(96, 200) + 3 * torch.eye(96, 200, device=DEV)
    o = orthogonalize(g, steps=40, coefficients=(1.5, -0.5, 0.0))
    u, _, vt = torch.linalg.svd(g.double().cpu(), full_matrices=False)
    assert (o.cpu().double() - u @ vt).norm() <= 96 ** 0.5 * (32 + 10 * 200 ** 0.5) * U * 2
    assert (o @ o.t() - torch.eye(96, device=DEV)).abs().max() < 1e-4


def test_scale_of_the_input():
    """Any power of two in front of the matrix changes nothing but eps' share."""
    g = matrix(90, 150)
    want = orthogonalize(g, eps=0.0)
    for e in (-60, -20, 20, 60):
        assert torch.equal(orthogonalize(g * 2.0 ** e, eps=0.0), want)
    check([g * 1e-7, g * 1e-6, g * 1e30])
    assert torch.equal(orthogonalize(torch.zeros(5, 9, device=DEV)), torch.zeros(5, 9, device=DEV))


def test_nan_and_inf_stay_in_their_matrix():
    a, b, c = matrix(70, 200), matrix(64, 64), matrix(300, 40)
    clean = orthogonalize([a, matrix(64, 64), c])
    for bad in (math.nan, math.inf, -math.inf):
        b[3, 5] = bad
        got = orthogonalize([a, b, c])
        assert torch.isnan(got[1]).any()
        assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype):
    base = matrix(140, 200, dtype=dtype)
    check([base.t(), base[::2], base[:, 1:], base[:, ::3], base[3:40, 5:9]])
    check([base[:1].expand(30, 200)], slope=COEFFICIENTS[0], alike=True)
    conv = base.reshape(140, 8, 5, 5)
    got = check([conv, conv.contiguous(memory_format=torch.channels_last)])
    assert torch.equal(got[0], got[1])
    one = orthogonalize(conv)
    assert one.shape == conv.shape
    shifted = torch.empty(140 * 200 + 1, dtype=base.dtype, device=DEV)[1:].view(140, 200).copy_(base)
    check([shifted])
    empty = orthogonalize([torch.empty(0, 5, device=DEV), torch.empty(5, 0, device=DEV)])
    assert [tuple(t.shape) for t in empty] == [(0, 5), (5, 0)]


def test_the_same_matrix_twice_and_again():
    g, h = matrix(256, 2304), matrix(65, 64)
    first = orthogonalize([g, h, g])
    assert torch.equal(first[0], first[2])
    for _ in range(3):
        for x, y in zip(orthogonalize([g, h, g]), first):
            assert torch.equal(x, y)
    assert not orthogonalize(g.clone().requires_grad_(True)).requires_grad


def test_coefficients_that_grow_are_refused():
    with pytest.raises(RuntimeError, match="invalid argument"):
        orthogonalize(matrix(8, 8), coefficients=(20.0, 0.0, 0.0))


def test_offsets_beyond_32_bits():
    gs = [matrix(64, 64, seed=i).half().repeat(128, 256) + torch.eye(8192, 16384, device=DEV).half() * (i + 1) for i in range(3)]
    got = orthogonalize(gs, steps=1)
    for g, o in zip(gs, got):
        want = iterate(g, 1)[0]
        assert (o.double() - want).norm() <= want.norm() * (2.0 ** -11 + 16 * U) + 2.0 ** -25 * g.numel() ** 0.5


def update_by_formula(w, g, m, lr, momentum, nesterov, decay, scale, steps=5):
    w, g, m = w.double(), g.double(), m.double()
    m = momentum * m + g
    u = g + momentum * m if nesterov else m
    rows, cols = w.size(0), w.numel() // w.size(0)
    s = 0.2 * math.sqrt(max(rows, cols)) if scale == "rms" else math.sqrt(max(1.0, rows / cols)) if scale == "spectral" else scale
    o, norms = iterate(u.contiguous(), steps)
    plain = iterate(u.contiguous(), steps, dtype=torch.float32)[0]
    tol = tolerances(u, norms, (plain.double() - o).norm().item(), steps, torch.float32)
    # (u itself is rounded to fp32 twice before the iteration: 2 u, carried through it as its first roundings are)
    tol += 3 * sum(4.0 ** (steps - i) * U * norms[i] for i in range(1))
    return (1 - lr * decay) * w - lr * s * o, m, lr * s * tol


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("nesterov,decay,scale", [(True, 0.01, "rms"), (False, 0.0, "spectral"), (True, 0.1, 0.7)])
def test_update(dtype, nesterov, decay, scale):
    t = TYPES[dtype]
    shapes = [(64, 64, 1, 1), (256, 256, 3, 3), (45, 256, 3, 3), (1, 9), (300, 20), (64, 7, 3, 5)]
    gen = torch.Generator().manual_seed(5)
    mk = lambda s: torch.randn(s, generator=gen).to(DEV)  # noqa: E731
    ws = [mk(s).to(t) for s in shapes]
    ws[1] = ws[1].contiguous(memory_format=torch.channels_last)
    ws[5] = ws[5].contiguous(memory_format=torch.channels_last)
    ms = [torch.empty_like(w, dtype=torch.float32).copy_(mk(s)) for w, s in zip(ws, shapes)]
    ref = [(w.double(), m.double()) for w, m in zip(ws, ms)]
    for turn in range(3):
        gs = [mk(s).to(t) for s in shapes]
        gs[1] = gs[1].contiguous(memory_format=torch.channels_last)  # (gs[5] is laid out otherwise than its weight)
        before = [(w.clone(), m.clone()) for w, m in zip(ws, ms)]
        versions = [w._version for w in ws]
        orthogonal_update_(ws, gs, ms, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=decay, scale=scale)
        assert all(w._version > v for w, v in zip(ws, versions))
        for w, g, m, (w0, m0) in zip(ws, gs, ms, before):
            want_w, want_m, tol = update_by_formula(w0, g, m0, 0.05, 0.9, nesterov, decay, scale)
            assert ((m.double() - want_m).abs() <= 3 * U * (want_m.abs() + m0.abs().double() + g.abs().double())).all()
            half = torch.finfo(t).eps / 2
            tol += (half + 4 * U) * want_w.norm().item() + torch.finfo(t).smallest_normal * w.numel() ** 0.5
            assert (w.double() - want_w).norm() <= tol
            assert w.stride() == w0.stride()
    assert len(ref) == len(ws)


def test_update_leaves_its_neighbours_alone():
    """Weights and momenta inside larger buffers: nothing before or behind them is written."""
    n, m, pad = 37, 91, 64
    store = [torch.full((n * m + 2 * pad,), 7.0, device=DEV) for _ in range(2)]
    w, b = (s[pad:pad + n * m].view(n, m) for s in store)
    g = matrix(n, m)
    keep = g.clone()
    orthogonal_update_([w], [g], [b], lr=0.1)
    for s in store:
        assert (s[:pad] == 7).all() and (s[pad + n * m:] == 7).all()
    assert torch.equal(g, keep) and not (w == 7).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(300, 1), (300, 3), (300, 4), (300, 5), (300, 6), (300, 7), (3, 301), (130, 129), (131, 130), (140, 131),
                                   (50, 61)], ids=str)
def test_rows_that_end_anywhere_from_any_element_on(shape, dtype):
    """Rows of any length, weights, gradients and momenta from an odd element on: the same bits as aligned ones, and nothing
    around them is written."""
    n, m = shape
    t = TYPES[dtype]
    w0, g0, b0 = matrix(n, m, dtype=dtype, seed=1), matrix(n, m, dtype=dtype, seed=2), matrix(n, m, seed=3)
    stores, views = [], []
    for k, x in enumerate((w0, g0, b0)):
        store = torch.full((n * m + 16,), 7.0, dtype=x.dtype, device=DEV)
        view = store[2 * k + 1:2 * k + 1 + n * m].view(n, m)
        view.copy_(x)
        stores.append(store), views.append(view)
    w, g, b = views
    assert torch.equal(orthogonalize(g), orthogonalize(g0))
    orthogonal_update_([w], [g], [b], lr=0.1, weight_decay=0.01)
    orthogonal_update_([w0], [g0], [b0], lr=0.1, weight_decay=0.01)
    assert torch.equal(w, w0) and torch.equal(b, b0) and torch.equal(g, g0)
    for k, store in enumerate(stores):
        assert (store[:2 * k + 1] == 7).all() and (store[2 * k + 1 + n * m:] == 7).all()
    check([g0])


def test_update_of_weights_that_need_gradients():
    w = torch.nn.Parameter(matrix(20, 30))
    (w * matrix(20, 30, seed=1)).sum().backward()
    before = w.detach().clone()
    orthogonal_update_([w], [w.grad], [torch.zeros_like(w)], lr=0.1)
    assert w.requires_grad and w.is_leaf and not torch.equal(w.detach(), before)


def test_streams_run_apart():
    lists = [[matrix(256, 2304, seed=i), matrix(15, 2304, seed=i), matrix(64, 64, seed=i)] for i in range(4)]
    want = [orthogonalize(l) for l in lists]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=DEV) for _ in range(2)]
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            got.append(orthogonalize(lists[i % 4]))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for x, y in zip(g, want[i % 4]):
            assert torch.equal(x, y)


def test_captured_and_replayed():
    shapes = [(64, 64), (256, 2304), (45, 2304)]
    ws = [matrix(*s) for s in shapes]
    ms = [torch.zeros_like(w) for w in ws]
    gs = [torch.zeros_like(w) for w in ws]
    e_ws, e_ms = [w.clone() for w in ws], [m.clone() for m in ms]
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        orthogonalize(gs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]  # (two graphs of one pool: each has its own workspace or its turn)
    for k, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if k else None):
            orthogonal_update_(ws, gs, ms, lr=0.02)
    for i in range(4):
        for g, s in zip(gs, shapes):
            g.copy_(matrix(*s, seed=30 + i))
        graphs[i % 2].replay()
        orthogonal_update_(e_ws, gs, e_ms, lr=0.02)
        torch.cuda.synchronize()
        for x, y in zip(ws + ms, e_ws + e_ms):
            assert torch.equal(x, y)


def one_large(rows, cols, large):
    g = matrix(rows, cols, seed=rows)
    u, _, v = torch.linalg.svd(g.double().cpu(), full_matrices=False)
    s = torch.ones(min(rows, cols), dtype=torch.float64)
    s[0] = large
    return ((u * s) @ v).float().to(DEV)


@pytest.mark.parametrize("steps", [3, 5, 7])
@pytest.mark.parametrize("rows", [2, 5, 15, 45, 65, 135, 192, 255, 256, 300])
def test_a_large_singular_value_in_a_long_list(rows, steps):
    """Beside as many tiles as a head's tower has, where wide matrices take their steps in groups: every matrix stays as close as
    it is alone.  (What a step rounds in the large value's direction is what a group carries over, see above.)"""
    tower = [matrix(256, 2304, seed=i) for i in range(8)]
    check([one_large(rows, cols, large) for cols in (600, 2304) for large in (9.0, 12.0, 20.0, 40.0)] + tower, steps=steps)


def test_neighbours_in_a_list_change_nothing_of_a_narrow_matrix_s_accuracy():
    """A head's predictions, their towers beside them: no further from 64 bits than 4 times what the same matrices alone are
    (single steps both times; parts of X X^t may differ), which their errors' random signs leave room for."""
    preds = [one_large(rows, 2304, 20.0) for rows in (5, 15, 45, 135)]
    tower = [matrix(256, 2304, seed=i) for i in range(8)]
    for g, beside, alone in zip(preds, orthogonalize(preds + tower), (orthogonalize(g) for g in preds)):
        want, norms = iterate(g)
        off = [(o.double() - want).norm().item() for o in (beside, alone)]
        assert off[0] <= 4 * off[1] + 4 * U * norms[-1], (tuple(g.shape), off)


MIXED = [(300, 500), (100, 900), (5, 700), (64, 64), (1100, 1300), (200, 210), (4097, 65), (15, 2304), (256, 256), (1, 5000)]


@pytest.mark.parametrize("steps,co,slope", [(s, COEFFICIENTS, 4.0) for s in (1, 2, 3, 4, 5, 6, 9)] +
                         [(7, (1.5, -0.5, 0.0), 1.5), (5, (15 / 8, -10 / 8, 3 / 8), 1.9)])
def test_narrow_and_wide_matrices_together(steps, co, slope):
    """Two chains of launches, the narrow one's pieces among the wide one's: more, as many and fewer of them than launches."""
    check([matrix(*s, seed=i) for i, s in enumerate(MIXED)], steps=steps, co=co, slope=slope)
    check([matrix(*s, dtype="bf16", seed=i) for i, s in enumerate(MIXED[::-1])], steps=steps, co=co, slope=slope)


@pytest.mark.parametrize("wide", [39, 40, 41])
def test_chains_that_end_anywhere_in_a_table(wide):
    shapes = [(260, 300 + i) for i in range(wide)]
    shapes[7:7] = [(100, 300), (64, 50), (3, 999)]
    check([matrix(*s, seed=i) for i, s in enumerate(shapes + [(200, 222)])])


def test_many_narrow_matrices_beside_a_wide_one():
    """A chain of its own work for the whole card, in tiles of 128, behind the wide one's."""
    check([matrix(200, 300, seed=i) for i in range(90)] + [matrix(1100, 1300)] + [matrix(130, 1000, seed=i) for i in range(90)])


def test_many_wide_matrices_beside_narrow_ones():
    """The wide ones in tiles of 128, quartered ones among them, with pieces of 64 along."""
    check([matrix(300, 400, seed=i) for i in range(52)] + [matrix(100, 700), matrix(9, 2000)] +
          [matrix(700, 900, seed=i) for i in range(13)])


def test_update_of_a_head():
    shapes = [(256, 2304)] * 8 + [(135, 2304), (45, 2304), (64, 100)]
    gen = torch.Generator().manual_seed(6)
    ws, gs, ms = ([torch.randn(s, generator=gen).to(DEV) for s in shapes] for _ in range(3))
    before = [(w.clone(), m.clone()) for w, m in zip(ws, ms)]
    orthogonal_update_(ws, gs, ms, lr=0.05, momentum=0.9, weight_decay=0.01)
    for w, g, m, (w0, m0) in zip(ws, gs, ms, before):
        want_w, want_m, tol = update_by_formula(w0, g, m0, 0.05, 0.9, True, 0.01, "rms")
        assert ((m.double() - want_m).abs() <= 3 * U * (want_m.abs() + m0.abs().double() + g.abs().double())).all()
        assert (w.double() - want_w).norm() <= tol + 5 * U * want_w.norm().item()


@pytest.mark.parametrize("steps,co", [(1, COEFFICIENTS), (5, COEFFICIENTS), (1, (1.5, -0.5, 0.0)), (6, (1.5, -0.5, 0.0))])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_bad_value_makes_its_whole_matrix_nan_and_no_other(bad, steps, co):
    """In every form: one launch for all steps, single steps, groups, tiles of 64 and of 128, pieces of one chain along with
    another's.  (An infinity leaves one NaN among zeros in the first X; its row and column of A are NaN, and so all of F X.)"""
    for shapes in ([(64, 64), (30, 100), (1, 9)], [(70, 200), (1, 4097), (300, 40)], [(300, 500), (257, 256)], MIXED,
                   [(256, 2304)] * 8 + [(135, 2304), (5, 2304)], [(300, 400)] * 60):
        ts = [matrix(*s, seed=i) for i, s in enumerate(shapes)]
        clean = orthogonalize(ts, steps=steps, coefficients=co)
        for k in {0, len(ts) // 2, len(ts) - 1}:
            n, m = shapes[k]
            one = list(ts)
            one[k] = ts[k].clone()
            one[k][n // 2, m - 1] = bad
            for i, (got, want) in enumerate(zip(orthogonalize(one, steps=steps, coefficients=co), clean)):
                if i == k:
                    assert torch.isnan(got).all(), (shapes[k], torch.isnan(got).sum())
                else:
                    assert torch.equal(got, want), (shapes[k], shapes[i])


def test_a_bad_gradient_spoils_its_weight_alone():
    shapes = [(64, 64), (135, 700), (300, 500), (1100, 1300)]
    ws, gs = [matrix(*s, seed=1) for s in shapes], [matrix(*s, seed=2) for s in shapes]
    clean, ms = [w.clone() for w in ws], [torch.zeros_like(w) for w in ws]
    orthogonal_update_(clean, gs, [m.clone() for m in ms], lr=0.1)
    for k in range(len(shapes)):
        got, bad = [w.clone() for w in ws], [g.clone() for g in gs]
        bad[k][2, 3] = math.inf
        orthogonal_update_(got, bad, [m.clone() for m in ms], lr=0.1)
        for i, (a, b) in enumerate(zip(got, clean)):
            assert torch.isnan(a).all() if i == k else torch.equal(a, b)


@pytest.mark.parametrize("shape", [(64, 64), (5, 700), (256, 2304), (1100, 1300)], ids=str)
def test_norms_far_below_eps(shape):
    """Values are held times 2^12 in fp16 pairs, whose second has steps of 2^-24: an entry is off by up to 2^-37 at first and
    after every step, and each step multiplies that by a (the cubic and quintic terms are nothing there)."""
    a = COEFFICIENTS[0]
    least = 2.0 ** -37 * sum(a ** k for k in range(6)) * math.sqrt(shape[0] * shape[1])
    for norm in (1e-8, 1e-9, 1e-10, 1e-12, 1e-15):
        g = matrix(*shape)
        g *= norm / g.norm()
        want, norms = iterate(g)
        plain = (iterate(g, dtype=torch.float32)[0].double() - want).norm().item()
        got = orthogonalize([g, matrix(256, 300)])[0]
        assert (got.double() - want).norm().item() <= tolerances(g, norms, plain, 5, torch.float32) + least, norm


@pytest.mark.parametrize("shape", [(65535, 32767), (1, 4194240), (4194240, 400)], ids=str)
def test_the_largest_matrices(shape):
    """Against the formula in 64 bits on three vectors, one step; the result is rounded to bf16, at most half a step an entry (a
    vector meets that error as a matrix of random signs: its norm is what it is of the entries)."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    g = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    o = orthogonalize(g, steps=1)
    norm = math.sqrt(sum(float(p.double().pow(2).sum()) for p in g.split(4096))) + 1e-7

    def of(m, v):
        return torch.cat([p.double() @ v for p in m.split(4096)])

    def turned(u):
        return sum(p.double().t() @ q for p, q in zip(g.split(4096), u.split(4096)))
    a, b, c = COEFFICIENTS
    v = torch.randn(shape[1], 3, generator=gen, device=DEV, dtype=torch.float64)
    x = of(g, v) / norm
    once = of(g, turned(x)) / norm ** 2
    want = a * x + b * once + c * of(g, turned(once)) / norm ** 2
    assert (of(o, v) - want).norm() <= want.norm() * (2.0 ** -8 + 64 * U)
    del g, o
    torch.cuda.empty_cache()


def test_two_threads_at_once():
    """Calls on two streams from two threads: mixed lists, small ones, updates in place."""
    import threading
    lists = [[matrix(*s, seed=i) for i, s in enumerate(shapes)] for shapes in (MIXED, [(64, 64), (20, 100)], [(256, 2304)] * 8 + [(135, 2304)])]
    want = [orthogonalize(l) for l in lists]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        stream = torch.cuda.Stream(device=DEV)
        with torch.cuda.stream(stream):
            for i in range(12):
                got = orthogonalize(lists[(i + k) % 3])
                bad.extend([(k, i)] * (not all(torch.equal(x, y) for x, y in zip(got, want[(i + k) % 3]))))
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad

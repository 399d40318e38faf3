"""CPU: what r3det.ops.orthogonalize refuses, at the Python boundary and at the C entries (which check before any launch)."""
import ctypes

import pytest
import torch

from r3det import _C
from r3det.ops.orthogonalize import orthogonal_update_, orthogonalize

W = torch.zeros(4, 6)


def test_refusals_of_orthogonalize():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        orthogonalize(W)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        orthogonalize([W, W])
    with pytest.raises(TypeError, match="Tensor"):
        orthogonalize([1.0])
    with pytest.raises(ValueError, match="two dimensions"):
        orthogonalize(torch.zeros(4))
    with pytest.raises(RuntimeError, match="fp32, fp16 or bf16"):
        orthogonalize(W.double())
    with pytest.raises(RuntimeError, match="one type"):
        orthogonalize([W, W.half()])
    with pytest.raises(ValueError, match="not taken"):
        orthogonalize(torch.empty(1, 1).expand(32769, 32769))
    for steps in (0, 65, 2.5, True):
        with pytest.raises(ValueError, match="steps"):
            orthogonalize(W, steps=steps)
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(W, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(W, eps=float("nan"))
    assert orthogonalize([]) == []


def test_refusals_of_the_update():
    ok = dict(params=[W.clone()], grads=[W], buffers=[W.clone()], lr=0.1)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        orthogonal_update_(**ok)
    for change, match in ((dict(grads=[]), "0 grads"), (dict(grads=[W[:2]]), "match its weight"),
                          (dict(buffers=[W[:, :3]]), "match its weight"), (dict(lr=-1.0), "negative"),
                          (dict(momentum=-0.1), "negative"), (dict(weight_decay=float("nan")), "negative"),
                          (dict(scale="mean"), "scale"), (dict(scale=None), "scale"), (dict(steps=0), "steps")):
        with pytest.raises(ValueError, match=match):
            orthogonal_update_(**{**ok, **change})
    for change, match in ((dict(grads=[W.half()]), "weight's type"), (dict(buffers=[W.half()]), "fp32"),
                          (dict(params=[torch.zeros(6, 4).t()]), "channels_last"),
                          (dict(buffers=[torch.zeros(6, 4).t()]), "laid out alike")):
        with pytest.raises(RuntimeError, match=match):
            orthogonal_update_(**{**ok, **change})
    w = W.clone()
    with pytest.raises(ValueError, match="twice"):
        orthogonal_update_([w, w], [W, W], [W.clone(), W.clone()], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        orthogonal_update_([W.clone(), W.clone()], [W, W], [w, w], lr=0.1)
    orthogonal_update_([], [], [], lr=0.1)


def test_weights_that_share_memory_are_refused():
    big = torch.zeros(10, 6)
    with pytest.raises(ValueError, match="shares memory"):
        orthogonal_update_([big[:4], big[3:7]], [W, W], [W.clone(), W.clone()], lr=0.1)
    with pytest.raises(ValueError, match="shares memory"):
        orthogonal_update_([big[:4]], [W], [big[2:6]], lr=0.1)
    with pytest.raises(ValueError, match="shares memory"):
        orthogonal_update_([big[4:8]], [big[1:5]], [W.clone()], lr=0.1)
    with pytest.raises(ValueError, match="shares memory"):
        orthogonal_update_([big[4:8]], [big[6:10]], [W.clone()], lr=0.1)
    for args in (([big[:4], big[4:8]], [W, W], [W.clone(), W.clone()]),   # neighbours, one gradient for two: nothing refused
                 ([big[4:8]], [big[:4]], [W.clone()])):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            orthogonal_update_(*args, lr=0.1)


def test_refusals_of_the_c_entries():
    L = _C.lib()
    ints = lambda *v: (ctypes.c_int * len(v))(*v)  # noqa: E731
    ptrs = lambda *v: (ctypes.c_void_p * len(v))(*v)  # noqa: E731
    far = 1 << 20  # (never followed: every call below ends at its checks)
    size = L.r3det_orthogonalize_workspace_bytes
    assert size(0, None, None) == 0
    for rows, cols in ((0, 4), (4, 0), (-1, 4), (32769, 32769), (1 << 16, 1 << 16), (1, 65536 * 64)):
        assert size(1, ints(rows), ints(cols)) == 0, (rows, cols)
    assert size(-1, ints(1), ints(1)) == 0 and size(1, None, ints(1)) == 0
    need = size(2, ints(4, 100), ints(6, 50))
    assert need > 0

    def run(count=2, src=ptrs(far, far), dst=ptrs(far, far), dtype=0, rows=ints(4, 100), cols=ints(6, 50), steps=5, a=3.4445,
            b=-4.775, c=2.0315, eps=1e-7, ws=far, n=need):
        return L.r3det_orthogonalize(count, src, dst, dtype, rows, cols, steps, a, b, c, eps, ws, n, None)
    assert run(count=0) == 0
    nan, inf = float("nan"), float("inf")
    for bad in (dict(count=-1), dict(src=None), dict(dst=None), dict(src=ptrs(far, None)), dict(dst=ptrs(None, far)), dict(dtype=3),
                dict(rows=ints(0, 100)), dict(cols=None), dict(steps=0), dict(steps=65), dict(a=nan), dict(b=inf), dict(c=nan),
                dict(a=20.0), dict(a=4.0, b=0.0, c=0.0), dict(b=-20.0), dict(eps=-1.0), dict(eps=nan), dict(ws=far + 8)):
        assert run(**bad) == -1, bad
    assert run(a=2.0, b=0.0, c=0.0, steps=3) == -1  # |X| doubles: X = 4 before the third step, whose A = 16 is over 15
    assert run(ws=None) == -3 and run(n=need - 1) == -3
    # coefficients that keep the iterates bounded pass this check (and end at the workspace's)
    for a, b, c, steps in ((1.5, -0.5, 0.0, 20), (2.0, -1.5, 0.5, 64), (15 / 8, -10 / 8, 3 / 8, 10), (3.4445, -4.7750, 2.0315, 10),
                           (2.0, 0.0, 0.0, 2), (0.0, 0.0, 0.0, 1)):
        assert run(a=a, b=b, c=c, steps=steps, n=0) == -3, (a, b, c)

    def update(bufs=ptrs(far, far), rates=(ctypes.c_float * 2)(1, 1), ws=far, n=0):
        return L.r3det_orthogonal_update(2, ptrs(far, far), ptrs(far, far), bufs, 0, ints(4, 100), ints(6, 50), rates, 1.0, 0.9,
                                         1, 5, 3.4445, -4.775, 2.0315, 1e-7, ws, n, None)
    assert update() == -3
    assert update(bufs=None) == -1 and update(rates=None) == -1 and update(bufs=ptrs(far, None)) == -1


def test_every_limit_is_refused_with_its_reason():
    """What the C entries do not take is refused by name in front of them, and nothing else is."""
    one = torch.empty(1, 1)
    L = _C.lib()
    for rows, cols, taken in ((1, 4194240, True), (1, 4194241, False), (4194241, 1, False), (5000000, 2, False), (32768, 65535, True),
                              (32769, 32769, False), (32768, 65536, False), (4194240, 511, True)):
        wide = (ctypes.c_int * 1)(rows), (ctypes.c_int * 1)(cols)
        assert (L.r3det_orthogonalize_workspace_bytes(1, *wide) > 0) == taken, (rows, cols)
        w = one.expand(rows, cols)
        with pytest.raises(RuntimeError if taken else ValueError, match="CUDA tensor" if taken else "not taken.*4194240"):
            orthogonalize([W, w])
    long = [torch.empty(1, 4194241) for _ in range(3)]
    with pytest.raises(ValueError, match="not taken"):
        orthogonal_update_(*([t] for t in long), lr=0.1)
    many = [torch.zeros(1, 1)] * 65537
    with pytest.raises(ValueError, match="at most 65536 matrices"):
        orthogonalize(many)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        orthogonalize(many[1:] + [torch.zeros(0, 3)])
    sizes = (ctypes.c_int * 65537)(*[1] * 65537)
    assert L.r3det_orthogonalize_workspace_bytes(65537, sizes, sizes) == 0
    assert L.r3det_orthogonalize_workspace_bytes(65536, sizes, sizes) > 0


def test_the_workspace_is_what_the_documentation_says():
    L = _C.lib()

    def size(*shapes):
        rows, cols = zip(*shapes)
        return L.r3det_orthogonalize_workspace_bytes(len(shapes), (ctypes.c_int * len(shapes))(*rows), (ctypes.c_int * len(shapes))(*cols))
    for shapes in ([(1, 1000000)], [(2048, 2048)], [(4096, 4096)], [(256, 2304)] * 8 + [(135, 2304)], [(300, 40000)], [(100, 70)] * 500):
        least = most = 0
        for r, c in shapes:
            n, m = (-(-s // 128) * 128 for s in sorted((r, c)))
            least += 8 * n * m + 24 * n * n
            most += 12 * n * m + 24 * n * n + 4 * n * n * -(-m // 512) + 4096 + n * m // 16  # (lists, diagonals, norms)
        assert least <= size(*shapes) <= most, (shapes, least, size(*shapes), most)
    assert size((64, 128), (128, 64), (5, 5)) == 256

"""Cases for timing the operators of a training step's two ends: the log probabilities a softmax classification loss is
made of (with entropies, best alternatives and the gradient), and the orthogonalised update of the weight matrices.

``own`` selects who computes a case: plain torch operations in 32 bits (False) or this package's operators (True)."""
import math
import os
import sys

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ the cases
def stages():
    """(rows, columns) of every trainable convolution weight of the R3Det-R50 detector: backbone stages 2-4, FPN, both
    heads and the feature refinement module's three convolutions."""
    got, width = [], 256
    for planes, blocks in ((128, 4), (256, 6), (512, 3)):
        got.append((4 * planes, width))  # the shortcut's projection
        for _ in range(blocks):
            got += [(planes, width), (planes, 9 * planes), (4 * planes, planes)]
            width = 4 * planes
    got += [(256, 512), (256, 1024), (256, 2048)] + [(256, 2304)] * 4 + [(256, 9 * 2048)]
    got += head(135, 45) + [(256, 1280), (256, 1280), (256, 256)] + head(15, 5)
    return got


def head(classes, boxes):
    """One head: two towers of four 3x3 convolutions over 256 channels, the class and the box prediction."""
    return [(256, 2304)] * 8 + [(classes, 2304), (boxes, 2304)]


def text(shapes):
    return " ".join("%dx%d" % s for s in shapes)


def shapes_of(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def listed():
    return [
        # the smallest update a training loop makes: one 1x1 convolution, where launches and latency count
        dict(name="update one 64x64", op="update", shapes=text([(64, 64)]), dtype="fp32"),
        # fine-tuning one detection head alone: equal wide matrices and two with few, odd rows
        dict(name="update one head", op="update", shapes=text(head(135, 45)), dtype="fp32"),
        # the optimiser step of the whole detector
        dict(name="update detector", op="update", shapes=text(stages()), dtype="fp32"),
        # weights kept in 16 bits, tall, wide, odd and single-row ones together
        dict(name="update ragged bf16", op="update", shapes=text([(1000, 777), (777, 1000), (1, 513), (129, 64), (65, 4097)]),
             dtype="bf16"),
        # one odd matrix, tall
        dict(name="orthogonalize odd 1025x511", op="orthogonalize", shapes=text([(1025, 511)]), dtype="bf16"),
        # a large square matrix in 32 bits, and a larger one held in 16
        dict(name="orthogonalize 2048x2048", op="orthogonalize", shapes=text([(2048, 2048)]), dtype="fp32"),
        dict(name="orthogonalize 4096x4096 fp16", op="orthogonalize", shapes=text([(4096, 4096)]), dtype="fp16"),
        # the classification loss of two 1024 x 1024 images: 9 anchors at every position of five levels, 15 classes and background
        dict(name="loss anchors", op="log_probs", rows=2 * 196416, classes=16, dtype="fp32", labels=True, top=0, masked=False,
             grad=True),
        # ranking the anchors of a batch of four at inference: the best two of 16 columns, no labels
        dict(name="rank anchors", op="log_probs", rows=4 * 196416, classes=16, dtype="fp32", labels=False, top=2, masked=False,
             grad=False),
        # one answer at a time over a long list of classes
        dict(name="one row of 50001", op="log_probs", rows=1, classes=50001, dtype="bf16", labels=True, top=8, masked=False,
             grad=False),
        # scoring a small batch with masked classes, some rows with nothing left, many alternatives
        dict(name="score 67x131072", op="log_probs", rows=67, classes=131072, dtype="fp32", labels=True, top=20, masked=True,
             grad=False),
        # training over a long list of classes
        dict(name="loss 4096x65536", op="log_probs", rows=4096, classes=65536, dtype="bf16", labels=True, top=0, masked=False,
             grad=True),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if rng.random() < 0.5:
        rows = size(1, 400_000)
        classes = size(2, min(160_000, 2 ** 28 // rows))
        grad = rng.random() < 0.5
        return dict(op="log_probs", rows=rows, classes=classes, dtype=dtype, labels=grad or rng.random() < 0.7,
                    top=0 if grad else min(classes, rng.randint(0, 20)), masked=rng.random() < 0.3, grad=grad)
    op = rng.choice(("update", "orthogonalize"))
    most = rng.choice((256, 1024, 4096))
    shapes = [(size(1, most), size(1, most)) for _ in range(1 if most == 4096 else rng.randint(1, 12))]
    return dict(op=op, shapes=text(shapes), dtype=dtype)


# ------------------------------------------------------------------------------------------------ the inputs
def gradient(shape, g):
    """A batch's gradient of a weight matrix: a few strong directions over noise."""
    n, m = shape
    r = min(n, m, 8)
    u, v = (torch.randn(s, generator=g, device="cuda") for s in ((n, r), (r, m)))
    return 1e-3 * (u @ v / math.sqrt(r) + 0.5 * torch.randn(n, m, generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = DTYPES[case["dtype"]]
    if case["op"] != "log_probs":
        shapes = shapes_of(case)
        grads = [gradient(s, g).to(t) for s in shapes]
        if case["op"] == "orthogonalize":
            return dict(case, grads=grads)
        # weights and momenta as views of one buffer each, as a training program keeps them
        total = sum(n * m for n, m in shapes)
        weights = torch.empty(total, dtype=t, device="cuda")
        momenta = torch.empty(total, dtype=torch.float32, device="cuda")
        state = dict(case, grads=grads, weights=weights, momenta=momenta, w=[], m=[])
        at = 0
        for n, m in shapes:
            w, b = (x[at:at + n * m].view(n, m) for x in (weights, momenta))
            w.copy_(torch.randn(n, m, generator=g, device="cuda") / math.sqrt(m))
            b.copy_(5 * gradient((n, m), g))
            state["w"].append(w)
            state["m"].append(b)
            at += n * m
        return state
    rows, classes = case["rows"], case["classes"]
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    if classes <= 64:  # anchors: nearly all of them are background, the last class
        labels = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.98, classes - 1, labels)
    logits = 2.5 * torch.randn(rows, classes, generator=g, device="cuda")
    logits.scatter_add_(1, labels[:, None], torch.rand(rows, 1, generator=g, device="cuda") * 8)
    if case["masked"]:  # classes that are not offered; every fifth row has none left
        logits.masked_fill_(torch.rand(rows, classes, generator=g, device="cuda") < 0.1, -math.inf)
        logits[3::5] = -math.inf
    state = dict(case, logits=logits.to(t), labels=labels if case["labels"] else None)
    if case["grad"]:
        state["logits"].requires_grad_(True)
        ignored = torch.rand(rows, generator=g, device="cuda") < 0.05
        state["labels"] = torch.where(ignored, -100, labels)
        weight = torch.rand(rows, generator=g, device="cuda") / rows
        state["d_log_prob"], state["d_entropy"] = -weight, -0.01 * weight
    return state


# ------------------------------------------------------------------------------------------------ the operators
def run(state):
    if own:
        return run_own(state)
    if state["op"] == "log_probs":
        return plain_log_probs(state)
    if state["op"] == "orthogonalize":
        return [plain_orthogonalize(x.float()).to(x.dtype) for x in state["grads"]]
    for w, b, d in zip(state["w"], state["m"], state["grads"]):
        d = d.float()
        b.mul_(MOMENTUM).add_(d)
        o = plain_orthogonalize(d + MOMENTUM * b)
        w.copy_(w.float() * (1 - LR * DECAY) - (LR * 0.2 * math.sqrt(max(w.shape))) * o)
    return [state["weights"], state["momenta"]]


def run_own(state):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "r3det-pytorch_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    if state["op"] == "orthogonalize":
        from r3det.ops.orthogonalize import orthogonalize
        return orthogonalize(state["grads"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    if state["op"] == "update":
        from r3det.ops.orthogonalize import orthogonal_update_
        orthogonal_update_(state["w"], state["grads"], state["m"], lr=LR, momentum=MOMENTUM, nesterov=True,
                           weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, scale="rms")
        return [state["weights"], state["momenta"]]
    from r3det.ops.log_probs import label_log_probs
    got = label_log_probs(state["logits"], state["labels"], top_k=state["top"], ignore_index=-100)
    out = dict(log_prob=got.log_prob, entropy=got.entropy)  # (log_prob: None without labels)
    if state["top"]:
        out.update(top_log_prob=got.top_log_prob, top_index=got.top_index)
    if state["grad"]:
        out["d_logits"], = torch.autograd.grad([got.log_prob, got.entropy], [state["logits"]],
                                               [state["d_log_prob"], state["d_entropy"]])
    return out


def plain_orthogonalize(x):
    tall = x.size(0) > x.size(1)
    x = x.t() if tall else x
    x = x / (x.norm() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        p = x @ x.t()
        p = b * p + c * (p @ p)
        x = a * x + p @ x
    return x.t() if tall else x


def plain_log_probs(state):
    """A row with no class left has the log probabilities -inf, the entropy 0 and no gradient."""
    raw, labels, top = state["logits"].detach().float(), state["labels"], state["top"]
    peak = raw.max(dim=1, keepdim=True).values
    peak = torch.where(peak == -math.inf, 0, peak)
    x = raw - peak
    e = x.exp()
    total = e.sum(dim=1, keepdim=True)
    log_total = total.log()
    p = e / torch.where(total == 0, 1, total)
    logp = torch.where(total == 0, -math.inf, x - log_total)
    terms = torch.where(p > 0, p * logp, 0)
    entropy = -terms.sum(dim=1)
    out = dict(log_prob=None, entropy=entropy)
    if labels is not None:
        counted = labels != -100
        at = torch.where(counted, labels, 0)[:, None]
        out["log_prob"] = torch.where(counted, logp.gather(1, at)[:, 0], 0)
    if top:
        # by value, the lowest index first among equals: both in one whole number, the value's bits in an order that sorts
        bits = (raw + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, -2 ** 31 - 1 - bits, bits)
        index = torch.arange(x.size(1), device=x.device)
        key = bits * 2 ** 32 + (2 ** 32 - 1 - index)
        best = key.topk(top, dim=1, sorted=True).values
        out["top_index"] = 2 ** 32 - 1 - best % 2 ** 32
        out["top_log_prob"] = logp.gather(1, out["top_index"])
    if state["grad"]:
        dl = torch.where(counted, state["d_log_prob"], 0)[:, None]
        dh = state["d_entropy"][:, None]
        d = -p * dl - dh * torch.where(p > 0, p * (logp + entropy[:, None]), 0)
        d.scatter_add_(1, at, dl)
        out["d_logits"] = torch.where(total == 0, 0, d).to(state["logits"].dtype)
    return out


# ------------------------------------------------------------------------------------------------ what a case needs
def work(case):
    size = {"fp32": 4, "fp16": 2, "bf16": 2}[case["dtype"]]
    if case["op"] == "log_probs":
        cells, rows = case["rows"] * case["classes"], case["rows"]
        n_bytes = cells * size + rows * (4 + 12 * case["labels"] + 12 * case["top"])
        if case["grad"]:
            n_bytes += cells * size + rows * 8
        return {"bytes": n_bytes, "flops": cells * (10 if case["grad"] else 5)}
    n_bytes = flops = 0
    for n, m in shapes_of(case):
        n, m = min(n, m), max(n, m)
        n_bytes += n * m * (2 * size if case["op"] == "orthogonalize" else 3 * size + 8)
        # a symmetric product has half its entries to compute: n n m for x x^t, n n n for its square, 2 n n m for the third
        flops += STEPS * (3 * n * n * m + n * n * n)
    return {"bytes": n_bytes, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "log_probs":
        z, y, k = s["logits"].detach().double(), s["labels"], case["top"]
        empty = (z == -math.inf).all(dim=1)
        q = torch.log_softmax(torch.where(empty[:, None], 0, z), dim=1)
        q[empty] = -math.inf
        w = q.exp()
        h = -torch.special.xlogy(w, w).sum(dim=1)
        out = dict(log_prob=None, entropy=h)
        if y is not None:
            used, row = y >= 0, torch.arange(len(y), device=y.device)
            out["log_prob"] = torch.where(used, q[row, y.clamp(min=0)], 0)
        if k:
            out.update(top_index=None, top_log_prob=q.sort(dim=1, descending=True).values[:, :k].contiguous())
        if case["grad"]:
            hot = s["d_log_prob"].double() * used
            slope = w * (torch.nan_to_num(q, neginf=0) + h[:, None])
            slope = -s["d_entropy"].double()[:, None] * slope - w * hot[:, None]
            slope[row, y.clamp(min=0)] += hot
            slope[empty] = 0
            out["d_logits"] = slope
        return out

    def orthogonal(x):
        wide = x if x.size(0) <= x.size(1) else x.t()
        wide = wide / (torch.sqrt((wide * wide).sum()) + EPS)
        a, b, c = COEFFICIENTS
        eye = torch.eye(wide.size(0), dtype=wide.dtype, device=wide.device)
        for _ in range(STEPS):
            gram = wide @ wide.t()
            wide = (a * eye + b * gram + c * gram @ gram) @ wide
        return wide if x.size(0) <= x.size(1) else wide.t()

    if case["op"] == "orthogonalize":
        return [orthogonal(x.double()).contiguous() for x in s["grads"]]
    ws, ms = [], []
    for w, b, d in zip(s["w"], s["m"], s["grads"]):
        b = MOMENTUM * b.double() + d.double()
        o = orthogonal(d.double() + MOMENTUM * b)
        ws.append((w.double() * (1 - LR * DECAY) - LR * 0.2 * math.sqrt(max(w.shape)) * o).reshape(-1))
        ms.append(b.reshape(-1))
    return [torch.cat(ws), torch.cat(ms)]

"""Cases of the operators of a training step over many classes: the classifier's softmax cross entropy taken in pieces of
the vocabulary, the orthogonalised update of weight matrices, and the optimiser step that applies it.

    linear_cross_entropy   loss of a linear classifier, [rows, features] x [classes, features], with its gradients, without
                           keeping the [rows, classes] logits; for evaluation the loss and the predicted class
    orthogonalize          Newton-Schulz iteration X <- a X + b (X X') X + c (X X')^2 X from X = G / |G|
    muon_step_             momentum, orthogonalisation and weight update of a list of matrices, in place

`run` computes them in their plain form, or, where `own` is true, through this repository's package.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
MOMENTUM, LR, WEIGHT_DECAY = 0.95, 0.02, 0.01
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# The matrices that a Mask R-CNN with a pyramid trains on a frozen backbone: lateral and output convolutions of four levels,
# the proposal head, the box head with 81 classes, the mask head; convolutions as [out, in * kh * kw].
HEADS = ([(256, 2048), (256, 1024), (256, 512), (256, 256)] + [(256, 2304)] * 4 + [(256, 2304), (3, 256), (12, 256)]
         + [(1024, 12544), (1024, 1024), (81, 1024), (324, 1024)] + [(256, 2304)] * 4 + [(256, 1024), (81, 256)])
# Matrices of odd sizes, one of a single row and one of a single column among them.
ODD = [(33, 65), (1, 129), (255, 77), (47, 47), (301, 1), (130, 517)]


def listed():
    return [
        # the box head's loss as the framework trains it: 2 images x 512 sampled RoIs, 1024 features, 81 classes
        {"name": "ce box head", "op": "ce", "train": True, "type": "fp32", "rows": 1024, "dim": 1024, "classes": 81, "ignored": 0.0},
        # the same head over a long-tailed list of classes; padded to a static number of RoIs
        {"name": "ce long tail", "op": "ce", "train": True, "type": "fp32", "rows": 1024, "dim": 1024, "classes": 1204, "ignored": 0.1},
        # odd sizes everywhere, a third of the rows padding that holds NaN
        {"name": "ce ragged", "op": "ce", "train": True, "type": "fp16", "rows": 777, "dim": 1001, "classes": 5003, "ignored": 0.33},
        # a language model's head in training
        {"name": "ce vocabulary", "op": "ce", "train": True, "type": "bf16", "rows": 8192, "dim": 4096, "classes": 50021, "ignored": 0.02},
        # evaluation of a few detections: latency alone
        {"name": "ce eval few", "op": "ce", "train": False, "type": "fp16", "rows": 7, "dim": 256, "classes": 81, "ignored": 0.0},
        # evaluation of a full image batch over a large list of classes
        {"name": "ce eval many", "op": "ce", "train": False, "type": "bf16", "rows": 2000, "dim": 1024, "classes": 21843, "ignored": 0.05},
        # one small projection
        {"name": "ns small", "op": "ns", "type": "fp32", "m": 64, "n": 256},
        # the box head's first layer, by far its largest matrix
        {"name": "ns first layer", "op": "ns", "type": "fp32", "m": 1024, "n": 12544},
        # a square layer
        {"name": "ns square", "op": "ns", "type": "fp32", "m": 2048, "n": 2048},
        # a tall matrix of odd sizes in 16 bits
        {"name": "ns tall odd", "op": "ns", "type": "bf16", "m": 5003, "n": 2001},
        # one optimiser step of everything trained on a frozen backbone
        {"name": "step heads", "op": "step", "type": "fp32", "mats": "heads"},
        # one optimiser step of small odd matrices in 16 bits
        {"name": "step odd", "op": "step", "type": "bf16", "mats": "odd"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "ns", "ns", "step"])
    if kind == "ce":
        while True:
            rows, dim, classes = _log(rng, 1, 8192), _log(rng, 16, 4096), _log(rng, 2, 50021)
            if rows * dim * classes <= 8192 * 4096 * 50021 // 8:
                break
        return {"op": "ce", "train": rng.random() < 0.7, "type": rng.choice(["fp32", "bf16", "fp16"]), "rows": rows,
                "dim": dim, "classes": classes, "ignored": rng.choice([0.0, 0.1, 0.5])}
    if kind == "ns":
        while True:
            m, n = _log(rng, 1, 12544), _log(rng, 1, 12544)
            if min(m, n) ** 2 * max(m, n) <= 1024 * 1024 * 12544:
                break
        return {"op": "ns", "type": rng.choice(["fp32", "bf16", "fp16"]), "m": m, "n": n}
    mats = []
    for _ in range(rng.randint(1, 8)):
        mats.append("%dx%d" % (_log(rng, 1, 1024), _log(rng, 1, 2304)))
    return {"op": "step", "type": rng.choice(["fp32", "bf16"]), "mats": ",".join(mats)}


def _shapes(case):
    named = {"heads": HEADS, "odd": ODD}
    if case["mats"] in named:
        return list(named[case["mats"]])
    return [tuple(int(v) for v in s.split("x")) for s in case["mats"].split(",")]


def _gradient(shape, gen, dev):
    """A gradient as training gives it: a few strong directions over a full-rank remainder."""
    m, n = shape
    rank = max(1, min(m, n) // 8)
    scale = torch.exp(-4.0 * torch.arange(rank, device=dev) / rank)
    strong = (torch.randn(m, rank, generator=gen, device=dev) * scale) @ torch.randn(rank, n, generator=gen, device=dev)
    return 1e-3 * (strong / math.sqrt(rank) + 0.7 * torch.randn(m, n, generator=gen, device=dev))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["type"]]
    if case["op"] == "ce":
        rows, dim, classes = case["rows"], case["dim"], case["classes"]
        weight = torch.randn(classes, dim, generator=gen, device=dev) / math.sqrt(dim)
        bias = 0.1 * torch.randn(classes, generator=gen, device=dev)
        labels = torch.randint(0, classes, (rows,), generator=gen, device=dev)
        # features after a ReLU, most rows leaning to their class as in a partly trained head
        lean = 6.0 * torch.rand(rows, 1, generator=gen, device=dev)
        x = torch.relu(torch.randn(rows, dim, generator=gen, device=dev)) + lean * weight[labels]
        padding = torch.rand(rows, generator=gen, device=dev) < case["ignored"]
        labels = torch.where(padding, torch.full_like(labels, -1), labels)
        x = torch.where(padding[:, None], torch.full_like(x, float("nan")), x)
        state = {"x": x.to(dt), "weight": weight.to(dt), "bias": bias.to(dt), "labels": labels}
        if case["train"]:
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_(True)
        return dict(state, op="ce", train=case["train"])
    if case["op"] == "ns":
        return {"op": "ns", "g": _gradient((case["m"], case["n"]), gen, dev).to(dt)}
    shapes = _shapes(case)
    return {"op": "step", "params": [(0.02 * torch.randn(s, generator=gen, device=dev)).to(dt) for s in shapes],
            "grads": [_gradient(s, gen, dev).to(dt) for s in shapes],
            "momenta": [5.0 * _gradient(s, gen, dev) for s in shapes]}


def _plain_ce(x, weight, bias, labels, train):
    real = labels >= 0
    xf = torch.where(real[:, None], x.detach(), torch.zeros_like(x.detach())).float()
    wf = weight.detach().float()
    logits = xf @ wf.t() + bias.detach().float()
    top = logits.max(dim=1, keepdim=True)[0]
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    index = labels.clamp_min(0)[:, None]
    losses = (torch.log(total) + top - logits.gather(1, index))[:, 0]
    count = real.sum().clamp_min(1).float()
    loss = torch.where(real, losses, torch.zeros_like(losses)).sum() / count
    if not train:
        places = torch.where(logits == top, torch.arange(logits.size(1), device=logits.device), logits.size(1))
        return loss, torch.where(real, places.min(dim=1)[0], -1)
    p = e / total
    p.scatter_add_(1, index, torch.full_like(index, -1, dtype=p.dtype))
    p = torch.where(real[:, None], p, torch.zeros_like(p)) / count
    return loss, (p @ wf).to(x.dtype), (p.t() @ xf).to(weight.dtype), p.sum(dim=0).to(bias.dtype)


def _plain_ns(g):
    """In float32; the caller rounds."""
    a, b, c = COEFFICIENTS
    x = g.float() if g.size(0) <= g.size(1) else g.float().t()
    norm = torch.sqrt((x.double() * x.double()).sum()).clamp_min(EPS)
    x = (x.double() / norm).float()
    for _ in range(STEPS):
        xxt = x @ x.t()
        x = a * x + (b * xxt + c * (xxt @ xxt)) @ x
    return x if g.size(0) <= g.size(1) else x.t()


def run(state):
    if state["op"] == "ce":
        x, weight, bias, labels, train = (state[k] for k in ("x", "weight", "bias", "labels", "train"))
        if own:
            from detectron_pytorch_amd.linear_cross_entropy import linear_cross_entropy

            if not train:
                return linear_cross_entropy(x, weight, bias, labels, ignore_index=-1, with_pred=True)
            loss = linear_cross_entropy(x, weight, bias, labels, ignore_index=-1)
            return (loss.detach(),) + torch.autograd.grad(loss, (x, weight, bias))
        return _plain_ce(x, weight, bias, labels, train)
    if state["op"] == "ns":
        if own:
            from detectron_pytorch_amd.orthogonalize import orthogonalize

            return orthogonalize(state["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        return _plain_ns(state["g"]).to(state["g"].dtype).contiguous()
    params, grads, momenta = state["params"], state["grads"], state["momenta"]
    if own:
        from detectron_pytorch_amd.muon import muon_step_

        muon_step_(params, grads, momenta, lr=LR, momentum=MOMENTUM, weight_decay=WEIGHT_DECAY, nesterov=True, steps=STEPS,
                   coefficients=COEFFICIENTS, eps=EPS)
        return params, momenta
    for p, g, buf in zip(params, grads, momenta):
        buf.copy_(MOMENTUM * buf + g.float())
        update = _plain_ns(g.float() + MOMENTUM * buf)
        scale = math.sqrt(max(1.0, p.size(0) / p.size(1)))
        p.copy_(p.float() * (1.0 - LR * WEIGHT_DECAY) - LR * scale * update)
    return params, momenta


def _ns_flops(m, n):
    """X X' and the polynomial's products are symmetric: half of each counts.  Two steps of the iteration can share one pass
    over the long side (products of the small side's matrices take the place of X's): the cheaper of the two counts."""
    m, n = min(m, n), max(m, n)
    one = 3.0 * m * m * n
    return min(STEPS * (one + m ** 3), 3 * one + (STEPS + 8) * float(m) ** 3)


def work(case):
    if case["op"] == "ce":
        size = 4 if case["type"] == "fp32" else 2
        r, d, v = case["rows"], case["dim"], case["classes"]
        inputs = (r * d + v * d + v) * size
        if case["train"]:
            return {"bytes": 2 * inputs + 8 * r + 4, "flops": 6.0 * r * d * v}
        return {"bytes": inputs + 16 * r + 4, "flops": 2.0 * r * d * v}
    if case["op"] == "ns":
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": 2.0 * case["m"] * case["n"] * size, "flops": _ns_flops(case["m"], case["n"])}
    size = 4 if case["type"] == "fp32" else 2
    shapes = _shapes(case)
    return {"bytes": float(sum(m * n * (3 * size + 8) for m, n in shapes)), "flops": sum(_ns_flops(m, n) for m, n in shapes)}


def _exact_ns(g):
    """The iteration as a polynomial in G G' that is applied once: p(X) = Q X with Q = product of (a + b A_k + c A_k A_k)."""
    a, b, c = COEFFICIENTS
    tall = g.size(0) > g.size(1)
    x = (g.t() if tall else g).double()
    x = x / torch.linalg.matrix_norm(x).clamp_min(EPS)
    eye = torch.eye(x.size(0), dtype=torch.float64, device=x.device)
    gram, q = x @ x.t(), eye
    for _ in range(STEPS):
        factor = a * eye + gram @ (b * eye + c * gram)
        q, gram = factor @ q, factor @ gram @ factor
    out = q @ x
    return out.t() if tall else out


def exact(case, seed):
    state = prepare(case, seed)
    if state["op"] == "ce":
        labels = state["labels"]
        keep = torch.nonzero(labels >= 0)[:, 0]
        leaves = [state["x"].detach()[keep].double(), state["weight"].detach().double(), state["bias"].detach().double()]
        grads = [torch.zeros(state[k].shape, dtype=torch.float64, device=labels.device) for k in ("x", "weight", "bias")]
        loss = torch.zeros((), dtype=torch.float64, device=labels.device)
        pred = torch.full_like(labels, -1)
        for at in range(0, keep.numel(), 1024):                       # rows in parts: the logits of all of them are large
            rows = keep[at:at + 1024]
            x = leaves[0][at:at + 1024]
            logits = torch.addmm(leaves[2], x, leaves[1].t())
            log_p = logits - torch.logsumexp(logits, dim=1, keepdim=True)
            loss -= log_p[torch.arange(rows.numel(), device=rows.device), labels[rows]].sum()
            pred[rows] = logits.argmax(dim=1)
            d = log_p.exp()
            d[torch.arange(rows.numel(), device=rows.device), labels[rows]] -= 1.0
            d /= keep.numel()
            if state["train"]:
                grads[0][rows] = d @ leaves[1]
                grads[1] += d.t() @ x
                grads[2] += d.sum(dim=0)
        loss = loss / max(1, keep.numel())
        return (loss, *grads) if state["train"] else (loss, pred)
    if state["op"] == "ns":
        return _exact_ns(state["g"])
    params, momenta = [], []
    for p, g, buf in zip(state["params"], state["grads"], state["momenta"]):
        buf = MOMENTUM * buf.double() + g.double()
        scale = math.sqrt(max(1.0, p.size(0) / p.size(1)))
        params.append((1.0 - LR * WEIGHT_DECAY) * p.double() - LR * scale * _exact_ns(g.double() + MOMENTUM * buf))
        momenta.append(buf)
    return params, momenta

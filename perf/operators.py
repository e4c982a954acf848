"""What the operators at the end of a training step cost, and what they should return.

Four operators of the library, each in a plain form made of elementary torch operations (``own = False``) and as a
user's program calls it (``own = True``):

xent    the cross entropy of every token's softmax over a large vocabulary, straight from the hidden states X and the
        classifier W, without the logits:  z = alpha X W^T,  lse = log sum exp z,  loss = lse - z[label]
grad    its gradients with respect to X and W, given those of loss and lse:
        P = gloss (softmax - onehot) + glse softmax,  gX = alpha P W,  gW = alpha P^T X
norm    the Euclidean norm of a group of tensors taken as one vector
clip    that norm and the group scaled down to a largest norm

Rows whose label is ``IGNORE`` have no target: loss, lse and gradients of such a row are zero.
"""
import math
import random

import torch

own = False

IGNORE = -100
TYPES = {"b": torch.bfloat16, "s": torch.float32}


def listed():
    return [
        # one generated token scored by the classifier: the classifier is read once, the latency of a decode step
        {"name": "xent-one-token", "op": "xent", "type": "b", "tokens": 1, "hidden": 4096, "vocab": 65536,
         "masked": 0.0, "pad": 0, "alpha": 1.0},
        # evaluation in single precision, odd sizes, rows that start anywhere, prompts without a target
        {"name": "xent-single-odd", "op": "xent", "type": "s", "tokens": 333, "hidden": 1000, "vocab": 20011,
         "masked": 0.25, "pad": 3, "alpha": 0.5},
        # an ordinary micro-batch
        {"name": "xent-ordinary", "op": "xent", "type": "b", "tokens": 2048, "hidden": 2048, "vocab": 32768,
         "masked": 0.0, "pad": 0, "alpha": 1.0},
        # a large micro-batch against a large vocabulary, a third of the tokens prompts
        {"name": "xent-large", "op": "xent", "type": "b", "tokens": 8192, "hidden": 4096, "vocab": 131072,
         "masked": 0.3, "pad": 0, "alpha": 1.0},
        # a handful of tokens with odd sizes and rows off alignment (a step on single answers)
        {"name": "grad-few-odd", "op": "grad", "type": "b", "tokens": 5, "hidden": 1001, "vocab": 30001,
         "masked": 0.0, "pad": 2, "alpha": 1.0, "glse": False},
        # single precision training
        {"name": "grad-single", "op": "grad", "type": "s", "tokens": 1024, "hidden": 1024, "vocab": 32000,
         "masked": 0.0, "pad": 0, "alpha": 1.0, "glse": False},
        # an ordinary micro-batch, half of it prompts, with a penalty on lse
        {"name": "grad-ordinary", "op": "grad", "type": "b", "tokens": 2048, "hidden": 2048, "vocab": 32768,
         "masked": 0.5, "pad": 0, "alpha": 1.0, "glse": True},
        # the large micro-batch, every token a target
        {"name": "grad-large", "op": "grad", "type": "b", "tokens": 8192, "hidden": 4096, "vocab": 131072,
         "masked": 0.0, "pad": 0, "alpha": 1.0, "glse": False},
        # the gradients of a small adapter: latency
        {"name": "norm-small", "op": "norm", "type": "s", "count": 12, "total": 1000003, "flat": False},
        # all gradients of a model of a billion parameters, views of flat buckets (tensors start anywhere)
        {"name": "norm-large", "op": "norm", "type": "b", "count": 200, "total": 1000000007, "flat": True},
        # small tensors of both types
        {"name": "clip-small", "op": "clip", "type": "mixed", "count": 30, "total": 500009, "flat": True,
         "max_norm": 1.0},
        # the gradients of a larger model, both types, tensors of their own
        {"name": "clip-large", "op": "clip", "type": "mixed", "count": 60, "total": 400000009, "flat": False,
         "max_norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["xent", "grad", "xent", "grad", "norm", "clip"])
    if op in ("norm", "clip"):
        total = _log_int(rng, 1000, 1000000000 if op == "norm" else 400000000)
        case = {"op": op, "type": rng.choice(["s", "b", "mixed"]), "count": _log_int(rng, 1, min(400, total // 4)),
                "total": total, "flat": rng.random() < 0.5}
        if case["type"] != "b":
            case["total"] = min(total, 400000000)
        if op == "clip":
            case["max_norm"] = rng.choice([0.5, 1.0, 1e6])
            if not case["flat"]:
                case["count"] = min(case["count"], 60)
        return case
    while True:
        tokens, hidden, vocab = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), _log_int(rng, 1000, 131072)
        if rng.random() < 0.5:                     # half the draws have the round sizes of a model
            hidden = max(64, hidden // 64 * 64)
        if tokens * hidden * vocab <= 8192 * 4096 * 131072 // 2:
            break
    case = {"op": op, "type": rng.choice(["b", "b", "s"]), "tokens": tokens, "hidden": hidden, "vocab": vocab,
            "masked": rng.choice([0.0, 0.0, 0.2, 0.6, 0.95]), "pad": rng.choice([0, 0, 1, 8]),
            "alpha": rng.choice([1.0, 0.7])}
    if op == "grad":
        case["glse"] = rng.random() < 0.5
    return case


def _targets(case):
    """Which rows have a target: sequences of 512 tokens, the first share of each of them a prompt."""
    at = torch.arange(case["tokens"])
    length = min(512, case["tokens"])
    return (at % length) >= min(length - 1, int(round(case["masked"] * length)))


def _sizes(case):
    """The lengths of the group's tensors: a few large ones, many small ones, the given total."""
    rng = random.Random(case["count"] * 1000003 + case["total"])
    weight = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(case["count"])]
    scale = (case["total"] - case["count"]) / sum(weight)
    sizes = [1 + int(w * scale) for w in weight]
    sizes[-1] += case["total"] - sum(sizes)
    return sizes


def _group_types(case):
    return ["sb"[i % 2] if case["type"] == "mixed" else case["type"] for i in range(case["count"])]


def _space(case):
    """Memory for the group: its tensors, and the buffers that they are views of (the tensors themselves where they
    stand alone; with flat buffers, one per type, in which they follow each other without gaps)."""
    sizes, types = _sizes(case), _group_types(case)
    if not case["flat"]:
        out = [torch.empty(n, dtype=TYPES[t], device="cuda") for n, t in zip(sizes, types)]
        return out, out
    out, flat = [None] * len(sizes), []
    for t in sorted(set(types)):
        mine = [i for i, u in enumerate(types) if u == t]
        flat.append(torch.empty(sum(sizes[i] for i in mine), dtype=TYPES[t], device="cuda"))
        for i, part in zip(mine, flat[-1].split([sizes[i] for i in mine])):
            out[i] = part
    return out, flat


def _group(case, seed):
    """Gradients: normal values whose scale differs from tensor to tensor."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    group, _ = _space(case)
    for i, x in enumerate(group):
        x.normal_(0.0, 10.0 ** -(1 + i % 3), generator=gen)
    return group


def _rows(rows, cols, pad, dtype, gen, scale):
    """A rows x cols window whose rows are cols + pad elements apart."""
    x = torch.empty(rows, cols + pad, dtype=dtype, device="cuda")
    x.normal_(0.0, scale, generator=gen)
    return x[:, :cols]


def _tokens_and_classifier(case, seed):
    """Normalised hidden states that lean towards their label's row of the classifier, as a trained model's do."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, h, v, dt = case["tokens"], case["hidden"], case["vocab"], TYPES[case["type"]]
    W = _rows(v, h, case["pad"], dt, gen, 2.0 / math.sqrt(h))
    X = _rows(t, h, case["pad"], dt, gen, 1.0)
    label = torch.randint(0, v, (t,), generator=gen, device="cuda", dtype=torch.int32)
    X += (1.5 * W[label.long()].float()).to(dt)
    label[~_targets(case).cuda()] = IGNORE
    return W, X, label, gen


def _gradients_in(case, gen, label):
    n = max(1, int(_targets(case).sum()))
    t = case["tokens"]
    gloss = torch.full((t,), 1.0 / n, device="cuda") * (0.5 + torch.rand(t, generator=gen, device="cuda"))
    glse = 1e-3 / n * torch.randn(t, generator=gen, device="cuda") if case["glse"] else None
    return gloss, glse


def prepare(case, seed):
    if case["op"] in ("norm", "clip"):
        group = _group(case, seed)
        state = {"case": case, "group": group}
        if own:
            from ulmblas_amd import blas
            state["handle"] = blas.TensorGroup(group)
            state["work"] = torch.empty(blas.gnrm2_worksize(state["handle"]), dtype=torch.uint8, device="cuda")
            state["norm"] = torch.empty(1, device="cuda")
        if case["op"] == "clip":
            out, state["flat"] = _space(case)
            state["out"] = blas.TensorGroup(out) if own else out
        return state
    W, X, label, gen = _tokens_and_classifier(case, seed)
    state = {"case": case, "W": W, "X": X, "label": label}
    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    if case["op"] == "grad":
        state["gloss"], state["glse"] = _gradients_in(case, gen, label)
        state["lse"] = _plain_xent(W, X, label, case["alpha"])[1]
    if own:
        from ulmblas_amd import blas
        if case["op"] == "xent":
            state["loss"], state["lse"] = torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
            size = blas.xent_worksize(case["type"], h, t, v)
        else:
            state["gW"] = torch.empty(v, h, dtype=W.dtype, device="cuda")
            state["gX"] = torch.empty(t, h, dtype=W.dtype, device="cuda")
            size = blas.xent_grad_worksize(case["type"], h, t, v)
        state["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return state


def _plain_xent(W, X, label, alpha):
    z = X.float() @ W.float().T
    z *= alpha
    top = z.max(dim=1, keepdim=True).values
    target = z.gather(1, label.long().clamp(min=0).unsqueeze(1)).squeeze(1)
    z -= top
    lse = z.exp_().sum(dim=1).log() + top.squeeze(1)
    has = label >= 0
    return torch.where(has, lse - target, 0.0), torch.where(has, lse, 0.0)


def _plain_grad(W, X, label, lse, gloss, glse, alpha):
    w, x = W.float(), X.float()
    P = x @ w.T
    P *= alpha
    P -= lse.unsqueeze(1)
    P.exp_()
    has = label >= 0
    P *= (gloss if glse is None else gloss + glse).unsqueeze(1)
    rows = torch.arange(label.numel(), device=label.device)
    P[rows, label.long().clamp(min=0)] -= gloss
    P *= torch.where(has, alpha, 0.0).unsqueeze(1)
    return (P.T @ x).to(W.dtype), (P @ w).to(X.dtype)


def _plain_norm(group):
    return torch.stack([x.float().square().sum(dtype=torch.float64) for x in group]).sum().sqrt().float().reshape(1)


def _plain_clip(group, norm, max_norm, out):
    factor = torch.where(norm > max_norm, max_norm / norm, torch.ones_like(norm))
    for x, y in zip(group, out):
        y.copy_(x.float() * factor)


def run(state):
    case = state["case"]
    if case["op"] in ("norm", "clip"):
        if not own:
            norm = _plain_norm(state["group"])
            if case["op"] == "norm":
                return {"norm": norm}
            _plain_clip(state["group"], norm, case["max_norm"], state["out"])
            return {"norm": norm, "out": state["flat"]}
        from ulmblas_amd import blas
        norm = blas.gpu_gnrm2(state["handle"], state["norm"], work=state["work"])
        if case["op"] == "norm":
            return {"norm": norm}
        blas.gpu_gclip(state["handle"], norm, case["max_norm"], out=state["out"])
        return {"norm": norm, "out": state["flat"]}
    W, X, label, alpha = state["W"], state["X"], state["label"], case["alpha"]
    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    if case["op"] == "xent":
        if not own:
            loss, lse = _plain_xent(W, X, label, alpha)
        else:
            from ulmblas_amd import blas
            loss, lse = blas.gpu_xent(case["type"], h, t, v, alpha, W, W.stride(0), X, X.stride(0), label, IGNORE,
                                      state["loss"], state["lse"], work=state["work"])
        return {"loss": loss, "lse": lse}
    if not own:
        gW, gX = _plain_grad(W, X, label, state["lse"], state["gloss"], state["glse"], alpha)
    else:
        from ulmblas_amd import blas
        gW, gX = blas.gpu_xent_grad(case["type"], h, t, v, alpha, W, W.stride(0), X, X.stride(0), label, IGNORE,
                                    state["lse"], state["gloss"], state["glse"], 0.0, state["gW"], h, state["gX"], h,
                                    work=state["work"])
    return {"gW": gW, "gX": gX}


def work(case):
    if case["op"] in ("norm", "clip"):
        size = {"s": 4, "b": 2}
        read = sum(n * size[t] for n, t in zip(_sizes(case), _group_types(case)))
        # the clipped group is the group read and written; the norm needs one more reading, since the factor
        # depends on every element
        return {"bytes": read + 4 if case["op"] == "norm" else 3 * read + 4,
                "flops": (2 if case["op"] == "norm" else 3) * case["total"]}
    size = 2 if case["type"] == "b" else 4
    t, h, v, n = case["tokens"], case["hidden"], case["vocab"], int(_targets(case).sum())
    operands = size * h * (v + n) + 4 * t
    product = 2 * n * h * v
    if case["op"] == "xent":
        return {"bytes": operands + 8 * t, "flops": product}
    return {"bytes": operands + 4 * t * (3 if case["glse"] else 2) + size * h * (v + t), "flops": 3 * product}


def exact(case, seed):
    if case["op"] in ("norm", "clip"):
        group = _group(case, seed)
        squares = 0.0
        for x in group:
            for part in x.split(1 << 26):
                d = part.double()
                squares += float(torch.dot(d, d))
        norm = math.sqrt(squares)
        out = {"norm": torch.tensor([norm], dtype=torch.float64, device="cuda")}
        if case["op"] == "clip":
            # the factor goes by the norm as it is handed over, in single precision
            handed = float(out["norm"].float())
            scaled = [x.double() * min(1.0, case["max_norm"] / handed) for x in group]
            if case["flat"]:
                types = _group_types(case)
                scaled = [torch.cat([x for x, u in zip(scaled, types) if u == t]) for t in sorted(set(types))]
            out["out"] = scaled
        return out
    W, X, label, gen = _tokens_and_classifier(case, seed)
    alpha, t = case["alpha"], case["tokens"]
    if case["op"] == "grad":
        gloss, glse = _gradients_in(case, gen, label)
        lse_in = _plain_xent(W, X, label, alpha)[1].double()
        gW = torch.zeros(W.shape, dtype=torch.float64, device="cuda")
        gX = torch.zeros(X.shape, dtype=torch.float64, device="cuda")
    w = W.double()
    loss = torch.zeros(t, dtype=torch.float64, device="cuda")
    lse = torch.zeros(t, dtype=torch.float64, device="cuda")
    targets = torch.nonzero(label != IGNORE).flatten()
    for rows in targets.split(1024):
        x, y = X[rows].double(), label[rows].long()
        z = alpha * torch.mm(x, w.t())
        here = torch.arange(rows.numel(), device="cuda")
        if case["op"] == "xent":
            l = torch.logsumexp(z, 1)
            lse[rows], loss[rows] = l, l - z[here, y]
            continue
        g = gloss[rows].double()
        both = g if glse is None else g + glse[rows].double()
        soft = torch.exp(z - lse_in[rows, None]) * both[:, None]
        soft[here, y] -= g
        gX[rows] = alpha * torch.mm(soft, w)
        gW.addmm_(soft.t(), x, alpha=alpha)
    return {"loss": loss, "lse": lse} if case["op"] == "xent" else {"gW": gW, "gX": gX}

"""The learner step's table and matrix operators, as they are called, with their plain forms.

Four kinds of case:

- ``embed``: rows of a table by index, times a scale (``pbg_b200.embedding.embedding``);
- ``embed_grad``: its gradient, the scaled sum of the incoming rows of each index
  (``pbg_b200.embedding.embedding_backward``), into a fresh table or added to the table's slice of a
  gradient that other parts of the step have written already;
- ``ortho``: a stack of matrices orthogonalised by five quintic Newton-Schulz steps
  (``pbg_b200.optim.orthogonalize``);
- ``muon``: one transition of an optimizer that orthogonalises the momentum of every matrix of a flat
  fp32 master (``pbg_b200.optim.FlatMuon``).

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits; with ``own`` true it
makes the framework's calls.
"""

import functools
import math
import os
import random
import sys

import torch

own = False

STEPS = 5
A, B, C = 3.4445, -4.7750, 2.0315
EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# Every matrix (count x rows x columns) of the queued policy/value network at d 128 with 2 layers, and at
# the default configuration's d 256 with 6 layers.
NETWORK_128 = ("12x128x128 10x128x512 4x512x512 3x512x928 2x384x128 2x512x88 2x512x407 2x512x131 1x128x6 1x3x128 "
               "1x6x128 1x128x90 1x128x248 1x128x52 1x128x32 1x512x96 1x32x512 1x512x9")
NETWORK_256 = ("36x256x256 14x256x1024 7x1024x1024 6x768x256 6x1024x88 6x1024x663 3x1024x2336 2x1024x259 1x256x6 "
               "1x3x256 1x12x256 1x1024x2816 1x256x90 1x256x376 1x256x52 1x256x32 1x1024x96 1x32x1024 1x1024x9")


def listed():
    return [
        # a serving step of a few rows: sixteen tokens of a bf16 vocabulary
        {"name": "embed_few", "op": "embed", "tokens": 16, "rows": 65536, "width": 1024, "type": "bf16", "out": "bf16",
         "scale": 32.0, "law": "uniform"},
        # the 64 history tokens of 1,280 decisions looking up the 13 public token types at d 128
        {"name": "embed_history", "op": "embed", "tokens": 81920, "rows": 13, "width": 128, "type": "f32", "out": "f32",
         "scale": 1.0, "law": "uniform"},
        # a training batch of long sequences over a large vocabulary, rows scaled by sqrt(width)
        {"name": "embed_vocabulary", "op": "embed", "tokens": 65536, "rows": 131072, "width": 2048, "type": "bf16",
         "out": "bf16", "scale": 45.254834, "law": "zipf"},
        # the 169 preflop class rows of width 32 over a small minibatch
        {"name": "grad_classes", "op": "embed_grad", "tokens": 512, "rows": 169, "width": 32, "type": "f32", "out": "f32",
         "scale": 1.0, "law": "uniform", "add": False},
        # the history tokens' gradient: 81,920 rows into 13, added into the flat gradient
        {"name": "grad_history", "op": "embed_grad", "tokens": 81920, "rows": 13, "width": 128, "type": "f32",
         "out": "f32", "scale": 1.0, "law": "uniform", "add": True},
        # one row of four (the streets) for every token of a large batch, an odd count
        {"name": "grad_streets", "op": "embed_grad", "tokens": 1000003, "rows": 4, "width": 128, "type": "bf16",
         "out": "f32", "scale": 1.0, "law": "uniform", "add": False},
        # a vocabulary's gradient with natural repeats, an odd number of rows
        {"name": "grad_vocabulary", "op": "embed_grad", "tokens": 65536, "rows": 50021, "width": 1024, "type": "bf16",
         "out": "f32", "scale": 32.0, "law": "zipf", "add": False},
        # one attention in-projection of the d 128 network
        {"name": "ortho_qkv", "op": "ortho", "batch": 1, "rows": 384, "cols": 128, "type": "f32", "out": "f32"},
        # a stack of feed-forward maps of the d 256 network
        {"name": "ortho_ffn", "op": "ortho", "batch": 14, "rows": 256, "cols": 1024, "type": "f32", "out": "f32"},
        # one wide matrix of a large model, bf16 in and out
        {"name": "ortho_large", "op": "ortho", "batch": 1, "rows": 4096, "cols": 4096, "type": "bf16", "out": "bf16"},
        # the whole optimizer step of the d 128 and of the d 256 network
        {"name": "muon_network_128", "op": "muon", "matrices": NETWORK_128, "nesterov": True, "adjust": "shape"},
        {"name": "muon_network_256", "op": "muon", "matrices": NETWORK_256, "nesterov": True, "adjust": "rms"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random):
    op = rng.choice(("embed", "embed_grad", "ortho", "muon"))
    if op in ("embed", "embed_grad"):
        width = _log(rng, 1, 4096)
        if rng.random() < 0.5:
            width = max(8, width // 8 * 8)
        case = {"op": op, "tokens": _log(rng, 1, min(1 << 20, (1 << 27) // width)),
                "rows": _log(rng, 2, min(1 << 17, (1 << 27) // width)), "width": width, "type": rng.choice(tuple(TYPES)),
                "scale": rng.choice((1.0, math.sqrt(width), 0.125)), "law": rng.choice(("uniform", "zipf"))}
        case["out"] = rng.choice((case["type"], "f32"))
        if op == "embed_grad":
            case["add"] = rng.random() < 0.5
        return case
    while True:
        if op == "ortho":
            case = {"op": op, "batch": _log(rng, 1, 16), "rows": _log(rng, 1, 4096), "cols": _log(rng, 1, 4096),
                    "type": rng.choice(tuple(TYPES)), "out": rng.choice(("bf16", "f32"))}
            if case["out"] == "f32" and min(case["rows"], case["cols"]) > 1024:
                continue
        else:
            case = {"op": op, "matrices": " ".join("%dx%dx%d" % (_log(rng, 1, 12), _log(rng, 2, 2816), _log(rng, 2, 2816))
                                                   for _ in range(rng.randint(1, 5))),
                    "nesterov": rng.random() < 0.7, "adjust": rng.choice(("shape", "rms"))}
        w = work(case)
        if w["flops"] <= 4.0e11 and w["bytes"] <= 1.2e9:
            return case


def _groups(case):
    return [tuple(int(v) for v in g.split("x")) for g in case["matrices"].split()]


def _index(case, gen):
    u = torch.rand(case["tokens"], generator=gen, device="cuda", dtype=torch.float64)
    rows = case["rows"]
    if case["law"] == "uniform":
        return (u * rows).long().clamp_(0, rows - 1)
    rank = torch.exp(u * math.log(rows + 1)).long().sub_(1).clamp_(0, rows - 1)  # p(rank) falls as 1 / rank
    return (rank * 7919) % rows  # frequent rows spread over the table


def _matrix(gen, count, rows, cols, noise=0.2):
    """Gradients as matrices have them: a low-rank part and noise."""
    r = max(1, min(rows, cols) // 8)
    low = torch.randn(count, rows, r, generator=gen, device="cuda") @ torch.randn(count, r, cols, generator=gen, device="cuda")
    return (low / math.sqrt(r) + noise * torch.randn(count, rows, cols, generator=gen, device="cuda")) * 1e-3


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case)
    if op == "embed":
        state["table"] = torch.randn(case["rows"], case["width"], generator=gen, device="cuda").to(TYPES[case["type"]])
        state["index"] = _index(case, gen)
    elif op == "embed_grad":
        state["grad"] = torch.randn(case["tokens"], case["width"], generator=gen, device="cuda").to(TYPES[case["type"]])
        state["index"] = _index(case, gen)
        if case["add"]:
            state["into"] = torch.randn(case["rows"], case["width"], generator=gen, device="cuda").to(TYPES[case["out"]])
    elif op == "ortho":
        state["x"] = _matrix(gen, case["batch"], case["rows"], case["cols"]).to(TYPES[case["type"]])
    else:
        groups = _groups(case)
        spans, at = [], 0
        for count, rows, cols in groups:
            spans.append((at, count, rows, cols))
            at += count * rows * cols
        state["spans"] = spans
        state["master"] = torch.cat([torch.randn(n * r * c, generator=gen, device="cuda") / math.sqrt(c) for n, r, c in groups])
        state["grad"] = torch.cat([_matrix(gen, n, r, c).reshape(-1) for n, r, c in groups])
        state["momentum"] = torch.cat([0.3 * _matrix(gen, n, r, c).reshape(-1) for n, r, c in groups])
        if own:  # the optimizer object that a program makes once
            state["step"] = _muon(state)
    if own:
        _package()
    return state


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ai-game-learning_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from pbg_b200 import embedding, optim

    return embedding, optim


def _muon(state):
    _, optim = _package()
    step = optim.FlatMuon(state["master"], [(at + i * r * c, r, c) for at, n, r, c in state["spans"] for i in range(n)],
                          lr=LR, momentum=MOMENTUM, decay=DECAY, nesterov=state["nesterov"], adjust=state["adjust"],
                          steps=STEPS, coefficients=(A, B, C), epsilon=EPS)
    step.grad.copy_(state["grad"])
    step.momentum.copy_(state["momentum"])
    return step


def _newton_schulz(x):
    """Five steps of x <- a x + (b G + c G^2) x with G = x x^T, from x over its norm; [batch, rows, cols] fp32."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + EPS)

    def step(x, _):
        g = x @ x.mT
        return A * x + (B * g + C * (g @ g)) @ x

    x = functools.reduce(step, range(STEPS), x)
    return x.mT if tall else x


def _adjust(rule, rows, cols):
    return math.sqrt(max(1.0, rows / cols)) if rule == "shape" else 0.2 * math.sqrt(max(rows, cols))


def _plain_muon(s):
    def group(at, count, rows, cols):
        span = slice(at, at + count * rows * cols)
        g, m, w = (s[k][span].view(count, rows, cols) for k in ("grad", "momentum", "master"))
        m.mul_(MOMENTUM).add_((1.0 - MOMENTUM) * g)
        u = MOMENTUM * m + (1.0 - MOMENTUM) * g if s["nesterov"] else m
        w.mul_(1.0 - LR * DECAY).sub_(LR * _adjust(s["adjust"], rows, cols) * _newton_schulz(u))

    [group(*span) for span in s["spans"]]
    return {"master": s["master"], "momentum": s["momentum"]}


def run(s):
    op = s["op"]
    if own:
        embedding, optim = _package()
        if op == "embed":
            return embedding.embedding(s["table"], s["index"], s["scale"], out_dtype=TYPES[s["out"]])
        if op == "embed_grad":
            if s["add"]:
                return embedding.embedding_backward(s["grad"], s["index"], s["rows"], s["scale"], out=s["into"],
                                                    accumulate=True)
            return embedding.embedding_backward(s["grad"], s["index"], s["rows"], s["scale"], out_dtype=TYPES[s["out"]])
        if op == "ortho":
            return optim.orthogonalize(s["x"], steps=STEPS, coefficients=(A, B, C), epsilon=EPS, out_dtype=TYPES[s["out"]])
        s["step"].step()
        return {"master": s["step"].master, "momentum": s["step"].momentum}
    if op == "embed":
        return (s["table"][s["index"]].float() * s["scale"]).to(TYPES[s["out"]])
    if op == "embed_grad":
        # sums of many rows lose what matters in 32 bits: 64 where a row collects 64 or more on average
        wide = torch.float64 if s["tokens"] >= 64 * s["rows"] else torch.float32
        sums = torch.zeros(s["rows"], s["width"], dtype=wide, device="cuda").index_add_(0, s["index"], s["grad"].to(wide))
        if s["add"]:
            return s["into"].copy_((s["into"].to(wide) + s["scale"] * sums).to(s["into"].dtype))
        return (s["scale"] * sums).to(TYPES[s["out"]])
    if op == "ortho":
        return _newton_schulz(s["x"].float()).to(TYPES[s["out"]])
    return _plain_muon(s)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        return s["table"].double().index_select(0, s["index"]).mul_(case["scale"])
    if op == "embed_grad":
        order = torch.argsort(s["index"], stable=True)
        counts = torch.bincount(s["index"], minlength=case["rows"])
        parts = []
        for a in range(0, case["width"], 64):  # a few columns at a time: the sorted rows in 64 bits
            g = s["grad"][:, a:a + 64][order].double()
            parts.append(torch.segment_reduce(g, "sum", lengths=counts, axis=0, unsafe=True))
        sums = torch.cat(parts, 1) * case["scale"]
        return s["into"].double() + sums if case["add"] else sums

    def polynomial(x):
        x = x.double()
        x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS)
        flip = x.shape[-1] < x.shape[-2]
        for _ in range(STEPS):  # odd powers of x, each from the last
            left = (lambda y: x @ (x.mT @ y)) if flip else (lambda y: (x @ x.mT) @ y)
            cube = left(x)
            x = A * x + B * cube + C * left(cube)
        return x

    if op == "ortho":
        return polynomial(s["x"])
    master, momentum = s["master"].double(), s["momentum"].double()
    momentum = MOMENTUM * momentum + (1.0 - MOMENTUM) * s["grad"].double()
    u = MOMENTUM * momentum + (1.0 - MOMENTUM) * s["grad"].double() if case["nesterov"] else momentum
    master = master * (1.0 - LR * DECAY)
    for at, count, rows, cols in s["spans"]:
        span = slice(at, at + count * rows * cols)
        update = polynomial(u[span].view(count, rows, cols))
        master[span] -= LR * _adjust(case["adjust"], rows, cols) * update.reshape(-1)
    return {"master": master, "momentum": momentum}


def _steps_flops(rows, cols):
    """Multiply-adds of the steps times two: the two symmetric products by halves."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m * m * m + 2.0 * m * m * n)


def work(case):
    op = case["op"]
    if op == "embed":
        n, e = case["tokens"] * case["width"], SIZE[case["type"]]
        return {"bytes": min(case["tokens"], case["rows"]) * case["width"] * e + 8 * case["tokens"] + n * SIZE[case["out"]],
                "flops": n}
    if op == "embed_grad":
        n, out = case["tokens"] * case["width"], SIZE[case["out"]]
        table = 2 * min(case["tokens"], case["rows"]) if case["add"] else case["rows"]
        return {"bytes": n * SIZE[case["type"]] + 8 * case["tokens"] + table * case["width"] * out, "flops": n}
    if op == "ortho":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": n * (SIZE[case["type"]] + SIZE[case["out"]]),
                "flops": case["batch"] * _steps_flops(case["rows"], case["cols"])}
    groups = _groups(case)
    return {"bytes": 20 * sum(n * r * c for n, r, c in groups),  # gradient, momentum and master read, the last two written
            "flops": sum(n * _steps_flops(r, c) for n, r, c in groups)}

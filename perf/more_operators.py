"""The calls at both ends of a student's training step: the embedding that its tokens come in by,
with its gradient, and the orthogonalised updates that its matrices are stepped by.

Every case is a dict of plain values with a "kind":

* orth  -- theseus.optim.orthogonalize: count matrices [rows, cols] brought near the orthogonal
           factor of their polar decomposition by Newton-Schulz products.
* muon  -- theseus.optim.FusedMuon.step: momentum, orthogonalised update, weight decay and step of
           the ten matrices of each TimeMix layer of a width.
* embed -- theseus.vocab.embedding: M rows of a table of V x D times a factor ("grads": False a
           lookup alone, True also the table's gradient).
"""
import math
import os
import sys

import torch

_PKG = os.path.join(os.getcwd(), "rwkv-theseus_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
WIDTHS = [768, 1024, 2048, 2560, 4096, 5120]  # heads x 64 of the layers in this repository's measurements
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, DECAY, MOMENTUM = 3e-4, 0.1, 0.95  # with updates scaled to the size of AdamW's


def listed():
    return [
        # the smallest: one head's 64 x 64 block, latency alone
        dict(name="orth_head", kind="orth", count=1, rows=64, cols=64, dtype="fp32"),
        # the four tall low-rank matrices of two layers' decay and gate inputs, as one batch
        dict(name="orth_lora", kind="orth", count=4, rows=2560, cols=128, dtype="fp32"),
        # odd sizes throughout, bfloat16 gradients
        dict(name="orth_ragged", kind="orth", count=1, rows=353, cols=1021, dtype="bf16"),
        # one projection of a middle width
        dict(name="orth_square", kind="orth", count=1, rows=2048, cols=2048, dtype="fp32"),
        # a step over one layer of the tests' width, and over two of a narrow model
        dict(name="muon_256", kind="muon", width=256, layers=1),
        dict(name="muon_768", kind="muon", width=768, layers=2),
        # the largest: the matrices of one layer of full width, 112 million parameters
        dict(name="muon_5120", kind="muon", width=5120, layers=1),
        # a serving step of one token: latency
        dict(name="embed_1", kind="embed", M=1, V=65536, D=5120, scale=1.0, weight="bf16", out="bf16", pad=False, grads=False),
        # a prompt batch out of a float32 table, scaled by sqrt(D) and rounded for the layers
        dict(name="embed_prompt", kind="embed", M=8192, V=65536, D=2560, scale=50.59644256269407, weight="fp32", out="bf16",
             pad=False, grads=False),
        # a short training step of a narrow student
        dict(name="embed_small", kind="embed", M=512, V=8192, D=256, scale=1.0, weight="fp32", out="bf16", pad=False, grads=True),
        # odd sizes throughout, a batch padded at its sequences' ends
        dict(name="embed_ragged", kind="embed", M=3001, V=50001, D=1001, scale=2.5, weight="bf16", out="bf16", pad=True, grads=True),
        # a micro-batch of 16384 tokens at the full width
        dict(name="embed_train", kind="embed", M=16384, V=65536, D=5120, scale=1.0, weight="bf16", out="bf16", pad=False, grads=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["orth", "orth", "muon", "embed", "embed"])
    if kind == "orth":
        rows, cols = _log(rng, 32, 5120), _log(rng, 32, 5120)
        return dict(kind=kind, count=rng.randint(1, max(1, min(8, (1 << 26) // (rows * cols)))), rows=rows, cols=cols,
                    dtype=rng.choice(["fp32", "fp32", "bf16"]))
    if kind == "muon":
        width = 64 * _log(rng, 2, 64)
        return dict(kind=kind, width=width, layers=rng.randint(1, max(1, min(3, (1 << 25) // (width * width)))))
    M, D, V = _log(rng, 1, 16384), rng.choice(WIDTHS + [256, rng.randint(100, 2000)]), _log(rng, 8192, 131072)
    V = min(V, 65536 * 5120 // D)
    return dict(kind=kind, M=M, V=V, D=D, scale=rng.choice([1.0, 1.0, math.sqrt(D)]), weight=rng.choice(["bf16", "fp32"]), out="bf16",
                pad=rng.random() < .3, grads=rng.random() < .7)


# ---------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _gradient(g, m, n):
    """A weight's gradient: a sum over directions of falling strength, and noise."""
    k = min(m, n, 512)
    s = torch.arange(1, k + 1, device="cuda").pow(-.5)
    return ((_randn(g, m, k) * s) @ _randn(g, k, n) + .05 * _randn(g, m, n)) * 1e-3


def _shapes(c):
    """The matrices of the case's TimeMix layers: four projections, and the two factors of the
    decay's, the in-context rate's and the gate's low-rank inputs."""
    C = c["width"]
    r = max(32, round(2.5 * math.sqrt(C) / 32) * 32)
    w = max(32, round(5 * math.sqrt(C) / 32) * 32)
    return ([(C, C)] * 4 + [(C, r), (r, C)] * 2 + [(C, w), (w, C)]) * c["layers"]


def prepare(case, seed):
    """Gradients whose singular values fall off over two orders of magnitude, parameters and
    momentum as they are in the middle of a run; tokens of a Zipf distribution over the table in
    no order, upstream gradients of normal size."""
    c, g = case, _gen(seed)
    if c["kind"] == "orth":
        x = torch.stack([_gradient(g, c["rows"], c["cols"]) for _ in range(c["count"])])
        return dict(c=c, x=x.to(DTYPES[c["dtype"]]))
    if c["kind"] == "muon":
        params, momenta = [], []
        for m, n in _shapes(c):
            p = (.02 * _randn(g, m, n)).requires_grad_()
            p.grad = _gradient(g, m, n)
            momenta.append(.5 * p.grad + .2 * _gradient(g, m, n))
            params.append(p)
        return dict(c=c, params=params, momenta=momenta)
    M, V, D = c["M"], c["V"], c["D"]
    odds = 1 / (torch.arange(V, device="cuda", dtype=torch.float64) + 2.7)
    u = torch.rand(M, generator=g, device="cuda", dtype=torch.float64) * odds.sum()
    ids = torch.randperm(V, generator=g, device="cuda")[torch.searchsorted(odds.cumsum(0), u).clamp_max(V - 1)]
    if c["pad"]:  # the last quarter of the tokens, but for some
        ids[M - M // 4:] = torch.where(torch.rand(M // 4, generator=g, device="cuda") < .9, 0, ids[M - M // 4:])
    weight = _randn(g, V, D).to(DTYPES[c["weight"]]).requires_grad_(c["grads"])
    s = dict(c=c, ids=ids, weight=weight, pad=0 if c["pad"] else None)
    if c["grads"]:
        s["up"] = (1e-2 * _randn(g, M, D)).to(DTYPES[c["out"]])
    return s


# ---------------------------------------------------------------------------- the calls
def run(s):
    if own:
        return {"orth": _orth_own, "muon": _muon_own, "embed": _embed_own}[s["c"]["kind"]](s, s["c"])
    with torch.no_grad():
        return {"orth": _orth_plain, "muon": _muon_plain, "embed": _embed_plain}[s["c"]["kind"]](s, s["c"])


def _orth_own(s, c):
    from theseus import optim
    return optim.orthogonalize(s["x"])


def _muon_own(s, c):
    from theseus import optim
    if "opt" not in s:  # the optimizer that a program keeps, in the middle of a run
        s["opt"] = optim.FusedMuon(s["params"], lr=LR, weight_decay=DECAY, momentum=MOMENTUM, scale="rms")
        for p, m in zip(s["params"], s["momenta"]):
            s["opt"].state[p]["momentum_buffer"] = m
    s["opt"].step()
    return {"params": [p.detach() for p in s["params"]], "momenta": s["momenta"]}


def _embed_own(s, c):
    from theseus import vocab
    out = vocab.embedding(s["ids"], s["weight"], scale=c["scale"], padding_idx=s["pad"], dtype=DTYPES[c["out"]])
    if not c["grads"]:
        return {"out": out}
    dweight, = torch.autograd.grad(out, (s["weight"],), s["up"])
    return {"out": out.detach(), "dweight": dweight}


def _polar(x):
    """Five Newton-Schulz products of [..., m, n] in float32, on the short side."""
    a, b, c = COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(EPS)
    for _ in range(STEPS):
        gram = x @ x.mT.contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT.contiguous() if tall else x


def _orth_plain(s, c):
    return _polar(s["x"].float()).to(torch.bfloat16)


def _muon_plain(s, c):
    for p, m in zip(s["params"], s["momenta"]):
        m.mul_(MOMENTUM).add_(p.grad, alpha=1 - MOMENTUM)
        update = _polar(MOMENTUM * m + (1 - MOMENTUM) * p.grad)
        p.mul_(1 - LR * DECAY).sub_(LR * .2 * math.sqrt(max(p.shape)) * update)
    return {"params": [p.detach() for p in s["params"]], "momenta": s["momenta"]}


def _embed_plain(s, c):
    out = {"out": (s["weight"][s["ids"]].float() * c["scale"]).to(DTYPES[c["out"]])}
    if c["grads"]:
        up = s["up"].float() * c["scale"]
        if c["pad"]:
            up = up * (s["ids"] != s["pad"]).unsqueeze(1)
        grad = torch.zeros(c["V"], c["D"], device=up.device).index_add_(0, s["ids"], up)
        out["dweight"] = grad.to(DTYPES[c["weight"]])
    return out


# ---------------------------------------------------------------------------- what cannot be done without
def _products(m, n):
    """Of the short side's Gram matrix and its square one triangle, and the product with x."""
    m, n = min(m, n), max(m, n)
    return STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)


def work(case):
    c = case
    if c["kind"] == "orth":
        m, n = c["rows"], c["cols"]
        return {"bytes": c["count"] * m * n * ((2 if c["dtype"] == "bf16" else 4) + 2), "flops": c["count"] * _products(m, n)}
    if c["kind"] == "muon":
        return {"bytes": sum(20 * m * n for m, n in _shapes(c)), "flops": sum(_products(m, n) for m, n in _shapes(c))}
    M, V, D = c["M"], c["V"], c["D"]
    size, to = 2 if c["weight"] == "bf16" else 4, 2 if c["out"] == "bf16" else 4
    moved = 8 * M + min(M, V) * D * size + M * D * to
    return {"bytes": moved + (M * D * to + V * D * size if c["grads"] else 0), "flops": M * D * (2 if c["grads"] else 1)}


# ---------------------------------------------------------------------------- 64 bits
def _polar64(x):
    """The same polynomials, p(s) = a s + b s^3 + c s^5 five times over, on one matrix."""
    a, b, c = COEFFICIENTS
    x = x.double()
    x = x / max(float(torch.linalg.matrix_norm(x)), EPS)
    flip = x.shape[0] < x.shape[1]
    x = x.t().contiguous() if flip else x
    eye = torch.eye(x.shape[1], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        s = torch.mm(x.t().contiguous(), x)
        x = torch.mm(x, torch.addmm(a * eye, s, b * eye + c * s))
    return x.t() if flip else x


@torch.no_grad()
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "orth":
        return torch.stack([_polar64(x) for x in s["x"]])
    if c["kind"] == "muon":
        momenta = [m.double().lerp_(p.grad.double(), 1 - MOMENTUM) for p, m in zip(s["params"], s["momenta"])]
        params = []
        for p, m in zip(s["params"], momenta):
            step = _polar64(torch.lerp(p.grad.double(), m, MOMENTUM)) * (.2 * LR * math.sqrt(max(p.shape)))
            params.append(p.detach().double() * (1 - LR * DECAY) - step)
        return {"params": params, "momenta": momenta}
    out = {"out": torch.nn.functional.embedding(s["ids"], s["weight"]).double() * c["scale"]}
    if c["grads"]:
        order = s["ids"].argsort(stable=True)
        if c["pad"]:
            order = order[s["ids"][order] != s["pad"]]
        out["dweight"] = torch.zeros(c["V"], c["D"], dtype=torch.float64, device="cuda").index_put_(
            (s["ids"][order],), s["up"][order].double() * c["scale"], accumulate=True)
    return out

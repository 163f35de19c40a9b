"""The vocabulary operators' calls: the losses that a student learns from over a large vocabulary,
and the top logits that a teacher hands over or a sampling step asks for.

Every case is a dict of plain values with a "kind":

* ce  -- theseus.vocab.linear_cross_entropy: softmax cross entropy of hidden @ weight^T.
* kd  -- theseus.vocab.linear_top_distillation: divergence from a teacher's top K logits.
* top -- theseus.vocab.top_logits: the K largest logits of each row, and its log-sum-exp.

M tokens, width D, vocabulary V.  "grads" says what a training step wants back: "none", "hidden"
(a frozen head) or "both"; "reduce" is the loss's reduction ("none": one loss a token, and with
gradients one upstream gradient a token).
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


def listed():
    return [
        # the log-probability of one token under a full-width head: latency and one read of the head
        dict(name="score_1", kind="ce", M=1, D=5120, V=65536, K=1, grads="none", reduce="none", T=1.0, dtype="bf16"),
        # scoring one token for each of 64 lanes
        dict(name="score_64", kind="ce", M=64, D=2560, V=65536, K=1, grads="none", reduce="none", T=1.0, dtype="bf16"),
        # validation: the losses of a ragged prompt, no gradients
        dict(name="valid_1500", kind="ce", M=1500, D=4096, V=131072, K=1, grads="none", reduce="none", T=1.0, dtype="bf16"),
        # the smallest training step: a narrow model, 64 tokens
        dict(name="ce_small", kind="ce", M=64, D=768, V=8192, K=1, grads="both", reduce="mean", T=1.0, dtype="bf16"),
        # odd sizes throughout, one upstream gradient for each token (weighted tokens)
        dict(name="ce_ragged", kind="ce", M=1021, D=2560, V=50001, K=1, grads="both", reduce="none", T=1.0, dtype="bf16"),
        # one micro-batch of 8 chunks of 512 tokens at the full width, head and hidden trained
        dict(name="ce_train", kind="ce", M=4096, D=5120, V=65536, K=1, grads="both", reduce="mean", T=1.0, dtype="bf16"),
        # a short distillation step of a narrow student
        dict(name="kd_small", kind="kd", M=200, D=1024, V=32768, K=16, grads="both", reduce="mean", T=1.0, dtype="bf16"),
        # distillation under a frozen head: the hidden states' gradient alone, softened logits
        dict(name="kd_frozen", kind="kd", M=2048, D=4096, V=131072, K=64, grads="hidden", reduce="mean", T=2.0, dtype="bf16"),
        # the largest: 8192 tokens at the full width, head and hidden trained
        dict(name="kd_train", kind="kd", M=8192, D=5120, V=65536, K=32, grads="both", reduce="mean", T=1.0, dtype="bf16"),
        # a sampling step of one token
        dict(name="top_1", kind="top", M=1, D=0, V=65536, K=50, grads="none", reduce="none", T=1.0, dtype="bf16"),
        # a ragged batch of float32 logits, part of the vocabulary masked out
        dict(name="top_masked", kind="top", M=333, D=0, V=50001, K=100, grads="none", reduce="none", T=2.0, dtype="fp32"),
        # the teacher's logits of a micro-batch of 4096 tokens
        dict(name="top_4096", kind="top", M=4096, D=0, V=65536, K=64, grads="none", reduce="none", T=1.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "kd", "kd", "top"])
    if kind == "top":
        M, V = _log(rng, 1, 4096), _log(rng, 8192, 131072)
        M = min(M, 4096 * 65536 // V)
        return dict(kind=kind, M=M, D=0, V=V, K=rng.randint(1, 128), grads="none", reduce="none",
                    T=rng.choice([1.0, 2.0]), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    M, D, V = _log(rng, 1, 8192), rng.choice(WIDTHS), _log(rng, 8192, 131072)
    grads = rng.choice(["none", "hidden", "both", "both"])
    reduce = "none" if grads == "none" else rng.choice(["mean", "mean", "none"])
    products = 1 + {"none": 0, "hidden": 1, "both": 2}[grads]
    M = max(1, min(M, 3 * 8192 * 5120 * 65536 // (products * D * V)))
    return dict(kind=kind, M=M, D=D, V=V, K=1 if kind == "ce" else rng.randint(4, 64), grads=grads, reduce=reduce,
                T=1.0 if kind == "ce" else rng.choice([1.0, 1.0, 2.0]), dtype="bf16")


# ---------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


PIECE = 1 << 26  # logits that making inputs and the 64-bit values hold at a time


def prepare(case, seed):
    """Normalised hidden states, a head whose logits spread by about 3 (a trained model's), labels
    sampled from the model's own softmax with one in twenty left out, or the top logits of a
    teacher near the student; for "top" the logits themselves, the highest sixteenth of a float32
    vocabulary masked."""
    c, g = case, _gen(seed)
    M, D, V, K = c["M"], c["D"], c["V"], c["K"]
    if c["kind"] == "top":
        x = (3 * _randn(g, M, V)).to(DTYPES[c["dtype"]])
        if c["dtype"] == "fp32":
            x[:, V - V // 16:] = -math.inf
        return dict(c=c, logits=x)
    wants = c["grads"]
    x = _randn(g, M, D).to(torch.bfloat16).requires_grad_(wants != "none")
    w = (_randn(g, V, D) * (3 / math.sqrt(D))).to(torch.bfloat16).requires_grad_(wants == "both")
    s = dict(c=c, x=x, w=w, up=None)
    if c["reduce"] == "none" and wants != "none":
        s["up"] = torch.rand(M, generator=g, device="cuda") / M
    rows = max(1, PIECE // V)
    with torch.no_grad():
        if c["kind"] == "ce":
            labels = torch.empty(M, dtype=torch.int64, device="cuda")
            for i in range(0, M, rows):
                z = (x[i:i + rows] @ w.t()).float()
                labels[i:i + rows] = (z - torch.rand(z.shape, generator=g, device="cuda").clamp_min(1e-20).log_()
                                      .neg_().log_()).argmax(-1)
            labels[torch.rand(M, generator=g, device="cuda") < .05] = -100
            s["labels"] = labels
        else:
            tv = torch.empty(M, K, dtype=torch.float32, device="cuda")
            ti = torch.empty(M, K, dtype=torch.int64, device="cuda")
            for i in range(0, M, rows):
                t = x[i:i + rows].float()
                z = ((t + .5 * _randn(g, *t.shape)).to(torch.bfloat16) @ w.t()).float()
                tv[i:i + rows], ti[i:i + rows] = z.topk(K, -1)
            s["tv"], s["ti"] = tv, ti
            s["tw"] = (torch.rand(M, generator=g, device="cuda") > .05).float()  # tokens that count
    return s


# ---------------------------------------------------------------------------- the calls
def run(s):
    c = s["c"]
    if c["kind"] == "top":
        return (_top_own if own else _top_plain)(s, c)
    return (_loss_own if own else _loss_plain)(s, c)


def _loss_own(s, c):
    from theseus import vocab
    x, w = s["x"], s["w"]
    if c["kind"] == "ce":
        loss = vocab.linear_cross_entropy(x, w, s["labels"], reduction=c["reduce"])
    else:
        loss = vocab.linear_top_distillation(x, w, s["tv"], s["ti"], temperature=c["T"], token_weight=s["tw"],
                                             reduction=c["reduce"])
    out = {"loss": loss.detach()}
    if c["grads"] == "both":
        out["dhidden"], out["dweight"] = torch.autograd.grad(loss, (x, w), s["up"])
    elif c["grads"] == "hidden":
        out["dhidden"], = torch.autograd.grad(loss, (x,), s["up"])
    return out


def _top_own(s, c):
    from theseus import vocab
    values, indices, lse = vocab.top_logits(s["logits"], c["K"], temperature=c["T"])
    return {"values": values, "indices": indices, "lse": lse}


@torch.no_grad()
def _loss_plain(s, c):
    T = c["T"]
    xf, wf = s["x"].float(), s["w"].float()
    z = xf @ wf.t()
    if T != 1.0:
        z /= T
    top = z.amax(-1, keepdim=True)
    lse = top + (z - top).exp_().sum(-1, keepdim=True).log_()
    if c["kind"] == "ce":
        keep = s["labels"] != -100
        j = s["labels"].clamp_min(0).unsqueeze(1)
        q, entropy, wt = torch.ones_like(z[:, :1]), 0.0, keep.float()
    else:
        t = s["tv"] / T
        e = (t - t.amax(-1, keepdim=True)).exp_()
        q = e / e.sum(-1, keepdim=True)
        j, wt, entropy = s["ti"], s["tw"], (q * q.log()).sum(-1)
    rows = T * T * (entropy - (q * z.gather(1, j)).sum(-1) + q.sum(-1) * lse.squeeze(1)) * wt
    if c["reduce"] == "mean":
        out, scale = {"loss": rows.sum() / wt.sum()}, wt / wt.sum()
    else:
        out, scale = {"loss": rows}, wt if s["up"] is None else wt * s["up"]
    if c["grads"] == "none":
        return out
    f = (T * scale).unsqueeze(1)
    gz = z.sub_(lse).exp_().mul_(f * q.sum(-1, keepdim=True)).scatter_add_(1, j, -f * q)
    out["dhidden"] = (gz @ wf).to(torch.bfloat16)
    if c["grads"] == "both":
        out["dweight"] = (gz.t() @ xf).to(torch.bfloat16)
    return out


def _top_plain(s, c):
    # keys that order as the logits do, ties by the lowest index
    x, V = s["logits"], c["V"]
    f = x.float()
    bits = (f + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    _, i = (order * V + torch.arange(V - 1, -1, -1, device=x.device)).topk(c["K"], -1)
    f = f / c["T"]
    top = f.amax(-1, keepdim=True)
    lse = (top + (f - top).exp_().sum(-1, keepdim=True).log_()).squeeze(1)
    return {"values": x.gather(1, i), "indices": i, "lse": lse}


# ---------------------------------------------------------------------------- what cannot be done without
def work(case):
    c = case
    M, D, V, K = c["M"], c["D"], c["V"], c["K"]
    if c["kind"] == "top":
        size = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": M * V * size + M * K * (size + 8) + 4 * M, "flops": 0}
    products = 1 + {"none": 0, "hidden": 1, "both": 2}[c["grads"]]
    target = 8 * M if c["kind"] == "ce" else M * (12 * K + 4)
    read = 2 * M * D + 2 * V * D + target + (4 * M if c["reduce"] == "none" and c["grads"] != "none" else 0)
    write = (4 * M if c["reduce"] == "none" else 4) + (2 * M * D if products > 1 else 0) + (2 * V * D if products > 2 else 0)
    return {"bytes": read + write, "flops": 2 * M * V * D * products}


# ---------------------------------------------------------------------------- 64 bits
@torch.no_grad()
def exact(case, seed):
    c, s = case, prepare(case, seed)
    M, D, V, T = c["M"], c["D"], c["V"], c["T"]
    piece = max(1, PIECE // V)
    if c["kind"] == "top":
        lse = torch.cat([torch.logsumexp(s["logits"][i:i + piece].double() / T, -1) for i in range(0, M, piece)])
        return {"values": None, "indices": None, "lse": lse}
    x, w = s["x"].double(), s["w"].double()
    if c["kind"] == "ce":
        wt = torch.where(s["labels"] == -100, 0.0, 1.0).double()
    else:
        wt = s["tw"].double()
    total = wt.sum() if c["reduce"] == "mean" else torch.ones((), device="cuda", dtype=torch.float64)
    up = wt / total if s["up"] is None else wt * s["up"].double()
    loss, dx, dw = [], [], torch.zeros(V if c["grads"] == "both" else 0, D, dtype=torch.float64, device="cuda")
    for i in range(0, M, piece):
        r = slice(i, i + piece)
        logp = torch.log_softmax(x[r] @ w.t() / T, -1)
        target = torch.zeros_like(logp)
        if c["kind"] == "ce":
            at = s["labels"][r]
            rows = torch.nonzero(at >= 0).squeeze(1)
            target[rows, at[rows]] = 1.0
            entropy = 0.0
        else:
            q = torch.softmax(s["tv"][r].double() / T, -1)
            target.scatter_add_(1, s["ti"][r], q)
            entropy = torch.special.entr(q).sum(-1).neg()
        loss.append(T * T * (entropy - (target * logp).sum(-1)) * wt[r])
        if c["grads"] != "none":
            gz = (logp.exp_() * target.sum(-1, keepdim=True) - target) * (T * up[r]).unsqueeze(1)
            dx.append(gz @ w)
            if c["grads"] == "both":
                dw += gz.t() @ x[r]
    loss = torch.cat(loss)
    out = {"loss": loss.sum() / total if c["reduce"] == "mean" else loss}
    if c["grads"] != "none":
        out["dhidden"] = torch.cat(dx)
    if c["grads"] == "both":
        out["dweight"] = dw
    return out

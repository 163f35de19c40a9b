"""The example that runs the vocabulary operators together, and sizes past 32-bit offsets."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

from theseus import vocab

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "distill_student.py"
    spec = importlib.util.spec_from_file_location("distill_student", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_the_student_learns_and_is_sampled():
    m = _example()
    student, ((kd0, ce0), (kd1, ce1)) = m.distill(steps=20, vocab=2000, width=128, batch=2, tokens=64)
    assert all(math.isfinite(x) for x in (kd0, ce0, kd1, ce1))
    assert ce1 < ce0 - .5 and kd1 < kd0  # (512 fixed tokens: a model this size takes them in within 20 steps)
    ids = m.sample(student, torch.tensor([3, 5], device="cuda"), 4)
    assert ids.shape == (2, 4) and int(ids.min()) >= 0 and int(ids.max()) < 2000


def test_a_step_matches_the_losses_over_full_logits():
    """The example's step against torch over full float32 logits: losses and the head's gradient."""
    m = _example()
    torch.manual_seed(1)
    V, k, T = 1000, 16, 2.0
    model, teacher = m.Model(V, 128).cuda(), m.Model(V, 128).cuda()
    ids = torch.randint(V, (2, 33), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        full = teacher.head(teacher(ids[:, :-1])[0])
        values, indices, lse = vocab.top_logits(full, k, temperature=T)
        h, _ = model(ids[:, :-1])
    w = model.head.weight.detach().clone().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        kd = vocab.linear_top_distillation(h, w, values, indices, temperature=T, teacher_lse=lse)
        ce = vocab.linear_cross_entropy(h, w, ids[:, 1:])
    (kd + ce).backward()
    wr = w.detach().to(torch.bfloat16).double().requires_grad_()
    z = (h.double() @ wr.t()).reshape(-1, V)
    q = torch.softmax(full.double() / T, -1).reshape(-1, V)
    top = torch.zeros_like(q).scatter_(1, indices.reshape(-1, k), 1.0)
    ref = (T * T * (top * q * (q.log() - torch.log_softmax(z / T, -1))).sum(-1).mean()
           + torch.nn.functional.cross_entropy(z, ids[:, 1:].reshape(-1)))
    ref.backward()
    assert abs(float((kd + ce).detach()) - float(ref.detach())) <= 1e-4 * float(ref.detach())
    # (each loss' gradient: G's and the result's rounding, 2^-8 each, and the sum's)
    assert float((w.grad.double() - wr.grad).norm()) <= 3 * 2.0 ** -8 * float(wr.grad.norm())


def test_offsets_past_32_bits():
    """A head of 4.6 GB (450001 x 5120) and logits of 4.5 GB (34000 x 65536): first and last entries."""
    print("  head of 450001 x 5120", flush=True)
    V, D, M = 450001, 5120, 3
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(V, D, dtype=torch.bfloat16, device="cuda")
    for i in range(0, V, 50000):
        n = min(50000, V - i)
        w[i:i + n] = torch.randn(n, D, generator=g, device="cuda") * .03
    w.requires_grad_()
    x = torch.randn(M, D, generator=g, device="cuda").bfloat16().requires_grad_()
    labels = torch.tensor([V - 1, 0, V - 2], device="cuda")
    loss = vocab.linear_cross_entropy(x, w, labels, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    with torch.no_grad():
        z = torch.cat([x.double() @ w[i:i + 50000].double().t() for i in range(0, V, 50000)], 1)
        lse = torch.logsumexp(z, 1)
        ref = lse - z.gather(1, labels[:, None]).squeeze(1)
        assert ((loss.double() - ref).abs() <= 1e-4).all()
        G = torch.exp(z - lse[:, None])
        G[torch.arange(M), labels] -= 1
        rx = sum(G[:, i:i + 50000] @ w[i:i + 50000].double() for i in range(0, V, 50000))
        assert float((dx.double() - rx).norm()) <= 2.0 ** -8 * float(rx.norm())
        for rows in (slice(0, 64), slice(V - 64, V), slice(419400, 419460)):  # (2^32 bytes lie in row 419430)
            rw = G[:, rows].t() @ x.double()
            assert float((dw[rows].double() - rw).norm()) <= 2.0 ** -8 * float(rw.norm())
    del w, dw, dx, z, G
    torch.cuda.empty_cache()
    print("  logits of 34000 x 65536", flush=True)
    x = torch.zeros(34000, 65536, dtype=torch.bfloat16, device="cuda")
    r = torch.arange(34000, device="cuda")
    x[r, (r * 7919) % 65536] = 3.0
    x[r, (r * 104729 + 1) % 65536] = 5.0
    v, i, _ = vocab.top_logits(x, 2)
    same = (r * 7919) % 65536 == (r * 104729 + 1) % 65536
    assert torch.equal(i[:, 0], (r * 104729 + 1) % 65536)
    assert torch.equal(i[~same, 1], ((r * 7919) % 65536)[~same])

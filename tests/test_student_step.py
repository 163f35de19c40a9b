"""A student's training step on the framework's own operators from its tokens to its updated weights: embedding,
TimeMix layer, vocabulary loss, their gradients, FusedMuon for the layer's matrices and FusedAdamW for the rest."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch
from torch import nn

from theseus.optim import FusedAdamW, FusedMuon, COEFFICIENTS
from theseus.timemix import TimeMix
from theseus.vocab import embedding, linear_cross_entropy

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class Student(nn.Module):
    def __init__(self, vocab, width):
        super().__init__()
        self.embed = nn.Parameter(torch.randn(vocab, width))
        self.mix = TimeMix(width, 0, 1)
        self.head = nn.Parameter(torch.randn(vocab, width) / math.sqrt(width))

    def loss(self, ids, rows):
        """``rows``: how the embedding is taken."""
        x = rows(ids[:, :-1], self.embed)
        with torch.autocast("cuda", dtype=BF):
            y, _ = self.mix(x)
            return linear_cross_entropy(x + y, self.head, ids[:, 1:], ignore_index=0)

    def matrices(self):
        return [p for p in self.mix.parameters() if p.dim() == 2 and p is not self.mix.r_k]


def _own(ids, table):
    return embedding(ids, table, padding_idx=0, dtype=BF)


def _torch(ids, table):
    return nn.functional.embedding(ids, table, padding_idx=0).to(BF)


def _polar(x):
    a, b, c = COEFFICIENTS
    x = x.double()
    x = x / x.norm()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for _ in range(5):
        s = x @ x.t().contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if tall else x


@pytest.mark.parametrize("vocab,width,batch,tokens", [(300, 128, 2, 50), (5000, 256, 3, 129)])
def test_a_step_from_tokens_to_weights(vocab, width, batch, tokens):
    print(f"  student vocab={vocab} width={width} {batch}x{tokens}", flush=True)
    torch.manual_seed(0)
    student = Student(vocab, width).cuda()
    with torch.no_grad():  # (output starts at zero, and the low-rank factors too: give every path a gradient)
        for p in student.mix.parameters():
            if not p.any():
                p.copy_(.02 * torch.randn_like(p))
    ids = torch.randint(1, vocab, (batch, tokens + 1), device="cuda")
    ids[0, tokens // 2:] = 0  # a padded sequence
    ids[1, :tokens // 2] = 7  # a frequent token
    matrices = student.matrices()
    rest = [p for p in student.parameters() if all(p is not m for m in matrices)]
    muon, adam = FusedMuon(matrices, lr=.01, scale="rms"), FusedAdamW(rest, lr=1e-3)

    loss = student.loss(ids, _torch)
    loss.backward()
    want = {n: p.grad for n, p in student.named_parameters()}
    student.zero_grad(set_to_none=True)
    own = student.loss(ids, _own)
    assert torch.equal(own, loss)  # (the same rows)
    own.backward()
    for n, p in student.named_parameters():
        if n == "embed":  # (torch adds the same bfloat16 rows, in another order)
            count = torch.bincount(ids[:, :-1].reshape(-1), minlength=vocab).double()
            assert (p.grad[0] == 0).all()
            err = (p.grad.double() - want[n].double()).norm(dim=1)
            mass = want[n].double().norm(dim=1) + 1e-3 * float(want[n].norm())
            assert (err <= 2 * (count + 1) * 2.0 ** -24 * mass * math.sqrt(width)).all()
        else:
            assert torch.equal(p.grad, want[n]), n

    old = {n: p.detach().double() for n, p in student.named_parameters()}
    norm = muon.step_after_backward(max_norm=math.inf)
    adam.step_after_backward(max_norm=1.0)
    assert abs(float(norm) ** 2 - sum(float(p.grad.double().square().sum()) for p in matrices)) <= 1e-5 * float(norm) ** 2
    moved = 0
    for n, p in student.named_parameters():
        new = p.detach().double()
        if any(p is m for m in matrices):
            step = .01 * .2 * math.sqrt(max(p.shape)) * _polar(p.grad)  # (a first step: the momentum is a multiple of the gradient)
            ref = old[n] * (1 - .01 * .1) - step
            assert float((new - ref).norm()) <= 6e-3 * float(step.norm()) + 3 * 2.0 ** -24 * float(ref.norm()), n
            moved += 1
        else:
            assert torch.isfinite(new).all()
    assert moved == len(matrices) == 10
    student.zero_grad(set_to_none=True)
    student.loss(ids, _own).backward()
    assert all(torch.isfinite(p.grad).all() for p in student.parameters())


def test_the_example_runs_with_both_optimizers():
    path = Path(__file__).resolve().parents[1] / "examples" / "distill_student.py"
    spec = importlib.util.spec_from_file_location("distill_student", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    for muon in (False, True):
        print(f"  example muon={muon}", flush=True)
        student, losses = m.distill(steps=3, vocab=1000, width=128, batch=2, tokens=40, muon=muon)
        assert all(math.isfinite(x) for pair in losses for x in pair)
        assert all(torch.isfinite(p).all() for p in student.parameters())
    ids = m.sample(student, torch.tensor([3, 5], device="cuda"), 3)
    assert ids.shape == (2, 3) and int(ids.min()) >= 0 and int(ids.max()) < 1000

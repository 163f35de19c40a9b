"""A student language model distilled from a teacher's top logits, and sampled from.

A frozen teacher and a student (embedding, one TimeMix layer, head) read the same tokens.  Of the
teacher's logits only each token's largest k and the row's log-sum-exp are kept (``top_logits``);
the student learns from them (``linear_top_distillation``) and from the next tokens
(``linear_cross_entropy``) without forming its own logits, its float32 parameters stepped by
``FusedAdamW``.  Afterwards it is sampled from one token at a time, ``top_logits`` again on the
logits of a step.

    python examples/distill_student.py [--steps 30] [--vocab 8192] [--width 256]
"""
import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "rwkv-theseus_amd"))

from theseus.optim import FusedAdamW  # noqa: E402
from theseus.timemix import TimeMix  # noqa: E402
from theseus.vocab import linear_cross_entropy, linear_top_distillation, top_logits  # noqa: E402


class Model(nn.Module):
    def __init__(self, vocab, width):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.mix = TimeMix(width, 0, 1)
        self.norm = nn.LayerNorm(width)
        self.head = nn.Linear(width, vocab, bias=False)

    def forward(self, ids, state=None):
        """Hidden states for the head [B,T,C] (bfloat16 under autocast) and the carried state."""
        x = self.embed(ids).to(torch.bfloat16)
        out, state = self.mix(x, state)
        return self.norm((x + out).float()).to(torch.bfloat16), state


def distill(steps=30, vocab=8192, width=256, batch=4, tokens=128, k=32, temperature=2.0, share=.5, seed=0, device="cuda"):
    """Returns the student, and the first and last steps' (distillation, cross entropy) losses."""
    torch.manual_seed(seed)
    teacher = Model(vocab, width).to(device).requires_grad_(False)
    teacher.head.weight.mul_(8)  # (an untrained head's logits hardly differ: give the teacher opinions)
    student = Model(vocab, width).to(device)
    opt = FusedAdamW(student.parameters(), lr=3e-3)
    ids = torch.randint(vocab, (batch, tokens + 1), device=device)
    losses = []
    for _ in range(steps):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            with torch.no_grad():
                h, _ = teacher(ids[:, :-1])
                values, indices, lse = top_logits(teacher.head(h), k, temperature=temperature)
            h, _ = student(ids[:, :-1])
            kd = linear_top_distillation(h, student.head.weight, values, indices, temperature=temperature, teacher_lse=lse)
            ce = linear_cross_entropy(h, student.head.weight, ids[:, 1:])
        (share * kd + (1 - share) * ce).backward()
        opt.step_after_backward(max_norm=1.0)
        opt.zero_grad(set_to_none=True)
        losses.append((kd.detach(), ce.detach()))
    return student, [tuple(float(x) for x in losses[i]) for i in (0, -1)]


@torch.no_grad()
def sample(model, start, count, k=8, temperature=.7):
    """``count`` tokens after ``start`` [B], each drawn from the top k of the model's softmax."""
    ids, state, out = start, None, []
    for _ in range(count):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            h, state = model(ids[:, None], state)
            values, indices, _ = top_logits(model.head(h[:, 0]), k)
        p = torch.softmax(values.float() / temperature, -1)
        ids = indices.gather(1, torch.multinomial(p, 1)).squeeze(1)
        out.append(ids)
    return torch.stack(out, 1)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--vocab", type=int, default=8192)
    ap.add_argument("--width", type=int, default=256)
    a = ap.parse_args()
    student, ((kd0, ce0), (kd1, ce1)) = distill(a.steps, a.vocab, a.width)
    print(f"distillation {kd0:.3f} -> {kd1:.3f}, cross entropy {ce0:.3f} -> {ce1:.3f} in {a.steps} steps")
    print("sampled:", sample(student, torch.zeros(1, dtype=torch.int64, device="cuda"), 16)[0].tolist())

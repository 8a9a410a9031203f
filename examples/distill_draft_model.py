"""A student distilled from a teacher's short lists, then used as its draft model.

The student is a frozen NF4 projection with a trainable LoRA adapter in front of a frozen
head, as in a QLoRA run; the teacher is the same network with a low-rank change that the
student does not know.  The teacher answers every context with its top logits and their
log-sum-exp (``top_logits``), the adapter is trained on them (``distilled_head``), and before
and after the training the student drafts tokens that the teacher verifies
(``verify_drafts``): the share it accepts is what the distillation is for.

    python examples/distill_draft_model.py [--steps 150] [--contexts 2048]
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from soupsuck_b200.head import distilled_head  # noqa: E402
from soupsuck_b200.kernels import dequantize_nf4, nf4_lora_linear, top_logits, verify_drafts  # noqa: E402
from soupsuck_b200.quantize import quantize_nf4  # noqa: E402


class Student:
    """hidden = x . (deq(W) + s B A)^T, logits = hidden . head^T."""

    def __init__(self, width, vocab, rank, gen):
        dev = "cuda"
        weight = torch.randn((width, width), device=dev, generator=gen) / math.sqrt(width)
        self.packed, self.state = quantize_nf4(weight.half())
        self.head = (torch.randn((vocab, width), device=dev, generator=gen) * 3 / math.sqrt(width)).half()
        self.a = (torch.randn((rank, width), device=dev, generator=gen) / math.sqrt(width)).requires_grad_()
        self.b = torch.zeros((width, rank), device=dev, requires_grad=True)

    def hidden(self, x):
        return nf4_lora_linear(x, self.packed, self.state, self.a, self.b, 1.0)


def draft_and_verify(student, x, teacher_probs, drafts, gen):
    """Share of drafted tokens that the teacher accepts, `drafts` places per context (every place
    sees the same context here)."""
    with torch.no_grad():
        q = torch.softmax(student.hidden(x).float() @ student.head.float().t(), -1)
        shape = (len(x), drafts, q.shape[1])
        race = torch.empty(shape, device="cuda").exponential_(generator=gen).clamp_min_(1e-30)
        tokens = (q[:, None] / race).argmax(-1)
        noise = torch.empty((len(x), q.shape[1]), device="cuda").exponential_(generator=gen).clamp_min_(1e-30)
        accepted, emitted = verify_drafts(teacher_probs[:, None].expand(-1, drafts + 1, -1), tokens,
                                          torch.rand((len(x), drafts), device="cuda", generator=gen), noise,
                                          q[:, None].expand(*shape))
    assert (emitted.gather(1, accepted[:, None]) >= 0).all()  # every context emits a token of its own
    return accepted.float().mean().item() / drafts


def run(steps=150, contexts=2048, width=256, vocab=5000, rank=16, listed=32, drafts=4, seed=0):
    """(accepted share before, accepted share after, first loss, last loss)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    student = Student(width, vocab, rank, gen)
    change = torch.randn((width, rank), device="cuda", generator=gen) @ torch.randn((rank, width), device="cuda", generator=gen)
    teacher = dequantize_nf4(student.packed, student.state).float() + change * (0.6 / width)
    x = torch.randn((contexts, width), device="cuda", generator=gen).half()
    logits = (x.float() @ teacher.t() @ student.head.float().t()).half()
    probs = torch.softmax(logits.float(), -1)

    values, indices, lse = top_logits(logits, listed)
    before = draft_and_verify(student, x, probs, drafts, gen)
    optimizer = torch.optim.Adam([student.a, student.b], lr=1e-2)
    first = last = None
    for _ in range(steps):
        loss, _ = distilled_head(student.hidden(x), student.head, indices, values, lse)
        optimizer.zero_grad()
        (loss * 4096).backward()  # the fp16 gradients' scale; Adam does not mind it
        optimizer.step()
        first = loss.item() if first is None else first
        last = loss.item()
    after = draft_and_verify(student, x, probs, drafts, gen)
    return before, after, first, last


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=150)
    parser.add_argument("--contexts", type=int, default=2048)
    args = parser.parse_args()
    before, after, first, last = run(args.steps, args.contexts)
    print(f"KL {first:.4f} -> {last:.4f}; drafted tokens accepted {before:.1%} -> {after:.1%}")


if __name__ == "__main__":
    main()

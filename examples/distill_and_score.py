"""Distils a language model's head from a teacher's top logits and scores text
with it: layer norm, head, distillation loss, and the log probabilities the
student gives a held-out text before and after.

    python examples/distill_and_score.py [--steps 60] [--vocab 65536]

The trunk's hidden states and the teacher are synthetic (random weights); what
runs is what a training step and an evaluation run after the trunk.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import rwkv7m_amd  # noqa: E402


def head_logits(hidden, norm_w, norm_b, head):
    """ln_out and the head's product: [B, T, C] -> [B, T, V]."""
    h = rwkv7m_amd.layer_norm(hidden, norm_w, norm_b)
    B, T, C = h.shape
    return F.linear(h.view(B * T, C), head).view(B, T, -1)


def score(hidden, params, tokens):
    """Log probabilities of each position's next token, the distribution's
    entropy and the three likeliest alternatives."""
    with torch.no_grad():
        logits = head_logits(hidden, *params)
        # position t predicts token t + 1: the last one has no target
        return rwkv7m_amd.token_logprobs(logits[:, :-1], tokens[:, 1:],
                                         top_k=3)


def run(steps=60, batch=4, length=65, width=768, vocab=65536, top=32,
        temperature=2.0, lr=0.02, seed=0, log=print):
    dev = "cuda"
    g = torch.Generator(dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    bf16 = torch.bfloat16
    teacher = (1.0 + 0.1 * normal(width), 0.1 * normal(width),
               (normal(vocab, width) * (3.0 / width ** 0.5)).to(bf16))
    # the student starts from the teacher's head with noise of its own size
    student = [torch.ones(width, device=dev), torch.zeros(width, device=dev),
               (teacher[2].float() + normal(vocab, width) *
                (3.0 / width ** 0.5)).to(bf16)]
    for p in student:
        p.requires_grad_()
    opt = torch.optim.Adam(student, lr=lr)

    hidden = (normal(batch, length, width) * 2.0).to(bf16)
    with torch.no_grad():
        logits = head_logits(hidden, *teacher)
        # the text is the teacher's own choice for each next position
        tokens = torch.cat([torch.zeros(batch, 1, dtype=torch.int64,
                                        device=dev),
                            logits[:, :-1].argmax(-1)], 1)
        teacher_logits, teacher_ids = logits.float().topk(top, -1)
    # the second half of the last sequence is padding
    mask = torch.ones(batch, length, device=dev)
    mask[-1, length // 2:] = 0.0
    weight = mask / mask.sum()

    before = score(hidden, student, tokens)
    losses = []
    for step in range(steps):
        opt.zero_grad(set_to_none=True)
        loss = rwkv7m_amd.distill_loss(
            head_logits(hidden, *student), teacher_ids, teacher_logits,
            weight, temperature=temperature).loss
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if step % 20 == 0:
            log(f"step {step:3d}  distillation loss {float(losses[-1]):.4f}")
    after = score(hidden, student, tokens)
    for name, r in (("before", before), ("after", after)):
        hit = (r.top_ids[..., 0] == tokens[:, 1:]).float().mean()
        log(f"{name:6s} log probability {float(r.logprobs.mean()):8.4f}  "
            f"entropy {float(r.entropy.mean()):7.4f}  "
            f"text is the likeliest {float(hit):.2f}")
    return torch.stack(losses), before, after


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--vocab", type=int, default=65536)
    args = ap.parse_args()
    run(steps=args.steps, vocab=args.vocab)

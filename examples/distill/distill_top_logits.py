"""Distil a Qwen3-MoE teacher into a student from the teacher's recorded top alternatives.

Three steps, as a training run would have them (here on random tokens and random-init models of the tiny
configuration, so that it runs anywhere):

1. the teacher scores the sequences once and records, per position, its most likely tokens with their
   log-probabilities (``ops.token_statistics(..., top=k)``): k ids and values in place of a vocabulary of logits;
2. the student trains on the records (``ops.distillation_loss``): KL over the alternatives and the rest of the mass,
   1 / tokens in the row weights so that the loss and its gradient take one pass over the logits;
3. held-out sequences are scored from the hidden states alone (``LMHead(..., mode="statistics")``):
   log-probability of the next token and entropy, no logits written.

    python examples/distill/distill_top_logits.py [--steps 30 --top 16 --temperature 1.0 --device cuda]

Prints one JSON line per step and one for the evaluation before and after.
"""

from __future__ import annotations

import argparse
import json
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[2]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

import torch  # noqa: E402

from tiny_dsv41_b200 import ops  # noqa: E402
from tiny_dsv41_b200.models.qwen import Qwen3MoeConfig, Qwen3MoeForCausalLM  # noqa: E402

IGNORE = -100


def next_tokens(ids: torch.Tensor) -> torch.Tensor:
    """The target of each position: the token after it, none at the last."""
    return torch.cat((ids[:, 1:], torch.full_like(ids[:, :1], IGNORE)), dim=1)


@torch.no_grad()
def record_teacher(teacher, ids, top: int, temperature: float) -> ops.TokenStatistics:
    return ops.token_statistics(teacher(ids).logits, next_tokens(ids), temperature=temperature, top=top)


def train_step(student, optimizer, ids, records, temperature: float) -> dict:
    logits = student(ids).logits
    scored = int(ids.shape[0] * (ids.shape[1] - 1))
    weights = torch.full(ids.shape, 1.0 / scored, device=ids.device)
    loss = ops.distillation_loss(logits, records.top_ids, records.top_log_probs, weights, temperature=temperature, tail=True)
    optimizer.zero_grad()
    loss.total.backward()
    optimizer.step()
    return {"loss": loss.total.item(), "worst_position": loss.rows.max().item()}


@torch.no_grad()
def evaluate(model, ids, temperature: float) -> dict:
    """Mean log-probability of the next token and mean entropy, from the hidden states."""
    targets = next_tokens(ids)
    hidden = model.model(ids).last_hidden_state
    scores = model.lm_head(hidden, targets, mode="statistics", temperature=temperature)
    tokens = (targets != IGNORE).sum()
    return {"log_prob": (scores.log_probs.sum() / tokens).item(), "entropy": (scores.entropy.sum() / tokens).item()}


def main(argv=None) -> list[dict]:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--steps", type=int, default=30)
    p.add_argument("--top", type=int, default=16, help="alternatives recorded per position")
    p.add_argument("--temperature", type=float, default=1.0)
    p.add_argument("--batch-size", type=int, default=4)
    p.add_argument("--seq-len", type=int, default=32)
    p.add_argument("--vocab-size", type=int, default=256)
    p.add_argument("--learning-rate", type=float, default=3e-3)
    p.add_argument("--seed", type=int, default=0)
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    args = p.parse_args(argv)
    config = Qwen3MoeConfig.tiny(num_hidden_layers=2, max_window_layers=2, vocab_size=args.vocab_size)
    dtype = torch.bfloat16 if args.device.startswith("cuda") else torch.float32

    def build(seed):
        torch.manual_seed(seed)
        return Qwen3MoeForCausalLM(config).to(args.device, dtype)

    teacher, student = build(args.seed), build(args.seed + 1)
    with torch.no_grad():  # a teacher with opinions: random-init logits are nearly flat
        teacher.lm_head.weight.mul_(20)
    generator = torch.Generator().manual_seed(args.seed)
    shape = (args.batch_size, args.seq_len)
    ids, held_out = (torch.randint(0, args.vocab_size, shape, generator=generator).to(args.device) for _ in range(2))
    optimizer = torch.optim.AdamW(student.parameters(), lr=args.learning_rate, weight_decay=0.0)
    rows = [{"event": "evaluate", "step": 0, **evaluate(student, held_out, args.temperature)}]
    print(json.dumps(rows[-1]), flush=True)
    records = record_teacher(teacher, ids, args.top, args.temperature)
    for step in range(1, args.steps + 1):
        rows.append({"event": "train", "step": step, **train_step(student, optimizer, ids, records, args.temperature)})
        print(json.dumps(rows[-1]), flush=True)
    rows.append({"event": "evaluate", "step": args.steps, **evaluate(student, held_out, args.temperature)})
    print(json.dumps(rows[-1]), flush=True)
    return rows


if __name__ == "__main__":
    main()

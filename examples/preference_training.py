"""A small policy trained on preferences, calibrated, and trained on its rewards.

    python examples/preference_training.py [--steps N] [--pairs N] [--state-bits 8|32]

The policy is a table of next-token logits with a low-rank update, its data pairs of answers in
which the chosen one follows a hidden rule (the next token is a fixed function of the last) more
often than the rejected one. The operators in the order in which such a program uses them:

1. ``token_logprobs`` scores the answers with the policy and with the frozen reference;
2. ``preference_loss`` compares the pairs, ``AdamW`` (8-bit states) makes the step;
3. ``fit_calibration`` and ``calibrate`` turn the margins of held-out pairs into probabilities that
   the chosen answer is the better one;
4. ``policy_loss`` trains further on sampled answers and their rewards, held near the reference by
   its KL term.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import Any

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import torchisotonic_b200 as ti  # noqa: E402

VOCAB, RANK, LENGTH, DEVICE = 211, 16, 24, "cuda"


class Policy(torch.nn.Module):
    """Next-token logits from the last token."""

    def __init__(self) -> None:
        super().__init__()
        self.embed = torch.nn.Embedding(VOCAB, RANK)
        self.head = torch.nn.Linear(RANK, VOCAB)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return self.head(self.embed(tokens))


def rule(tokens: torch.Tensor) -> torch.Tensor:
    return (7 * tokens + 3) % VOCAB


def answers(n: int, follow: float, gen: torch.Generator) -> torch.Tensor:
    """n sequences whose tokens follow the rule with probability ``follow``."""
    out = torch.randint(0, VOCAB, (n, LENGTH), generator=gen, device=DEVICE)
    keep = torch.rand(n, LENGTH, generator=gen, device=DEVICE) < follow
    for t in range(1, LENGTH):
        out[:, t] = torch.where(keep[:, t], rule(out[:, t - 1]), out[:, t])
    return out


def pair_batch(pairs: int, gen: torch.Generator) -> torch.Tensor:
    return torch.cat([answers(pairs, 0.6, gen), answers(pairs, 0.2, gen)])


def scores(policy: Policy, tokens: torch.Tensor) -> torch.Tensor:
    """Token log-probabilities of every sequence, packed back to back. (The logits are cut along
    their length, in the forward without a copy.)"""
    return ti.token_logprobs(policy(tokens)[:, :-1], tokens[:, 1:]).flatten()


def sample(policy: Policy, n: int, gen: torch.Generator) -> torch.Tensor:
    tokens = torch.randint(0, VOCAB, (n, 1), generator=gen, device=DEVICE)
    for _ in range(LENGTH - 1):
        p = torch.softmax(policy(tokens[:, -1]).float(), -1)
        tokens = torch.cat([tokens, torch.multinomial(p, 1, generator=gen)], 1)
    return tokens


def main(argv: list[str] | None = None) -> dict[str, Any]:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--pairs", type=int, default=128)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    gen = torch.Generator(device=DEVICE).manual_seed(1)
    policy, reference = Policy().to(DEVICE), Policy().to(DEVICE)
    reference.load_state_dict(policy.state_dict())
    offsets = torch.arange(0, (2 * args.pairs + 1) * (LENGTH - 1), LENGTH - 1, device=DEVICE)
    out: dict[str, Any] = {"loss": [], "reward": []}

    opt = ti.AdamW(policy.parameters(), lr=2e-2, state_bits=args.state_bits)
    for _ in range(args.steps):
        tokens = pair_batch(args.pairs, gen)
        with torch.no_grad():
            ref = scores(reference, tokens)
        loss, _ = ti.preference_loss(scores(policy, tokens), ref, offsets, beta=0.1)
        opt.zero_grad()
        loss.backward()
        opt.step()
        out["loss"].append(float(loss.detach()))

    # margins of held-out pairs, shown in either order: the curve from a margin to the probability
    # that the first answer shown is the better one
    margins, first_better = [], []
    for _ in range(20):
        tokens = pair_batch(args.pairs, gen)
        with torch.no_grad():
            _, rewards = ti.preference_loss(scores(policy, tokens), scores(reference, tokens),
                                            offsets, beta=0.1)
        m = rewards[0] - rewards[1]
        swap = torch.rand(args.pairs, generator=gen, device=DEVICE) < 0.5
        margins.append(torch.where(swap, -m, m))
        first_better.append((~swap).float())
    m, better = torch.cat(margins), torch.cat(first_better)
    xs, curve = ti.fit_calibration(m, better)
    out["curve"] = curve
    out["accuracy"] = float(((m > 0).float() == better).float().mean())
    out["probability"] = ti.calibrate(torch.tensor([-1.0, 0.0, 1.0], device=DEVICE), xs, curve)

    # on from here with rewards: how often an answer follows the rule
    reference.load_state_dict(policy.state_dict())
    opt = ti.AdamW(policy.parameters(), lr=1e-2, state_bits=args.state_bits)
    for _ in range(args.steps):
        with torch.no_grad():
            tokens = sample(policy, args.pairs, gen)
            old, ref = scores(policy, tokens), scores(reference, tokens)
        reward = (tokens[:, 1:] == rule(tokens[:, :-1])).float()
        advantages = (reward - reward.mean()).flatten()
        for _ in range(2):
            logits = policy(tokens)[:, :-1]
            got = ti.policy_loss(logits, tokens[:, 1:], old.view_as(reward),
                                 advantages.view_as(reward), ref_logps=ref.view_as(reward),
                                 kl_coef=0.01)
            opt.zero_grad()
            got.loss.backward()
            opt.step()
        out["reward"].append(float(reward.mean()))
    print(f"preference loss {out['loss'][0]:.3f} -> {out['loss'][-1]:.3f}, held-out accuracy "
          f"{out['accuracy']:.3f}")
    print("probability that the first is better at margins -1, 0, 1:",
          [round(v, 3) for v in out["probability"].tolist()])
    print(f"reward {out['reward'][0]:.3f} -> {out['reward'][-1]:.3f}")
    return out


if __name__ == "__main__":
    main()

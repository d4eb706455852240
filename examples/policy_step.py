"""A policy trained on replayed positions with the training operators.

    python examples/policy_step.py [--positions 256] [--steps 20]

Positions of seeded games become the trainer's device batch
(gpu_batch.make_batch); a small residual network over their public features
gives logits over the engine's list of legal actions of each. Its blocks use
train_layers: norms with gate and residual scale, linear layers and GELU whose
inputs are kept in 8 bits, and the clipped policy loss with a KL term towards
the starting policy. As there is no game result here, the advantage is a
seeded preference for some actions, which the policy then learns.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "war-chest-bot-9000-_b200"))
import warchest_b200 as wc  # noqa: E402
from warchest_b200 import gpu_batch, train_layers as layers  # noqa: E402

ACTIONS = 512  # the longest list of legal actions the engine hands out
WIDTH, HIDDEN, BLOCKS = 96, 192, 2


def legal_count(root):
    """How many actions are legal in the state that a root starts with: the one prefix that reads as a state (where a
    state ends does not depend on what follows it, so no shorter or longer one does)."""
    for end in range(64, len(root)):
        try:
            return len(wc.legal_actions(root[:end]))
        except wc.SolveError:
            continue
    raise ValueError("no state at the start of the root")


def positions(n):
    """Replay rows of n positions and how many legal actions each has."""
    rows, counts, seed = [], [], 0
    while len(rows) < n:
        seed += 1
        try:
            root = wc.generate_root(seed, plies=(0, 6, 12, 20)[seed % 4])
            rows.append(np.frombuffer(wc.pack_row(root), np.uint8))
        except wc.SolveError:
            continue
        counts.append(legal_count(root))
    return np.stack(rows), np.asarray(counts)


class Net:
    """The device's parameters: float32 masters, bfloat16 activations."""

    def __init__(self, features, device):
        g = torch.Generator(device=device).manual_seed(0)
        new = lambda *s: (torch.randn(*s, generator=g, device=device) / s[0] ** 0.5).requires_grad_()  # noqa: E731
        flat = lambda v: torch.full((WIDTH,), v, device=device, requires_grad=True)  # noqa: E731
        self.stem, self.head = new(features, WIDTH), new(WIDTH, ACTIONS)
        self.first = (flat(1.0), flat(0.0))
        self.blocks = []
        for _ in range(BLOCKS):
            self.blocks.append({"up": new(WIDTH, HIDDEN), "bias": torch.zeros(HIDDEN, device=device, requires_grad=True),
                                "down": new(HIDDEN, WIDTH), "post": (flat(1.0), flat(0.0)), "pre": (flat(1.0), flat(0.0)),
                                "gate": torch.full((1, WIDTH), 0.5, dtype=torch.bfloat16, device=device, requires_grad=True)})

    def parameters(self):
        out = [self.stem, self.head, *self.first]
        for b in self.blocks:
            out += [b["up"], b["bias"], b["down"], *b["post"], *b["pre"], b["gate"]]
        return out

    def logits(self, features):
        y = layers.linear8(features.to(torch.bfloat16), self.stem)
        # the first block's norm: nothing comes back into the stream yet
        y, n, n8 = layers.block_norm(y, torch.zeros_like(y), pre=self.first, pack=True)
        for b in self.blocks:
            h = layers.linear8(layers.gelu8(layers.linear8(n, b["up"], x8=n8), b["bias"]), b["down"])
            y, n, n8 = layers.block_norm(y, h, gate=b["gate"], residual_scale=0.9, post=b["post"], pre=b["pre"], pack=True)
        return layers.linear8(n, self.head, x8=n8)


def train(n, steps, device="cuda:0", rate=3e-3):
    rows, counts = positions(n)
    seg = np.arange(2 * n, dtype=np.int64)
    parts = (rows, np.zeros((n, 10), np.uint8), np.zeros((2 * n, 15), np.uint8), (seg % 2).astype(np.uint8),
             np.ones(2 * n, np.float32), np.zeros(2 * n, np.float32), seg)
    x = gpu_batch.make_batch(parts, None, device)[0]
    batch = x.shape[0]  # two views of every position
    legal = torch.arange(ACTIONS, device=device) < torch.as_tensor(np.repeat(counts, 2), device=device)[:, None]
    taste = torch.randn(ACTIONS, generator=torch.Generator(device=device).manual_seed(1), device=device)
    net = Net(x.shape[1], device)
    opt = torch.optim.Adam(net.parameters(), lr=rate)
    weights = torch.full((batch,), 1.0 / batch, device=device)
    start, gains = None, []
    g = torch.Generator(device=device).manual_seed(2)
    for _ in range(steps):
        with torch.no_grad():
            z = net.logits(x).float().masked_fill(~legal, -torch.inf)
            lp = torch.log_softmax(z, 1)
            actions = torch.multinomial(lp.exp(), 1, generator=g)[:, 0]
            old = lp.gather(1, actions[:, None])[:, 0].contiguous()
            start = lp if start is None else start
            ref = start.gather(1, actions[:, None])[:, 0].contiguous()
            gains.append(float((lp.exp() * taste).sum(1).mean()))
            advantage = taste[actions] - (lp.exp() * taste).sum(1)
        for _ in range(2):  # two steps on each batch of actions: the second's ratios are no longer 1
            opt.zero_grad()
            r = layers.policy_loss(net.logits(x), actions, old, advantage, weights=weights, ref_logp=ref, legal=legal,
                                   kl_coef=0.01, entropy_coef=0.001)
            r.loss.backward()
            opt.step()
    return gains


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--positions", type=int, default=256)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    gains = train(a.positions, a.steps)
    print("expected preference of the policy: " + " ".join("%.3f" % v for v in gains))


if __name__ == "__main__":
    main()

"""Trains a small decoder and its engram on text, with nothing of the size of the logits in memory:

  1. the decoder's states go to head_cross_entropy with its tied head;
  2. the dense weights (decoder, head, the engram's projections) take a DenseAdamW step with 8-bit moments, the tables a
     row-wise one on their sparse row gradients;
  3. the frozen decoder's log-probabilities, what preference and policy losses take as their reference, come from
     head_token_logps.

    python examples/train_engram_text.py [--steps 30] [--device cuda]

The text is random sequences in which some tokens follow from the two before them; what it shows is the calls.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from micro_engram_fork_amd import MicroEngram, attach_engram, losses  # noqa: E402
from micro_engram_fork_amd.optim import DenseAdamW  # noqa: E402
from micro_engram_fork_amd.rows import RowTables  # noqa: E402

VOCAB, DIM = 4001, 192


class Layer(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = nn.RMSNorm(DIM)
        self.up, self.down = nn.Linear(DIM, 2 * DIM, bias=False), nn.Linear(2 * DIM, DIM, bias=False)

    def forward(self, x):
        return x + self.down(torch.nn.functional.silu(self.up(self.norm(x))))


class Decoder(nn.Module):
    """A decoder without attention that ends in its states; the head is the embedding."""

    def __init__(self):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, DIM)
        self.layers = nn.ModuleList(Layer() for _ in range(2))
        self.norm = nn.RMSNorm(DIM)
        nn.init.normal_(self.embed.weight, std=0.05)

    def forward(self, input_ids):
        x = self.embed(input_ids)
        for layer in self.layers:
            x = layer(x)
        return self.norm(x)


class Trained:
    def __init__(self, device, dtype=torch.bfloat16, state_bits=8, seed=0):
        torch.manual_seed(seed)
        self.decoder = Decoder().to(device, dtype)
        self.engram = MicroEngram(DIM, table_size=8191, engram_dim=32, num_heads=4, orders=(2, 3), vocab_size=VOCAB, gate="scalar_sqrt",
                                  seed=seed)
        self.ids = None
        attach_engram(self.decoder, self.engram, 0, get_ids=lambda: (self.ids, None))
        self.engram.shard_rows(0, 1)
        self.tables = RowTables([("layers.0.micro_engram.", self.engram)], lazy=True, rowwise=True, sparse_grads=True, seed=seed)
        # the engram is a submodule by now: its dense parameters are among the decoder's
        self.dense = DenseAdamW(self.decoder.parameters(), lr=2e-3, weight_decay=0.01, state_bits=state_bits, seed=seed)

    def states(self, ids, engram=True):
        self.ids = ids if engram else None
        return self.decoder(ids)

    def loss(self, ids, targets):
        return losses.head_cross_entropy(self.states(ids), self.decoder.embed.weight, targets, z_loss=1e-4)

    def step(self, ids, targets):
        loss = self.loss(ids, targets)
        loss.backward()
        self.tables.step(2e-2)
        self.dense.step()
        self.tables.zero_grad()
        self.dense.zero_grad()
        return loss.detach()


def text(batch, length, device, gen):
    """(tokens, what each predicts): every third token follows from the two before it, and only those are trained."""
    ids = torch.randint(0, VOCAB, (batch, length + 1), generator=gen, device=device)
    for at in range(2, length + 1, 3):
        ids[:, at] = (ids[:, at - 1] * 31 + ids[:, at - 2] * 17 + 5) % VOCAB
    targets = ids[:, 1:].clone()
    targets[:, torch.arange(length, device=device) % 3 != 1] = losses.IGNORE_INDEX
    return ids[:, :-1], targets


def main(steps=30, device="cuda"):
    model = Trained(device)
    gen = torch.Generator(device=device).manual_seed(1)
    ids, targets = text(8, 96, device, gen)
    history = torch.stack([model.step(ids, targets) for _ in range(steps)]).tolist()
    print(f"cross entropy {history[0]:.3f} -> {history[-1]:.3f}")
    with torch.no_grad():
        head = model.decoder.embed.weight
        with_engram = losses.head_token_logps(model.states(ids), head, targets)
        without = losses.head_token_logps(model.states(ids, engram=False), head, targets)
    print(f"mean log-probability with the engram {with_engram.sum() / (targets >= 0).sum():.3f}, without it "
          f"{without.sum() / (targets >= 0).sum():.3f}")
    return history, with_engram, without


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=30)
    parser.add_argument("--device", default="cuda")
    args = parser.parse_args()
    main(args.steps, args.device)

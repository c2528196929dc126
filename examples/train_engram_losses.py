"""Trains one engram inside a small frozen decoder with each of the losses over logits, one after the
other, as a training program uses them:

  1. distillation from the top logits of a teacher that knows facts the decoder does not;
  2. preference pairs, the reference being the same decoder without its engram's rows;
  3. sampled answers with advantages (clipped policy loss with a KL term to the state before).

    python examples/train_engram_losses.py [--steps 30] [--device cuda]

Everything is random and small; what it shows is the calls. The decoder's weights stay frozen: only
the engram's tables (row-wise Adam on their sparse row gradients) and its two projections learn.
"""
import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from micro_engram_fork_amd import MicroEngram, attach_engram, losses  # noqa: E402
from micro_engram_fork_amd.rows import RowTables  # noqa: E402

VOCAB, DIM = 4000, 256


class Layer(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm = nn.RMSNorm(DIM)
        self.up, self.down = nn.Linear(DIM, 2 * DIM, bias=False), nn.Linear(2 * DIM, DIM, bias=False)

    def forward(self, x):
        return x + self.down(torch.nn.functional.silu(self.up(self.norm(x))))


class Decoder(nn.Module):
    """A decoder without attention: embedding, two layers, tied head."""

    def __init__(self):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, DIM)
        self.layers = nn.ModuleList(Layer() for _ in range(2))
        self.norm = nn.RMSNorm(DIM)
        nn.init.normal_(self.embed.weight, std=0.1)

    def forward(self, input_ids, position_ids=None):
        x = self.embed(input_ids)
        for layer in self.layers:
            x = layer(x)
        return torch.nn.functional.linear(self.norm(x), self.embed.weight)


class Trained:
    """The decoder with its engram, which can be left out (the reference policy)."""

    def __init__(self, device, seed=0):
        torch.manual_seed(seed)
        self.decoder = Decoder().to(device, torch.bfloat16).requires_grad_(False)
        self.engram = MicroEngram(DIM, table_size=8191, engram_dim=32, num_heads=4, orders=(2, 3), vocab_size=VOCAB,
                                  gate="scalar_sqrt", seed=seed)
        self.ids = None
        attach_engram(self.decoder, self.engram, 0, get_ids=lambda: (self.ids, None))
        self.engram.shard_rows(0, 1)
        self.tables = RowTables([("layers.0.micro_engram.", self.engram)], lazy=True, rowwise=True, sparse_grads=True, seed=seed)
        self.dense = torch.optim.AdamW(self.engram.parameters(), lr=5e-3, weight_decay=0.0)

    def logits(self, ids, engram=True):
        self.ids = ids if engram else None
        return self.decoder(ids)

    def step(self, loss):
        loss.backward()
        self.tables.step(2e-2)
        self.dense.step()
        self.tables.zero_grad()
        self.dense.zero_grad()


def next_targets(ids):
    """What each position predicts; the last one predicts nothing."""
    targets = torch.full_like(ids, losses.IGNORE_INDEX)
    targets[:, :-1] = ids[:, 1:]
    return targets


def facts(ids):
    """The token that, for the teacher, follows each pair of tokens."""
    before = torch.cat([ids[:, :1], ids[:, :-1]], dim=1)
    return (ids * 31 + before * 17 + 5) % VOCAB


def distill(model, ids, steps, top=16):
    with torch.no_grad():
        teacher = model.logits(ids, engram=False).float()
        teacher.scatter_add_(2, facts(ids).unsqueeze(2), torch.full((*ids.shape, 1), 8.0, device=ids.device))
        values, tokens = teacher.topk(top, dim=-1)
        lse = teacher.logsumexp(-1)
        del teacher
    history = []
    for _ in range(steps):
        loss = losses.distill_loss(model.logits(ids), tokens, values, teacher_lse=lse)
        model.step(loss)
        history.append(loss.detach())
    return torch.stack(history).tolist()


def preference(model, chosen, rejected, steps):
    ids = torch.cat([chosen, rejected])
    targets = next_targets(ids)
    with torch.no_grad():
        ref = losses.token_logps(model.logits(ids, engram=False), targets)
    history, margins = [], []
    for _ in range(steps):
        loss, up, down = losses.preference_loss(model.logits(ids), targets, ref, beta=0.5)
        model.step(loss)
        history.append(loss.detach())
        margins.append((up - down).mean())
    return torch.stack(history).tolist(), torch.stack(margins).tolist()


def policy(model, prompts, steps, answer=8):
    """Answers sampled from the model; tokens under VOCAB / 8 are what is rewarded."""
    history = []
    for _ in range(steps):
        with torch.no_grad():
            ids = prompts
            for _ in range(answer):
                q = torch.softmax(model.logits(ids)[:, -1].float(), dim=-1)
                ids = torch.cat([ids, torch.multinomial(q, 1)], dim=1)
            targets = next_targets(ids)
            targets[:, :prompts.shape[1] - 1] = losses.IGNORE_INDEX
            rewards = (ids[:, prompts.shape[1]:] < VOCAB // 8).float().mean(1)
            old = losses.token_logps(model.logits(ids), targets)
            ref = losses.token_logps(model.logits(ids, engram=False), targets)
        advantages = (rewards - rewards.mean()) / (rewards.std() + 1e-4)
        for _ in range(2):
            loss, _, stats = losses.policy_loss(model.logits(ids), targets, old, advantages, ref_logps=ref,
                                                clip_high=0.28, kl_coef=0.01, reduction="sequence")
            model.step(loss)
        history.append(rewards.mean())
    return torch.stack(history).tolist()


def main(steps=30, device="cuda"):
    model = Trained(device)
    gen = torch.Generator(device=device).manual_seed(1)

    def tokens(*shape):
        return torch.randint(0, VOCAB, shape, generator=gen, device=device)

    ids = tokens(4, 64)
    kl = distill(model, ids, steps)
    print(f"distillation: KL to the teacher {kl[0]:.3f} -> {kl[-1]:.3f}")
    loss, margin = preference(model, tokens(8, 24), tokens(8, 24), steps)
    print(f"preference: loss {loss[0]:.3f} -> {loss[-1]:.3f}, reward margin {margin[0]:.3f} -> {margin[-1]:.3f}")
    reward = policy(model, tokens(1, 12).expand(64, 12).contiguous(), steps)
    print(f"policy: mean reward {reward[0]:.3f} -> {sum(reward[-5:]) / len(reward[-5:]):.3f}")
    return kl, loss, margin, reward


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=30)
    parser.add_argument("--device", default="cuda")
    args = parser.parse_args()
    main(args.steps, args.device)

"""The dense end of a training step as one: states of a decoder with an engram, the cross entropy from its tied head,
gradients of everything, the step of all dense weights beside that of the tables."""
import importlib.util
import os

import pytest
import torch

import adamw_reference as ref
import head_reference
from micro_engram_fork_amd import losses

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("train_engram_text", os.path.join(ROOT, "examples", "train_engram_text.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_runs():
    history, with_engram, without = _example().main(steps=4)
    assert len(history) == 4 and all(x == x for x in history)
    assert with_engram.shape == without.shape == (8, 96) and bool(torch.isfinite(with_engram).all())


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.bfloat16, 32), (torch.float32, 32)])
def test_a_step(dtype, bits):
    example = _example()
    model = example.Trained("cuda", dtype, bits, seed=3)
    ids, targets = example.text(4, 60, "cuda", torch.Generator(device="cuda").manual_seed(2))
    head = model.decoder.embed.weight
    # the states' and head's own gradients, from the loss alone, against the definition
    states = model.states(ids)
    h, w = states.detach().requires_grad_(), head.detach().requires_grad_()
    loss = losses.head_cross_entropy(h, w, targets, z_loss=1e-4)
    gh, gw = torch.autograd.grad(loss, (h, w))
    want = head_reference.head(h.detach().reshape(-1, example.DIM), w.detach(), targets.reshape(-1), dtype, z_loss=1e-4)
    for got, name in ((loss.detach(), "loss"), (gh, "hidden"), (gw, "weight")):
        value, bound = want[name]
        assert bool(((got.double().reshape(value.shape) - value).abs() <= bound).all()), name
    # through the whole decoder: what autograd makes of those two
    dense = [p for p in model.decoder.parameters()]
    tied = next(i for i, p in enumerate(dense) if p is head)
    states.backward(gh)
    through = [None if p.grad is None else p.grad.clone() for p in dense]
    rows = {t: tuple(x.clone() for x in t.sparse_grad) for t in model.tables.params() if getattr(t, "sparse_grad", None) is not None}
    model.tables.zero_grad(), model.dense.zero_grad()
    full = model.loss(ids, targets)
    assert torch.equal(full.detach(), loss.detach())
    full.backward()
    assert rows
    for t, (r, g) in rows.items():
        assert torch.equal(t.sparse_grad[0], r) and torch.equal(t.sparse_grad[1], g)
    for i, (p, g) in enumerate(zip(dense, through)):
        if i == tied:
            # two uses add up in the parameter's type, in either order
            assert torch.equal(p.grad, g + gw) or torch.equal(p.grad, gw + g)
        elif g is not None:
            assert torch.equal(p.grad, g)
    # the step of the dense weights
    before = [(p.detach().double().cpu().reshape(-1), p.grad.double().cpu().reshape(-1)) for p in dense if p.grad is not None]
    live = [p for p in dense if p.grad is not None]
    streams = {id(p): i for i, p in enumerate(p for g in model.dense.param_groups for p in g["params"])}
    model.tables.step(2e-2)
    model.dense.step()
    group = model.dense.param_groups[0]
    for p, (p0, g0) in zip(live, before):
        zero = torch.zeros_like(p0)
        (value, _, _), (err, _, _) = ref.step(p0, g0, zero, zero, 1, group["lr"], group["betas"], group["eps"], group["weight_decay"])
        got = p.detach().double().cpu().reshape(-1)
        if dtype is torch.float32:
            assert bool(((got - value).abs() <= err).all())
        else:
            r = ref.noise(p0.numel(), model.dense.seed, 1, streams[id(p)])
            a, b = value - err, value + err
            lo, hi = ref.bf16_stochastic(torch.minimum(a.abs(), b.abs()), r), ref.bf16_stochastic(torch.maximum(a.abs(), b.abs()), r)
            assert bool(((got.abs() >= lo) | (a * b <= 0)).all()) and bool((got.abs() <= hi).all())


def test_a_captured_step_replays_as_eager_ones():
    """Loss, gradients of states and head, and the step of the head with its own count: one graph of a head's training."""
    from micro_engram_fork_amd.optim import DenseAdamW

    def make():
        gen = torch.Generator(device="cuda").manual_seed(4)
        w = torch.nn.Parameter((torch.randn(1500, 128, device="cuda", generator=gen) / 8).bfloat16())
        opt = DenseAdamW([w], lr=1e-2, state_bits=8, seed=9, capturable=True)
        return w, opt
    hidden = torch.randn(200, 128, device="cuda").bfloat16()
    targets = torch.randint(0, 1500, (200,), device="cuda")

    def step(w, opt):
        loss = losses.head_cross_entropy(hidden, w, targets)
        w.grad, = torch.autograd.grad(loss, w)
        opt.step()
        return loss.detach()
    (a, eager), (b, opt) = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b, opt)
    torch.cuda.current_stream().wait_stream(side)
    step(a, eager)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(b, opt)
    for k in range(4):
        with torch.no_grad():
            hidden.copy_(torch.randn(200, 128, device="cuda"))
            targets.copy_(torch.randint(-1, 1500, (200,), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step(a, eager)
        torch.cuda.synchronize()
        assert torch.equal(captured, want) and torch.equal(a, b), k

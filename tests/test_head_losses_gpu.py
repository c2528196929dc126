"""head_cross_entropy and head_token_logps against their definitions in float64 (head_reference)."""
import pytest
import torch

import head_reference as ref
from micro_engram_fork_amd import losses

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32

# rows, vocabulary, width: single ones, ends of tiles and slabs (64 / 128 / 256 rows, 256 columns, 64 deep) and past them
SIZES = [(1, 1, 1), (1, 2, 8), (1, 700, 64), (2, 65, 3), (5, 257, 64), (16, 256, 128), (63, 1000, 72), (64, 255, 200), (65, 300, 129),
         (128, 513, 100), (129, 254, 64), (130, 1001, 129), (200, 2049, 264), (257, 777, 192), (300, 4100, 65), (512, 512, 512)]


def _inputs(n, vocab, dim, dtype, seed=0, masked=0.2):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    hidden = torch.randn(n, dim, device=DEV, generator=gen).to(dtype)
    weight = (2.0 / dim ** 0.5 * torch.randn(vocab, dim, device=DEV, generator=gen)).to(dtype)
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen)
    if n > 1:
        targets[torch.rand(n, device=DEV, generator=gen) < masked] = -100
    return hidden, weight, targets


def _close(got, want, what=""):
    value, bound = want
    got = got.detach().double().reshape(value.shape)
    assert got.device == value.device
    bad = ~((got - value).abs() <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - value).abs() / bound).nan_to_num(9e9).max()):.3g} bounds"


def _check_logps(hidden, weight, targets, flat=None, **kw):
    """All of head_token_logps; flat: (hidden, targets) as rows where they have another shape."""
    h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    upstream = torch.randn(targets.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
    logps = losses.head_token_logps(h, w, targets, **kw)
    assert logps.shape == targets.shape and logps.dtype is torch.float32
    gh, gw = torch.autograd.grad(logps, (h, w), upstream)
    rows, t = flat or (hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1))
    want = ref.head(rows, weight, t, hidden.dtype, upstream=upstream.reshape(-1), **kw)
    _close(logps, want["logps"], "logps")
    _close(gh, want["hidden"], "hidden")
    _close(gw, want["weight"], "weight")
    with torch.no_grad():
        assert torch.equal(losses.head_token_logps(hidden, weight, targets, **kw), logps.detach())
    return gh, gw


def _check_ce(hidden, weight, targets, reduction="mean", label_smoothing=0.0, upstream=None, **kw):
    h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = losses.head_cross_entropy(h, w, targets, reduction=reduction, label_smoothing=label_smoothing, **kw)
    assert loss.shape == () and loss.dtype is torch.float32
    gh, gw = torch.autograd.grad(loss, (h, w), None if upstream is None else torch.tensor(upstream, device=DEV))
    rows, t = hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1)
    want = ref.head(rows, weight, t, hidden.dtype, smoothing=label_smoothing, mean=reduction == "mean", **kw)
    _close(loss, want["loss"], "loss")
    f = 1.0 if upstream is None else upstream
    _close(gh, tuple(abs(f) * x if i else f * x for i, x in enumerate(want["hidden"])), "hidden")
    _close(gw, tuple(abs(f) * x if i else f * x for i, x in enumerate(want["weight"])), "weight")
    return loss, gh, gw


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_logps(n, vocab, dim, dtype):
    _check_logps(*_inputs(n, vocab, dim, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_cross_entropy(n, vocab, dim, dtype):
    _check_ce(*_inputs(n, vocab, dim, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [3, 150])
@pytest.mark.parametrize("kw", [dict(label_smoothing=0.1), dict(z_loss=1e-2), dict(temperature=0.5), dict(temperature=3.0), dict(reduction="sum"),
                                dict(scale=-2.5), dict(upstream=0.37), dict(label_smoothing=1.0), dict(ignore_index=7),
                                dict(label_smoothing=0.3, z_loss=1e-3, temperature=1.7, reduction="sum", scale=0.01, upstream=-3.0)])
def test_cross_entropy_options(kw, n, dtype):
    hidden, weight, targets = _inputs(n, 611, 128, dtype)
    targets[1] = 7
    _check_ce(hidden, weight, targets, **kw)


@pytest.mark.parametrize("n", [3, 150])
def test_logps_options(n):
    hidden, weight, targets = _inputs(n, 611, 128, BF16)
    targets[1] = 7
    _check_logps(hidden, weight, targets, temperature=0.7, ignore_index=7)
    _check_logps(hidden, weight, targets.int(), temperature=2.0)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [40, 260])
def test_rows_that_do_not_count_are_not_read(n, dtype):
    hidden, weight, targets = _inputs(n, 300, 64, dtype)
    targets[:3] = torch.tensor([-100, 300, -1])
    out = targets.clone()
    out[(out < 0) | (out >= 300)] = -100
    clean = [x.clone() for x in _check_ce(hidden, weight, out)]
    hidden[(targets < 0) | (targets >= 300)] = float("nan")
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = losses.head_cross_entropy(h, w, targets)
    for a, b in zip((loss, *torch.autograd.grad(loss, (h, w))), clean):
        assert torch.equal(a.detach(), b.detach())


@pytest.mark.parametrize("n", [0, 1, 5, 200])
def test_no_row_counts(n):
    hidden, weight, _ = _inputs(n, 90, 72, BF16)
    targets = torch.full((n,), -100, device=DEV)
    h, w = hidden.fill_(float("nan")).requires_grad_(), weight.requires_grad_()
    for loss in (losses.head_cross_entropy(h, w, targets), losses.head_token_logps(h, w, targets).sum()):
        gh, gw = torch.autograd.grad(loss, (h, w))
        assert float(loss) == 0 and gh.shape == h.shape and gw.shape == w.shape
        assert not gh.any() and not gw.any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [6, 170])
def test_layouts_of_hidden_states(n, dtype):
    """Next-token views, three dims that are no two strides, values that are not next to each other, rows at odd places."""
    long, weight, _ = _inputs(2 * (n + 1), 200, 96, dtype)
    targets = torch.randint(0, 200, (2, n), device=DEV)
    _check_logps(long.view(2, n + 1, 96)[:, :-1], weight, targets)
    _check_logps(long.view(n + 1, 2, 96).transpose(0, 1)[:, 1:], weight, targets)
    apart = torch.randn(2, n, 192, device=DEV).to(dtype)[..., ::2]
    _check_logps(apart, weight, targets)
    odd = torch.randn(2 * n * 97 + 1, device=DEV).to(dtype)[1:].view(2, n, 97)[..., :96]
    _check_logps(odd, weight, targets)
    deep = torch.randn(2, 3, n, 96, device=DEV).to(dtype).transpose(1, 2)
    _check_logps(deep, weight, torch.randint(0, 200, (2, n, 3), device=DEV))
    _check_logps(long[0], weight, targets[0, 0])  # one row, no leading dims


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [6, 170])
def test_layouts_of_the_head(n, dtype):
    hidden, _, targets = _inputs(n, 200, 96, dtype)
    wide = torch.randn(230, 104, device=DEV).to(dtype)
    _check_logps(hidden, wide[:200, :96], targets)            # rows 16 bytes aligned
    _check_logps(hidden, wide[20:220, 3:99], targets)         # rows at odd places
    _check_logps(hidden, torch.randn(200, 97, device=DEV).to(dtype)[:, 1:], targets)
    _check_logps(hidden, torch.randn(96, 200, device=DEV).to(dtype).t(), targets)
    _check_logps(hidden, torch.randn(1, 96, device=DEV).to(dtype).expand(200, 96), targets)


@pytest.mark.parametrize("n", [4, 140])
def test_likely_targets_keep_the_digits_of_what_remains(n):
    """The target carries all but 1e-4 to 1e-9: loss and gradient are as exact, relatively, as the others' weight."""
    dim, vocab = 64, 500
    gen = torch.Generator(device=DEV).manual_seed(3)
    weight = torch.randn(vocab, dim, device=DEV, generator=gen) / 8
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen)
    row = weight[targets]
    hidden = row / row.square().sum(1, keepdim=True) * torch.linspace(16, 27, n, device=DEV)[:, None]
    logps = losses.head_token_logps(hidden, weight, targets)
    z = hidden.double() @ weight.double().t()
    d = z - z.gather(1, targets[:, None])
    d.scatter_(1, targets[:, None], -float("inf"))
    want = -torch.log1p(d.exp().sum(1))
    assert float(want.abs().max()) < 1e-2
    # a logit's absolute error is the others' relative one
    bound = 2 * 3 * (dim + 8) * 2.0 ** -24 * (hidden.double().abs() @ weight.double().abs().t()).amax(1) + 1e-5
    assert bool(((logps.double() - want).abs() <= bound * want.abs()).all())


@pytest.mark.parametrize("n", [4, 140])
def test_logits_of_any_size(n):
    hidden, weight, targets = _inputs(n, 300, 64, FP32)
    _check_logps(hidden * 300, weight, targets)   # differences in the thousands
    _check_logps(hidden * 1e-6, weight, targets)
    hidden[0, 0] = float("inf")
    targets[0] = 5
    assert bool(torch.isnan(losses.head_token_logps(hidden, weight, targets)[0]))
    hidden[0, 0] = float("nan")
    logps = losses.head_token_logps(hidden, weight, targets)
    assert bool(torch.isnan(logps[0])) and bool(torch.isfinite(logps[1:]).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [7, 150])
def test_one_gradient_alone(n, dtype):
    hidden, weight, targets = _inputs(n, 400, 128, dtype)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    gh, gw = torch.autograd.grad(losses.head_cross_entropy(h, w, targets), (h, w))
    assert torch.equal(torch.autograd.grad(losses.head_cross_entropy(h, w.detach(), targets), h)[0], gh)
    assert torch.equal(torch.autograd.grad(losses.head_cross_entropy(h.detach(), w, targets), w)[0], gw)


@pytest.mark.parametrize("n", [9, 150])
def test_gradients_against_differences(n):
    hidden, weight, targets = _inputs(n, 150, 64, FP32)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    gh, gw = torch.autograd.grad(losses.head_cross_entropy(h, w, targets, z_loss=0.01, label_smoothing=0.1), (h, w))
    gen = torch.Generator(device=DEV).manual_seed(1)
    step = 2.0 ** -6
    for x, g in ((h, gh), (w, gw)):
        d = torch.randn(x.shape, device=DEV, generator=gen)
        with torch.no_grad():
            up, down = (float(losses.head_cross_entropy(*(y + s * step * d if y is x else y for y in (h, w)), targets, z_loss=0.01,
                                                        label_smoothing=0.1)) for s in (1, -1))
        # third derivatives of the loss along d are at most the cube of the logits' change, here about 1 per row
        # (std sqrt(1) or 2 sqrt(64) / 8): step^2; and the two losses' own error over the step
        change = d.norm() / d.numel() ** 0.5 * (2.0 if x is h else 8.0)
        bound = float(change) ** 3 * step ** 2 + 2 * 2e-5 / (2 * step)
        assert abs((up - down) / (2 * step) - float((g * d).sum())) <= bound


@pytest.mark.parametrize("n,vocab,dim,dtype", [(16_400, 20_001, 64, BF16), (5_500, 20_001, 64, FP32), (150, 4_500, 33_000, FP32), (3, 9_000, 33_001, BF16)])
def test_more_than_one_piece(n, vocab, dim, dtype):
    """Vocabularies that go through in pieces: of the gradient, of the laid-out head."""
    _check_ce(*_inputs(n, vocab, dim, dtype), label_smoothing=0.1)


def test_many_rows_and_sequences_of_two_uses():
    """One head used for two batches: gradients add up."""
    (h1, w, t1), (h2, _, t2) = _inputs(1000, 999, 128, BF16), _inputs(64, 999, 128, BF16, seed=4)
    w = w.requires_grad_()
    one, = torch.autograd.grad(losses.head_cross_entropy(h1, w, t1), w)
    two, = torch.autograd.grad(losses.head_cross_entropy(h2, w, t2), w)
    both, = torch.autograd.grad(losses.head_cross_entropy(h1, w, t1) + losses.head_cross_entropy(h2, w, t2), w)
    assert torch.equal(both, one + two) or torch.equal(both, two + one)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [50, 300])
def test_the_same_bits_every_time(n, dtype):
    hidden, weight, targets = _inputs(n, 5000, 192, dtype)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    first = None
    for _ in range(5):
        loss = losses.head_cross_entropy(h, w, targets)
        got = [loss.detach(), *torch.autograd.grad(loss, (h, w))]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("n", [20, 200])
def test_captured_forward_and_backward(n):
    """Replays on new inputs, rows that count among them, equal eager calls."""
    hidden, weight, targets = _inputs(n, 700, 128, BF16)
    h, w = hidden.requires_grad_(), weight.requires_grad_()

    def step():
        loss = losses.head_cross_entropy(h, w, targets, z_loss=1e-3)
        logps = losses.head_token_logps(h, w, targets)
        return [loss, logps, *torch.autograd.grad(loss + logps.sum(), (h, w))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        new = _inputs(n, 700, 128, BF16, seed=20 + k, masked=0.2 * k)
        with torch.no_grad():
            h.copy_(new[0]), w.copy_(new[1]), targets.copy_(new[2])
        graph.replay()
        torch.cuda.synchronize()
        got = [x.detach().clone() for x in captured]
        want = [x.detach() for x in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_two_streams_at_once():
    cases = [_inputs(300, 3000, 256, BF16, seed=k) for k in range(4)]
    want = [losses.head_token_logps(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for s, c in zip(streams, cases):
        with torch.cuda.stream(s):
            got.append(losses.head_token_logps(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_changed_inputs_are_noticed():
    hidden, weight, targets = _inputs(10, 100, 64, BF16)
    h = hidden.requires_grad_()
    loss = losses.head_cross_entropy(h, weight, targets)
    weight.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_no_second_derivatives_and_a_second_backward():
    hidden, weight, targets = _inputs(10, 100, 64, BF16)
    h = hidden.requires_grad_()
    loss = losses.head_cross_entropy(h, weight, targets)
    one, = torch.autograd.grad(loss, h, retain_graph=True)
    two, = torch.autograd.grad(loss, h)
    assert torch.equal(one, two)
    g, = torch.autograd.grad(losses.head_cross_entropy(h, weight, targets), h, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_against_the_losses_over_logits():
    """The log-probabilities are those of token_logps on the fp32 logits."""
    hidden, weight, targets = _inputs(200, 1000, 256, FP32)
    a = losses.head_token_logps(hidden, weight, targets)
    b = losses.token_logps((hidden.double() @ weight.double().t()).float(), targets)
    # the logits here are rounded once (2^-24 of up to 16), there as the reference's bound has it
    assert float((a - b).abs().max()) <= 3 * 264 * 2.0 ** -24 * float((hidden.abs() @ weight.abs().t()).max()) * 2 + 1e-5


def test_compiled():
    hidden, weight, targets = _inputs(40, 300, 64, BF16)
    h = hidden.requires_grad_()

    @torch.compile(backend="aot_eager")
    def f(h):
        return losses.head_cross_entropy(h * 2, weight, targets)
    g, = torch.autograd.grad(f(h), h)
    want, = torch.autograd.grad(losses.head_cross_entropy(h * 2, weight, targets), h)
    assert torch.equal(g, want)


# ---- the hidden states' gradient alone, from the forward's exponentials ------------------------------------------
@pytest.fixture
def leaves_unit(monkeypatch):
    """Calls of any size take that way, not those alone that are large enough for it to pay."""
    from micro_engram_fork_amd import _lib, head_ops
    as_it_is = head_ops.unit_elements
    monkeypatch.setattr(head_ops, "unit_elements", lambda n, vocab, dim, dtype, gradients:
                        n * -(-dim // 4) * 4 if (dtype, gradients) == (_lib.ME_BF16, head_ops.OF_HIDDEN)
                        else as_it_is(n, vocab, dim, dtype, gradients))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_hidden_alone_at_the_ends_of_tiles(n, vocab, dim, dtype, leaves_unit):
    _check_hidden_alone(*_inputs(n, vocab, dim, dtype))


LARGE = [(130, 40_001, 264, BF16), (700, 33_000, 1_024, BF16), (70, 33_000, 1_000, FP32), (300, 20_001, 520, FP32), (3, 70_000, 2_048, BF16),
         (9_000, 40_000, 64, BF16)]


def _check_hidden_alone(hidden, weight, targets, upstream=None, label_smoothing=0.0, reduction="mean", **kw):
    """Both losses and their gradients of hidden, where these leave what the backward scales."""
    h = hidden.detach().requires_grad_()
    loss = losses.head_cross_entropy(h, weight, targets, label_smoothing=label_smoothing, reduction=reduction, **kw)
    want = ref.head(hidden, weight, targets, hidden.dtype, smoothing=label_smoothing, mean=reduction == "mean", **kw)
    _close(loss, want["loss"], "loss")
    _close(torch.autograd.grad(loss, h)[0], want["hidden"], "hidden of the loss")
    up = torch.randn(targets.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
    kw.pop("z_loss", None), kw.pop("scale", None)
    logps = losses.head_token_logps(h, weight, targets, **kw)
    want = ref.head(hidden, weight, targets, hidden.dtype, upstream=up, **kw)
    _close(logps, want["logps"], "logps")
    _close(torch.autograd.grad(logps, h, up)[0], want["hidden"], "hidden of logps")


@pytest.mark.parametrize("n,vocab,dim,dtype", LARGE)
def test_hidden_alone(n, vocab, dim, dtype, leaves_unit):
    _check_hidden_alone(*_inputs(n, vocab, dim, dtype))


@pytest.mark.parametrize("n", [100, 300])
@pytest.mark.parametrize("kw", [dict(label_smoothing=0.1), dict(z_loss=1e-2, temperature=0.5), dict(reduction="sum", scale=-2.5, ignore_index=7),
                                dict(label_smoothing=0.3, z_loss=1e-3, temperature=1.7, scale=0.01)])
def test_hidden_alone_options(kw, n, leaves_unit):
    hidden, weight, targets = _inputs(n, 40_000, 1_024, BF16)
    targets[1] = 7
    _check_hidden_alone(hidden, weight, targets, **kw)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [40, 300])
def test_hidden_alone_of_unlikely_targets(n, dtype, leaves_unit):
    """Rows whose target is so unlikely that exponentials around it would overflow, between ordinary ones, and rows
    that are not finite: each as it should be, and the others untouched by them."""
    hidden, weight, targets = _inputs(n, 33_000, 1_024, dtype, masked=0.3)
    some = torch.arange(n, device=DEV) % 7 == 3
    hidden[some] *= 60.0
    _check_hidden_alone(hidden, weight, targets)
    _check_hidden_alone(hidden * 30, weight, targets)
    h = hidden.clone()
    h[5, 1], targets[5] = float("nan"), 3
    h[6, 2], targets[6] = float("inf"), 4
    h.requires_grad_()
    logps = losses.head_token_logps(h, weight, targets)
    assert bool(torch.isnan(logps[5])) and bool(torch.isnan(logps[6]))
    up = torch.ones_like(logps)
    g, = torch.autograd.grad(logps, h, up)
    clean = torch.ones(n, dtype=torch.bool, device=DEV)
    clean[5] = clean[6] = False
    want = ref.head(hidden, weight, torch.where(clean, targets, -100), dtype, upstream=up)
    assert bool(torch.isnan(g[5]).any()) and bool(torch.isnan(g[6]).any())
    assert bool(((g.double() - want["hidden"][0]).abs() <= want["hidden"][1])[clean].all())


def test_hidden_alone_strides_and_odd_heads(leaves_unit):
    hidden, weight, _ = _inputs(400, 40_000, 1_000, BF16)
    targets = torch.randint(0, 39_990, (2, 199), device=DEV)
    view = hidden.view(2, 200, 1_000)[:, :-1, 1:]
    odd = weight[5:39_995, 1:]
    h = view.detach().requires_grad_()
    logps = losses.head_token_logps(h, odd, targets)
    up = torch.randn(targets.shape, device=DEV)
    want = ref.head(view.reshape(-1, 999), odd, targets.reshape(-1), BF16, upstream=up.reshape(-1))
    _close(logps, want["logps"])
    _close(torch.autograd.grad(logps, h, up)[0], want["hidden"])


@pytest.mark.parametrize("n", [100, 300])
def test_hidden_alone_without_counted_rows(n, leaves_unit):
    hidden, weight, targets = _inputs(n, 40_000, 1_024, BF16)
    h = hidden.fill_(float("nan")).requires_grad_()
    loss = losses.head_cross_entropy(h, weight, torch.full_like(targets, -100))
    assert float(loss.detach()) == 0 and not torch.autograd.grad(loss, h)[0].any()


def test_hidden_alone_captured_and_twice(leaves_unit):
    hidden, weight, targets = _inputs(300, 40_000, 1_024, BF16)
    h = hidden.requires_grad_()

    def step():
        loss = losses.head_cross_entropy(h, weight, targets, label_smoothing=0.1)
        return [loss, *torch.autograd.grad(loss, h, retain_graph=True), *torch.autograd.grad(3 * loss, h)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        new = _inputs(300, 40_000, 1_024, BF16, seed=30 + k, masked=0.25 * k)
        with torch.no_grad():
            h.copy_(new[0] * (60 if k == 2 else 1)), weight.copy_(new[1]), targets.copy_(new[2])
        graph.replay()
        torch.cuda.synchronize()
        got = [x.detach().clone() for x in captured]
        want = [x.detach() for x in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_hidden_alone_under_saved_tensor_hooks(leaves_unit):
    hidden, weight, targets = _inputs(300, 40_000, 1_024, BF16)
    h = hidden.requires_grad_()
    want, = torch.autograd.grad(losses.head_cross_entropy(h, weight, targets), h)
    with torch.autograd.graph.save_on_cpu():
        loss = losses.head_cross_entropy(h, weight, targets)
    assert torch.equal(torch.autograd.grad(loss, h)[0], want)


def test_large_calls_for_hidden_alone_take_that_way():
    from micro_engram_fork_amd import _lib, head_ops
    hidden, weight, targets = _inputs(700, 33_000, 2_048, BF16)
    assert head_ops.unit_elements(700, 33_000, 2_048, _lib.ME_BF16, head_ops.OF_HIDDEN) == 700 * 2_048
    _check_hidden_alone(hidden, weight, targets)


@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [12, 140])
def test_gradients_of_likely_targets(n, dtype, alone, leaves_unit):
    """Rows whose target carries all but 1e-3 to 1e-9: their gradients, as small as that, keep their digits (the reference's
    bound is relative to the others' weight)."""
    dim, vocab = 128, 700
    gen = torch.Generator(device=DEV).manual_seed(5)
    weight = (torch.randn(vocab, dim, device=DEV, generator=gen) / 8).to(dtype)
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen)
    row = weight[targets].float()
    hidden = (row / row.square().sum(1, keepdim=True) * torch.linspace(14, 27, n, device=DEV)[:, None]).to(dtype)
    h, w = hidden.requires_grad_(), weight.requires_grad_(not alone)
    logps = losses.head_token_logps(h, w, targets)
    up = torch.rand(n, device=DEV, generator=gen) + 0.5
    grads = torch.autograd.grad(logps, (h,) if alone else (h, w), up)
    want = ref.head(hidden.detach(), weight.detach(), targets, dtype, upstream=up)
    assert float(want["hidden"][0].abs().amax(1).min()) < 1e-8
    _close(grads[0], want["hidden"], "hidden")
    if not alone:
        _close(grads[1], want["weight"], "weight")


def test_heads_of_rows_of_very_different_sizes():
    """fp32 rows of the head from 1e-6 to 1e3 of the others: each is a part of the sums as it should be."""
    hidden, weight, targets = _inputs(150, 600, 128, FP32)
    weight *= torch.logspace(-6, 3, 600, device=DEV)[torch.randperm(600, device=DEV)][:, None]
    hidden /= 300
    _check_logps(hidden, weight, targets)
    hidden *= torch.logspace(-4, 1, 150, device=DEV)[:, None]
    _check_logps(hidden, weight, targets)


# ---- few rows of fp32, whose logits are kept ------------------------------------------------------------------------
@pytest.mark.parametrize("n,vocab,dim", [(9, 1_000, 512), (31, 8_191, 100), (32, 20_001, 64), (33, 257, 1_023), (64, 3_000, 2_050), (90, 3_423, 1_000),
                                         (96, 140_000, 36), (97, 511, 33), (128, 40_003, 260), (128, 700, 4_097), (2, 150_001, 129), (7, 600, 1_500), (8, 900, 2_300),
                                         (129, 5_000, 68), (193, 70_001, 40), (384, 3_001, 200), (1_000, 515, 77), (1_024, 16_000, 24)])
def test_few_rows_of_fp32(n, vocab, dim):
    """Tiles of 32 to 128 rows, one and more of them, splits of either reduction, heads whose rows start and end anywhere."""
    _check_logps(*_inputs(n, vocab, dim, FP32))
    _check_hidden_alone(*_inputs(n, vocab, dim, FP32, seed=1))


@pytest.mark.parametrize("n", [5, 100])
@pytest.mark.parametrize("kw", [dict(label_smoothing=0.1, z_loss=1e-2), dict(temperature=0.4, reduction="sum", scale=-2.0, upstream=0.3)])
def test_few_rows_of_fp32_options(kw, n):
    _check_ce(*_inputs(n, 5_001, 130, FP32), **kw)


@pytest.mark.parametrize("n", [6, 77])
def test_few_rows_of_fp32_twice_and_captured(n):
    """A second backward finds the logits as they were; replays, with eager work between them, give the eager bits."""
    hidden, weight, targets = _inputs(n, 3_001, 257, FP32)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = losses.head_cross_entropy(h, w, targets)
    want = torch.autograd.grad(loss, (h, w), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (h, w)), want))
    del loss
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(losses.head_cross_entropy(h, w, targets), (h, w))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch.autograd.grad(losses.head_cross_entropy(h, w, targets), (h, w))
    for _ in range(3):
        for g in got:
            g.zero_()
        graph.replay()
        torch.autograd.grad(losses.head_cross_entropy(h, w, targets), (h, w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [4, 60, 140])
@pytest.mark.parametrize("dim", [64, 66, 67])
def test_what_lies_between_rows_of_the_head_is_not_used(dim, n, dtype):
    """Rows that are apart, of lengths that end inside of 16 bytes, with NaN between them and behind the last one's end."""
    hidden, weight, targets = _inputs(n, 300, dim, dtype)
    apart = torch.full((300, 72), float("nan"), device=DEV, dtype=dtype)
    apart[:, :dim] = weight
    _check_logps(hidden, apart[:, :dim], targets)
    _check_hidden_alone(hidden, apart[:, :dim], targets)


@pytest.mark.parametrize("n,vocab,dim", [(385, 70_001, 72), (1_025, 300, 129), (1_100, 2_049, 264), (1_500, 7_000, 65), (1_025, 9_000, 33_000)])
def test_more_rows_of_fp32(n, vocab, dim):
    """In parts: tiles of 64 rows and of 256, more than one piece of the head."""
    _check_logps(*_inputs(n, vocab, dim, FP32))
    _check_ce(*_inputs(n, vocab, dim, FP32, seed=1), label_smoothing=0.1, z_loss=1e-3)


def test_few_rows_of_fp32_whose_forward_kept_nothing():
    """The operators' own call: the logits are made again."""
    from micro_engram_fork_amd import head_ops
    hidden, weight, targets = _inputs(40, 700, 96, FP32)
    up = torch.randn(40, device=DEV)
    logps, saved = head_ops.head_logps(hidden, weight, targets, -100, 1.0, head_ops.NO_GRADIENT)
    gh, gw = head_ops.head_backward(hidden, weight, targets, saved, None, up, -100, 1.0, True, 0.0, 0.0, 1.0, 0, True, True)
    want = ref.head(hidden, weight, targets, FP32, upstream=up)
    _close(gh, want["hidden"], "hidden")
    _close(gw, want["weight"], "weight")


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_compiled_for_any_number_of_rows(dtype):
    hidden, weight, targets = _inputs(300, 700, 72, dtype)
    h = hidden.requires_grad_()

    @torch.compile(backend="aot_eager", dynamic=True)
    def f(h, t):
        return losses.head_cross_entropy(h * 2, weight, t)
    for n in (300, 40, 17):
        g, = torch.autograd.grad(f(h[:n], targets[:n]), h)
        want, = torch.autograd.grad(losses.head_cross_entropy(h[:n] * 2, weight, targets[:n]), h)
        assert torch.equal(g, want), n


def test_offsets_past_32_bits():
    """Heads of more than 4 GiB, and their gradient: the last rows are where they belong."""
    try:
        _check_logps(*_inputs(12, 262_144, 4_200, FP32))
        torch.cuda.empty_cache()
        _check_hidden_alone(*_inputs(390, 262_144, 4_200, FP32))
        torch.cuda.empty_cache()
        _check_hidden_alone(*_inputs(70, 420_001, 5_376, BF16))
    finally:
        torch.cuda.empty_cache()

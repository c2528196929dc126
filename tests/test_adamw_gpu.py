"""DenseAdamW against AdamW in float64 with the same rounding noise (adamw_reference)."""
import pytest
import torch

import adamw_reference as ref
from micro_engram_fork_amd.optim import DenseAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"
SEED = (123 << 32) + 77
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 8, 9, 127, 128, 129, 255, 2047, 2048, 2049, 4095, 4096, 4097, 10_001, 0, (3, 5, 7), (64, 33)]


def _tensors(sizes, dtype, gdtype, offset=0, seed=0):
    """Parameters that start `offset` values into their own buffers, with gradients likewise."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    params = []
    for size in sizes:
        shape = size if isinstance(size, tuple) else (size,)
        n = int(torch.Size(shape).numel())

        def piece(std, kind):
            x = torch.randn(n + offset, device=DEV, generator=gen) * std
            x = x * torch.exp(2 * torch.randn(n + offset, device=DEV, generator=gen)) if std != 1 else x
            return x.to(kind)[offset:].view(shape)
        p = torch.nn.Parameter(piece(1, dtype))
        g = piece(1e-3, gdtype)
        if dtype is gdtype:
            p.grad = g
        else:
            p.fp32_grad = g
        params.append(p)
    return params


def _grad(p):
    g = getattr(p, "fp32_grad", None)
    return (p.grad if g is None else g).detach()


def _state(opt, p, bits):
    """(m, v) in float64, flat, of a parameter that has state."""
    s = opt.state[p]
    if bits == 32:
        return s["exp_avg"].double().cpu().reshape(-1), s["exp_avg_sq"].double().cpu().reshape(-1)
    return (ref.values(s["exp_avg"].cpu(), s["exp_avg_scale"].cpu(), torch.float8_e4m3fn),
            ref.values(s["exp_avg_sq"].cpu(), s["exp_avg_sq_scale"].cpu(), torch.float8_e5m2))


def _check_codes(codes, scale, x, err, r, fmt, second):
    """Codes and scales of a rounded moment against its exact value and that value's error."""
    codes, scale = codes.view(torch.uint8).long().reshape(-1), scale.view(torch.uint8).long()
    low, high = (x.abs() - err).clamp(min=0), x.abs() + err
    for bound, ok in ((ref.block_exponent(low), torch.ge), (ref.block_exponent(high), torch.le)):
        assert bool(ok(scale, (bound - fmt[2]).clamp(min=0)).all())
    each = scale.repeat_interleave(ref.BLOCK)[:codes.numel()]
    at_least, at_most = ref.magnitude(low, r, each, fmt), ref.magnitude(high, r, each, fmt)
    if second:
        at_least, at_most = torch.where(low > 0, at_least.clamp(min=1), at_least), torch.where(high > 0, at_most.clamp(min=1), at_most)
        assert bool((codes < 128).all())
    else:
        negative = codes >= 128
        codes = codes & 127
        sure = (codes > 0) & (x.abs() > err)
        assert bool((negative == (x < 0))[sure].all())
    assert bool((codes >= at_least).all()) and bool((codes <= at_most).all())


def _check_step(opt, params, before, t, bits, sr=True):
    """before: (p, g, m, v) of each parameter, float64, ahead of the step that ended at count t."""
    for stream, (p, (p0, g0, m0, v0)) in enumerate(zip(params, before)):
        if p0.numel() == 0:
            continue
        (want, m, v), (ep, em, ev) = ref.step(p0, g0, m0, v0, t, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
        r = ref.noise(p0.numel(), SEED, t, stream)
        got = p.detach().double().cpu().reshape(-1)
        if p.dtype is torch.float32:
            assert bool(((got - want).abs() <= ep).all())
        elif sr:
            # more magnitude rounds to no less
            a, b = want - ep, want + ep
            small, large = torch.minimum(a.abs(), b.abs()), torch.maximum(a.abs(), b.abs())
            same = a * b > 0
            lo, hi = ref.bf16_stochastic(small, r), ref.bf16_stochastic(large, r)
            assert bool(((got.abs() >= lo) | ~same).all()) and bool((got.abs() <= hi).all())
        else:
            assert bool(((got - want).abs() <= ep + 2.0 ** -8 * want.abs() / (1 - 2.0 ** -8)).all())
        s = opt.state[p]
        if bits == 32:
            assert bool(((s["exp_avg"].double().cpu().reshape(-1) - m).abs() <= em + 2.0 ** -149).all())
            assert bool(((s["exp_avg_sq"].double().cpu().reshape(-1) - v).abs() <= ev + 2.0 ** -149).all())
        else:
            turned = ((r << 8) | (r >> 8)) & 0xFFFF
            _check_codes(s["exp_avg"].cpu(), s["exp_avg_scale"].cpu(), m, em, turned, ref.E4M3, False)
            _check_codes(s["exp_avg_sq"].cpu(), s["exp_avg_sq_scale"].cpu(), v, ev, 0xFFFF - r, ref.E5M2, True)


def _before(opt, params, bits):
    out = []
    for p in params:
        p0 = p.detach().double().cpu().reshape(-1)
        m, v = _state(opt, p, bits) if opt.state[p] else (torch.zeros_like(p0), torch.zeros_like(p0))
        out.append((p0, _grad(p).double().cpu().reshape(-1), m, v))
    return out


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,gdtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
def test_three_steps(dtype, gdtype, bits, offset):
    params = _tensors(SIZES, dtype, gdtype, offset)
    opt = DenseAdamW(params, state_bits=bits, seed=SEED, **HYPER)
    for t in range(1, 4):
        before = _before(opt, params, bits)
        opt.step()
        _check_step(opt, params, before, t, bits)
        for p in params:
            _grad(p).mul_(-0.7)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_holds(bits):
    params = _tensors([5 + 37 * i for i in range(97)], torch.bfloat16, torch.bfloat16)
    opt = DenseAdamW(params, state_bits=bits, seed=SEED, **HYPER)
    before = _before(opt, params, bits)
    opt.step()
    _check_step(opt, params, before, 1, bits)


def test_bf16_gradients_of_fp32_parameters_through_the_c_entry():
    """The one pair of types that torch's grads cannot have, but the entry point takes."""
    from micro_engram_fork_amd import ops
    p = torch.randn(1000, device=DEV)
    g = torch.randn(1000, device=DEV).bfloat16()
    m, v = torch.zeros(1000, device=DEV), torch.zeros(1000, device=DEV)
    p0 = p.double().cpu()
    arrays = [ops.ptr_array([x.data_ptr()]) for x in (p, m, v)] + [None, None]
    ops.adamw_launch(p.device, 1, arrays, ops.ptr_array([g.data_ptr()]), ops.i64_array([1000]), ops.f64_array([1.0]), None,
                     ops.i32_array([0]), ops.ME_F32, ops.ME_BF16, 32, lr=HYPER["lr"], betas=HYPER["betas"], eps=HYPER["eps"],
                     weight_decay=HYPER["weight_decay"], stochastic_rounding=True, seed=SEED)
    zero = torch.zeros(1000, dtype=torch.float64)
    (want, _, _), (err, _, _) = ref.step(p0, g.double().cpu(), zero, zero, 1, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
    assert bool(((p.double().cpu() - want).abs() <= err).all())


def test_round_to_nearest_weights():
    params = _tensors([3000], torch.bfloat16, torch.bfloat16)
    opt = DenseAdamW(params, stochastic_rounding=False, seed=SEED, **HYPER)
    before = _before(opt, params, 32)
    opt.step()
    _check_step(opt, params, before, 1, 32, sr=False)


def test_a_parameter_without_gradient_stays_and_counts_apart():
    params = _tensors([300, 400], torch.float32, torch.float32)
    held, params[0].grad = params[0].grad, None
    opt = DenseAdamW(params, seed=SEED, **HYPER)
    was = params[0].detach().clone()
    opt.step()
    assert torch.equal(params[0], was) and not opt.state[params[0]]
    params[0].grad = held
    before = _before(opt, params, 32)
    opt.step()
    _check_step(opt, params[:1], before[:1], 1, 32)
    assert float(opt.state[params[0]]["step"]) == 1 and float(opt.state[params[1]]["step"]) == 2


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_gradient_that_is_not_finite_spoils_its_own_value_only(bits, bad):
    params = _tensors([300], torch.float32, torch.float32)
    params[0].grad[130] = bad
    opt = DenseAdamW(params, state_bits=bits, seed=SEED, **HYPER)
    for _ in range(2):
        opt.step()
    spoiled = ~torch.isfinite(params[0])
    assert spoiled.nonzero().flatten().tolist() == [130]
    m, v = _state(opt, params[0], bits)
    assert [i for i in range(300) if not torch.isfinite(m[i])] == [130] == [i for i in range(300) if not torch.isfinite(v[i])]


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_leave_zero_moments(bits):
    p = torch.nn.Parameter(torch.ones(257, device=DEV))
    p.grad = torch.zeros_like(p)
    opt = DenseAdamW([p], lr=0.5, weight_decay=0.5, state_bits=bits)
    opt.step()
    assert torch.equal(p, torch.full_like(p, 0.75))
    m, v = _state(opt, p, bits)
    assert not m.any() and not v.any()


@pytest.mark.parametrize("size", [1e-30, 1e-17, 1.0, 1e17])
def test_gradients_of_any_size(size):
    """Squares from the smallest fp32 holds to near its largest: scales reach their ends."""
    params = _tensors([1000], torch.float32, torch.float32)
    params[0].grad.mul_(size)
    opt = DenseAdamW(params, state_bits=8, seed=SEED, **HYPER)
    for t in (1, 2):
        before = _before(opt, params, 8)
        opt.step()
        _check_step(opt, params, before, t, 8)
    assert bool(torch.isfinite(params[0]).all())


def test_second_moments_in_8_bits_follow_their_mean():
    """After gradients of one size have settled, 64 times smaller ones bring each moment down, by stochastic rounding
    alone: a step of a thousandth is far less than half a code. The mean over 65,536 values is within five
    standard errors (a value's own spread is below its size)."""
    n, beta2 = 65_536, 0.999
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    p.grad = torch.ones_like(p)
    opt = DenseAdamW([p], lr=0.0, betas=(0.9, beta2), state_bits=8, weight_decay=0.0, seed=5)
    want = 0.0
    for t in range(600):
        if t == 200:
            p.grad.fill_(1 / 64)
        opt.step()
        want = beta2 * want + (1 - beta2) * float(p.grad[0]) ** 2
        if t in (199, 599):
            m, v = _state(opt, p, 8)
            assert abs(float(v.mean()) / want - 1) < 5 / n ** 0.5
            assert abs(float(m.mean()) / float(p.grad[0]) - 1) < 0.05 / n ** 0.5 * 100  # first moments follow at once


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_loaded_state_goes_on_exactly(bits):
    a = _tensors([1000, 129], torch.bfloat16, torch.bfloat16)
    opt = DenseAdamW(a, state_bits=bits, seed=SEED, **HYPER)
    opt.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    other = DenseAdamW(b, state_bits=bits, seed=SEED, **HYPER)
    other.load_state_dict(opt.state_dict())
    for s, t in zip(opt.state.values(), other.state.values()):
        assert {k: x.dtype for k, x in s.items()} == {k: x.dtype for k, x in t.items()}
        assert all(x is not t[k] for k, x in s.items())
    opt.step(), other.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k, x in opt.state[p].items():
            y = other.state[q][k]
            assert torch.equal(x.contiguous().view(torch.uint8) if x.dim() else x, y.contiguous().view(torch.uint8) if y.dim() else y)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_as_eager_ones(bits):
    def make():
        params = _tensors([1000, 129, (40, 50)], torch.bfloat16, torch.bfloat16)
        return params, DenseAdamW(params, state_bits=bits, seed=SEED, capturable=True, **HYPER)
    (a, eager), (b, opt) = make(), make()
    eager.step(), opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        for p, q in zip(a, b):
            p.grad.mul_(-0.9), q.grad.mul_(-0.9)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q), k
            assert float(opt.state[q]["step"]) == float(eager.state[p]["step"]) == k + 2
            for name in ("exp_avg", "exp_avg_sq"):
                x, y = eager.state[p][name], opt.state[q][name]
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_capturable_steps_are_those_of_host_counts():
    a, b = (_tensors([5000], torch.float32, torch.float32) for _ in range(2))
    one, two = DenseAdamW(a, seed=SEED, **HYPER), DenseAdamW(b, seed=SEED, capturable=True, **HYPER)
    for t in range(1, 4):
        before = _before(two, b, 32)
        one.step(), two.step()
        _check_step(two, b, before, t, 32)


def test_a_step_under_capture_needs_capturable():
    params = _tensors([64], torch.float32, torch.float32)
    for opt in (DenseAdamW(params), DenseAdamW(params, capturable=True)):  # the second has no states yet
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(graph):
                opt.step()
        torch.cuda.synchronize()


def test_steps_on_another_stream_and_version_counters():
    params = _tensors([100_000], torch.float32, torch.float32)
    opt = DenseAdamW(params, seed=SEED, **HYPER)
    before, version = _before(opt, params, 32), params[0]._version
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    _check_step(opt, params, before, 1, 32)
    assert params[0]._version > version


def test_gradients_of_other_strides_and_what_changes_between_steps():
    p = torch.nn.Parameter(torch.randn(40, 30, device=DEV))
    opt = DenseAdamW([p], seed=SEED, **HYPER)
    for t in (1, 2, 3):
        p.grad = torch.randn(30, 40, device=DEV).t()
        before = _before(opt, [p], 32)
        opt.step()
        _check_step(opt, [p], before, t, 32)
        p.data = p.data.clone()  # another place


def test_groups_and_fp32_grad():
    a, = _tensors([200], torch.bfloat16, torch.float32)
    b, = _tensors([300], torch.float32, torch.float32)
    opt = DenseAdamW([{"params": [a], "state_bits": 8}, {"params": [b]}], seed=SEED, **HYPER)
    before = _before(opt, [a, b], 32)
    opt.step()
    _check_step(opt, [a], before[:1], 1, 8)
    (want, _, _), (err, _, _) = ref.step(*before[1], 1, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
    assert bool(((b.detach().double().cpu() - want).abs() <= err).all())
    opt.zero_grad(set_to_none=False)
    assert not a.fp32_grad.any() and not b.grad.any()
    opt.zero_grad()
    assert a.fp32_grad is None and b.grad is None
    was = a.detach().clone()
    opt.step()
    assert torch.equal(a, was)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_changes_between_steps_is_noticed(bits):
    """Each of these ends the reuse of what the step before prepared: every step is as one from scratch."""
    params = _tensors([300, 129, 50], torch.bfloat16, torch.bfloat16)
    opt = DenseAdamW(params, state_bits=bits, seed=SEED, **HYPER)
    counts = [0, 0, 0]

    def step():
        live = [k for k, p in enumerate(params) if p.grad is not None or getattr(p, "fp32_grad", None) is not None]
        before = {k: _before(opt, [params[k]], bits)[0] for k in live}
        held = [p.detach().clone() for p in params]
        opt.step()
        for k, p in enumerate(params):
            if k not in live:
                assert torch.equal(p, held[k])
                continue
            counts[k] += 1
            assert float(opt.state[p]["step"]) == counts[k]
            _check_one(opt, p, before[k], counts[k], bits, k)
    step(), step()
    params[1].grad = None                                              # one rests
    step(), step()
    params[1].grad = torch.randn_like(params[1])                       # and comes back, another rests
    params[0].grad = None
    step()
    params[0].fp32_grad = torch.randn(params[0].shape, device=DEV)     # a wide gradient
    step(), step()
    params[0].fp32_grad = params[0].fp32_grad[::1].clone()             # another tensor
    step()
    params[2].data = torch.randn(50, device=DEV).bfloat16()            # another place
    step()
    s = opt.state[params[2]]
    s["exp_avg"] = s["exp_avg"].clone()                                # other states
    step()
    opt.state[params[2]] = dict(s)
    step()
    s["step"].fill_(99.0)                                              # no longer the parameter's own
    opt.state[params[1]]["step"] = torch.tensor(7.0)                   # another count
    counts[1] = 7
    opt.state[params[2]]["step"] = torch.tensor(float(counts[2]))
    step()
    params[1].grad = torch.randn(129 * 2, device=DEV).bfloat16()[::2]  # strides
    step()
    opt.param_groups[0]["lr"] = HYPER["lr"]
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3, device=DEV))]})
    step()


def _check_one(opt, p, before, t, bits, stream):
    """_check_step of one parameter with the noise of its place."""
    noise = ref.noise
    try:
        ref.noise = lambda n, seed, step, _: noise(n, seed, step, stream)
        _check_step(opt, [p], [before], t, bits)
    finally:
        ref.noise = noise


def test_the_state_of_torchs_adamw_goes_on():
    """bf16 parameters whose moments torch keeps in bf16: they go on in fp32 from there."""
    p = torch.nn.Parameter(torch.randn(700, device=DEV).bfloat16())
    p.grad = torch.randn(700, device=DEV).bfloat16()
    torchs = torch.optim.AdamW([p], **HYPER)
    torchs.step()
    opt = DenseAdamW([p], seed=SEED)
    opt.load_state_dict(torchs.state_dict())
    assert opt.state[p]["exp_avg"].dtype is torch.float32
    assert torch.equal(opt.state[p]["exp_avg"], torchs.state[p]["exp_avg"].float())
    before = _before(opt, [p], 32)
    opt.step()
    _check_step(opt, [p], before, 2, 32)


@pytest.mark.parametrize("bits", [8, 32])
def test_more_values_than_32_bits_count(bits):
    """A first step moves each value with a gradient by the learning rate, against its sign, and no other."""
    p = torch.nn.Parameter(torch.zeros(2_200_000_123, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros_like(p)
    at = torch.tensor([0, 4_095, 2_147_483_647, 2_147_483_648, 2_199_999_990, 2_200_000_122], device="cuda")
    p.grad[at] = torch.tensor([1.0, -1.0, 2.0, -3.0, 1.0, -0.5], device="cuda", dtype=torch.bfloat16)
    DenseAdamW([p], lr=2.0 ** -7, state_bits=bits, weight_decay=0.0, seed=1).step()
    with torch.no_grad():
        # m / (sqrt(v) + eps) is 1 but for eps / |g|, the quotient's roundings and that of the weight, 2^-7 at most
        assert torch.allclose(p[at].float(), -(2.0 ** -7) * p.grad[at].float().sign(), rtol=2.0 ** -7 + 1e-6, atol=0.0)
        assert int(p.count_nonzero()) == len(at)
    del p
    torch.cuda.empty_cache()

"""What the losses over a decoder's head refuse, and the shapes that tracing sees."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from micro_engram_fork_amd import _lib, head_ops, losses

CALLS = [losses.head_cross_entropy, losses.head_token_logps]


def _args(rows=(2, 3), vocab=11, dim=8, dtype=torch.bfloat16):
    return torch.zeros(*rows, dim, dtype=dtype), torch.zeros(vocab, dim, dtype=dtype), torch.zeros(rows, dtype=torch.long)


@pytest.mark.parametrize("call", CALLS)
def test_shapes_and_types(call):
    hidden, weight, targets = _args()
    for bad in ((hidden[..., :7], weight, targets), (hidden, weight[0], targets), (hidden, weight[:0], targets),
                (hidden, weight[None], targets), (hidden, weight, targets[:, :2]), (hidden, weight, targets[..., None])):
        with pytest.raises(ValueError, match="micro_engram"):
            call(*bad)
    for bad in ((hidden.float(), weight, targets), (hidden, weight.float(), targets), (hidden.half(), weight.half(), targets),
                (hidden.double(), weight.double(), targets), (hidden, weight, targets.float()), (hidden, weight, targets.to(torch.int16))):
        with pytest.raises(TypeError, match="micro_engram"):
            call(*bad)
    with pytest.raises(ValueError, match="temperature"):
        call(*_args(), temperature=0.0)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        call(*_args())


@pytest.mark.parametrize("bad", [dict(label_smoothing=-0.1), dict(label_smoothing=1.1), dict(z_loss=-1.0), dict(z_loss=float("nan")),
                                 dict(scale=float("inf")), dict(reduction="none"), dict(reduction="sequence"), dict(temperature=float("nan"))])
def test_options(bad):
    with pytest.raises(ValueError, match="micro_engram"):
        losses.head_cross_entropy(*_args(), **bad)


def test_c_entry_checks():
    """The C entry refuses what its kernels do not hold, before any launch."""
    p = 4096  # an address that is not read

    def logps(dtype=_lib.ME_BF16, n=4, dim=8, vocab=11, stride=8, tdtype=_lib.ME_I64, temperature=1.0, size=1 << 40, ws=p, saved=p):
        _lib.call("me_head_logps", p, dtype, n, dim, max(n, 1), 0, dim, p, vocab, stride, p, tdtype, -100, temperature, p, saved, None, ws, size, None)
    for bad in (dict(dtype=_lib.ME_I32), dict(n=-1), dict(n=1 << 25), dict(dim=0), dict(dim=65537), dict(vocab=0), dict(vocab=1 << 22),
                dict(stride=7), dict(stride=1 << 23), dict(tdtype=_lib.ME_F32), dict(temperature=0.0), dict(temperature=float("nan")),
                dict(size=16), dict(ws=None), dict(saved=None), dict(ws=p + 8)):
        with pytest.raises(_lib.EngramLibError):
            logps(**bad)


def test_fake_shapes():
    with FakeTensorMode():
        hidden, weight, targets = _args()
        out, saved = head_ops.head_logps(hidden, weight, targets, -100, 1.0, head_ops.NO_GRADIENT)
        assert out.shape == (2, 3) and out.dtype is torch.float32
        loss, saved = head_ops.head_ce(hidden, weight, targets, -100, 1.0, 0.0, 0.0, 1.0, 0, head_ops.NO_GRADIENT)
        assert loss.shape == () and saved.shape == (16 + 5 * 6,)
        both = head_ops.head_backward(hidden, weight, targets, saved, None, loss, -100, 1.0, False, 0.0, 0.0, 1.0, 0, True, True)
        assert [g.shape for g in both] == [hidden.shape, weight.shape] and both[1].dtype is torch.bfloat16
        one, = head_ops.head_backward(hidden, weight, targets, saved, None, loss, -100, 1.0, False, 0.0, 0.0, 1.0, 0, False, True)
        assert one.shape == weight.shape


def test_what_a_forward_leaves_for_the_gradient_of_hidden_alone():
    """Nothing for small calls; fp32 values of every row, in whole fours, for those worth it."""
    of = head_ops.OF_HIDDEN
    assert head_ops.unit_elements(64, 300, 64, _lib.ME_BF16, of) == 0
    assert head_ops.unit_elements(0, 262_144, 5_376, _lib.ME_BF16, of) == 0
    assert head_ops.unit_elements(3, 262_144, 5_375, _lib.ME_BF16, of) == 3 * 5_376
    assert head_ops.unit_elements(3, 262_144, 5_375, _lib.ME_BF16, head_ops.OF_WEIGHT) == 0
    assert head_ops.unit_elements(3, 262_144, 5_375, _lib.ME_BF16, head_ops.NO_GRADIENT) == 0
    for of in (head_ops.OF_HIDDEN, head_ops.OF_WEIGHT):  # few rows of fp32: their logits
        assert head_ops.unit_elements(384, 262_144, 64, _lib.ME_F32, of) == 384 * (262_144 + 64)
        assert head_ops.unit_elements(385, 262_144, 64, _lib.ME_F32, of) == 262_144 * 64 + 262_144 + 256 + 4  # the head in parts
        assert head_ops.unit_elements(385, 262_144, 1_025, _lib.ME_F32, of) == 0
        assert head_ops.unit_elements(1024, 301, 64, _lib.ME_F32, of) == 1024 * 320
        assert head_ops.unit_elements(1025, 301, 64, _lib.ME_F32, of) == 301 * 64 + 304 + 256 + 4
        assert head_ops.unit_elements(0, 301, 64, _lib.ME_F32, of) == 0
    with FakeTensorMode():
        hidden, weight, targets = _args(rows=(4096,), vocab=32_000, dim=1_024)
        _, saved, unit = head_ops.head_ce(hidden, weight, targets, -100, 1.0, 0.0, 0.0, 1.0, 0, head_ops.OF_HIDDEN)
        assert unit.shape == (4096 * 1024,) and unit.dtype is torch.float32


class _Reached(Exception):
    pass


class _Wrapped(torch.Tensor):
    """A tensor subclass without memory of its own, which ends a call at the first of this library's ops that it reaches."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        if func.namespace == "micro_engram_amd":
            raise _Reached(func.name())
        res = func(*(a.inner if isinstance(a, cls) else a for a in args), **(kwargs or {}))
        return cls(res) if isinstance(res, torch.Tensor) else res


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("call", CALLS)
def test_tensor_subclasses_go_through_the_ops(call, which, grad):
    args = list(_args())
    args[0].requires_grad_(grad)
    args[which] = _Wrapped(args[which])
    with pytest.raises(_Reached):
        call(*args)


@pytest.mark.parametrize("n,vocab,dim,apart", [((1 << 24) + 1, 4, 8, 8), (4, (1 << 21) + 1, 8, 8), (4, 4, 65_537, 65_537), (1 << 24, 4, 32_768, 32_768),
                                               (4, 4, 8, (1 << 22) + 8), (4, 4, 8, 7)])
def test_sizes_past_the_limits(n, vocab, dim, apart):
    """Refused when the workspace is asked for, before any is allocated."""
    for dtype in (_lib.ME_F32, _lib.ME_BF16):
        with pytest.raises(RuntimeError, match="must be"):
            head_ops.workspace_bytes(n, vocab, dim, dtype, 0, apart, 0, False)

"""Arguments of the losses that decide what the kernels read: shapes that do not hold what a call would read are
refused, shapes that do reach the GPU's own check."""
import pytest
import torch

from micro_engram_fork_amd import _lib, loss_ops, losses


def _policy(shape, advantages, sequences=None):
    """policy_loss on targets of `shape`, packed as `sequences` sequences where that is given."""
    n = int(torch.Size(shape).numel())
    cu = None if sequences is None else torch.linspace(0, n, sequences + 1).long()
    return losses.policy_loss(torch.zeros(*shape, 11), torch.zeros(shape, dtype=torch.long), torch.zeros(shape),
                              torch.zeros(advantages), cu_seqlens=cu)


@pytest.mark.parametrize("shape,advantages,sequences", [
    ((10,), (1,), 3), ((10,), (1, 1), 3), ((1, 10), (1, 1), 3), ((1, 10), (1,), 5), ((2, 5), (2, 1), 5), ((2, 5), (2,), 3),
    ((2, 5), (5, 1), 4), ((2, 3, 4), (2, 3, 1), 5), ((10,), (4,), 5), ((10,), (6, 1), 5),
    ((2, 3, 4), (5,), None), ((2, 3), (3, 1), None), ((4,), (2,), None),
])
def test_advantages_of_another_number_of_sequences_are_refused(shape, advantages, sequences):
    with pytest.raises(ValueError, match="advantages"):
        _policy(shape, advantages, sequences)


@pytest.mark.parametrize("shape,advantages,sequences", [
    ((10,), (10,), 3), ((10,), (3,), 3), ((10,), (3, 1), 3), ((1, 10), (1, 10), 3), ((1, 10), (3,), 3), ((1, 10), (3, 1), 3),
    ((2, 5), (2, 1), 2), ((10,), (1,), 1), ((2, 5), (2, 1), None), ((2, 5), (2,), None), ((2, 3, 4), (2, 3, 1), None),
    ((2, 3, 4), (6,), None), ((2, 3, 4), (6, 1), None), ((4,), (1,), None), ((4,), (4,), None),
])
def test_advantages_of_the_tokens_or_the_sequences_pass(shape, advantages, sequences):
    with pytest.raises(RuntimeError, match="only on the GPU"):
        _policy(shape, advantages, sequences)


class _Reached(Exception):
    pass


class _Wrapped(torch.Tensor):
    """A tensor subclass without memory of its own (as sharded or quantised tensors are), which ends a call at the
    first of this library's ops that it reaches."""

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


def _loss_with(name, wrapped, grad):
    """The loss with its argument `wrapped` as such a subclass."""
    rows, vocab = (2, 3), 11
    args = dict(logits=torch.zeros(*rows, vocab, requires_grad=grad))
    if name == "distill_loss":
        args.update(teacher_ids=torch.zeros(*rows, 2, dtype=torch.long), teacher_logits=torch.zeros(*rows, 2),
                    teacher_lse=torch.zeros(rows), mask=torch.ones(rows, dtype=torch.bool))
    else:
        args["targets"] = torch.zeros(rows, dtype=torch.long)
    if name == "preference_loss":
        args.update(ref_logps=torch.zeros(rows), cu_seqlens=torch.tensor([0, 3, 6]))
    if name == "policy_loss":
        args.update(old_logps=torch.zeros(rows), advantages=torch.zeros(2), ref_logps=torch.zeros(rows),
                    cu_seqlens=torch.tensor([0, 3, 6]))
    args[wrapped] = _Wrapped(args[wrapped])
    return getattr(losses, name)(**args)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name,wrapped", [
    ("token_logps", "targets"), ("preference_loss", "targets"), ("preference_loss", "ref_logps"), ("preference_loss", "cu_seqlens"),
    ("policy_loss", "old_logps"), ("policy_loss", "advantages"), ("policy_loss", "ref_logps"), ("policy_loss", "cu_seqlens"),
    ("distill_loss", "teacher_ids"), ("distill_loss", "teacher_logits"), ("distill_loss", "teacher_lse"), ("distill_loss", "mask"),
])
def test_tensor_subclasses_in_any_argument_reach_the_op(name, wrapped, grad):
    # not the kernels with the subclass's own address, which is none: an optional argument would count as not given
    with pytest.raises(_Reached, match="micro_engram_amd::" + name.replace("_loss", "")):
        _loss_with(name, wrapped, grad)


@pytest.fixture
def entry_calls(monkeypatch):
    """The losses without their kernels: names of the library's entry points in the order of their calls."""
    names = []
    monkeypatch.setattr(loss_ops, "call", lambda name, *args: names.append(name))
    monkeypatch.setattr(loss_ops, "require_gpu", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(loss_ops, "stream_of", lambda device: 0)
    monkeypatch.setattr(loss_ops, "workspace_bytes", lambda *sizes: 256)
    return names


def _plain_loss(name, logits):
    rows = logits.shape[:-1]
    targets, values = torch.zeros(rows, dtype=torch.long), torch.zeros(rows)
    if name == "token_logps":
        return losses.token_logps(logits, targets)
    if name == "preference_loss":
        return losses.preference_loss(logits, targets, values)[0]
    if name == "policy_loss":
        return losses.policy_loss(logits, targets, values, values)[0]
    return losses.distill_loss(logits, targets[..., None], values[..., None])


NAMES = ["token_logps", "preference_loss", "policy_loss", "distill_loss"]


@pytest.mark.parametrize("name", NAMES)
def test_an_upstream_gradient_of_a_subclass_reaches_the_op(entry_calls, name):
    logits = torch.zeros(2, 3, 11, requires_grad=True)
    loss = _plain_loss(name, logits)
    with pytest.raises(_Reached, match="backward"):
        torch.autograd.grad(loss, logits, _Wrapped(torch.full(loss.shape, 3.0)))
    assert len(entry_calls) == 1
    torch.autograd.grad(_plain_loss(name, logits), logits, torch.full(loss.shape, 3.0))
    assert len(entry_calls) == 3 and entry_calls[2].endswith("_backward")


@pytest.mark.parametrize("name", NAMES)
def test_saved_tensor_hooks_get_all_that_a_backward_needs(entry_calls, name):
    # hooks that move saved tensors off the GPU, or make them again, find the logits nowhere else in the graph
    packed, logits = [], torch.zeros(2, 3, 11, requires_grad=True)

    def pack(t):
        packed.append(t.shape)
        return t.clone()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        loss = _plain_loss(name, logits * 1)
    assert torch.Size((2, 3, 11)) in packed
    assert loss.grad_fn.run is None  # the prepared call would hold them
    torch.autograd.grad(loss, logits, torch.ones(loss.shape))
    assert len(entry_calls) == 2 and entry_calls[1].endswith("_backward")
    loss = _plain_loss(name, logits * 1)
    assert loss.grad_fn.run is not None


@pytest.mark.parametrize("shape", [(2, 3, 0, 10), (2, 0, 3, 10), (0, 2, 3, 10), (2, 2, 0, 3, 10), (2, 0, 10), (0, 10)])
def test_row_layout_of_no_rows(shape):
    logits, args = loss_ops.row_layout(torch.zeros(shape))
    assert logits.shape == shape and args[2:5] == (0, 10, max(1, shape[-2]))


@pytest.mark.parametrize("name", NAMES)
def test_logits_of_no_rows_in_many_dims(entry_calls, name):
    logits = torch.zeros(2, 3, 0, 10, requires_grad=True)
    loss = _plain_loss(name, logits)
    assert torch.autograd.grad(loss, logits, torch.ones(loss.shape))[0].shape == logits.shape


def _entry_args(name, n, vocab, dtype):
    """Arguments of entry point `name` for n rows, with addresses that no refused call reads."""
    at, logits, targets = 64, (64, dtype, n, vocab, n, 0, vocab), (64, _lib.ME_I64, -100)
    space = (at, 1 << 62, None)
    return {
        "me_token_logps": (*logits, *targets, 1.0, at, at, *space),
        "me_token_logps_backward": (*logits, *targets, 1.0, at, at, 1.0, None, 0, at, None),
        "me_preference": (*logits, *targets, at, at, _lib.ME_I64, 1, 0, 0, 0.1, 0.0, 0, at, at, at, at, at, *space),
        "me_policy": (*logits, *targets, at, at, 0, None, None, 0, 1, n, 0.2, 0.2, 0.0, 1.0, 1.0, 0, at, at, at, at, at, at, *space),
        "me_distill": (*logits, at, _lib.ME_I64, at, _lib.ME_F32, 1, None, None, 1.0, 1.0, 0, at, at, at, at, at, *space),
        "me_distill_backward": (*logits, at, _lib.ME_I64, 1, 1.0, at, at, at, None, 0, at, None),
    }[name]


@pytest.mark.parametrize("name", ["me_token_logps", "me_token_logps_backward", "me_preference", "me_policy", "me_distill",
                                  "me_distill_backward"])
@pytest.mark.parametrize("n,vocab,dtype", [((1 << 26) - 16, 64, _lib.ME_BF16), ((1 << 24) - 16, 4096, _lib.ME_F32),
                                           (1 << 23, 8200, _lib.ME_BF16), ((1 << 31) - 1, 2, _lib.ME_BF16)])
def test_rows_past_what_a_launch_holds_are_refused(name, n, vocab, dtype):
    # a launch of 2^32 threads runs only those past the 32 bits that count them, without an error
    with pytest.raises(_lib.EngramLibError, match="too many rows"):
        _lib.call(name, *_entry_args(name, n, vocab, dtype))

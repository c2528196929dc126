"""Host side of the losses over logits: refusals with a message before anything reaches the GPU, shapes under
tracing, workspace sizes, and the float64 reference itself on small cases worked out by hand."""
import math

import pytest
import torch

import loss_reference as ref64
from micro_engram_fork_amd import _lib, loss_ops, losses


def _call(**kw):
    base = dict(logits=torch.zeros(2, 3, 11), targets=torch.zeros(2, 3, dtype=torch.long))
    base.update(kw)
    return base


@pytest.mark.parametrize("kw,error,text", [
    (dict(logits=torch.zeros(2, 3, 11, dtype=torch.float16)), TypeError, "bf16 or fp32"),
    (dict(logits=torch.zeros(2, 3, 0)), ValueError, "vocab"),
    (dict(targets=torch.zeros(2, 4, dtype=torch.long)), ValueError, "do not match"),
    (dict(targets=torch.zeros(2, 3)), TypeError, "int32 or int64"),
    (dict(temperature=0.0), ValueError, "temperature"),
    (dict(temperature=float("nan")), ValueError, "temperature"),
    (dict(), RuntimeError, "only on the GPU"),
])
def test_token_logps_refusals(kw, error, text):
    with pytest.raises(error, match=text):
        losses.token_logps(**_call(**kw))


@pytest.mark.parametrize("kw,error,text", [
    (dict(ref_logps=torch.zeros(2, 4)), ValueError, "ref_logps"),
    (dict(ref_logps=torch.zeros(2, 3, dtype=torch.long)), TypeError, "floating"),
    (dict(loss_type="other"), ValueError, "loss_type"),
    (dict(beta=0.0), ValueError, "beta"),
    (dict(label_smoothing=1.5), ValueError, "label_smoothing"),
    (dict(loss_type="ipo", label_smoothing=0.1), ValueError, "sigmoid"),
    (dict(cu_seqlens=torch.tensor([0, 2, 4, 6])), ValueError, "no pairs"),
    (dict(cu_seqlens=torch.zeros(2, 2, dtype=torch.long)), ValueError, "cu_seqlens"),
    (dict(cu_seqlens=torch.tensor([0.0, 3.0, 6.0])), TypeError, "cu_seqlens"),
    (dict(logits=torch.zeros(6, 11), targets=torch.zeros(6, dtype=torch.long), ref_logps=torch.zeros(6)), ValueError, "packed"),
    (dict(logits=torch.zeros(3, 2, 11), targets=torch.zeros(3, 2, dtype=torch.long), ref_logps=torch.zeros(3, 2)), ValueError,
     "no pairs"),
    (dict(), RuntimeError, "only on the GPU"),
])
def test_preference_refusals(kw, error, text):
    with pytest.raises(error, match=text):
        losses.preference_loss(**_call(**{"ref_logps": torch.zeros(2, 3), **kw}))


@pytest.mark.parametrize("kw,error,text", [
    (dict(old_logps=torch.zeros(2)), ValueError, "old_logps"),
    (dict(advantages=torch.zeros(3)), ValueError, "advantages"),
    (dict(advantages=torch.zeros(2, dtype=torch.long)), TypeError, "floating"),
    (dict(reduction="mean"), ValueError, "reduction"),
    (dict(clip_low=-0.1), ValueError, "clip_low"),
    (dict(kl_coef=0.1), ValueError, "ref_logps"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(), RuntimeError, "only on the GPU"),
])
def test_policy_refusals(kw, error, text):
    with pytest.raises(error, match=text):
        losses.policy_loss(**_call(**{"old_logps": torch.zeros(2, 3), "advantages": torch.zeros(2), **kw}))


@pytest.mark.parametrize("kw,error,text", [
    (dict(teacher_ids=torch.zeros(2, 4, 5, dtype=torch.long)), ValueError, "teacher_ids"),
    (dict(teacher_ids=torch.zeros(2, 3, 5)), TypeError, "int32 or int64"),
    (dict(teacher_logits=torch.zeros(2, 3, 4)), ValueError, "teacher_logits"),
    (dict(teacher_logits=torch.zeros(2, 3, 5, dtype=torch.float64)), TypeError, "teacher_logits"),
    (dict(teacher_ids=torch.zeros(2, 3, 0, dtype=torch.long), teacher_logits=torch.zeros(2, 3, 0)), ValueError, "entries"),
    (dict(teacher_ids=torch.zeros(2, 3, 1025, dtype=torch.long), teacher_logits=torch.zeros(2, 3, 1025)), ValueError, "entries"),
    (dict(teacher_ids=torch.zeros(2, 3, 11, dtype=torch.long), teacher_logits=torch.zeros(2, 3, 11),
          teacher_lse=torch.zeros(2, 3)), ValueError, "no rest"),
    (dict(mask=torch.zeros(2, 3)), ValueError, "mask"),
    (dict(reduction="token"), ValueError, "reduction"),
    (dict(), RuntimeError, "only on the GPU"),
])
def test_distill_refusals(kw, error, text):
    base = dict(logits=torch.zeros(2, 3, 11), teacher_ids=torch.zeros(2, 3, 5, dtype=torch.long), teacher_logits=torch.zeros(2, 3, 5))
    with pytest.raises(error, match=text):
        losses.distill_loss(**{**base, **kw})


def _logits_args(n=4, vocab=10, dtype=_lib.ME_F32):
    return 64, dtype, n, vocab, n, 0, vocab


def test_c_entries_refuse_bad_arguments_before_the_gpu():
    targets = (64, _lib.ME_I64, -100)
    with pytest.raises(_lib.EngramLibError, match="vocab"):
        _lib.call("me_token_logps", *_logits_args(vocab=0), *targets, 1.0, 64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="vocab"):
        _lib.call("me_token_logps", *_logits_args(vocab=1 << 40), *targets, 1.0, 64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="bf16 or fp32"):
        _lib.call("me_token_logps", *_logits_args(dtype=_lib.ME_I32), *targets, 1.0, 64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="n out of range"):
        _lib.call("me_token_logps", *_logits_args(n=-1), *targets, 1.0, 64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="temperature"):
        _lib.call("me_token_logps", *_logits_args(), *targets, 0.0, 64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="targets"):
        _lib.call("me_token_logps", *_logits_args(), None, _lib.ME_I64, -100, 1.0, 64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="workspace"):
        _lib.call("me_token_logps", *_logits_args(), *targets, 1.0, 64, None, 64, 16, None)
    with pytest.raises(_lib.EngramLibError, match="workspace"):
        _lib.call("me_token_logps", *_logits_args(), *targets, 1.0, 64, None, None, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="null"):
        _lib.call("me_token_logps_backward", *_logits_args(), *targets, 1.0, 64, 64, 1.0, None, 0, None, None)
    with pytest.raises(_lib.EngramLibError, match="upstream"):
        _lib.call("me_token_logps_backward", *_logits_args(), *targets, 1.0, 64, 64, 1.0, None, 1, 64, None)
    with pytest.raises(_lib.EngramLibError, match="sequences"):
        _lib.call("me_preference", *_logits_args(), *targets, 64, None, 0, 1, 3, 0, 0.1, 0.0, 0, 64, 64, 64, 64, 64, 64,
                  1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="kind"):
        _lib.call("me_preference", *_logits_args(), *targets, 64, None, 0, 1, 2, 9, 0.1, 0.0, 0, 64, 64, 64, 64, 64, 64,
                  1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="reduction"):
        _lib.call("me_policy", *_logits_args(), *targets, 64, 64, 0, None, None, 0, 1, 4, 0.2, 0.2, 0.0, 1.0, 1.0, 7, 64, 64,
                  64, 64, 64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="top"):
        _lib.call("me_distill", *_logits_args(), 64, _lib.ME_I64, 64, _lib.ME_F32, 2000, None, None, 1.0, 1.0, 0, 64, 64, 64,
                  64, None, 64, 1 << 20, None)
    with pytest.raises(_lib.EngramLibError, match="no rest"):
        _lib.call("me_distill", *_logits_args(), 64, _lib.ME_I64, 64, _lib.ME_F32, 10, 64, None, 1.0, 1.0, 0, 64, 64, 64, 64,
                  None, 64, 1 << 20, None)


def test_workspace_grows_with_the_rows():
    small, large = loss_ops.workspace_bytes(1, 262_144), loss_ops.workspace_bytes(8192, 262_144)
    assert 0 < small < large < 64 << 20


def test_row_layout_reads_views_in_place():
    base = torch.zeros(3, 6, 20)
    view, args = loss_ops.row_layout(base[:, 1:, :17])
    assert args[2:] == (15, 17, 5, 120, 20) and args[0] == base.data_ptr() + 80
    assert loss_ops.row_layout(base[0, :, :17])[1][2:] == (6, 17, 6, 0, 20)
    assert loss_ops.row_layout(base[0, 0])[1][2:] == (1, 20, 1, 0, 0)
    moved, args = loss_ops.row_layout(base.transpose(1, 2))  # values apart: copied
    assert moved.is_contiguous() and args[2:] == (60, 6, 20, 120, 6)
    four, args = loss_ops.row_layout(base.view(3, 2, 3, 20)[:, :, 1:])
    assert args[2:] == (12, 20, 2, 60, 20) and args[0] == base.data_ptr() + 80


def test_fake_tensors_reach_the_ops():
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 3, 50, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        t = torch.empty(2, 3, dtype=torch.long, device="cuda")
        rows = torch.empty(2, 3, device="cuda")
        out = losses.token_logps(x, t)
        assert isinstance(out, FakeTensor) and out.shape == (2, 3) and out.dtype == torch.float32
        loss, chosen, rejected = losses.preference_loss(x, t, rows)
        assert loss.shape == () and chosen.shape == (1,) and rejected.shape == (1,)
        loss, logps, stats = losses.policy_loss(x, t, rows, rows)
        assert loss.shape == () and logps.shape == (2, 3) and stats.shape == (2,)
        top = torch.empty(2, 3, 4, dtype=torch.long, device="cuda")
        assert losses.distill_loss(x, top, top.float()).shape == ()


def test_reference_by_hand():
    # two tokens of probabilities 1/4 and 3/4
    x = torch.tensor([[0.0, math.log(3.0)]], dtype=torch.float64)
    t = torch.tensor([0])
    assert float(ref64.token_logps(x, t)) == pytest.approx(math.log(0.25))
    assert float(ref64.token_logps(x, torch.tensor([-100]))) == 0
    ok, w = torch.tensor([True]), torch.ones(1, dtype=torch.float64)
    loss, _, stats = ref64.policy(x, t, torch.tensor([math.log(0.125)]), torch.ones(1).double(), torch.tensor([math.log(0.25)]), w,
                                  ok, 0.2, 0.2, 1.0, 1.0)
    assert float(loss) == pytest.approx(-1.2) and stats.tolist() == pytest.approx([0.0, 1.0], abs=1e-9)
    loss, chosen, rejected = ref64.preference(x.repeat(2, 1), torch.tensor([1, 0]), torch.zeros(2), [0, 1, 2], 1.0, "sigmoid")
    assert float(loss) == pytest.approx(math.log(1 + 1 / 3)) and float(chosen) == pytest.approx(math.log(0.75))
    full = ref64.distill(x, torch.tensor([[0, 1]]), torch.zeros(1, 2), None, ok, w, 1.0)
    assert float(full) == pytest.approx(0.5 * math.log(0.5 / 0.25) + 0.5 * math.log(0.5 / 0.75))
    rest = ref64.distill(x, torch.tensor([[0]]), torch.zeros(1, 1), torch.tensor([math.log(2.0)]), ok, w, 1.0)
    assert float(rest) == pytest.approx(float(full))

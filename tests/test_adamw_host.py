"""What DenseAdamW refuses, and its reference's own roundings."""
import pytest
import torch

import adamw_reference as ref
from micro_engram_fork_amd.optim import DenseAdamW


def _param(dtype=torch.float32):
    p = torch.nn.Parameter(torch.zeros(4, dtype=dtype))
    p.grad = torch.zeros_like(p)
    return p


@pytest.mark.parametrize("bad", [dict(state_bits=16), dict(state_bits="8"), dict(lr=-1.0), dict(lr=float("nan")), dict(eps=-1e-8), dict(eps=1e-40), dict(eps=1e-60),
                                 dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(betas=(0.9,)), dict(weight_decay=-1.0)])
def test_hyperparameters(bad):
    with pytest.raises(ValueError, match="micro_engram"):
        DenseAdamW([_param()], **bad)
    opt = DenseAdamW([_param()])
    with pytest.raises(ValueError, match="micro_engram"):
        opt.add_param_group({"params": [_param()], **bad})
    assert len(opt.param_groups) == 1


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_parameter_types(dtype):
    with pytest.raises(TypeError, match="bf16 or fp32"):
        DenseAdamW([_param(dtype)])


def test_parameters_on_the_cpu_are_refused():
    with pytest.raises(RuntimeError, match="only on the GPU"):
        DenseAdamW([_param()]).step()


def test_gradients():
    p = _param(torch.bfloat16)
    p.fp32_grad = torch.zeros(4, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="fp32_grad"):
        DenseAdamW([p]).step()
    p.fp32_grad = torch.zeros(5)
    with pytest.raises(ValueError, match="shape and device"):
        DenseAdamW([p]).step()
    p = _param()
    p.sparse_grad = (torch.zeros(1, dtype=torch.long), torch.zeros(1, 4))
    with pytest.raises(ValueError, match="LazyAdamW"):
        DenseAdamW([p]).step()
    p = torch.nn.Parameter(torch.zeros(4, 2))
    p.grad = torch.zeros(4, 2).to_sparse()
    with pytest.raises(ValueError, match="dense"):
        DenseAdamW([p]).step()


def test_no_gradients_no_step():
    p = torch.nn.Parameter(torch.zeros(4))
    assert DenseAdamW([p]).step(lambda: 3.0) == 3.0


def test_the_reference_rounds_to_torchs_codes():
    """With noise of one half, codes of exactly representable values are torch's own."""
    for kind, fmt in ((torch.float8_e4m3fn, ref.E4M3), (torch.float8_e5m2, ref.E5M2)):
        codes = torch.arange(0, 0x78 if kind is torch.float8_e4m3fn else 0x78)
        x = codes.to(torch.uint8).view(kind).float().double()
        for r in (0, 32768, 65535):
            assert torch.equal(ref.magnitude(x, torch.full_like(codes, r), torch.full_like(codes, 127), fmt), codes)


def test_philox_known_answer():
    """The published vectors of Philox4x32-10 (Salmon et al., Random123's kat_vectors)."""
    import numpy as np
    out = ref.philox(np.zeros((1, 4), dtype=np.uint64), (0, 0))[0]
    assert [int(x) for x in out] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = np.full((1, 4), 0xFFFFFFFF, dtype=np.uint64)
    out = ref.philox(ones, (0xFFFFFFFF, 0xFFFFFFFF))[0]
    assert [int(x) for x in out] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_a_parameter_twice():
    p = _param()
    with pytest.raises(ValueError, match="twice"):
        with pytest.warns(UserWarning):
            DenseAdamW([p, p])


def test_copies_and_older_states_have_every_setting():
    import copy
    import pickle
    opt = DenseAdamW([_param()], state_bits=8, seed=11)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.seed == 11 and other.param_groups[0]["state_bits"] == 8
    state = torch.optim.AdamW([_param()], lr=0.25).state_dict()
    opt.load_state_dict(state)
    group = opt.param_groups[0]
    assert group["lr"] == 0.25 and group["seed"] == 11 and group["state_bits"] == 8
    saved = DenseAdamW([_param()], seed=5).state_dict()
    opt.load_state_dict(saved)
    assert opt.seed == 5 and opt.param_groups[0]["state_bits"] == 32


@pytest.mark.parametrize("torchs", [lambda p: torch.optim.AdamW(p, amsgrad=True), lambda p: torch.optim.AdamW(p, maximize=True), torch.optim.Adam])
def test_states_of_other_formulas_are_refused(torchs):
    """And nothing of them is taken."""
    p = _param()
    state = torchs([p]).state_dict()
    if torchs is torch.optim.Adam and "decoupled_weight_decay" not in state["param_groups"][0]:
        pytest.skip("this torch's Adam does not say so")
    opt = DenseAdamW([p], lr=0.25)
    with pytest.raises(ValueError, match="not supported"):
        opt.load_state_dict(state)
    assert opt.param_groups[0]["lr"] == 0.25 and "amsgrad" not in opt.param_groups[0]
    plain = torch.optim.AdamW([p], lr=0.5)
    opt.load_state_dict(plain.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5

"""Arguments of the losses that decide what the kernels read: shapes that do not hold what a call would read are
refused, shapes that do reach the GPU's own check."""
import pytest
import torch

from micro_engram_fork_amd import losses


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

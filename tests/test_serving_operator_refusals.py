"""The operators of a serving step refuse tensors that are not on a GPU before they look at anything else: there is no CPU path."""

import pytest
import torch

from matricxon_b200.ops import kernels
from matricxon_b200.ops.library import KernelLibraryError


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_step_tables():
    with pytest.raises(KernelLibraryError, match="CUDA"):
        kernels.step_tables(ints(2), ints(2), ints(2), ints(2, 4), ints(4), ints(1), 16, 8, ints(2), ints(2), ints(3), ints(2),
                            ints(2, 4), ints(1), ints(1))


def test_paged_attention_shared():
    with pytest.raises(KernelLibraryError, match="CUDA"):
        kernels.paged_attention_shared(torch.zeros(2, 128), 128, torch.zeros(4, 2, 1, 16, 128), ints(2, 4), ints(3), ints(2), ints(2),
                                       ints(2), ints(2), ints(2), 2, 1, 1, 128, None, 1.0, torch.zeros(2, 128), ints(1), max_q_len=1,
                                       max_shared_len=16, max_own_len=16)


def test_adjust_logits():
    with pytest.raises(KernelLibraryError, match="CUDA"):
        kernels.adjust_logits(torch.zeros(2, 8), torch.zeros(2, 8))


def test_the_new_status_bit_has_words():
    assert "does not fit" in kernels.describe_status(16) and kernels.describe_status(0) == "no error"

"""Infinities in rows of adapters whose ranks are padded, in the kernels of few and of many rows."""
import pytest
import torch

from lora_inf_cases import RANKS, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ranks", RANKS)
@pytest.mark.parametrize("tokens", [1, 40, 300, 1500])
@pytest.mark.parametrize("interleaved", [False, True])
def test_padded_ranks_add_no_nan(tokens, ranks, interleaved):
    check("cuda", torch.bfloat16, tokens, ranks, slices=(72, 72) if interleaved else (64, 24, 40), interleaved=interleaved)


@pytest.mark.parametrize("tokens", [17, 900])
@pytest.mark.parametrize("max_rank", [64, 192])
def test_stacks_of_larger_ranks(tokens, max_rank):
    check("cuda", torch.bfloat16, tokens, [3, 0, 17], max_rank=max_rank)
    check("cuda", torch.bfloat16, tokens, [2, 5], max_rank=max_rank, slices=(72, 72), interleaved=True)

"""Infinities in rows of adapters whose ranks are padded."""
import pytest
import torch

from lora_inf_cases import RANKS, check


@pytest.mark.parametrize("ranks", RANKS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_padded_ranks_add_no_nan(ranks, interleaved):
    check("cpu", torch.float32, 40, ranks, slices=(24, 24) if interleaved else (64, 24, 40), interleaved=interleaved)

"""What is loaded beside a token's own adapter does not change its result."""
import pytest
import torch

from lora_cases import make_case, slots_of
from omni_npu_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [5, 700, 1024, 2847, 8192])
@pytest.mark.parametrize("interleaved", [False, True])
def test_results_keep_their_bits_when_other_adapters_come_and_go(tokens, interleaved):
    k, slices = 2048, [256, 256] if interleaved else [256, 64, 64]
    x, y, ad = make_case(tokens, 4, [16], k, slices, interleaved, device="cuda", seed=tokens)
    _, _, large = make_case(1, 4, [128], k, slices, interleaved, device="cuda", seed=1)
    stack = ops.LoraStack(8, 128, k, slices, device="cuda", interleaved=interleaved)
    plan = ops.lora_plan(slots_of(tokens, 4, seed=tokens).to("cuda"), 8)
    apply = ops.lora_gated if interleaved else ops.lora_add
    for i, factors in enumerate(ad):
        stack.load(i, *factors)
    want = apply(y, x, stack, plan)
    for i, factors in enumerate(large):
        stack.load(4 + i, *factors)
        assert torch.equal(apply(y, x, stack, plan), want)
    for i in range(8):
        if i % 2 and i > 3:
            stack.clear(i)
    assert torch.equal(apply(y, x, stack, plan), want)

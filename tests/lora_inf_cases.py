"""Adapters of rows that hold infinities, shared by the tests of both devices."""
import torch

from lora_cases import exact, load, make_case, slots_of
from omni_npu_b200 import ops

# ranks that are padded, of one slice after another and of the adapters in turn
RANKS = [[1], [2, 1], [5], [3, 0, 17], [16], [24, 1, 2], [33, 4]]


def kinds(t):
    """0 finite, 1 and -1 the infinities, 2 NaN."""
    return torch.where(t.isnan(), 2, torch.where(t.isinf(), t.sign(), 0)).to(torch.int8)


def check(device, dtype, tokens, ranks, k=264, slices=(64, 24, 40), max_rank=None, interleaved=False):
    """Where an input row holds an infinity, results are infinite or NaN where the definition's are: a product with the padding
    of a rank adds no NaN.  Other rows keep their values."""
    slices = list(slices)
    x, y, ad = make_case(tokens, 3, ranks, k, slices, interleaved, device=device, seed=tokens, dtype=dtype)
    if interleaved:                                            # factors of the up columns alone: the gate stays finite
        ad = [([None, a[1]], [None, b[1]], s) for a, b, s in ad]
    slots = slots_of(tokens, 3, seed=tokens).to(device)
    bad = torch.arange(0, tokens, 3, device=device)
    x[bad, bad * 7 % k] = torch.where(bad % 2 == 0, float("inf"), -float("inf")).to(dtype)
    stack = load(ops, ad, max_rank or max(max(ranks), 1), k, slices, device, interleaved, dtype)
    plan = ops.lora_plan(slots, 3)
    z, _ = exact(x, y, ad, slots, slices, interleaved)
    if interleaved:
        v = z.view(tokens, -1, 2, 8)
        g, u = v[:, :, 0].reshape(tokens, -1), v[:, :, 1].reshape(tokens, -1)
        z, out = g * torch.sigmoid(g) * u, ops.lora_gated(y, x, stack, plan)
    else:
        out = ops.lora_add(y, x, stack, plan)
    assert torch.equal(kinds(out), kinds(z))
    if tokens > 16 and any(0 < r < 3 for r in ranks):
        assert bool(out[bad].isinf().any())
    fine = ~z.isfinite().all(dim=1)
    assert bool(fine.any()) == bool((slots[bad] >= 0).any())

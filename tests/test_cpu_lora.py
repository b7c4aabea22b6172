import pytest
import torch

from omni_npu_b200 import ops
from lora_cases import check_silu, check_sum, exact, load, make_case, slots_of


@pytest.mark.parametrize("tokens,num_slots,ranks,k,slices", [
    (1, 1, [4], 16, [8]), (9, 3, [1, 8, 0, 16], 40, [16, 8, 24]), (5, 2, [0], 16, [8, 8])])
def test_add_matches_64_bits(tokens, num_slots, ranks, k, slices):
    x, y, ad = make_case(tokens, num_slots, ranks, k, slices)
    slots = slots_of(tokens, num_slots)
    st, plan = load(ops, ad, 16, k, slices, "cpu"), ops.lora_plan(slots, num_slots)
    z, bound = exact(x, y, ad, slots, slices)
    out = ops.lora_add(y, x, st, plan)
    check_sum(out, z, bound)
    same = y.clone()
    assert ops.lora_add(same, x, st, plan, out=same) is same and torch.equal(same, out)


def test_gated_matches_64_bits():
    x, y, ad = make_case(11, 2, [4, 8], 24, [24, 24])
    slots = slots_of(11, 2)
    z, bound = exact(x, y, ad, slots, [24, 24], interleaved=True)
    check_silu(ops.lora_gated(y, x, load(ops, ad, 8, 24, [24, 24], "cpu", True), ops.lora_plan(slots, 2)), z, bound)


def test_a_slot_is_replaced_and_cleared():
    x, y, ad = make_case(4, 2, [8, 3], 16, [8, 16])
    slots = torch.tensor([0, 1, 0, -1], dtype=torch.int32)
    st, plan = load(ops, ad, 16, 16, [8, 16], "cpu"), ops.lora_plan(slots, 2)
    st.load(0, *ad[1])
    z, bound = exact(x, y, [ad[1], ad[1]], slots, [8, 16])
    check_sum(ops.lora_add(y, x, st, plan), z, bound)
    st.clear(0)
    z, bound = exact(x, y, [([None] * 2, [None] * 2, 1.0), ad[1]], slots, [8, 16])
    check_sum(ops.lora_add(y, x, st, plan), z, bound)


def test_no_tokens():
    x, y, ad = make_case(0, 1, [4], 16, [8])
    st = load(ops, ad, 4, 16, [8], "cpu")
    assert ops.lora_add(y, x, st, ops.lora_plan(torch.zeros(0, dtype=torch.int32), 1)).shape == (0, 8)


def test_refusals():
    for kw in (dict(num_slots=0), dict(num_slots=513), dict(max_rank=0), dict(max_rank=257), dict(in_features=12),
               dict(slices=[12]), dict(slices=[]), dict(slices=[8] * 5), dict(slices=[8, 16], interleaved=True),
               dict(slices=[8], interleaved=True), dict(slices=[0])):
        with pytest.raises(ValueError):
            ops.LoraStack(**{**dict(num_slots=1, max_rank=8, in_features=16, slices=[8]), **kw})
    st = ops.LoraStack(2, 8, 16, [8, 8])
    a, b = torch.zeros(4, 16), torch.zeros(8, 4)
    for slot, fa, fb in ((2, [a, a], [b, b]), (-1, [a, a], [b, b]), (0, [a], [b]), (0, [a, None], [b, b]), (0, [a, a], [b, b[:, :3]]),
                         (0, [a, a], [b, b[:4]]), (0, [a[:, :8], a], [b, b]), (0, [torch.zeros(17, 16), a], [torch.zeros(8, 17), b]),
                         (0, [torch.zeros(0, 16), a], [torch.zeros(8, 0), b])):
        with pytest.raises(ValueError):
            st.load(slot, fa, fb)
    with pytest.raises(ValueError):
        st.clear(2)
    for slots, n in ((torch.zeros(3), 2), (torch.zeros(3, 1, dtype=torch.int32), 2), (torch.zeros(6, dtype=torch.int32)[::2], 2),
                     (torch.tensor([2], dtype=torch.int32), 2), (torch.tensor([-2], dtype=torch.int32), 2),
                     (torch.zeros(1, dtype=torch.int32), 0)):
        with pytest.raises(ValueError):
            ops.lora_plan(slots, n)
    plan = ops.lora_plan(torch.zeros(3, dtype=torch.int32), 2)
    x, y = torch.zeros(3, 16).bfloat16(), torch.zeros(3, 16).bfloat16()
    both = ops.LoraStack(2, 8, 16, [8, 8], interleaved=True)
    for fn, args in ((ops.lora_add, (y, x[:, :8], st, plan)), (ops.lora_add, (y[:, :8], x, st, plan)), (ops.lora_add, (y[:2], x[:2], st, plan)),
                     (ops.lora_add, (y, x, both, plan)), (ops.lora_gated, (y, x, st, plan)),
                     (ops.lora_add, (y, x, st, ops.lora_plan(torch.zeros(3, dtype=torch.int32), 1))),
                     (ops.lora_add, (y, x, st, plan, y[:, :8])), (ops.lora_add, (y, x, st, plan, y.float()))):
        with pytest.raises(ValueError):
            fn(*args)


def test_copy_blocks_whole_and_in_part():
    g = torch.Generator().manual_seed(0)
    caches = [torch.randn(6, 2, 4, 8, generator=g).bfloat16(), torch.randn(6, 4, 16, generator=g).bfloat16()]
    want = [c.clone() for c in caches]
    for c in want:
        c[3] = c[0]
        c[5][..., :2, :] = c[0][..., :2, :]
    cache = ops.CacheBlocks(caches)
    ops.copy_blocks(cache, [(0, 3), (1, 4)][:1])
    ops.copy_blocks(cache, [(0, 5, 2), (2, 1, 0)])
    ops.copy_blocks(cache, [])
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("pairs", [[(0, 6)], [(-1, 2)], [(0, 2, 5)], [(0, 2, -1)], [(0, 2), (1, 2)], [(0, 1), (1, 2)], [(3, 3)],
                                   [(0,)], [(0, 1, 2, 3)]])
def test_copy_blocks_refusals(pairs):
    cache = ops.CacheBlocks([torch.zeros(6, 2, 4, 8).bfloat16()])
    with pytest.raises(ValueError):
        ops.copy_blocks(cache, pairs)


def test_cache_blocks_refusals():
    t = torch.zeros(6, 2, 4, 8).bfloat16()
    for tensors in ([], [t, t[:5]], [t, torch.zeros(6, 2, 3, 8).bfloat16()], [torch.zeros(6, 2, 4, 4).bfloat16()], [t.transpose(1, 2)],
                    [torch.zeros(6, 4)], [t[..., :4]], [torch.zeros(0, 2, 4, 8)], [torch.zeros(6, 2, 0, 8)], [torch.zeros(6, 2, 4, 0)]):
        with pytest.raises(ValueError):
            ops.CacheBlocks(tensors)

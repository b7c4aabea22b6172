"""Adapter and page-copy kernels against 64 bits."""
import pytest
import torch

from omni_npu_b200 import ops
from lora_cases import check_silu, check_sum, exact, load, make_case, slots_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run_add(tokens, num_slots, ranks, k, slices, slots, max_rank=None, seed=0):
    x, y, ad = make_case(tokens, num_slots, ranks, k, slices, device=DEV, seed=seed)
    st = load(ops, ad, max_rank or max(max(ranks), 1), k, slices, DEV)
    slots = slots.to(DEV)
    out = ops.lora_add(y, x, st, ops.lora_plan(slots, num_slots))
    z, bound = exact(x, y, ad, slots, slices)
    check_sum(out, z, bound)
    same = y.clone()
    ops.lora_add(same, x, st, ops.lora_plan(slots, num_slots), out=same)
    assert torch.equal(same, out)


@pytest.mark.parametrize("num_slots", [1, 3, 33, 512])
@pytest.mark.parametrize("tokens", [1, 2, 31, 33, 256, 257, 1000, 5001])
def test_plan_groups_every_token_once(tokens, num_slots):
    slots = slots_of(tokens, num_slots, none=0.3)
    plan = ops.lora_plan(slots.to(DEV), num_slots)
    tiles = plan.tiles.tolist()
    order = plan.order.tolist()
    want, want_tiles = [], []
    for s in [*range(num_slots), -1]:
        mine = (slots == s).nonzero().flatten().tolist()
        for i in range(0, len(mine), plan.rows):
            want_tiles.append([s, len(want) + i, min(plan.rows, len(mine) - i), 0])
        want += mine
    assert order == want and tiles == want_tiles


@pytest.mark.parametrize("k,slices", [(8, [8]), (24, [8, 16]), (152, [40, 8, 104]), (4096, [512, 128, 128]), (1032, [64, 8, 32, 24]),
                                      (14336, [256])])
@pytest.mark.parametrize("tokens", [1, 5, 16, 17, 128, 257, 333])
def test_add(tokens, k, slices):
    run_add(tokens, 3, [16, 8, 33], k, slices, slots_of(tokens, 3, seed=tokens))


@pytest.mark.parametrize("ranks", [[1], [8, 0, 64], [128, 4], [256], [0, 0, 16], [65, 129]])
@pytest.mark.parametrize("tokens", [7, 300])
def test_ranks_and_missing_slices(tokens, ranks):
    run_add(tokens, 4, ranks, 520, [64, 24, 40], slots_of(tokens, 4))


@pytest.mark.parametrize("tokens", [3, 64, 700])
def test_no_adapters_at_all(tokens):
    run_add(tokens, 2, [0], 64, [32], torch.zeros(tokens, dtype=torch.int32))
    run_add(tokens, 2, [16], 64, [32], torch.full((tokens,), -1, dtype=torch.int32))


@pytest.mark.parametrize("tokens,contiguous", [(128, False), (513, True), (2000, True), (1999, False)])
def test_many_adapters(tokens, contiguous):
    run_add(tokens, 200, [8, 16, 24], 256, [128], slots_of(tokens, 200, contiguous=contiguous))


@pytest.mark.parametrize("act", [ops.SILU, ops.GELU_TANH, ops.RELU, (1.702, 7.0)])
@pytest.mark.parametrize("tokens,n,k", [(1, 8, 8), (17, 24, 64), (128, 1000, 136), (333, 2816, 1024), (70, 40, 4096)])
def test_gated(tokens, n, k, act):
    x, y, ad = make_case(tokens, 3, [8, 16, 0, 40], k, [n, n], device=DEV)
    slots = slots_of(tokens, 3).to(DEV)
    out = ops.lora_gated(y, x, load(ops, ad, 40, k, [n, n], DEV, True), ops.lora_plan(slots, 3), act=act)
    z, bound = exact(x, y, ad, slots, [n, n], interleaved=True)
    if act == ops.SILU:
        check_silu(out, z, bound)
        return
    v, e = z.view(tokens, -1, 2, 8), bound.view(tokens, -1, 2, 8)
    want = ops.ref.gated_act(v[:, :, 0], v[:, :, 1], act).reshape(tokens, -1)
    # the functions' slopes are at most 1.2 in the gate and, times it, in the up column; one more step for the fp32 function
    size = (v.abs().amax(dim=2) + 1).reshape(tokens, -1)
    lim = e.amax(dim=2).reshape(tokens, -1) * 3 * size + 2.0 ** -8 * want.abs() + 2.0 ** -20 * size * size
    assert bool(((out.double() - want).abs() <= lim).all())


def test_rows_apart_and_beside_other_data():
    """Views of wider rows; what lies beside the result's columns stays."""
    x, y, ad = make_case(40, 2, [16], 64, [48], device=DEV)
    slots = slots_of(40, 2).to(DEV)
    st, plan = load(ops, ad, 16, 64, [48], DEV), ops.lora_plan(slots, 2)
    z, bound = exact(x, y, ad, slots, [48])
    wide = torch.full((40, 64 + 48 + 16), 7.0, device=DEV, dtype=torch.bfloat16)
    wide[:, :64], wide[:, 64:112] = x, y
    out = ops.lora_add(wide[:, 64:112], wide[:, :64], st, plan, out=wide[:, 64:112])
    check_sum(out, z, bound)
    assert torch.equal(wide[:, :64], x) and bool((wide[:, 112:] == 7).all())


def test_values_of_other_rows_do_not_spread():
    """Infinities and NaN of a token stay in its row; those of an unused slot and of empty slots stay there."""
    x, y, ad = make_case(48, 3, [16], 128, [64], device=DEV)
    slots = slots_of(48, 2).to(DEV)
    slots[5], slots[6] = 0, -1
    x[5], x[6], y[7] = float("nan"), float("inf"), float("-inf")
    st = load(ops, ad[:2] + [([torch.full_like(t, float("nan")) for t in ad[2][0]], ad[2][1], 1.0)], 16, 128, [64], DEV)
    out = ops.lora_add(y, x, st, ops.lora_plan(slots, 3))
    keep = torch.tensor([i not in (5, 7) for i in range(48)], device=DEV)
    z, bound = exact(x, y, ad, slots, [64])
    check_sum(out[keep], z[keep], bound[keep])
    assert torch.equal(out[6], y[6]) and bool(out[5].isnan().all()) and bool((out[7] == float("-inf")).all())


def test_a_row_does_not_depend_on_the_rows_beside_it():
    x, y, ad = make_case(128, 4, [16, 32], 4096, [256, 64], device=DEV)
    slots = slots_of(128, 4).to(DEV)
    st = load(ops, ad, 32, 4096, [256, 64], DEV)
    full = ops.lora_add(y, x, st, ops.lora_plan(slots, 4))
    for n in (1, 3, 50):
        assert torch.equal(ops.lora_add(y[:n], x[:n], st, ops.lora_plan(slots[:n].clone(), 4)), full[:n])


def test_captured_and_replayed_with_other_slots_and_factors():
    x, y, ad = make_case(24, 3, [16, 8], 256, [64, 32], device=DEV)
    slots = slots_of(24, 3).to(DEV)
    st = load(ops, ad, 16, 256, [64, 32], DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.lora_add(y, x, st, ops.lora_plan(slots, 3))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                       # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.lora_add(y, x, st, ops.lora_plan(slots, 3)))
        graphs.append(g)
    for step in range(3):
        slots.copy_(slots_of(24, 3, seed=step))
        x.copy_(torch.randn_like(x.float()))
        st.load(step, *ad[(step + 1) % 3])
        ad[step] = ad[(step + 1) % 3]
        for g in graphs:
            g.replay()
        z, bound = exact(x, y, ad, slots, [64, 32])
        for o in outs:
            check_sum(o, z, bound)


def test_streams_side_by_side():
    cases = [make_case(t, 2, [16], 512, [128], device=DEV, seed=t) for t in (40, 300)]
    sts = [load(ops, c[2], 16, 512, [128], DEV) for c in cases]
    slots = [slots_of(c[0].shape[0], 2).to(DEV) for c in cases]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.lora_add(cases[i][1], cases[i][0], sts[i], ops.lora_plan(slots[i], 2)))
    torch.cuda.synchronize()
    for i, (x, y, ad) in enumerate(cases):
        z, bound = exact(x, y, ad, slots[i], [128])
        for o in outs[i]:
            check_sum(o, z, bound)


def test_slots_out_of_range_are_reported():
    x, y, ad = make_case(6, 2, [16], 64, [32], device=DEV)
    st = load(ops, ad, 16, 64, [32], DEV)
    slots = torch.tensor([0, 2, -5, 1, 1 << 30, -1], dtype=torch.int32, device=DEV)
    out = ops.lora_add(y, x, st, ops.lora_plan(slots, 2))
    with pytest.raises(RuntimeError):
        ops.check_status()
    z, bound = exact(x, y, ad, torch.tensor([0, -1, -1, 1, -1, -1], device=DEV), [32])
    check_sum(out, z, bound)


def test_refusals_on_the_device():
    x, y, ad = make_case(6, 2, [16], 64, [32], device=DEV)
    st, plan = load(ops, ad, 16, 64, [32], DEV), ops.lora_plan(slots_of(6, 2).to(DEV), 2)
    with pytest.raises(ValueError):
        ops.LoraStack(1, 8, 64, [32], device=DEV, dtype=torch.float32)
    with pytest.raises(ValueError):
        ops.lora_add(y, x.cpu(), st, plan)
    wide = torch.zeros(6, 100, device=DEV, dtype=torch.bfloat16)
    for bad_y, bad_x, out in ((y.float(), x, None), (y, x.float(), None), (y, wide[:, 4:68], None), (y, wide[:, 1:65], None),
                              (y.t().contiguous().t(), x, None), (y, wide[:, :64], wide[:, 8:40]),
                              (wide[:, :32], x, wide[:, 8:40])):
        with pytest.raises(ValueError):
            ops.lora_add(bad_y, bad_x, st, plan, out=out)
    # a plan of other tokens or slots, x of another width (the buffers' sizes are the same), another device's plan
    other = ops.LoraStack(2, 16, 56, [32], device=DEV)
    for t, n in ((5, 2), (7, 2), (6, 1), (6, 3)):
        with pytest.raises(ValueError):
            ops.lora_add(y, x, st, ops.lora_plan(torch.zeros(t, dtype=torch.int32, device=DEV), n))
    with pytest.raises(ValueError):
        ops.lora_add(y, x, other, plan)
    with pytest.raises(ValueError):
        ops.lora_add(y, x, st, ops.lora_plan(torch.zeros(6, dtype=torch.int32), 2))
    both = ops.LoraStack(2, 16, 64, [16, 16], device=DEV, interleaved=True)
    with pytest.raises(ValueError):
        ops.lora_add(y, x, both, plan)
    with pytest.raises(ValueError):
        ops.lora_gated(y, x, st, plan)
    torch.cuda.synchronize()


@pytest.mark.parametrize("shape,dims", [((9, 2, 16), (64, 64)), ((30, 4, 64), (192, 128)), ((7, 1, 1), (8, 8)), ((12, 8, 16), (128, 128))])
@pytest.mark.parametrize("layers", [1, 5])
def test_copy_blocks(shape, dims, layers):
    blocks, heads, page = shape
    caches = [torch.randn(blocks, heads, page, d, device=DEV).bfloat16() for _ in range(layers) for d in dims]
    caches.append(torch.randn(blocks, page, 576, device=DEV).bfloat16())
    want = [c.clone() for c in caches]
    pairs = [(0, blocks - 1, page), (0, blocks - 2, (page + 1) // 2), (2, blocks - 3, 0), (1, 3, max(1, page - 1))]
    for c in want:
        for s, d, n in pairs:
            c[d, ..., :n, :] = c[s, ..., :n, :]
    ops.copy_blocks(ops.CacheBlocks(caches), pairs)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("num", [1, 16, 17, 256, 257, 2048, 2500])
def test_copy_many_blocks(num):
    c = torch.randint(0, 1 << 15, (2 * num, 2, 4, 8), device=DEV, dtype=torch.int16)
    want = c.clone()
    perm = torch.randperm(2 * num)
    want[perm[:num].to(DEV)] = c[perm[num:].to(DEV)]
    ops.copy_blocks(ops.CacheBlocks([c]), list(zip(perm[num:].tolist(), perm[:num].tolist())))
    assert torch.equal(c, want)


def test_copy_in_views_of_a_larger_pool_past_4_gib():
    pool = torch.zeros(70000, 2, 2, 16, 512, dtype=torch.bfloat16, device=DEV)       # 4.6 GB; keys and values interleaved
    k, v = pool[:, 0], pool[:, 1]
    k[69999] = torch.randn(2, 16, 512, device=DEV)
    v[69999] = torch.randn(2, 16, 512, device=DEV)
    ops.copy_blocks(ops.CacheBlocks([k, v]), [(69999, 0), (69999, 69998, 3)])
    assert torch.equal(pool[0], pool[69999]) and torch.equal(pool[69998, :, :, :3], pool[69999, :, :, :3])
    assert not bool(pool[69998, :, :, 3:].any()) and not bool(pool[1:69998].any())


def test_copy_is_captured():
    c = torch.randn(4, 2, 16, 64, device=DEV).bfloat16()
    cache = ops.CacheBlocks([c])
    ops.copy_blocks(cache, [(0, 1)])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.copy_blocks(cache, [(0, 3, 5)])
    c[0] = torch.randn(2, 16, 64, device=DEV)
    kept = c[3, :, 5:].clone()
    g.replay()
    assert torch.equal(c[3, :, :5], c[0, :, :5]) and torch.equal(c[3, :, 5:], kept)


@pytest.mark.parametrize("pairs", [[(0, 6)], [(-1, 2)], [(0, 2, 5)], [(0, 2, -1)], [(0, 2), (1, 2)], [(0, 1), (1, 2)], [(1, 2), (0, 1)],
                                   [(3, 3)], [(0,)], [(0, 1, 2, 3)], [(0, 1 << 40)]])
def test_copy_blocks_refusals(pairs):
    c = torch.randn(6, 2, 4, 8, device=DEV).bfloat16()
    want, cache = c.clone(), ops.CacheBlocks([c])
    with pytest.raises(ValueError):
        ops.copy_blocks(cache, pairs)
    assert torch.equal(c, want)


@pytest.mark.parametrize("contiguous", [False, True])
@pytest.mark.parametrize("k,slices,ranks", [(8, [8], [16]), (40, [16, 24], [1, 0, 17]), (1032, [64, 8], [33, 128]),
                                            (4096, [256, 72, 64], [16, 0, 64, 100]), (14336, [64], [8, 256])])
@pytest.mark.parametrize("tokens", [769, 1000, 2177])
def test_many_rows(tokens, k, slices, ranks, contiguous):
    """Tiles of 128 rows: rows that follow one another, or gathered; ends of K inside a slab; parts of K; 16 to 500 joined ranks."""
    run_add(tokens, 4, ranks, k, slices, slots_of(tokens, 4, seed=tokens, contiguous=contiguous))
    if contiguous:                                             # no gaps: whole tiles follow one another
        run_add(tokens, 4, ranks, k, slices, slots_of(tokens, 4, none=0, contiguous=True))


@pytest.mark.parametrize("stride", [0, 64, 256, 264])
def test_many_rows_of_any_stride(stride):
    tokens, k = 900, 256
    _, y, ad = make_case(tokens, 2, [16, 48], k, [72], device=DEV)
    data = torch.randn(tokens * max(stride, 8) + k, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    x = torch.as_strided(data, (tokens, k), (stride, 1))
    slots = slots_of(tokens, 2, none=0, contiguous=True).to(DEV)
    out = ops.lora_add(y, x, load(ops, ad, 48, k, [72], DEV), ops.lora_plan(slots, 2))
    z, bound = exact(x, y, ad, slots, [72])
    check_sum(out, z, bound)


@pytest.mark.parametrize("contiguous", [False, True])
@pytest.mark.parametrize("tokens,n,k,ranks", [(800, 104, 520, [16, 0, 40]), (1500, 1000, 2048, [32]), (900, 1000, 256, [64, 0, 0, 8]),
                                              (1300, 520, 264, [128, 16, 0, 100, 128]), (800, 96, 128, [150, 0]), (1000, 200, 64, [256, 17])])
def test_gated_many_rows(tokens, n, k, ranks, contiguous):
    x, y, ad = make_case(tokens, 3, ranks, k, [n, n], device=DEV)
    slots = slots_of(tokens, 3, contiguous=contiguous).to(DEV)
    out = ops.lora_gated(y, x, load(ops, ad, max(ranks), k, [n, n], DEV, True), ops.lora_plan(slots, 3))
    z, bound = exact(x, y, ad, slots, [n, n], interleaved=True)
    check_silu(out, z, bound)


def test_many_rows_keep_their_values_to_themselves():
    """NaN of a row of a tile, and of the rows behind a tile's last, stay in their rows."""
    tokens, k = 1000, 256
    x, y, ad = make_case(tokens, 2, [16], k, [64], device=DEV)
    slots = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    slots[:300], slots[400:777] = 0, 1
    bad = torch.tensor([3, 129, 300, 301, 777, 500], device=DEV)
    x[bad] = float("nan")
    out = ops.lora_add(y, x, load(ops, ad, 16, k, [64], DEV), ops.lora_plan(slots, 2))
    z, bound = exact(x, y, ad, slots, [64])
    keep = torch.ones(tokens, dtype=torch.bool, device=DEV)
    keep[torch.tensor([3, 129, 500], device=DEV)] = False
    check_sum(out[keep], z[keep], bound[keep])
    assert bool(out[~keep].isnan().all())


@pytest.mark.parametrize("ranks", [[16], [48], [64, 16], [128], [200, 0, 40]])
def test_many_rows_in_and_out_of_place(ranks):
    """Both ways give the same; rows without an adapter keep their bits."""
    tokens, k, slices = 3000, 128, [328, 64]
    x, y, ad = make_case(tokens, 2, ranks, k, slices, device=DEV)
    slots = slots_of(tokens, 2, none=0.5).to(DEV)
    st, plan = load(ops, ad, max(ranks), k, slices, DEV), ops.lora_plan(slots, 2)
    out = ops.lora_add(y, x, st, plan)
    z, bound = exact(x, y, ad, slots, slices)
    check_sum(out, z, bound)
    assert torch.equal(out[slots < 0].view(torch.int16), y[slots < 0].view(torch.int16))
    assert torch.equal(ops.lora_add(y, x, st, plan, out=y), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
@pytest.mark.parametrize("max_rank", [32, 128])
@pytest.mark.parametrize("k,slices,interleaved", [(8, [8], False), (40, [72, 8, 136], False), (264, [40, 40], True), (520, [16, 24, 8, 64], False)])
def test_factors_are_laid_out_as_on_the_host(dtype, max_rank, k, slices, interleaved):
    gen = torch.Generator().manual_seed(k)
    host = ops.LoraStack(3, max_rank, k, slices, interleaved=interleaved)
    card = ops.LoraStack(3, max_rank, k, slices, device=DEV, interleaved=interleaved)
    for slot, ranks in enumerate([[1, 16, 17, 32], [max_rank, 0, 5, 8], [0, 9, 0, max_rank]]):
        a = [torch.randn(r, k, generator=gen).to(dtype) if r else None for r in ranks[: len(slices)]]
        b = [torch.randn(n, r, generator=gen).to(dtype) if r else None for n, r in zip(slices, ranks)]
        host.load(slot, a, b, 0.3)
        if slot == 0:                                          # other strides
            a = [t if t is None else t.t().contiguous().t() for t in a]
            b = [t if t is None else torch.cat([t, t], 1)[:, t.shape[1]:] for t in b]
        card.load(slot, [t if t is None or slot == 2 else t.to(DEV) for t in a], [t if t is None else t.to(DEV) for t in b], 0.3)
    assert torch.equal(card.a.cpu(), host.a) and torch.equal(card.b.cpu(), host.b) and torch.equal(card.ranks.cpu(), host.ranks)
    card.load(0, [None] * len(slices), [None] * len(slices))   # nothing left but the scale
    assert card.ranks[0].tolist() == [0] * len(slices) + [0x3F800000]

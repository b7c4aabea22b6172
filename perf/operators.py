"""What requests of one server have of their own beside what they share, measured on one GPU.

Requests share a projection's weights and bring a low-rank adapter of their own (``add``: the attention and down
projections; ``gated``: the joined gate / up projection, whose activation follows the adapter), and the samples of one
prompt share its cache pages and bring copies of those that they go on to write (``pages``).

``prepare`` gives what a serving program has in hand: activations, the base product's result, the loaded adapters and
the step's grouping of tokens by adapter (made once a step and used by every layer), or the cache and the list of copies
that the scheduler made.  Sizes are those of the framework's presets and its benchmark's batches.
"""
import math
import random

import torch

own = False

HEADS = 8                    # key heads of the dense presets' caches


def _nums(text):
    return [int(v) for v in text.split()]


def listed():
    return [
        # one user's decode step: a single token through the joined query / key / value projection
        dict(name="add_token", kind="add", tokens=1, adapters=1, ranks="16", k=4096, slices="4096 1024 1024",
             plain=0, prompts=False),
        # a decode batch whose requests use adapters of mixed ranks, some none
        dict(name="add_decode_mixed", kind="add", tokens=128, adapters=31, ranks="8 16 32 64", k=4096,
             slices="4096 1024 1024", plain=16, prompts=False),
        # the same batch with an adapter for each request, down projection: the most adapter weights a step reads
        dict(name="add_decode_each", kind="add", tokens=128, adapters=128, ranks="16", k=14336, slices="4096",
             plain=0, prompts=False),
        # a prompt step with the whole token budget: eight prompts of eight adapters
        dict(name="add_prompt_8192", kind="add", tokens=8192, adapters=8, ranks="16", k=4096,
             slices="4096 1024 1024", plain=0, prompts=True),
        # an uneven chunk of prompts with large ranks, one prompt without an adapter
        dict(name="add_prompt_ragged", kind="add", tokens=2847, adapters=4, ranks="64 33 128", k=2048,
             slices="4096 512 512", plain=402, prompts=True),
        # gate / up of a lightly loaded server
        dict(name="gated_decode_16", kind="gated", tokens=16, adapters=4, ranks="16", k=4096, slices="14336 14336",
             plain=2, prompts=False),
        # gate / up of a small model, an odd number of prompt tokens
        dict(name="gated_prompt_odd", kind="gated", tokens=333, adapters=3, ranks="8 16", k=1024, slices="2816 2816",
             plain=0, prompts=True),
        # gate / up of the full token budget
        dict(name="gated_prompt_8192", kind="gated", tokens=8192, adapters=8, ranks="32", k=4096,
             slices="14336 14336", plain=0, prompts=True),
        # a second sample of one prompt: the last page, partly filled, in every layer
        dict(name="pages_fork_one", kind="pages", layers=32, heads=HEADS, page=16, dims="128 128", pool=64, pairs=1,
             rows="5"),
        # many samples of several prompts that become decoding requests in one step
        dict(name="pages_fork_127", kind="pages", layers=32, heads=HEADS, page=16, dims="128 128", pool=512, pairs=127,
             rows="1 7 12 15"),
        # a cache with other pages and with values narrower than keys
        dict(name="pages_fork_wide", kind="pages", layers=27, heads=4, page=64, dims="192 128", pool=128, pairs=37,
             rows="63 17 64"),
        # whole pages of long sequences that get a copy of their own
        dict(name="pages_whole_512", kind="pages", layers=16, heads=HEADS, page=16, dims="128 128", pool=2048,
             pairs=512, rows="16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["add", "add", "gated", "pages"])
    if kind == "pages":
        page = rng.choice([8, 16, 32, 64])
        pairs = _spread(rng, 1, 400)
        heads = rng.choice([1, 2, 4, 8])
        dims = rng.choice(["128 128", "64 64", "192 128", "96 96", "256 256"])
        layers = rng.randint(1, 32)
        page_bytes = layers * heads * page * sum(_nums(dims)) * 2
        pairs = max(1, min(pairs, (1 << 29) // page_bytes))
        return dict(kind="pages", layers=layers, heads=heads, page=page, dims=dims,
                    pool=2 * pairs + rng.randint(1, 64), pairs=pairs, rows=" ".join(str(rng.randint(1, page)) for _ in range(4)))
    prompts = rng.random() < 0.5
    tokens = _spread(rng, 130, 8192) if prompts else _spread(rng, 1, 256)
    adapters = _spread(rng, 1, min(tokens, 12 if prompts else 64))
    ranks = rng.choice(["8", "16", "32", "64", "8 16 64", "4 24", "1 128"])
    plain = 0 if tokens == adapters else rng.choice([0, rng.randint(0, (tokens - adapters) // 2)])
    k = 8 * _spread(rng, 16, 512)
    if kind == "gated":
        n = 8 * _spread(rng, 32, 1792)
        slices = f"{n} {n}"
    else:
        slices = " ".join(str(8 * _spread(rng, 16, 512)) for _ in range(rng.randint(1, 3)))
    return dict(kind=kind, tokens=tokens, adapters=adapters, ranks=ranks, k=k, slices=slices, plain=plain,
                prompts=prompts)


def _ranks(case):
    ranks = _nums(case["ranks"])
    return [ranks[i % len(ranks)] for i in range(case["adapters"])]


def _slots(case, seed):
    """Adapter of each token, -1 for none: every adapter has a token at least.  Prompts lie one after another."""
    rng = random.Random(seed * 7919 + case["tokens"])
    n, used = case["tokens"] - case["plain"], case["adapters"]
    if case["prompts"]:
        cuts = sorted(rng.sample(range(1, n), used - 1))
        runs = [(i, b - a) for i, (a, b) in enumerate(zip([0] + cuts, cuts + [n]))]
        if case["plain"]:
            runs.insert(rng.randrange(used + 1), (-1, case["plain"]))
        return [s for s, c in runs for _ in range(c)]
    slots = list(range(used)) + [rng.randrange(used) for _ in range(n - used)] + [-1] * case["plain"]
    rng.shuffle(slots)
    return slots


def _pairs(case, seed):
    """(source page, destination page, rows) of distinct destinations that are nobody's source."""
    rng = random.Random(seed * 104729 + case["pairs"])
    pages = rng.sample(range(case["pool"]), min(case["pool"], 2 * case["pairs"]))
    dst = pages[:case["pairs"]]
    src = pages[case["pairs"]:]
    rows = _nums(case["rows"])
    return [(rng.choice(src), d, rows[i % len(rows)]) for i, d in enumerate(dst)]


def _adapters(case, seed, gen):
    out = []
    for r in _ranks(case):
        a = [(torch.rand(r, case["k"], generator=gen, device="cuda") * 2 - 1) * math.sqrt(3.0 / case["k"])
             for _ in _nums(case["slices"])]
        b = [torch.randn(n, r, generator=gen, device="cuda") * 0.1 for n in _nums(case["slices"])]
        out.append(([t.bfloat16() for t in a], [t.bfloat16() for t in b], 2.0 * 16 / max(r, 8)))
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "pages":
        caches = [torch.randn(case["pool"], case["heads"], case["page"], d, generator=gen, device="cuda",
                              dtype=torch.bfloat16) for _ in range(case["layers"]) for d in _nums(case["dims"])]
        st = dict(kind="pages", caches=caches, pairs=_pairs(case, seed))
        if own:
            from omni_npu_b200 import ops
            st["cache"] = ops.CacheBlocks(caches)
        return st
    t, slices = case["tokens"], _nums(case["slices"])
    x = torch.randn(t, case["k"], generator=gen, device="cuda").bfloat16()
    y = torch.randn(t, sum(slices), generator=gen, device="cuda").bfloat16()
    adapters = _adapters(case, seed, gen)
    slots = _slots(case, seed)
    st = dict(kind=case["kind"], x=x, y=y, slices=slices)
    if own:
        from omni_npu_b200 import ops
        stack = ops.LoraStack(case["adapters"], max(_ranks(case)), case["k"], slices, device="cuda",
                              interleaved=case["kind"] == "gated")
        for i, (a, b, scale) in enumerate(adapters):
            stack.load(i, a, b, scale)
        st["stack"] = stack
        st["plan"] = ops.lora_plan(torch.tensor(slots, dtype=torch.int32, device="cuda"), case["adapters"])
        return st
    host = torch.tensor(slots)
    st["adapters"] = adapters
    st["groups"] = [(host == i).nonzero().flatten().cuda() for i in range(case["adapters"])]
    return st


def _own(st):
    from omni_npu_b200 import ops
    if st["kind"] == "pages":
        ops.copy_blocks(st["cache"], st["pairs"])
        return st["caches"]
    if st["kind"] == "gated":
        return ops.lora_gated(st["y"], st["x"], st["stack"], st["plan"])
    return ops.lora_add(st["y"], st["x"], st["stack"], st["plan"])


def run(st):
    if own:
        return _own(st)
    if st["kind"] == "pages":
        dev = st["caches"][0].device
        page = st["caches"][0].shape[2]
        src, dst, rows = (torch.tensor(c, device=dev) for c in zip(*st["pairs"]))
        kept = torch.arange(page, device=dev)[None, :] < rows[:, None]
        for c in st["caches"]:
            c[dst] = torch.where(kept[:, None, :, None], c[src], c[dst])
        return st["caches"]
    x = st["x"].float()
    # gate and up columns lie in alternating groups of eight
    t, n = st["y"].shape
    y = st["y"].float().view(t, -1, 2, 8).transpose(1, 2).reshape(t, n) if st["kind"] == "gated" else st["y"].float()
    for rows, (a, b, scale) in zip(st["groups"], st["adapters"]):
        xs = x[rows]
        y[rows] += torch.cat([(xs @ p.float().t()) @ q.float().t() for p, q in zip(a, b)], dim=1) * scale
    if st["kind"] == "gated":
        gate, up = y[:, : n // 2], y[:, n // 2:]
        y = gate / (1 + torch.exp(-gate)) * up
    return y.bfloat16()


def exact(case, seed):
    if case["kind"] == "pages":
        return None
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, slices = case["tokens"], _nums(case["slices"])
    x = torch.randn(t, case["k"], generator=gen, device="cuda").bfloat16().double()
    y = torch.randn(t, sum(slices), generator=gen, device="cuda").bfloat16().double()
    slots = torch.tensor(_slots(case, seed), device="cuda")
    cols, at = [], 0
    for s, n in enumerate(slices):
        j = torch.arange(n, device="cuda")
        cols.append(j // 8 * 16 + s * 8 + j % 8 if case["kind"] == "gated" else at + j)
        at += n
    delta = torch.zeros_like(y)
    for i, (a, b, scale) in enumerate(_adapters(case, seed, gen)):
        mine = torch.where(slots == i)[0]
        for p, q, c in zip(a, b, cols):
            h = torch.einsum("tk,rk->tr", x[mine], p.double())
            delta[mine[:, None], c[None, :]] = scale * torch.einsum("tr,nr->tn", h, q.double())
    y += delta
    if case["kind"] == "gated":
        g, u = y[:, cols[0]], y[:, cols[1]]
        return g * torch.sigmoid(g) * u
    return y


def work(case):
    if case["kind"] == "pages":
        rows = _nums(case["rows"])
        rows = sum(rows[i % len(rows)] for i in range(case["pairs"]))
        return {"bytes": 2 * 2 * rows * case["layers"] * case["heads"] * sum(_nums(case["dims"])) + 12 * case["pairs"], "flops": 0}
    t, k, slices = case["tokens"], case["k"], _nums(case["slices"])
    n = sum(slices)
    ranks, mine = _ranks(case), t - case["plain"]
    out = n // 2 if case["kind"] == "gated" else n
    weights = sum(ranks) * (len(slices) * k + n)
    mean = sum(ranks) / len(ranks)
    return {"bytes": 2 * (mine * k + t * n + t * out + weights) + 4 * t,
            "flops": int(2 * mine * mean * (len(slices) * k + n))}

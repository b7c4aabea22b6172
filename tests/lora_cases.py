"""Inputs, 64-bit results and error bounds shared by the adapter tests."""
import torch


def make_case(tokens, num_slots, ranks, k, slices, interleaved=False, device="cpu", seed=0, dtype=torch.bfloat16):
    """(x, y, adapters): adapters[i] = (factors A, factors B, scale) of slot i, with None for rank 0."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, k, generator=gen).to(dtype).to(device)
    y = torch.randn(tokens, sum(slices), generator=gen).to(dtype).to(device)
    adapters = []
    for i in range(num_slots):
        a, b = [], []
        for j, n in enumerate(slices):
            r = ranks[(i * len(slices) + j) % len(ranks)]
            a.append((torch.randn(r, k, generator=gen) / k ** 0.5).to(dtype).to(device) if r else None)
            b.append((torch.randn(n, r, generator=gen) / 4).to(dtype).to(device) if r else None)
        adapters.append((a, b, 0.5 + 0.37 * i))
    return x, y, adapters


def columns(slices, i, interleaved, device):
    j = torch.arange(slices[i], device=device)
    return j // 8 * 16 + i * 8 + j % 8 if interleaved else sum(slices[:i]) + j


def exact(x, y, adapters, slots, slices, interleaved=False):
    """(z, bound): y + scale B (A x) in 64 bits, and how far fp32 sums of h may move it.

    The sum over K is a chain of at most K / 16 matrix instructions (two per 32 of K in one warp), then 8 warps and 8
    parts: each addition rounds or cuts off 2^-23 of what has been added in absolute value at most, and the products inside an
    instruction count as one more.  h goes on as two bf16, 2^-17 of it, and the sum over the rank is a chain of
    2 r / 16 instructions."""
    z, bound = y.double(), torch.zeros_like(y, dtype=torch.float64)
    for s, (a, b, scale) in enumerate(adapters):
        rows = (slots == s).nonzero().flatten()
        for i in range(len(slices)):
            if a[i] is None or not len(rows):
                continue
            c = columns(slices, i, interleaved, y.device)
            ad, bd, xd = a[i].double(), b[i].double(), x[rows].double()
            z[rows[:, None], c[None, :]] += scale * ((xd @ ad.t()) @ bd.t())
            mass = (xd.abs() @ ad.abs().t()) @ bd.abs().t() * abs(scale)
            k, r = ad.shape[1], ad.shape[0]
            bound[rows[:, None], c[None, :]] = mass * (2.0 ** -23 * (2 * (k / 16 + 24) + 2 * (r / 8 + 8)) + 2.0 ** -17)
    return z, bound


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_sum(out, z, bound):
    err = (out.double() - z).abs()
    lim = half_step(out.dtype) * (z.abs() + bound) + bound
    assert bool((err <= lim).all()), f"off by {float((err - lim).max())}, {float((err / lim.clamp_min(1e-30)).max())} of the bound"


def check_silu(out, z, bound):
    """silu'(g) <= 1.1; the exponential and the division of the fp32 function cost (4 + 1.5 |g|) 2^-22 of the result."""
    t = z.shape[0]
    v, e = z.view(t, -1, 2, 8), bound.view(t, -1, 2, 8)
    g, u, eg, eu = (w.reshape(t, -1) for w in (v[:, :, 0], v[:, :, 1], e[:, :, 0], e[:, :, 1]))
    want = g * torch.sigmoid(g) * u
    lim = 1.1 * eg * (u.abs() + eu) + (g * torch.sigmoid(g)).abs() * eu + want.abs() * (4 + 1.5 * g.abs()) * 2.0 ** -22
    lim = half_step(out.dtype) * (want.abs() + lim) + lim + 1e-38
    err = (out.double() - want).abs()
    assert bool((err <= lim).all()), f"off by {float((err - lim).max())}, {float((err / lim).max())} of the bound"


def load(ops, adapters, max_rank, k, slices, device, interleaved=False, dtype=torch.bfloat16):
    st = ops.LoraStack(len(adapters), max_rank, k, slices, device=device, interleaved=interleaved, dtype=dtype)
    for i, (a, b, scale) in enumerate(adapters):
        if any(p is not None for p in a):
            st.load(i, a, b, scale)
    return st


def slots_of(tokens, num_slots, seed=0, none=0.2, contiguous=False):
    g = torch.Generator().manual_seed(seed + 91)
    s = torch.randint(0, num_slots, (tokens,), generator=g)
    if contiguous:
        s = s.sort().values
    s[torch.rand(tokens, generator=g) < none] = -1
    return s.to(torch.int32)

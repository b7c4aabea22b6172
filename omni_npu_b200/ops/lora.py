"""Low-rank adapters of many requests beside a shared projection.

A projection's weights are shared; a request may bring factors A [r, K] and B [N, r] of its own that add
``scale * B (A x)`` to the projection's result for its tokens.  :class:`LoraStack` holds the factors of one projection for
every adapter slot of the server, :func:`lora_plan` groups a step's tokens by slot once, and :func:`lora_add` and
:func:`lora_gated` apply them to the result of the shared product.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import SILU, _C, _act_kind, _count, device_state, ref

MAX_SLOTS, MAX_SLICES, MAX_RANK, LANES_RANK = 512, 4, 256, 32

# Tokens of one adapter that are taken together.  Up to this many tokens of a step: tiles of 16, one matrix instruction high,
# through kernels that stream the factors; above, tiles of 128.  The rule sees the number of tokens alone.  Us, tiles of 128 / 16:
# 200 tokens of 8 adapters of rank 16, 4096 to 4096 + 1024 + 1024 12.3 / 8.1, 14336 to 4096 17.8 / 8.5; 768 tokens 16.7 / 13.9 and
# 20.8 / 14.7; 1000 tokens 17.1 / 19.1.  Where it loses: 768 tokens of 8 of rank 64 21.1 / 26.5 (taken in 16), 1000 tokens 14336
# to 4096 21.8 / 16.3 (taken in 128).  A row's result does not depend on the rows beside it as long as these are no more.
FEW_TOKENS, FEW_ROWS, MANY_ROWS = 768, 16, 128


def _padded(t: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    if tuple(t.shape) != (rows, cols):
        t = torch.nn.functional.pad(t, (0, cols - t.shape[1], 0, rows - t.shape[0]))
    return t.contiguous()


class LoraStack:
    """Factors of one projection [sum(slices), in_features] for ``num_slots`` adapters of rank up to ``max_rank``.

    ``slices``: columns of the parts of a joined projection (query, key and value; gate and up), each with factors of its
    own.  ``interleaved``: two equal slices whose columns alternate in groups of eight, gate first, as the gated products
    store them.  Slots start empty: tokens of an empty slot get the shared product alone.  Factors are finite.

    The kernels are chosen, and the work is dealt, by ``max_rank`` and ``num_slots``: neither larger than needed."""

    def __init__(self, num_slots: int, max_rank: int, in_features: int, slices: Sequence[int], device=None,
                 dtype: torch.dtype = torch.bfloat16, interleaved: bool = False) -> None:
        slices = [int(n) for n in slices]
        if not 1 <= num_slots <= MAX_SLOTS:
            raise ValueError(f"LoraStack: {num_slots} slots, 1 to {MAX_SLOTS} are possible")
        if not 1 <= max_rank <= MAX_RANK:
            raise ValueError(f"LoraStack: rank {max_rank}, 1 to {MAX_RANK} are possible")
        if not 1 <= len(slices) <= MAX_SLICES or any(n <= 0 or n % 8 for n in slices):
            raise ValueError(f"LoraStack: slices {slices}, one to {MAX_SLICES} multiples of 8 are possible")
        if in_features <= 0 or in_features % 8:
            raise ValueError(f"LoraStack: {in_features} input features are not a multiple of 8")
        if interleaved and (len(slices) != 2 or slices[0] != slices[1]):
            raise ValueError("LoraStack: interleaved columns are those of two equal slices")
        device = torch.device(device if device is not None else "cpu")
        if device.type == "cuda" and dtype != torch.bfloat16:
            raise ValueError("LoraStack: factors on a GPU are bf16")
        self.num_slots, self.in_features, self.slices, self.interleaved = num_slots, in_features, slices, interleaved
        self.out_features = sum(slices)
        self.max_rank = (max_rank + 15) // 16 * 16
        self.dtype = dtype
        with torch.inference_mode(False):
            # in the order of the matrix instructions (csrc/lora/lora.cu), K in whole 32, columns in whole blocks
            self._k = (in_features + 31) // 32
            self.a = torch.zeros(num_slots, len(slices) * self.max_rank * self._k * 32, dtype=dtype, device=device)
            self._lanes = self.max_rank <= LANES_RANK
            self._block = 32 if interleaved or self._lanes else 64
            self.b = torch.zeros(num_slots, sum((n + self._block - 1) // self._block for n in slices) * self._block * self.max_rank,
                                 dtype=dtype, device=device)
            # of every slot the ranks and the bits of the scale
            self.ranks = torch.zeros(num_slots, len(slices) + 1, dtype=torch.int32, device=device)
        self.device = self.a.device
        self._ranks = [[0] * len(slices) for _ in range(num_slots)]
        self._padded = [[0] * len(slices) for _ in range(num_slots)]       # in whole 16, as the factors lie
        self._scales = [0.0] * num_slots
        self.sizes = [in_features, self.max_rank, 0, *slices]

    def load(self, slot: int, a: Sequence[Optional[torch.Tensor]], b: Sequence[Optional[torch.Tensor]],
             scale: float = 1.0) -> None:
        """Put an adapter into ``slot``: ``a[i]`` [r, in_features] and ``b[i]`` [slices[i], r] of each slice, or None for a
        slice that it leaves as it is.  Steps launched before keep the slot's earlier contents, later ones see these
        (stream order)."""
        self._check_slot(slot)
        if len(a) != len(self.slices) or len(b) != len(self.slices):
            raise ValueError(f"LoraStack.load: {len(self.slices)} slices need as many factors")
        ranks = []
        for i, (p, q) in enumerate(zip(a, b)):
            if (p is None) != (q is None):
                raise ValueError(f"LoraStack.load: slice {i} has one factor of two")
            if p is None:
                ranks.append(0)
                continue
            r = p.shape[0] if p.dim() == 2 else -1
            if p.dim() != 2 or q.dim() != 2 or p.shape[1] != self.in_features or tuple(q.shape) != (self.slices[i], r):
                raise ValueError(f"LoraStack.load: slice {i} has factors {tuple(p.shape)} and {tuple(q.shape)}, expected "
                                 f"(r, {self.in_features}) and ({self.slices[i]}, r)")
            if not 1 <= r <= self.max_rank:
                raise ValueError(f"LoraStack.load: rank {r}, at most {self.max_rank}")
            ranks.append(r)
        padded = [(r + 15) // 16 * 16 for r in ranks]
        if self.device.type == "cuda":
            _count(1)
            _C().lora_pack(self.a, self.b, self.ranks, slot, [self._here(p) for p in a], [self._here(q) for q in b], self.slices,
                           self.in_features, self._lanes, self._block, scale)
        else:
            with torch.inference_mode():
                for p, view in zip(a, self._views_a(slot, padded)):
                    if view is not None:
                        view.copy_(_padded(p, view.shape[0] * 8, self._k * 32).view(view.shape))
                for q, view in zip(b, self._views_b(slot, padded)):
                    if view is not None:
                        view.copy_(_padded(q, view.shape[0] * self._block,
                                           view.shape[5] * (16 if self._lanes else 8)).view(view.shape))
                row = torch.tensor(ranks + [0], dtype=torch.int32)
                row[-1:].view(torch.float32).fill_(scale)
                self.ranks[slot].copy_(row)
        self._scales[slot] = float(scale)
        self._set_ranks(slot, ranks)

    def _here(self, t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        """A factor on the stack's device, of a type that the packing kernel reads."""
        if t is None:
            return None
        if t.device != self.device:
            t = t.to(self.device)
        return t if t.dtype in (torch.bfloat16, torch.float16, torch.float32) else t.to(self.dtype)

    def _views_a(self, slot: int, ranks):
        """A of each slice as [ranks, K] in the shape (rank / 8, 8, K / 32, 4, 8) over its packed place."""
        total = sum(ranks) // 8
        packed = self.a[slot, : total * 8 * self._k * 32].view(self._k, total, 4, 8, 8)   # k32, r8, k8, rank, 8
        at = 0
        for r in ranks:
            yield packed[:, at: at + r // 8].permute(1, 3, 0, 2, 4) if r else None
            at += r // 8

    def _views_b(self, slot: int, ranks):
        """B of each slice as [columns, rank] over its packed place: (columns / 32, 4, 2, 2, 2, rank / 16, 2, 4, 2) in the order
        of lanes, else (columns / block, block / 32, 4, 4, 2, rank / 8, 8)."""
        at = 0
        for r, n in zip(ranks, self.slices):
            c = (n + self._block - 1) // self._block
            packed = self.b[slot, at: at + c * self._block * r]
            if not r:
                yield None
            elif self._lanes:                                 # n32, r16, j / 2, i / 2, i % 2, q, j % 2, half, 2
                yield packed.view(c, r // 16, 2, 4, 2, 4, 2, 2, 2).permute(0, 3, 2, 6, 4, 1, 7, 5, 8)
            else:                                             # block, r8, 32 columns, j, i / 2, i % 2, 8
                yield packed.view(c, r // 8, self._block // 32, 4, 4, 2, 8).permute(0, 2, 4, 3, 5, 1, 6)
            at += c * self._block * r

    def clear(self, slot: int) -> None:
        """Empty a slot."""
        self._check_slot(slot)
        with torch.inference_mode():
            self.ranks[slot].zero_()
        self._set_ranks(slot, [0] * len(self.slices))

    def reset(self) -> None:
        """Empty every slot, whatever the memory holds."""
        with torch.inference_mode():
            self.ranks.zero_()
        for slot in range(self.num_slots):
            self._set_ranks(slot, [0] * len(self.slices))

    def factors(self, slot: int):
        """(A, B) of each slice of a slot (ranks padded to 16), None where it has none."""
        ranks = self._padded[slot]
        return [None if a is None else (a.reshape(r, -1)[:, : self.in_features], b.reshape(-1, r)[:n])
                for a, b, r, n in zip(self._views_a(slot, ranks), self._views_b(slot, ranks), ranks, self.slices)]

    def columns(self, i: int) -> torch.Tensor:
        """Where the columns of slice ``i`` lie in the projection's result."""
        j = torch.arange(self.slices[i], device=self.device)
        return j // 8 * 16 + i * 8 + j % 8 if self.interleaved else sum(self.slices[:i]) + j

    def _set_ranks(self, slot: int, ranks) -> None:
        self._ranks[slot] = ranks
        self._padded[slot] = [(r + 15) // 16 * 16 for r in ranks]
        used = [sum(r) for r in self._padded if any(r)]
        # input features; largest rank; mean of the loaded adapters' ranks, the slices' together (only speed depends on it); slices
        self.sizes = [self.in_features, self.max_rank, sum(used) // max(1, len(used)), *self.slices]

    def _check_slot(self, slot: int) -> None:
        if not 0 <= slot < self.num_slots:
            raise ValueError(f"LoraStack: slot {slot} of {self.num_slots}")


class LoraPlan:
    """A step's tokens grouped by adapter slot (:func:`lora_plan`)."""

    __slots__ = ("slots", "num_slots", "num_tokens", "rows", "buffer", "status")

    def __init__(self, slots: torch.Tensor, num_slots: int, rows: int = 0, buffer: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> None:
        self.slots, self.num_slots, self.num_tokens, self.rows, self.buffer = slots, num_slots, slots.shape[0], rows, buffer
        self.status = status                                  # where the device's kernels report (on a GPU)

    @property
    def order(self) -> torch.Tensor:
        """Tokens by slot, those without an adapter last (on a GPU)."""
        return self.buffer[: self.num_tokens]

    @property
    def tiles(self) -> torch.Tensor:
        """[tiles, 4]: slot, first place in ``order`` and number of tokens of every tile (on a GPU; reads their number back)."""
        t = self.num_tokens
        at = (t + 1 + 3) // 4 * 4
        return self.buffer[at: at + 4 * int(self.buffer[t])].view(-1, 4)


def lora_plan(slots: torch.Tensor, num_slots: int) -> LoraPlan:
    """Group tokens by adapter: ``slots`` int32 [T], the slot of each token or -1 for the shared weights alone.  The plan is
    made on the device (it may be captured, and follows ``slots`` at every replay) and serves every projection of the step.
    A slot outside -1 .. num_slots - 1 counts as -1 and is reported by :func:`check_status`."""
    if slots.dim() != 1 or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError("lora_plan: slots are a contiguous int32 vector")
    if not 1 <= num_slots <= MAX_SLOTS:
        raise ValueError(f"lora_plan: {num_slots} slots, 1 to {MAX_SLOTS} are possible")
    t = slots.shape[0]
    if not slots.is_cuda:
        if t and (int(slots.min()) < -1 or int(slots.max()) >= num_slots):
            raise ValueError(f"lora_plan: slots outside -1 .. {num_slots - 1}")
        return LoraPlan(slots, num_slots)
    rows = FEW_ROWS if t <= FEW_TOKENS else MANY_ROWS
    status = device_state(slots.device).status
    if t == 0:
        return LoraPlan(slots, num_slots, rows, slots.new_empty(4), status)
    _count(1)
    return LoraPlan(slots, num_slots, rows, _C().lora_plan(slots, num_slots, rows, status), status)


def _check(what: str, y: torch.Tensor, x: torch.Tensor, stack: LoraStack, plan: LoraPlan) -> None:
    if y.dim() != 2 or x.dim() != 2 or x.shape[1] != stack.in_features or y.shape[1] != stack.out_features \
            or x.shape[0] != y.shape[0]:
        raise ValueError(f"{what}: x {tuple(x.shape)} and y {tuple(y.shape)} do not fit a projection of "
                         f"{stack.in_features} to {stack.out_features}")
    if plan.num_tokens != x.shape[0] or plan.num_slots != stack.num_slots:
        raise ValueError(f"{what}: a plan of {plan.num_tokens} tokens and {plan.num_slots} slots for {x.shape[0]} tokens and "
                         f"{stack.num_slots} slots")
    if not x.device == y.device == stack.device == plan.slots.device:
        raise ValueError(f"{what}: tensors on {x.device}, {y.device}, {stack.device} and {plan.slots.device}")


def _launch(y, x, stack: LoraStack, plan: LoraPlan, out, kind, alpha, limit) -> torch.Tensor:
    if plan.num_tokens:
        _count(2)
    return _C().lora(x, y, out, stack.a, stack.b, stack.ranks, plan.buffer,
                     [plan.num_tokens, plan.num_slots, plan.rows, kind] + stack.sizes, alpha, limit, plan.status)


def lora_add(y: torch.Tensor, x: torch.Tensor, stack: LoraStack, plan: LoraPlan,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y + scale * B (A x)`` with the factors of each token's adapter: y [T, sum(slices)] is the shared product of
    x [T, in_features].  ``out`` may be ``y`` itself (rows without an adapter are then not touched)."""
    if stack.interleaved:
        raise ValueError("lora_add: the stack's columns are interleaved (lora_gated)")
    if x.is_cuda and plan.buffer is not None:
        return _launch(y, x, stack, plan, out, 0, 0.0, 0.0)
    _check("lora_add", y, x, stack, plan)
    if out is not None and (out.shape != y.shape or out.dtype != y.dtype or out.device != y.device):
        raise ValueError("lora_add: out has another shape, type or device than y")
    z = ref.lora_sum(y, x, stack, plan.slots).to(y.dtype)
    return z if out is None else out.copy_(z)


def lora_gated(y: torch.Tensor, x: torch.Tensor, stack: LoraStack, plan: LoraPlan, act=SILU) -> torch.Tensor:
    """``act(gate) * up`` of z = y + scale * B (A x), y [T, 2 I] being the shared gate / up product without its activation
    (columns in alternating groups of eight, an ``interleaved`` stack): [T, I].  ``act`` as in :func:`gemm`."""
    if not stack.interleaved:
        raise ValueError("lora_gated: the stack's columns are not interleaved")
    if x.is_cuda and plan.buffer is not None:
        return _launch(y, x, stack, plan, None, *_act_kind(True, act))
    _check("lora_gated", y, x, stack, plan)
    z = ref.lora_sum(y, x, stack, plan.slots).view(y.shape[0], -1, 2, 8)
    return ref.gated_act(z[:, :, 0], z[:, :, 1], act).reshape(y.shape[0], -1).to(y.dtype)

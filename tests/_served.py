"""Requests with rows in a shuffled page pool (float32 or int8) on the CPU, and what attending them gives in 64 bits."""

from __future__ import annotations

import torch

D = 128
SCALE = D ** -0.5


def quantized(x: torch.Tensor, slot: int) -> torch.Tensor:
    """Float32 rows ``[..., heads, 128]`` as slots ``[..., slot]`` of an int8 pool, each step rounded as IEEE says."""
    top = x.abs().amax(dim=-1)
    scale = top * (torch.tensor(1.0) / torch.tensor(127.0))
    scale = torch.where(scale == 0, torch.ones(()), scale)
    whole = torch.round(x / scale[..., None]).clamp(-127, 127)
    lost = ~torch.isfinite(x).all(dim=-1)
    scale = torch.where(lost, torch.full((), float("nan")), scale)
    out = torch.zeros(*x.shape[:-2], slot, dtype=torch.int8)
    heads = x.shape[-2]
    out[..., :128 * heads] = torch.where(lost[..., None], torch.zeros(()), whole).to(torch.int8).flatten(-2)
    out[..., 128 * heads:132 * heads] = scale.contiguous().view(torch.int8)
    return out


def values(slots: torch.Tensor, heads: int) -> torch.Tensor:
    """What slots stand for: float64 ``[..., heads, 128]``."""
    scale = slots[..., 128 * heads:132 * heads].contiguous().view(torch.float32).double()
    return slots[..., :128 * heads].unflatten(-1, (heads, D)).double() * scale[..., None]


def masks_of(parents: list[int]) -> list[int]:
    """The bits of every node's ancestors and its own, for one tree."""
    out: list[int] = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else 0) | 1 << i)
    return out


def signed(bits: int) -> int:
    return bits - (1 << 64) if bits >> 63 else bits


class Served:
    """Chunks of new tokens of requests with cached rows; ``lead`` and ``tail`` token rows belong to no chunk."""

    def __init__(self, seed, chunks, cached, *, heads=2, page_size=128, layers=2, spare=2, lead=0, tail=0, int8=True,
                 slot=None) -> None:
        g = self.g = torch.Generator().manual_seed(seed)
        self.chunks, self.cached, self.heads, self.page_size, self.layers = chunks, cached, heads, page_size, layers
        self.int8, self.lead = int8, lead
        per = [-(-(c + k) // page_size) for c, k in zip(chunks, cached)]
        pages = sum(per) + spare + 1
        order = torch.randperm(pages - 1, generator=g).tolist()
        self.table = torch.full((len(chunks), max(max(per), 1) + 1), pages - 1, dtype=torch.int32)
        for i, k in enumerate(per):
            self.table[i, :k] = torch.tensor(order[:k], dtype=torch.int32)
            order = order[k:]
        rows = torch.randn(pages, 2, layers, page_size, heads, D, generator=g)
        self.slot = slot or -(-132 * heads // 128) * 128
        self.pool = quantized(rows, self.slot) if int8 else rows
        if int8:  # what lies behind a slot's scales is nobody's
            self.pool[..., 132 * heads:] = 77
        self.offsets = torch.tensor([lead + sum(chunks[:i]) for i in range(len(chunks) + 1)], dtype=torch.int32)
        self.tokens = lead + sum(chunks) + tail
        self.qkv = torch.randn(self.tokens, 3, heads, D, generator=g)
        self.attend_max = max(1, max(c + k for c, k in zip(chunks, cached)))

    def each(self):
        """(request, token row, place in the chunk) of every chunk's token."""
        for i, c in enumerate(self.chunks):
            for j in range(c):
                yield i, int(self.offsets[i]) + j, j

    def positions(self) -> torch.Tensor:
        p = torch.zeros(self.tokens, dtype=torch.int32)
        for i, t, j in self.each():
            p[t] = self.cached[i] + j
        return p

    def place(self, i: int, row: int) -> tuple[int, int]:
        return int(self.table[i, row // self.page_size]), row % self.page_size

    def rows_of(self, pool, i, count, layer) -> tuple[torch.Tensor, torch.Tensor]:
        """Request i's first rows' keys and values, float64 [count, heads, D]."""
        per = [pool[int(p), :, layer] for p in self.table[i][:-(-count // self.page_size)]]
        if not per:
            return (torch.zeros(0, self.heads, D, dtype=torch.float64),) * 2
        rows = torch.cat(per, dim=1)[:, :count]
        rows = values(rows, self.heads) if self.int8 else rows.double()
        return rows[0], rows[1]

    def stored(self, layer, k, v, where=None) -> torch.Tensor:
        """The pool with the new rows in it; ``where`` each token's row (None: behind the cached ones)."""
        pool = self.pool.clone()
        for i, t, j in self.each():
            page, slot = self.place(i, self.cached[i] + j if where is None else where[t])
            for side, x in enumerate((k, v)):
                if not self.int8:
                    pool[page, side, layer, slot] = x[t]
                else:
                    pool[page, side, layer, slot, :132 * self.heads] = quantized(x[t], self.slot)[:132 * self.heads]
        return pool

    def want(self, pool, layer, q, *, seen=None, scale=SCALE) -> torch.Tensor:
        """Every token over the rows that ``seen(i, j)`` names (None: those up to its own), float64; 0 where there are
        none, and at tokens of no chunk."""
        out = torch.zeros(self.tokens, self.heads, D, dtype=torch.float64)
        for i, c in enumerate(self.chunks):
            if c == 0:
                continue
            keys, vals = self.rows_of(pool, i, self.cached[i] + c, layer)
            for j in range(c):
                rows = list(range(self.cached[i] + j + 1)) if seen is None else seen(i, j)
                if not rows:
                    continue
                t = int(self.offsets[i]) + j
                s = torch.einsum("hd,rhd->hr", q[t].double(), keys[rows]) * scale
                out[t] = torch.einsum("hr,rhd->hd", torch.softmax(s, dim=1), vals[rows])
        return out


def far(got: torch.Tensor, want: torch.Tensor) -> float:
    """The largest error of a token over that token's largest output (a token that must be 0 has to be)."""
    if got.numel() == 0:
        return 0.0
    err = (got.double() - want).abs().flatten(1).amax(dim=1)
    top = want.abs().flatten(1).amax(dim=1)
    return float(torch.where(top > 0, err / top, torch.where(err > 0, torch.inf, 0.0)).nan_to_num(torch.inf).max())

"""The paged cache's operators: attention of a chunk of new tokens, and the copying, forking, resizing and
compacting of a cache's pages, at the served decoder's sizes (10 attention heads of 128, 12 layers, pages of
128 rows).

The pool is fp32 ``[pages, 2 (k, v), layers, 128, heads, 128]``; its last page is the null page, which an unset
entry of a request's row of the lookup table names.  A case is a dict of plain values:

``kind``      ``attention`` (``paged_chunk_attention``, or with ``rope`` ``paged_chunk_attention_qkv``), ``copy``
              (``copy_pages``), ``fork`` (``fork_pages``), ``resize`` (``resize_pages``) or ``compact``
              (``compact_pages``).
``requests``  requests of the call (fork, resize and compact: rows of the lookup table).
``tokens``    the longest chunk (attention); ``cached`` the most rows a request has in the cache before it.
``ragged``    whether the chunks' lengths differ.
``layers``    layers of the pool.
``pairs``     pages copied (copy), ``partial`` whether only their first rows.
``children``  requests forked (fork); ``length`` the longest request's rows (fork, resize, compact); ``shared``
              how many of its first rows a child shares with its parent.
``pages``     pages of the pool (resize).
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PKG = str(Path(__file__).resolve().parent.parent / "unlimited-ocr-max_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

HEADS, D, PAGE, H = 10, 128, 128, 1280
LAYERS = 12
LAYER = 1  # of the attention cases' pool of two
SCALE = D ** -0.5
DEV = "cuda:0"


def listed() -> list[dict]:
    return [
        # Four draft tokens of one request checked at once: the smallest call, bound by latency.
        {"name": "chunk-b1-t4", "kind": "attention", "requests": 1, "tokens": 4, "cached": 300, "ragged": False,
         "rope": True},
        # Draft tokens of a full batch, late in the answers: the cache's bytes count.
        {"name": "chunk-b8-t7", "kind": "attention", "requests": 8, "tokens": 7, "cached": 1150, "ragged": True,
         "rope": False},
        # Eight prompts of up to 512 tokens (a page of 273 image rows and an instruction, and longer ones).
        {"name": "prompts-b8-t512", "kind": "attention", "requests": 8, "tokens": 512, "cached": 0, "ragged": True,
         "rope": True},
        # A further piece of a long document's prompt: the largest call.
        {"name": "chunk-b1-t2048", "kind": "attention", "requests": 1, "tokens": 2048, "cached": 14001,
         "ragged": False, "rope": False},
        # One page set aside before it is written to.
        {"name": "copy-1", "kind": "copy", "pairs": 1, "layers": LAYERS, "partial": False},
        # The last, part filled pages of many requests.
        {"name": "copy-24-partial", "kind": "copy", "pairs": 24, "layers": LAYERS, "partial": True},
        # One request's prompt continued three ways: the prompt's full pages are shared.
        {"name": "fork-3", "kind": "fork", "requests": 4, "children": 3, "length": 345, "shared": 291,
         "layers": LAYERS},
        # A beam step of a full batch of requests with four beams each; half of the beams change their parent.
        {"name": "fork-16-of-32", "kind": "fork", "requests": 32, "children": 16, "length": 640, "shared": 512,
         "layers": 4},
        # Two requests end and two begin in a small server.
        {"name": "resize-b8", "kind": "resize", "requests": 8, "length": 640, "pages": 81},
        # The same in a large one, with long requests.
        {"name": "resize-b256", "kind": "resize", "requests": 256, "length": 4000, "pages": 6001},
        # A small pool after its first requests ended.
        {"name": "compact-b6", "kind": "compact", "requests": 6, "length": 291, "layers": 2},
        # A full batch's pool, all layers, before part of it is given back.
        {"name": "compact-b24", "kind": "compact", "requests": 24, "length": 640, "layers": LAYERS},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng) -> dict:
    kind = rng.choice(["attention", "attention", "attention", "copy", "fork", "resize", "compact"])
    if kind == "attention":
        while True:
            case = {"kind": kind, "requests": _log_int(rng, 1, 8), "tokens": _log_int(rng, 1, 2048),
                    "cached": rng.choice([0, _log_int(rng, 1, 14001), _log_int(rng, 1, 14001)]),
                    "ragged": rng.random() < 0.5, "rope": rng.random() < 0.5}
            largest = work(listed()[3])
            cost = work(case)
            if cost["flops"] <= largest["flops"] and case["requests"] * (case["cached"] + case["tokens"]) <= 40000:
                return case
    if kind == "copy":
        return {"kind": kind, "pairs": _log_int(rng, 1, 24), "layers": rng.randint(1, LAYERS),
                "partial": rng.random() < 0.5}
    if kind == "fork":
        requests = _log_int(rng, 2, 32)
        length = _log_int(rng, 1, 640)
        return {"kind": kind, "requests": requests, "children": rng.randint(1, requests // 2), "length": length,
                "shared": rng.randint(0, length), "layers": rng.randint(1, 4)}
    if kind == "resize":
        requests = _log_int(rng, 1, 256)
        length = _log_int(rng, 1, 4000)
        return {"kind": kind, "requests": requests, "length": length,
                "pages": requests * -(-length // PAGE) + rng.randint(1, 500)}
    return {"kind": kind, "requests": _log_int(rng, 1, 24), "length": _log_int(rng, 1, 640),
            "layers": rng.randint(1, LAYERS)}


# ------------------------------------------------------------------------------------------ inputs


class _Draws:
    """Seeded tensors on the GPU."""

    def __init__(self, seed: int) -> None:
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, *shape: int) -> torch.Tensor:
        return torch.randn(shape, generator=self.g, device=DEV)

    def pages(self, n: int) -> list[int]:
        return torch.randperm(n, generator=self.g, device=DEV).tolist()

    def ints(self, low: int, high: int, n: int) -> list[int]:
        """n whole numbers of [low, high]."""
        return torch.randint(low, high + 1, (n,), generator=self.g, device=DEV).tolist()


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _spread(most: int, n: int, ragged: bool) -> list[int]:
    """n lengths: the first is the longest, the others down to a third of it."""
    return [max(1, most - (i * 2 * most) // (3 * n)) if ragged else most for i in range(n)]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Each request's chunk and the rows before it."""
    n = case["requests"]
    cached = [c if case["cached"] else 0 for c in _spread(case["cached"], n, True)]
    return _spread(case["tokens"], n, case["ragged"]), cached


def _pages_of(length: int) -> int:
    return -(-length // PAGE)


def _angles(rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 10000.0 ** -(torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    angle = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
    angle = torch.cat([angle, angle], dim=1)
    return angle.cos().float(), angle.sin().float()


def _attention_state(case: dict, seed: int) -> dict:
    d = _Draws(seed)
    chunk, cached = _lengths(case)
    cols = max(_pages_of(c + t) for c, t in zip(cached, chunk))
    used = sum(_pages_of(c + t) for c, t in zip(cached, chunk))
    order = iter(d.pages(used))
    table = [[next(order) if p < _pages_of(c + t) else used for p in range(cols)] for c, t in zip(cached, chunk)]
    offsets = [sum(chunk[:i]) for i in range(len(chunk) + 1)]
    state = {"pool": d.normal(used + 1, 2, 2, PAGE, HEADS, D), "table": _i32(table), "cached": _i32(cached),
             "offsets": _i32(offsets), "qkv": d.normal(offsets[-1], 3 * H), "most": max(chunk), "total": offsets[-1],
             "attend": max(c + t for c, t in zip(cached, chunk)), "rope": case["rope"]}
    state["positions"] = _i32([c + i for c, t in zip(cached, chunk) for i in range(t)])
    state["cos"], state["sin"] = _angles(state["attend"])
    return state


def _copy_state(case: dict, seed: int) -> dict:
    d = _Draws(seed)
    n = case["pairs"]
    order = d.pages(2 * n + 3)
    return {"pool": d.normal(2 * n + 4, 2, case["layers"], PAGE, HEADS, D), "src": _i32(order[:n]),
            "dst": _i32(order[n:2 * n]), "rows": _i32(d.ints(1, PAGE, n)) if case["partial"] else None}


def _requests(d: _Draws, case: dict, pages: int, cols: int, held: list[int]) -> tuple[torch.Tensor, torch.Tensor]:
    """A lookup table and the pages' counts: each request holds pages of its own, as many as `held` says."""
    order = iter(d.pages(pages - 1))
    table = [[next(order) if c < n else pages - 1 for c in range(cols)] for n in held]
    counts = torch.zeros(pages, dtype=torch.int32, device=DEV)
    flat = torch.tensor(table, device=DEV).flatten()
    counts[flat[flat < pages - 1]] = 1
    return _i32(table), counts


def _fork_state(case: dict, seed: int) -> dict:
    d = _Draws(seed)
    n, kids = case["requests"], case["children"]
    cols = _pages_of(case["length"])
    lengths = _spread(case["length"], n, True)
    order = d.pages(n)
    children, parents = order[:kids], [order[kids + i % (n - kids)] for i in range(kids)]
    # a child's old pages are released; its new ones come from those free before
    held = [_pages_of(x) for x in lengths]
    copied = [_pages_of(lengths[p]) - min(case["shared"] // PAGE, _pages_of(lengths[p])) for p in parents]
    pages = sum(held) + kids * cols + 4
    table, counts = _requests(d, case, pages, cols, held)
    return {"pool": d.normal(pages, 2, case["layers"], PAGE, HEADS, D), "table": table, "counts": counts,
            "parents": _i32(parents), "children": _i32(children), "lengths": _i32([lengths[p] for p in parents]),
            "shared": _i32([case["shared"]] * kids), "copied": sum(copied)}


def _resize_state(case: dict, seed: int) -> dict:
    d = _Draws(seed)
    n, pages = case["requests"], case["pages"]
    cols = _pages_of(case["length"])
    now = d.ints(1, case["length"], n)
    then = [x if k % 4 else d.ints(0, case["length"], 1)[0] for k, x in enumerate(now)]  # one in four changes
    table, counts = _requests(d, case, pages, cols, [_pages_of(x) for x in now])
    return {"table": table, "counts": counts, "lengths": _i32(then)}


def _compact_state(case: dict, seed: int) -> dict:
    d = _Draws(seed)
    held = [_pages_of(x) for x in _spread(case["length"], case["requests"], True)]
    pages = 2 * sum(held) + 1  # about half of the pages were freed
    table, counts = _requests(d, case, pages, max(held), held)
    live = sum(held)
    return {"pool": d.normal(pages, 2, case["layers"], PAGE, HEADS, D), "table": table, "counts": counts,
            "live": live, "moved": int((counts[live:] > 0).sum())}


def prepare(case: dict, seed: int) -> dict:
    make = {"attention": _attention_state, "copy": _copy_state, "fork": _fork_state, "resize": _resize_state,
            "compact": _compact_state}[case["kind"]]
    return {"kind": case["kind"], **make(case, seed)}


# ------------------------------------------------------------------------------------------ the plain forms


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = D // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _plain_attention(s: dict) -> dict:
    q, k, v = s["qkv"].view(s["total"], 3, HEADS, D).unbind(1)
    if s["rope"]:
        at = s["positions"].long()
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    offsets, cached, table = s["offsets"].long(), s["cached"].long(), s["table"].long()
    token = torch.arange(s["total"], device=DEV)
    request = (token[:, None] >= offsets[None, 1:]).sum(dim=1)
    inside = token - offsets[request]
    row = cached[request] + inside
    page = table[request, row // PAGE]
    s["pool"][page, 0, LAYER, row % PAGE] = k
    s["pool"][page, 1, LAYER, row % PAGE] = v
    n = table.shape[0]
    keys, values = (s["pool"][table, j, LAYER].flatten(1, 2)[:, :s["attend"]] for j in (0, 1))  # [n, rows, heads, D]
    padded = q.new_zeros(n, s["most"], HEADS, D)
    padded[request, inside] = q
    last = cached[:, None] + torch.arange(s["most"], device=DEV)[None, :]
    seen = torch.arange(s["attend"], device=DEV)[None, None, :] <= last[:, :, None]
    score = padded.permute(0, 2, 1, 3).contiguous() @ keys.permute(0, 2, 3, 1).contiguous() * SCALE
    score = score.masked_fill(~seen[:, None], -math.inf)
    weight = torch.exp(score - score.amax(dim=3, keepdim=True))
    weight = weight / weight.sum(dim=3, keepdim=True)
    weight = weight @ values.permute(0, 2, 1, 3).contiguous()  # [n, heads, most, D]
    return {"out": weight.permute(0, 2, 1, 3)[request, inside], "pool": s["pool"]}


def _copy_rows(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, rows: torch.Tensor) -> None:
    """The first rows[i] rows of page src[i], all layers, into page dst[i]."""
    slot = torch.arange(PAGE, device=DEV)
    kept = (slot[None, :] < rows[:, None])[:, None, None, :, None, None]
    pool[dst] = torch.where(kept, pool[src], pool[dst])


def _plain_copy(s: dict) -> dict:
    src, dst = s["src"].long(), s["dst"].long()
    if s["rows"] is None:
        s["pool"][dst] = s["pool"][src]
    else:
        _copy_rows(s["pool"], src, dst, s["rows"])
    return {"pool": s["pool"]}


def _free_pages(counts: torch.Tensor) -> torch.Tensor:
    """The pages nobody holds in ascending order (then the others); the null page is nobody's to take."""
    taken = (counts > 0).int()
    taken[-1] = 2
    return torch.sort(taken, stable=True).indices


def _plain_fork(s: dict) -> dict:
    table, counts = s["table"].clone(), s["counts"].clone()
    null, (n, cols) = counts.shape[0] - 1, table.shape
    column = torch.arange(cols, device=DEV)[None, :]
    need = (s["lengths"][:, None] + PAGE - 1) // PAGE
    old = table[s["parents"].long()]
    held = (column < need) & (old != null)
    share = held & (column < s["shared"][:, None] // PAGE)
    copy = held & ~share
    rank = copy.flatten().int().cumsum(0).view_as(copy) - 1
    fresh = _free_pages(counts)[rank.clamp(min=0)].int()
    new = torch.where(copy, fresh, torch.where(share, old, null))
    # the pages to copy, first in (child, column) order
    at = torch.sort((~copy).flatten().int(), stable=True).indices[:s["copied"]]
    rows = (s["lengths"][:, None] - column * PAGE).clamp(max=PAGE).flatten()[at]
    _copy_rows(s["pool"], old.flatten()[at].long(), new.flatten()[at].long(), rows)
    gone = table[s["children"].long()].flatten().long()
    counts.index_add_(0, new.flatten().long(), torch.ones_like(new.flatten()))
    counts.index_add_(0, gone, -torch.ones_like(gone, dtype=torch.int32))
    counts[null] = s["counts"][null]
    table[s["children"].long()] = new
    return {"pool": s["pool"], "table": table, "counts": counts, "missing": copy.new_zeros(1, dtype=torch.int32)}


def _plain_resize(s: dict) -> dict:
    table, counts = s["table"].clone(), s["counts"].clone()
    null, (n, cols) = counts.shape[0] - 1, table.shape
    need = torch.arange(cols, device=DEV)[None, :] < (s["lengths"][:, None] + PAGE - 1) // PAGE
    gone = (~need) & (table != null)
    counts.index_add_(0, table.flatten().long(), -gone.flatten().int())
    wanted = need & (table == null)
    free = _free_pages(counts)
    rank = wanted.flatten().int().cumsum(0).view_as(wanted) - 1
    served = wanted & (rank < (counts[:-1] <= 0).sum())
    fresh = free[rank.clamp(min=0)].int()
    counts.index_add_(0, torch.where(served, fresh, null).flatten().long(), served.flatten().int())
    table = torch.where(served, fresh, torch.where(need, table, null))
    return {"table": table, "counts": counts, "missing": (wanted & ~served).sum().int().view(1)}


def _plain_compact(s: dict) -> dict:
    counts, pool = s["counts"], s["pool"]
    null = counts.shape[0] - 1
    live = (counts > 0).int()
    live[null] = 0
    number = torch.arange(null + 1, device=DEV)
    first = number < live.sum()
    source = torch.sort((~((live > 0) & ~first)).int(), stable=True).indices[:s["moved"]]
    hole = torch.sort((~((live == 0) & first)).int(), stable=True).indices[:s["moved"]]
    pool[hole] = pool[source]
    remap = torch.where(live > 0, number, -1)
    remap[source] = hole
    remap[null] = null
    moved = counts.clone()
    moved[hole] = counts[source]
    moved[source] = 0
    return {"pool": pool, "table": remap[s["table"].long()].int(), "counts": moved, "remap": remap.int()}


# ------------------------------------------------------------------------------------------ the calls


def _own_run(s: dict) -> dict:
    import uocr_moe

    kind = s["kind"]
    if kind == "attention":
        kv = uocr_moe.PagedChunk(kv_blocks=s["pool"], lookup_table=s["table"], cache_lengths=s["cached"],
                                 chunk_offsets=s["offsets"], attend_max=s["attend"])
        if s["rope"]:
            out = uocr_moe.paged_chunk_attention_qkv(s["qkv"], s["positions"], s["cos"], s["sin"], heads=HEADS, kv=kv,
                                                     layer_idx=LAYER, scale=SCALE)
        else:
            q, k, v = s["qkv"].view(s["total"], 3, HEADS, D).unbind(1)
            out = uocr_moe.paged_chunk_attention(q, k, v, kv=kv, layer_idx=LAYER, scale=SCALE)
        return {"out": out, "pool": s["pool"]}
    if kind == "copy":
        return {"pool": uocr_moe.copy_pages(s["pool"], s["src"], s["dst"], rows=s["rows"])}
    if kind == "fork":
        table, counts, missing = uocr_moe.fork_pages(s["pool"], s["counts"], s["table"], s["parents"], s["children"],
                                                     s["lengths"], s["shared"])
        return {"pool": s["pool"], "table": table, "counts": counts, "missing": missing}
    if kind == "resize":
        table, counts, missing = uocr_moe.resize_pages(s["counts"], s["table"], s["lengths"], page_size=PAGE)
        return {"table": table, "counts": counts, "missing": missing}
    table, counts, remap = uocr_moe.compact_pages(s["pool"], s["counts"], s["table"])
    return {"pool": s["pool"], "table": table, "counts": counts, "remap": remap}


def run(state: dict) -> dict:
    if own:
        return _own_run(state)
    plain = {"attention": _plain_attention, "copy": _plain_copy, "fork": _plain_fork, "resize": _plain_resize,
             "compact": _plain_compact}[state["kind"]]
    return plain(state)


# ------------------------------------------------------------------------------------------ what a pass needs


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "attention":
        chunk, cached = _lengths(case)
        tokens = sum(chunk)
        pairs = sum(t * c + t * (t + 1) // 2 for t, c in zip(chunk, cached))
        # q, k and v read, the output and the new rows written; the cached rows read once
        return {"bytes": 4 * H * (6 * tokens + 2 * sum(cached)), "flops": 4.0 * H * pairs}
    slot = 2 * H * 4  # bytes of one layer's k and v rows
    if kind == "copy":
        rows = PAGE // 2 if case["partial"] else PAGE
        return {"bytes": 2 * case["pairs"] * rows * case["layers"] * slot, "flops": 0}
    n, cols = case["requests"], _pages_of(case["length"])
    if kind == "resize":
        return {"bytes": 4 * (2 * n * cols + 2 * case["pages"] + n + 1), "flops": 0}
    lengths = _spread(case["length"], n, True)
    if kind == "fork":
        tables = 4 * (2 * n * cols + 4 * case["children"])
        mean = sum(max(0, x - case["shared"] // PAGE * PAGE) for x in lengths) / n
        return {"bytes": tables + 2 * case["children"] * mean * case["layers"] * slot, "flops": 0}
    live = sum(_pages_of(x) for x in lengths)
    return {"bytes": 4 * (2 * n * cols + 6 * live) + live * PAGE * case["layers"] * slot, "flops": 0}


# ------------------------------------------------------------------------------------------ the 64-bit values


def _exact_attention(case: dict, seed: int) -> dict:
    s = _attention_state(case, seed)
    pool = s["pool"].double()
    chunk, cached = _lengths(case)
    out = torch.empty(s["total"], HEADS, D, dtype=torch.float64, device=DEV)
    begin = 0
    for pages, t, c in zip(s["table"].tolist(), chunk, cached):
        qkv = s["qkv"][begin:begin + t].double()
        parts = []
        for j in range(3):
            x = qkv[:, j * H:(j + 1) * H].reshape(t, HEADS, D)
            if s["rope"] and j < 2:
                cos, sin = (m[c:c + t, None, :].double() for m in (s["cos"], s["sin"]))
                low, high = x[..., :D // 2], x[..., D // 2:]
                x = torch.cat([low * cos[..., :D // 2] - high * sin[..., :D // 2],
                               high * cos[..., D // 2:] + low * sin[..., D // 2:]], dim=2)
            parts.append(x)
        for j in (0, 1):
            for p in range(c // PAGE, (c + t - 1) // PAGE + 1):
                low, high = max(c, p * PAGE), min(c + t, (p + 1) * PAGE)
                pool[pages[p], j, LAYER, low - p * PAGE:high - p * PAGE] = parts[1 + j][low - c:high - c]
        at = torch.tensor(pages[:_pages_of(c + t)], device=DEV)
        hidden = torch.ones(t, c + t, dtype=torch.bool, device=DEV).triu(c + 1)
        for h in range(HEADS):
            keys, values = (pool[at, j, LAYER, :, h].reshape(-1, D)[:c + t] for j in (0, 1))
            score = torch.mm(parts[0][:, h].contiguous(), keys.t()) * SCALE
            out[begin:begin + t, h] = torch.mm(torch.softmax(score.masked_fill_(hidden, -math.inf), dim=1), values)
        begin += t
    return {"out": out, "pool": pool}


def _exact_pages(case: dict, seed: int) -> dict:
    """The page operators one page at a time, on lists."""
    s = prepare(case, seed)
    pool = s["pool"].double() if "pool" in s else None
    if case["kind"] == "copy":
        rows = s["rows"].tolist() if s["rows"] is not None else [PAGE] * case["pairs"]
        for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), rows):
            pool[b, :, :, :n] = pool[a, :, :, :n]
        return {"pool": pool}
    table, counts = s["table"].tolist(), s["counts"].tolist()
    null, cols = len(counts) - 1, len(table[0])
    if case["kind"] == "compact":
        live = [p for p in range(null) if counts[p] > 0]
        holes = [p for p in range(len(live)) if counts[p] <= 0]
        remap = [p if counts[p] > 0 else -1 for p in range(null)] + [null]
        for p in live:
            if p >= len(live):
                remap[p] = holes.pop(0)
                pool[remap[p]] = pool[p]
                counts[remap[p]], counts[p] = counts[p], 0
        return {"pool": pool, "table": _i32([[remap[p] for p in row] for row in table]), "counts": _i32(counts),
                "remap": _i32(remap)}
    missing = 0
    if case["kind"] == "fork":
        free = [p for p in range(null) if counts[p] <= 0]
        rows = [list(r) for r in table]
        for a, b, length, shared in zip(*(s[k].tolist() for k in ("parents", "children", "lengths", "shared"))):
            for c in range(cols):
                old, page = rows[a][c], null
                if c * PAGE < length and old != null:
                    if (c + 1) * PAGE <= shared:
                        page = old
                    else:
                        page = free.pop(0)
                        n = min(PAGE, length - c * PAGE)
                        pool[page, :, :, :n] = pool[old, :, :, :n]
                    counts[page] += 1
                if rows[b][c] != null:
                    counts[rows[b][c]] -= 1
                table[b][c] = page
        return {"pool": pool, "table": _i32(table), "counts": _i32(counts), "missing": _i32([missing])}
    lengths = s["lengths"].tolist()
    for row, length in zip(table, lengths):
        for c in range(_pages_of(length), cols):
            if row[c] != null:
                counts[row[c]] -= 1
                row[c] = null
    free = [p for p in range(null) if counts[p] <= 0]
    for row, length in zip(table, lengths):
        for c in range(_pages_of(length)):
            if row[c] == null:
                if free:
                    row[c] = free.pop(0)
                    counts[row[c]] = 1
                else:
                    missing += 1
    return {"table": _i32(table), "counts": _i32(counts), "missing": _i32([missing])}


def exact(case: dict, seed: int) -> dict:
    return _exact_attention(case, seed) if case["kind"] == "attention" else _exact_pages(case, seed)

"""GPU tests of the served operators as they are used: prompts into an int8 pool, beams over it, drafts verified against it,
the decoder's step on it.

A token's output follows from its sequence alone, so what a run with forks, rejections and cut prompts left in the pages is
held against the same tokens sent as one prompt into pages of their own: each of the two outputs is within 1e-5 of a token's
largest output (the attention's bar), so they are within 2e-5 of one another, and the pool's rows are equal.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from _gpu import DEV, layer_weights, n, t
from _served import D, SCALE, quantized, values

pytestmark = pytest.mark.gpu

BAR = 1e-5
HEADS, LAYERS, P, VOCAB = 3, 2, 128, 97


def _uocr():
    import uocr_moe

    return uocr_moe


def _on(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


class Model:
    """A row of q, k and v for each token, and logits from the attention's output."""

    def __init__(self, seed: int) -> None:
        g = torch.Generator().manual_seed(seed)
        self.rows = torch.randn(VOCAB, 3 * HEADS * D, generator=g).to(DEV)
        self.head = torch.randn(HEADS * D, VOCAB, generator=g).to(DEV)
        self.cos, self.sin = (torch.from_numpy(x).to(DEV) for x in
                              _uocr().rope_tables(head_dim=D, seq_len=2048, theta=10000.0))

    def chunk(self, tokens, positions, kv, layer=1) -> torch.Tensor:
        return _uocr().paged_chunk_attention_qkv(self.rows[tokens.long()], positions, self.cos, self.sin, heads=HEADS, kv=kv,
                                                 layer_idx=layer, scale=SCALE)

    def decode(self, tokens, positions, kv, layer=1) -> torch.Tensor:
        return _uocr().paged_decode_attention_qkv(self.rows[tokens.long()], positions, self.cos, self.sin, heads=HEADS, kv=kv,
                                                  layer_idx=layer, scale=SCALE)

    def logits(self, out) -> torch.Tensor:
        return out.flatten(1) @ self.head

    def alone(self, tokens: list[int], pool) -> tuple[torch.Tensor, torch.Tensor]:
        """The tokens as one prompt in pages 0, 1, ... of an empty pool like ``pool``: (every token's output, that pool)."""
        cols = -(-len(tokens) // P)
        own = torch.zeros(cols + 1, *pool.shape[1:], dtype=pool.dtype, device=DEV)
        kv = _uocr().PagedChunk(kv_blocks=own, lookup_table=_on([list(range(cols))]), cache_lengths=_on([0]),
                                chunk_offsets=_on([0, len(tokens)]), attend_max=len(tokens))
        return self.chunk(_on(tokens), torch.arange(len(tokens), dtype=torch.int32, device=DEV), kv), own


def _near(got: torch.Tensor, want: torch.Tensor) -> None:
    assert float((got - want).abs().max()) <= 2 * BAR * float(want.abs().max())


def _rows(pool, table, length, layer=1) -> torch.Tensor:
    """A request's rows of a layer, [2, length, ...], from its pages."""
    pages = pool[table[:-(-length // P)].long(), :, layer]
    return pages.transpose(0, 1).flatten(1, 2)[:, :length]


def test_beams_over_an_int8_pool() -> None:
    """Prompts, forked to beams; steps of decode, n-gram guard, selection and fork, over a page's end."""
    u = _uocr()
    m = Model(1)
    beams, prompts = 4, [[int(x) for x in torch.randint(2, VOCAB, (k,), generator=torch.Generator().manual_seed(k))]
                         for k in (125, 40, 260)]
    rows, cols, pages, eos, width = beams * len(prompts), 4, 40, 1, 6
    pool = u.int8_kv_blocks(pages, LAYERS, P, HEADS)
    table = torch.full((rows, cols), pages - 1, dtype=torch.int32, device=DEV)
    table[:] = -1
    counts = torch.zeros(pages, dtype=torch.int32, device=DEV)
    first = torch.arange(0, rows, beams, device=DEV)
    want_rows = torch.zeros(rows, dtype=torch.int32, device=DEV)
    want_rows[first] = _on([len(p) for p in prompts])
    table, counts, missing = u.resize_pages(counts, table, want_rows, page_size=P)
    assert int(missing) == 0
    offsets = [0]
    for p in prompts:
        offsets.append(offsets[-1] + len(p))
    kv = u.PagedChunk(kv_blocks=pool, lookup_table=table[first].contiguous(), cache_lengths=_on([0, 0, 0]),
                      chunk_offsets=_on(offsets), attend_max=260)
    out = m.chunk(_on([x for p in prompts for x in p]), _on([i for p in prompts for i in range(len(p))]), kv)
    lengths = _on([len(p) for p in prompts]).repeat_interleave(beams)
    children = torch.arange(rows, dtype=torch.int32, device=DEV)
    parents = first.to(torch.int32).repeat_interleave(beams)
    table, counts, missing = u.fork_pages(pool, counts, table, parents, children, lengths, lengths)
    assert int(missing) == 0
    logits = m.logits(out[_on(offsets[1:]).long() - 1]).repeat_interleave(beams, dim=0).contiguous()
    scores = torch.full((rows,), -math.inf, device=DEV)
    scores[first] = 0.0
    history = torch.stack([_on(prompts[r // beams][-width:]) for r in range(rows)])
    ended, words = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV)
    said: list[list[int]] = [[] for _ in range(rows)]
    for step in range(8):
        guarded = u.ngram_block(logits, history, 2)
        best = u.beam_select(guarded, scores, beams=beams, eos=eos, ended=ended, lengths=words, alpha=0.6, history=history)
        # selection, in 64 bits
        keys = scores.double()[:, None] + guarded.double().log_softmax(dim=1)
        stay = ended.bool()
        keys[stay] = -math.inf
        keys[stay, eos] = scores.double()[stay]
        ranks = keys / (words.double() + (~stay).double()).clamp(min=1)[:, None] ** 0.6
        for r in range(len(prompts)):
            mine = slice(r * beams, r * beams + beams)
            order = torch.argsort(ranks[mine].flatten(), descending=True, stable=True)[:beams].cpu()
            assert best.tokens[mine].tolist() == (order % VOCAB).tolist()
            assert best.parents[mine].tolist() == (order // VOCAB + r * beams).tolist()
        tokens, from_rows = best.tokens.tolist(), best.parents.tolist()
        over = ended.tolist()
        said = [said[p] + ([] if over[p] else [x]) for p, x in zip(from_rows, tokens)]
        scores, ended, words, history = best.scores, best.ended, best.lengths, best.history
        assert words.tolist() == [len(x) for x in said]
        table, counts, missing = u.fork_pages(pool, counts, table, best.parents, children, lengths, lengths)
        assert int(missing) == 0
        table, counts, missing = u.resize_pages(counts, table, lengths + 1, page_size=P)
        assert int(missing) == 0
        kv = u.PagedKv(kv_blocks=pool, lookup_table=table, attend_lengths=lengths, attend_max=int(lengths.max()) + 1,
                       write_index=lengths)
        out = m.decode(best.tokens, lengths, kv)
        logits = m.logits(out)
        lengths = lengths + 1
    checked = 0
    for r in range(rows):
        if int(ended[r]):
            continue
        checked += 1
        sequence = prompts[r // beams] + said[r]
        assert len(sequence) == int(lengths[r])
        want, own = m.alone(sequence, pool)
        _near(out[r], want[-1])
        assert torch.equal(_rows(pool, table[r], len(sequence)), _rows(own, torch.arange(4), len(sequence)))
    assert checked >= 3


@pytest.mark.parametrize("int8", [True, False], ids=["int8", "fp32"])
def test_drafts_over_either_pool(int8) -> None:
    """Trees of drafts, some of whose branches are what the model says: masks, attention, acceptance, step after step."""
    u = _uocr()
    m = Model(2)
    g = torch.Generator().manual_seed(3)
    prompts = [[int(x) for x in torch.randint(0, VOCAB, (k,), generator=g)] for k in (120, 7, 250)]
    cols, pages = 4, 14
    pool = u.int8_kv_blocks(pages, LAYERS, P, HEADS) if int8 else \
        torch.zeros(pages, 2, LAYERS, P, HEADS, D, device=DEV)
    order = torch.randperm(pages - 1, generator=g)[:12].to(torch.int32).view(3, cols).to(DEV)
    for r, p in enumerate(prompts):  # all but the last token, which is the first tree's root
        for layer in range(LAYERS):
            kv = u.PagedChunk(kv_blocks=pool, lookup_table=order[r:r + 1], cache_lengths=_on([0]), chunk_offsets=_on([0, len(p) - 1]),
                              attend_max=len(p) - 1)
            m.chunk(_on(p[:-1]), torch.arange(len(p) - 1, dtype=torch.int32, device=DEV), kv, layer)
    cached = _on([len(p) - 1 for p in prompts])
    said = [list(p) for p in prompts]

    def says(sequence: list[int]) -> tuple[int, torch.Tensor]:
        out, _ = m.alone(sequence, pool)
        return int(m.logits(out[-1:]).argmax()), out[-1]

    for step in range(3):
        parents, tokens, depth, offsets = [], [], [], [0]
        for r in range(3):
            right = [said[r][-1]]
            for _ in range((2, 0, 4)[(r + step) % 3]):
                right.append(says(said[r] + right[1:])[0])
            tree = [(-1, right[0], 0)]
            path = 0
            for k, x in enumerate(right[1:]):  # a wrong child before the right one
                tree.append((path, (x + 1) % VOCAB, k + 1))
                tree.append((path, x, k + 1))
                path = len(tree) - 1
            tree.append((path, VOCAB, len(right)))  # what nobody says
            parents += [a for a, _, _ in tree]
            tokens += [b for _, b, _ in tree]
            depth += [c for _, _, c in tree]
            offsets.append(len(parents))
        chunk_offsets = _on(offsets)
        masks = u.draft_masks(_on(parents), chunk_offsets)
        positions = _on(depth) + cached.repeat_interleave(chunk_offsets.diff())
        kv = u.PagedChunk(kv_blocks=pool, lookup_table=order, cache_lengths=cached, chunk_offsets=chunk_offsets,
                          attend_max=int((cached + chunk_offsets.diff()).max()), visible=masks)
        drafted = _on(tokens)
        for layer in range(LAYERS):
            out = m.chunk(drafted.clamp(max=VOCAB - 1), positions, kv, layer)
        answers = m.logits(out).argmax(dim=1).to(torch.int32)
        counts, path, following, lengths = u.accept_drafts(kv, _on(parents), drafted, answers)
        assert counts.tolist() == [1 + (2, 0, 4)[(r + step) % 3] for r in range(3)]
        for r in range(3):
            taken = path[offsets[r]:offsets[r] + int(counts[r])].tolist()
            assert taken == [0] + [2 * (k + 1) for k in range(int(counts[r]) - 1)]
            said[r] += [tokens[offsets[r] + x] for x in taken[1:]]
            assert int(lengths[r]) == len(said[r])
            answer, want = says(said[r])
            assert int(following[r]) == answer
            _near(out[offsets[r] + taken[-1]], want)
            _, own = m.alone(said[r], pool)
            for layer in range(LAYERS):
                assert torch.equal(_rows(pool, order[r], len(said[r]), layer), _rows(own, torch.arange(cols), len(said[r])))
            said[r].append(answer)
        cached = lengths
    last = _on([s[-1] for s in said])
    kv = u.PagedKv(kv_blocks=pool, lookup_table=order, attend_lengths=cached, attend_max=int(cached.max()) + 1, write_index=cached)
    out = m.decode(last, cached, kv)
    for r in range(3):
        _near(out[r], says(said[r])[1])


def test_a_page_converted_serves_as_it_was() -> None:
    """Rows of a float32 pool, quantised into an int8 one, are those that its own writes give; and back, their values."""
    u = _uocr()
    m = Model(4)
    tokens = [int(x) for x in torch.randint(0, VOCAB, (200,), generator=torch.Generator().manual_seed(5))]
    _, wide = m.alone(tokens, torch.zeros(1, 2, LAYERS, P, HEADS, D, device=DEV))
    _, narrow = m.alone(tokens, u.int8_kv_blocks(1, LAYERS, P, HEADS))
    got = u.int8_kv_blocks(4, LAYERS, P, HEADS)
    u.quantize_pages(wide, _on([0, 1]), got, _on([3, 0]), rows=_on([128, 72]))
    assert torch.equal(got[[3, 0], :, 1], narrow[:2, :, 1])
    back = torch.zeros_like(wide)
    u.dequantize_pages(got, _on([3, 0]), back, _on([0, 1]))
    # half a step of a row's scale, and the product's rounding
    steps = wide.abs().amax(dim=-1, keepdim=True) / 127
    assert bool(((back - wide).abs()[:2] <= 0.5 * steps[:2] * (1 + 2 ** -14)).all())


def test_the_decoders_step_on_an_int8_pool(oracle) -> None:
    """As over a float32 pool (1e-4 of the chain in 64 bits), of the keys and values that the int8 pool holds: those are
    the chain's own to half a step of a row's scale, and the 1e-4 of the projections before it."""
    from test_gpu_decoder import E, FFN, HID, _decoder_weights, _norm64, _rel, _rope64
    from test_gpu_decoder import HEADS as H
    from test_gpu_decoder import LAYERS as L
    from test_gpu_decoder import VOCAB as V

    u = _uocr()
    w, moes = _decoder_weights(oracle)
    gw = {k: t(v) for k, v in w.items()}
    for i, layer in moes.items():
        gw.update({f"layers.{i}.mlp.{k}": v for k, v in layer_weights(layer).items()})
    cfg = u.DecoderConfig(hidden_size=HID, num_attention_heads=H, num_hidden_layers=L, intermediate_size=FFN,
                          first_k_dense_replace=1, vocab_size=V,
                          moe=u.MoeConfig(hidden_size=HID, moe_intermediate_size=128, n_routed_experts=E, num_experts_per_tok=6,
                                          n_shared_experts=2, int8_experts=True))
    dec = u.Decoder(cfg, gw, max_seq_len=1024)
    cos_t, sin_t = oracle.rope_tables(head_dim=D, seq_len=1024, theta=10000.0)
    rng = np.random.default_rng(8)
    slot = 1408
    pool = quantized(torch.from_numpy(0.5 * rng.standard_normal((6, 2, L, P, H, D))).float(), slot).to(DEV)
    table = np.array([[3, 0, 5], [1, 4, 5]], np.int32)
    for write in ([39, 199], [40, 200]):
        hidden = rng.standard_normal((2, HID)).astype(np.float32)
        kv = u.PagedKv(kv_blocks=pool, lookup_table=t(table), attend_lengths=_on(write), attend_max=max(write) + 1,
                       write_index=_on(write))
        before = pool.clone()
        apart = before.clone()
        other = u.PagedKv(kv_blocks=apart, lookup_table=kv.lookup_table, attend_lengths=kv.attend_lengths,
                          attend_max=kv.attend_max, write_index=kv.write_index)
        normed = dec.decode(t(hidden), positions=_on(write), kv=kv)
        assert torch.equal(dec.decode(t(hidden), positions=_on(write), kv=other, fuse_norm=False), normed)
        assert torch.equal(apart, pool)
        held = values(pool.cpu(), H).numpy()  # [pages, 2, L, P, H, D]
        pos = np.array(write, np.int32)
        where = [(table[b, r // P], r % P) for b, r in enumerate(write)]
        x, delta = hidden.astype(np.float64), None
        for i in range(L):
            p = f"layers.{i}."
            if delta is not None:
                x = x + delta
            a = _norm64(x, w[p + "input_layernorm.weight"])
            q, k, v = (oracle.dense_f64(a, w[f"{p}self_attn.{c}_proj.weight"]).reshape(2, H, D) for c in "qkv")
            q, k = _rope64(q, pos, cos_t, sin_t), _rope64(k, pos, cos_t, sin_t)
            for side, mine in enumerate((k, v)):
                for b, (page, at) in enumerate(where):
                    half = np.abs(mine[b]).max(axis=-1, keepdims=True) / 254
                    assert bool((np.abs(held[page, side, i, at] - mine[b]) <= half + 1e-4 * np.abs(mine[b]).max()).all())
            out = np.zeros((2, H, D))
            for b, r in enumerate(write):
                rows = held[table[b, :-(-(r + 1) // P)], :, i].swapaxes(0, 1).reshape(2, -1, H, D)[:, :r + 1]
                s = np.einsum("hd,rhd->hr", q[b], rows[0]) / math.sqrt(D)
                e = np.exp(s - s.max(axis=1, keepdims=True))
                out[b] = np.einsum("hr,rhd->hd", e / e.sum(axis=1, keepdims=True), rows[1])
            x = x + oracle.dense_f64(out.reshape(2, HID), w[p + "self_attn.o_proj.weight"])
            a = _norm64(x, w[p + "post_attention_layernorm.weight"])
            if i == 0:
                gate = oracle.dense_f64(a, w[p + "mlp.gate_proj.weight"])
                up = oracle.dense_f64(a, w[p + "mlp.up_proj.weight"])
                delta = oracle.dense_f64(gate / (1 + np.exp(-gate)) * up, w[p + "mlp.down_proj.weight"])
            else:
                delta = oracle.moe_layer_f64(a, moes[i])
        assert _rel(n(normed), _norm64(x + delta, w["norm.weight"])) <= 1e-4
        # nothing but the new rows is written
        same = pool == before
        for page, at in where:
            same[page, :, :, at, :132 * H] = True
        assert bool(same.all())


# ------------------------------------------------------------------------------------------ what the wrappers refuse


def _good():
    u = _uocr()
    x = torch.zeros(4, HEADS, D, device=DEV)
    kv = dict(kv_blocks=u.int8_kv_blocks(3, LAYERS, P, HEADS), lookup_table=_on([[0, 1]]), cache_lengths=_on([5]),
              chunk_offsets=_on([0, 4]), attend_max=9, visible=None)
    return u, x, kv


@pytest.mark.parametrize(("change", "message"), [
    (lambda kv: {"kv_blocks": kv["kv_blocks"][..., :-4]}, "an int8 pool must be a contiguous"),
    (lambda kv: {"kv_blocks": kv["kv_blocks"][:, :1].contiguous()}, "an int8 pool must be a contiguous"),
    (lambda kv: {"kv_blocks": kv["kv_blocks"].cpu()}, "an int8 pool must be a contiguous"),
    (lambda kv: {"kv_blocks": kv["kv_blocks"][..., :256].contiguous()}, "has slots of 256 bytes, too few for 3 heads"),
    (lambda kv: {"kv_blocks": kv["kv_blocks"].view(torch.uint8)}, "kv_blocks must be a contiguous f32"),
    (lambda kv: {"lookup_table": kv["lookup_table"].long()}, "lookup_table"),
    (lambda kv: {"cache_lengths": kv["cache_lengths"].float()}, "cache_lengths"),
    (lambda kv: {"cache_lengths": _on([5, 5])}, "metadata is not for"),
    (lambda kv: {"chunk_offsets": _on([0, 2, 4])}, "metadata is not for"),
    (lambda kv: {"visible": _on([1, 1, 1, 1])}, "visible"),
    (lambda kv: {"visible": _on([1, 1, 1], torch.int64)}, "3 masks for 4 tokens"),
])
def test_wrapper_refusals(change, message) -> None:
    u, x, kv = _good()
    with pytest.raises((TypeError, ValueError), match=message):
        u.paged_chunk_attention(x, x, x, kv=u.PagedChunk(**{**kv, **change(kv)}), layer_idx=0, scale=1.0)


def test_more_wrapper_refusals() -> None:
    u, x, kv = _good()
    chunk = u.PagedChunk(**kv)
    with pytest.raises(ValueError, match="out must be"):
        u.paged_chunk_attention(x, x, x, kv=chunk, layer_idx=0, scale=1.0, out=torch.zeros(3, HEADS, D, device=DEV))
    with pytest.raises(u.UocrError, match="out must not overlap the inputs"):
        u.paged_chunk_attention(x, x.clone(), x.clone(), kv=chunk, layer_idx=0, scale=1.0, out=x)
    with pytest.raises(u.UocrError, match="layer 2 is not in the pool's 2 layers"):
        u.paged_chunk_attention(x, x, x, kv=chunk, layer_idx=2, scale=1.0)
    with pytest.raises(u.UocrError, match="attend_max 257 is not in"):
        u.paged_chunk_attention(x, x, x, kv=u.PagedChunk(**{**kv, "attend_max": 257}), layer_idx=0, scale=1.0)
    with pytest.raises(ValueError, match="q must be an fp32"):
        u.paged_chunk_attention(x.half(), x, x, kv=chunk, layer_idx=0, scale=1.0)
    logits = torch.zeros(4, 9, device=DEV)
    with pytest.raises(ValueError, match="must have 4 rows"):
        u.beam_select(logits, torch.zeros(3, device=DEV), beams=2, eos=0)
    with pytest.raises(u.UocrError, match="eos 9 is not in the vocabulary"):
        u.beam_select(logits, torch.zeros(4, device=DEV), beams=2, eos=9)
    with pytest.raises(TypeError, match="must be torch.float32"):
        u.beam_select(logits.double(), torch.zeros(4, device=DEV), beams=2, eos=0)
    with pytest.raises(ValueError, match="must have one length"):
        u.accept_drafts(chunk, _on([-1, 0, 0, 0]), _on([1, 2, 3]), _on([1, 2, 3, 4]))
    with pytest.raises(ValueError, match="out must have 4 words"):
        u.draft_masks(_on([-1, 0, 0, 0]), _on([0, 4]), out=torch.zeros(3, dtype=torch.int64, device=DEV))


def test_the_librarys_own_workspace(monkeypatch) -> None:
    """Entries that are given no workspace take the library's: the results of calls with one."""
    u = _uocr()
    from uocr_moe import ops

    g = torch.Generator().manual_seed(9)
    calls = []
    for tokens, cached in ((40, 3000), (600, 5000)):
        cols = -(-(tokens + cached) // P)
        pool = quantized(torch.randn(cols, 2, 1, P, HEADS, D, generator=g), 512)
        qkv = torch.randn(tokens, 3, HEADS, D, generator=g).to(DEV)
        for masks in (None, torch.full((tokens,), -1, dtype=torch.int64, device=DEV)):
            calls.append(lambda pool=pool, qkv=qkv, masks=masks, tokens=tokens, cached=cached, cols=cols: u.paged_chunk_attention(
                *qkv.unbind(1), layer_idx=0, scale=SCALE, kv=u.PagedChunk(
                    kv_blocks=pool.to(DEV), lookup_table=_on([list(range(cols))]), cache_lengths=_on([cached]),
                    chunk_offsets=_on([0, tokens]), attend_max=tokens + cached, visible=masks)))
        calls.append(lambda pool=pool, qkv=qkv, cached=cached, cols=cols: u.paged_decode_attention(
            *qkv[:1].unbind(1), layer_idx=0, scale=SCALE, kv=u.PagedKv(
                kv_blocks=pool.to(DEV), lookup_table=_on([list(range(cols))]), attend_lengths=_on([cached]),
                attend_max=cached + 1, write_index=_on([7]))))
    logits = torch.randn(8, 5000, generator=g).to(DEV)
    calls.append(lambda: torch.stack([x.float() for x in u.beam_select(logits, torch.zeros(8, device=DEV), beams=4, eos=0)[:4]]))
    want = [call() for call in calls]
    monkeypatch.setattr(ops, "_workspace", lambda *a: None)
    for _ in range(2):
        assert all(torch.equal(call(), x) for call, x in zip(calls, want))

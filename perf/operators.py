"""Operators of batched serving: the paged key/value cache, the attention that reads it, and the rules on the logits.

A batch holds sequences of different lengths.  Each has `past` positions in the cache and brings `new` tokens, whose
keys and values are quantised into the pages of its table (`store`), attended to together with the past (`attend`) and
read back where a prefix is used again (`load`); the logits of each row then take the row's penalties, biases and
grammar mask (`edit`).

`listed()` names the fixed cases, `draw()` gives others of the same ranges.  With `own` false an operator runs in its
plain form (elementary torch operations in 32 bits), with `own` true through the library's entry points.  `exact()`
restates a case in float64 from the operator's definition.

The cache.  A page holds `page` positions of every KV head.  Per head and per 16 positions it has a block: the 16 keys,
the 16 values, and in the 8-bit formats the 16 + 16 float32 scales of the rows.  A row x of a head is stored as f16, or
as round(x / scale) with scale = clamp(max|x| / top, 2^-40, 2^60), where the 8-bit type is int8 (top 127) or e4m3 (top
448).  Within a block element d of key i lies at ((d // E)·16 + i)·E + d % E, E elements filling 16 bytes; element d of
value i, d = 16M·D + 16m + l with M = 4 (8 bits) or 2 (f16), at (((D·4 + i // 4)·16 + l)·M + m)·4 + i % 4.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

F64 = torch.float64
GROUP = 16                    # positions of a block
TOP = dict(i8=127.0, f8=448.0)
SMALLEST, LARGEST = 2.0 ** -40, 2.0 ** 60
NO_MASK = 0xFFFFFFFF
IN_FLIGHT = 3                 # recordings that a serving loop has queued at most


# --- the cases ----------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # One token's keys and values of each of eight sequences: what every decode step stores in every layer.
        dict(name="store_tokens", kind="store", fmt="i8", kv=8, hd=64, page=16, decodes=8, chunks=0, chunk=0, past=2000),
        # Four long prompts of a prefill step.
        dict(name="store_chunks", kind="store", fmt="f8", kv=8, hd=128, page=64, decodes=0, chunks=4, chunk=2048,
             past=5000),
        # A short system prompt read back for a request that continues it.
        dict(name="load_short", kind="load", fmt="f16", kv=2, hd=256, page=32, decodes=1, chunks=0, chunk=0, past=77),
        # The prefix of a 30,000-token document.
        dict(name="load_prefix", kind="load", fmt="i8", kv=8, hd=64, page=64, decodes=1, chunks=0, chunk=0, past=30001),
        # A single user's next token: nothing but latency.
        dict(name="attend_token", kind="attend", fmt="i8", heads=32, kv=8, hd=64, page=16, decodes=1, chunks=0, chunk=0,
             past=600),
        # The next tokens of 64 users with ragged contexts.
        dict(name="attend_tokens", kind="attend", fmt="i8", heads=32, kv=8, hd=64, page=64, decodes=64, chunks=0,
             chunk=0, past=16384),
        # The same of the small model, whose key heads serve two query heads, with an unquantised cache.
        dict(name="attend_tokens_f16", kind="attend", fmt="f16", heads=16, kv=8, hd=64, page=32, decodes=16, chunks=0,
             chunk=0, past=32768),
        # Five drafted tokens each to verify, heads of 256.
        dict(name="attend_drafts", kind="attend", fmt="f8", heads=8, kv=2, hd=256, page=16, decodes=0, chunks=12,
             chunk=5, past=4096),
        # A prefill batch deep in a long prompt, unquantised.
        dict(name="attend_chunk", kind="attend", fmt="f16", heads=32, kv=8, hd=64, page=64, decodes=0, chunks=1,
             chunk=512, past=7680),
        # A step that serves decoding users and two users' prompts at once.
        dict(name="attend_mixed", kind="attend", fmt="i8", heads=32, kv=8, hd=128, page=16, decodes=8, chunks=2,
             chunk=1024, past=16384),
        # One user's logits: penalties over a short answer and a grammar's mask.
        dict(name="edit_row", kind="edit", rows=1, vocab=65536, history=600, bias=8),
        # The logits of a large batch with long histories.
        dict(name="edit_rows", kind="edit", rows=96, vocab=151936, history=4096, bias=300),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    kind = rng.choice(["store", "load", "attend", "attend", "attend", "edit"])
    if kind == "edit":
        rows = _log_int(rng, 1, 96)
        return dict(kind=kind, rows=rows, vocab=_log_int(rng, 1000, 151936), history=_log_int(rng, 1, 8192),
                    bias=rng.choice([0, 1, _log_int(rng, 2, 600)]))
    hd, kv = rng.choice([64, 64, 128, 256]), rng.choice([1, 2, 4, 8])
    case = dict(kind=kind, fmt=rng.choice(["f16", "i8", "f8"]), kv=kv, hd=hd, page=rng.choice([16, 16, 32, 48, 64, 128]))
    if kind == "load":
        return dict(case, decodes=1, chunks=0, chunk=0, past=_log_int(rng, 1, min(32768, 2 ** 24 // (kv * hd))))
    if kind == "store":
        n = _log_int(rng, 1, 8)
        return dict(case, decodes=rng.randint(0, 16), chunks=n, chunk=_log_int(rng, 1, 8192 // n), past=_log_int(rng, 1, 8192))
    case["heads"] = kv * rng.choice([1, 2, 3, 4, 6, 8])
    past = _log_int(rng, 1, 32768)
    decodes = _log_int(rng, 1, max(1, min(64, 400_000_000 // (past * _position_bytes(case)))))
    style = rng.choice(["tokens", "chunk", "drafts", "mixed"])
    wide = max(1, case["heads"] * hd // 1024)  # the products grow with it
    if style == "tokens":
        return dict(case, decodes=decodes, chunks=0, chunk=0, past=past)
    if style == "drafts":
        return dict(case, decodes=0, chunks=max(1, decodes // 2), chunk=rng.randint(2, 17), past=past)
    chunk = _log_int(rng, 17, max(18, min(2048, 16_000_000 // (past + 2048) // wide)))
    return dict(case, decodes=0 if style == "chunk" else min(8, decodes), chunks=1 if style == "chunk" else 2,
                chunk=chunk, past=past)


def _position_bytes(case: dict) -> int:
    return case["kv"] * 2 * (2 * case["hd"] if case["fmt"] == "f16" else case["hd"] + 4)


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """The past positions and the new tokens of the batch's sequences, decoding and prompt ones shuffled."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    seqs = []
    for i in range(case["decodes"]):
        seqs.append((case["past"] if i == 0 else _log_int(rng, max(1, case["past"] // 8), case["past"]), 1))
    for i in range(case["chunks"]):
        seqs.append((case["past"] if i == 0 else rng.randint(0, case["past"]),
                     case["chunk"] if i == 0 else rng.randint((case["chunk"] + 1) // 2, case["chunk"])))
    if case["kind"] == "load":
        seqs = [(p, 0) for p, _ in seqs]
    rng.shuffle(seqs)
    return [p for p, _ in seqs], [n for _, n in seqs]


def _edit_lengths(case: dict) -> tuple[list[int], list[int]]:
    """Tokens of history and biases of each row."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    history = [case["history"]] + [rng.randint(0, case["history"]) for _ in range(case["rows"] - 1)]
    return history, [case["bias"]] + [rng.choice([0, rng.randint(0, case["bias"])]) for _ in range(case["rows"] - 1)]


def work(case: dict) -> dict:
    if case["kind"] == "edit":
        history, bias = _edit_lengths(case)
        masked = sum(r % 4 != 3 for r in range(case["rows"]))
        return dict(bytes=8 * case["rows"] * case["vocab"] + masked * case["vocab"] // 8 + 4 * sum(history) + 8 * sum(bias),
                    flops=2 * case["rows"] * case["vocab"])
    past, new = _lengths(case)
    kv, hd = case["kv"], case["hd"]
    position = _position_bytes(case)
    if case["kind"] == "attend":
        seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
        return dict(bytes=position * (sum(past) + sum(new)) + 8 * sum(new) * case["heads"] * hd,
                    flops=4 * seen * case["heads"] * hd)
    moved = sum(new) if case["kind"] == "store" else sum(past)
    return dict(bytes=moved * (position + 8 * kv * hd), flops=moved * kv * hd * 4)


# --- inputs -----------------------------------------------------------------------

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(gen, positions: int, kv: int, hd: int) -> torch.Tensor:
    """Rows of keys or values: normal, of a magnitude of its own per position and head."""
    size = torch.exp(0.4 * torch.randn(positions, kv, 1, generator=gen, device="cuda"))
    return torch.randn(positions, kv, hd, generator=gen, device="cuda").mul_(size)


def _quantise(x: torch.Tensor, fmt: str):
    """(values in the cache's type, scales or None) of rows x [..., hd]."""
    if fmt == "f16":
        return x.half(), None
    scale = (x.abs().amax(-1) / TOP[fmt]).clamp(SMALLEST, LARGEST)
    y = (x / scale[..., None]).clamp(-TOP[fmt], TOP[fmt])
    return (torch.round(y).to(torch.int8) if fmt == "i8" else y.to(torch.float8_e4m3fn)), scale


def _block_bytes(case: dict) -> int:
    return 2 * GROUP * case["hd"] * (2 if case["fmt"] == "f16" else 1) + (0 if case["fmt"] == "f16" else 8 * GROUP)


def _parts(pool: torch.Tensor, case: dict):
    """The keys [.., hd/E, 16, E], the values [.., D, 4, 16, M, 4] and the scales [.., 2, 16] (or None) of the blocks'
    bytes [.., block]; the elements as int8 or int16."""
    half = case["fmt"] == "f16"
    size, kind, per = (2, torch.int16, 8) if half else (1, torch.int8, 16)
    n, m = GROUP * case["hd"] * size, per // 4
    k = pool[..., :n].view(kind).unflatten(-1, (case["hd"] // per, GROUP, per))
    v = pool[..., n:2 * n].view(kind).unflatten(-1, (case["hd"] // (16 * m), 4, 16, m, 4))
    return k, v, None if half else pool[..., 2 * n:].view(torch.float32).unflatten(-1, (2, GROUP))


def _elements(bits: torch.Tensor, fmt: str) -> torch.Tensor:
    return bits.view(torch.float16) if fmt == "f16" else bits.view(torch.float8_e4m3fn) if fmt == "f8" else bits


def _pack(k, v, case: dict) -> torch.Tensor:
    """The blocks [groups, kv, bytes] of quantised rows, each (values [16·groups, kv, hd], scales)."""
    blocks = torch.zeros(k[0].shape[0] // GROUP, case["kv"], _block_bytes(case), dtype=torch.uint8, device="cuda")
    kp, vp, scales = _parts(blocks, case)
    per = kp.shape[-1]
    bits = kp.dtype
    kp.copy_(k[0].view(bits).reshape(-1, GROUP, case["kv"], case["hd"] // per, per).permute(0, 2, 3, 1, 4))
    vp.copy_(v[0].view(bits).reshape(-1, 4, 4, case["kv"], case["hd"] // (4 * per), per // 4, 16).permute(0, 3, 4, 1, 6, 5, 2))
    if scales is not None:
        scales.copy_(torch.stack([k[1], v[1]]).reshape(2, -1, GROUP, case["kv"]).permute(1, 3, 0, 2))
    return blocks


class State:
    """What a program keeps between calls."""


def _pages(case: dict, lengths: list[int], seed: int):
    """Each sequence's pages out of a pool that other sequences use too: (lists, pages of the pool)."""
    need = [-(-n // case["page"]) for n in lengths]
    total = sum(need) + 1 + sum(need) // 8
    order = np.random.default_rng(seed).permutation(total)[:sum(need)]
    return [a.tolist() for a in np.split(order, np.cumsum(need)[:-1])], total


def _dense(case: dict, seed: int):
    """The cache inputs of a case: quantised keys and values of all positions (each sequence padded to whole blocks),
    where each sequence's rows begin among them, and the new tokens' rows and queries."""
    past, new = _lengths(case)
    gen = _generator(seed)
    groups = [-(-(p + n) // GROUP) for p, n in zip(past, new)]
    begins = (GROUP * np.cumsum([0] + groups)).tolist()
    s = State()
    s.past, s.new, s.begins = past, new, begins
    tokens = sum(new)
    s.k_new = _rows(gen, tokens, case["kv"], case["hd"])
    s.v_new = _rows(gen, tokens, case["kv"], case["hd"])
    if case["kind"] == "attend":
        s.q = 1.5 * torch.randn(tokens, case["heads"], case["hd"], generator=gen, device="cuda")
    if case["kind"] != "store":
        s.k = _quantise(_rows(gen, begins[-1], case["kv"], case["hd"]), case["fmt"])
        s.v = _quantise(_rows(gen, begins[-1], case["kv"], case["hd"]), case["fmt"])
    return s


def _fill(case: dict, seed: int, blocks: int) -> torch.Tensor:
    """Bytes of blocks that belong to other sequences: finite in every format."""
    raw = torch.randint(0, 0x40, (blocks, case["kv"], _block_bytes(case)), generator=_generator(seed + 1), device="cuda")
    return raw.to(torch.uint8)


def _mask_rows(gen, rows: int, vocab: int) -> torch.Tensor:
    """Allowed tokens: nearly all, one in a hundred, or (one row in sixteen) none; every fourth row has no mask."""
    share = torch.tensor([0.98, 0.01, 0.5, 0.0], device="cuda").repeat((rows + 3) // 4)[:rows]
    share[5::16] = 0.0
    return torch.rand(rows, vocab, generator=gen, device="cuda") < share[:, None]


def _edit_inputs(case: dict, seed: int):
    gen, s = _generator(seed), State()
    rows, vocab = case["rows"], case["vocab"]
    s.history_len, s.bias_len = _edit_lengths(case)
    s.logits = 3 * torch.randn(rows, vocab, generator=gen, device="cuda")
    rand = lambda n: torch.rand(n, generator=gen, device="cuda")  # noqa: E731
    s.history = (vocab * rand(sum(s.history_len)) ** 4).long().clamp_(max=vocab - 1)
    s.bias_tokens = (vocab * rand(sum(s.bias_len))).long().clamp_(max=vocab - 1)
    s.bias = 8 * rand(sum(s.bias_len)) - 4
    s.repeat, s.presence, s.frequency = 1 + 0.3 * rand(rows), 0.5 * rand(rows), 0.2 * rand(rows)
    s.allowed = _mask_rows(gen, rows, vocab)
    return s


# --- the state -----------------------------------------------------------------------

_HIP = None


def _hip():
    """The process's one device context, as a program opens it."""
    global _HIP
    if _HIP is None:
        from bobcat_amd.backend import Hip
        _HIP = Hip()
    return _HIP


class _Memory:
    """A device buffer's memory for torch (the array interface), which keeps the buffer."""

    def __init__(self, buffer, nbytes: int):
        self.buffer = buffer
        self.__cuda_array_interface__ = dict(shape=(nbytes,), typestr="|u1", strides=None, version=3,
                                             data=(buffer.device_ptr, False))


def _place(t: torch.Tensor):
    """A tensor in a buffer of the library's context: (the view, the tensor over the buffer's memory)."""
    hip = _hip()
    buffer = hip.new_buffer(max(16, t.numel() * t.element_size()))
    hip._buffers.remove(buffer)  # freed with its last view, not with the context
    there = torch.as_tensor(_Memory(buffer, t.numel() * t.element_size()), device="cuda").view(t.dtype).view(t.shape)
    there.copy_(t)
    return buffer.at(0), there


def prepare(case: dict, seed: int) -> State:
    if case["kind"] == "edit":
        s = _prepare_edit(case, seed)
    else:
        s = _prepare_cache(case, seed)
    s.case = case
    torch.cuda.synchronize()
    return s


def _prepare_cache(case: dict, seed: int) -> State:
    d, s = _dense(case, seed), State()
    per_page = case["page"] // GROUP
    lengths = [p + n for p, n in zip(d.past, d.new)]
    pages, total = _pages(case, lengths, seed)
    s.pool = _fill(case, seed, total * per_page)
    if case["kind"] != "store":
        # Block g of a sequence is block g % per_page of its page g // per_page.
        where = [np.asarray(pg, np.int64)[g // per_page] * per_page + g % per_page
                 for pg, n in zip(pages, lengths) for g in [np.arange(-(-n // GROUP))]]
        s.pool[torch.from_numpy(np.concatenate(where)).cuda()] = _pack(d.k, d.v, case)
    s.pool = s.pool.view(total, per_page, case["kv"], -1).transpose(1, 2).contiguous()  # [page, head, block of 16, bytes]
    widest = max(len(pg) for pg in pages)
    s.table = torch.tensor([pg + [0] * (widest - len(pg)) for pg in pages], device="cuda")
    s.past, s.new = (torch.tensor(x, device="cuda") for x in (d.past, d.new))
    s.rows = torch.repeat_interleave(torch.arange(len(d.new), device="cuda"), s.new)  # the sequence of each new token
    s.step = torch.arange(sum(d.new), device="cuda") - (torch.cumsum(s.new, 0) - s.new)[s.rows]
    s.most_new, s.longest = max(d.new), max(lengths)
    s.k, s.v = d.k_new, d.v_new
    s.q = getattr(d, "q", None)
    if own:
        hip = _hip()
        s.plan = hip.kv_plan(case["fmt"], case["kv"], case["hd"], case["page"], total, case.get("heads", case["kv"]))
        s.plan.set(d.past, d.new, pages)
        s.at_pool, s.pool = _place(s.pool)
        if case["kind"] == "store":
            s.at_k, s.k = _place(s.k)
            s.at_v, s.v = _place(s.v)
        elif case["kind"] == "load":
            s.at_k, s.k_out = _place(torch.zeros(d.past[0], case["kv"], case["hd"], device="cuda"))
            s.at_v, s.v_out = _place(torch.zeros(d.past[0], case["kv"], case["hd"], device="cuda"))
        else:
            s.at_q, s.q = _place(s.q)
            s.at_out, s.out = _place(torch.zeros_like(s.q))
    return s


def _prepare_edit(case: dict, seed: int) -> State:
    d, s = _edit_inputs(case, seed), State()
    rows, vocab = case["rows"], case["vocab"]
    words = -(-vocab // 32)
    bits = torch.zeros(rows, 32 * words, dtype=torch.int32, device="cuda")
    bits[:, :vocab] = d.allowed
    s.masks = (bits.view(rows, words, 32) << torch.arange(32, device="cuda", dtype=torch.int32)).sum(-1).to(torch.int32)
    s.mask_of = torch.arange(rows, device="cuda")
    s.mask_of[3::4] = NO_MASK
    s.logits, s.history, s.bias_tokens, s.bias = d.logits, d.history, d.bias_tokens, d.bias
    s.repeat, s.presence, s.frequency = d.repeat, d.presence, d.frequency
    s.history_row = torch.repeat_interleave(torch.arange(rows), torch.tensor(d.history_len)).cuda()
    s.bias_row = torch.repeat_interleave(torch.arange(rows), torch.tensor(d.bias_len)).cuda()
    if own:
        from bobcat_amd.backend import LOGIT_ROW
        table = np.zeros(rows, LOGIT_ROW)
        table["history_at"], table["history_len"] = np.cumsum([0] + d.history_len[:-1]), d.history_len
        table["bias_at"], table["bias_len"] = np.cumsum([0] + d.bias_len[:-1]), d.bias_len
        table["mask"] = s.mask_of.cpu().numpy()
        for name in ("repeat", "presence", "frequency"):
            table[name] = getattr(d, name).cpu().numpy()
        s.at_table, s.row_table = _place(torch.from_numpy(table.view(np.uint8)).cuda())
        s.at_logits, s.logits = _place(s.logits)
        s.at_out, s.out = _place(torch.zeros_like(s.logits))
        s.at_masks, s.masks = _place(s.masks)
        s.at_history, s.history = _place(s.history.int())
        s.at_bias_tokens, s.bias_tokens = _place(s.bias_tokens.int())
        s.at_bias, s.bias = _place(s.bias)
    return s


# --- one pass -----------------------------------------------------------------------

def run(state: State):
    kind = state.case["kind"]
    if own:
        hip = _hip()
        hip.begin()
        out = _OWN[kind](hip, state, state.case)
        ticket = hip.commit()
        if ticket > IN_FLIGHT:
            hip.wait(ticket - IN_FLIGHT)  # a serving loop keeps a few steps queued
        return out
    return _PLAIN[kind](state, state.case)


def _own_store(hip, s, c):
    width = c["kv"] * c["hd"]
    hip.kv_store(s.plan, s.at_pool, s.at_k, width, s.at_v, width)
    return _stored(s.pool, c)


def _own_load(hip, s, c):
    hip.kv_load(s.plan, s.at_pool, 0, 0, s.k_out.shape[0], s.at_k, s.at_v)
    return [s.k_out, s.v_out]


def _own_attend(hip, s, c):
    hip.attention_paged(s.plan, s.at_pool, s.at_q, c["heads"] * c["hd"], s.at_out, c["heads"] * c["hd"])
    return s.out


def _own_edit(hip, s, c):
    hip.logits_edit(s.at_logits, s.at_out, c["rows"], c["vocab"], s.at_table, history=s.at_history,
                    n_history=s.history.numel(), bias_tokens=s.at_bias_tokens, bias_values=s.at_bias,
                    n_bias=s.bias.numel(), masks=s.at_masks, n_masks=c["rows"])
    return s.out


def _stored(pool, c):
    """The cache as the values that it holds, with the rows' scales."""
    k, v, scales = _parts(pool, c)
    return [_elements(k, c["fmt"]), _elements(v, c["fmt"])] + ([] if scales is None else [scales])


def _plain_store(s, c):
    k, v, scales = _parts(s.pool, c)
    position = s.past[s.rows] + s.step
    page = s.table[s.rows, position // c["page"]]
    block, i = position % c["page"] // GROUP, position % GROUP
    per, tokens = k.shape[-1], s.k.shape[0]
    (kq, ks), (vq, vs) = _quantise(s.k, c["fmt"]), _quantise(s.v, c["fmt"])
    k[page, :, block, :, i, :] = kq.view(k.dtype).view(tokens, c["kv"], -1, per)
    v[page, :, block, :, i // 4, :, :, i % 4] = vq.view(v.dtype).view(tokens, c["kv"], -1, per // 4, 16).transpose(-1, -2)
    if scales is not None:
        scales[page, :, block, 0, i] = ks
        scales[page, :, block, 1, i] = vs
    return _stored(s.pool, c)


def _gathered(s, c):
    """The keys and values [sequence, kv, positions, hd] of the tables' pages, in float32."""
    blocks = s.pool[s.table].permute(0, 2, 1, 3, 4)  # [sequence, kv, page, block, bytes]
    k, v, scales = _parts(blocks, c)
    k, v = _elements(k, c["fmt"]).float(), _elements(v, c["fmt"]).float()
    k = k.transpose(-3, -2).reshape(*k.shape[:4], GROUP, c["hd"])                 # E pieces of a key side by side
    v = v.permute(0, 1, 2, 3, 5, 8, 4, 7, 6).reshape(*v.shape[:4], GROUP, c["hd"])  # key (4 + 4), then D, m, l
    if scales is not None:
        k, v = k * scales[..., 0, :, None], v * scales[..., 1, :, None]
    return k.flatten(2, 4), v.flatten(2, 4)


def _plain_load(s, c):
    k, v = _gathered(s, c)
    n = s.longest
    return [k[0, :, :n].transpose(0, 1).contiguous(), v[0, :, :n].transpose(0, 1).contiguous()]


def _plain_attend(s, c):
    k, v = _gathered(s, c)
    n, group, longest = s.past.numel(), c["heads"] // c["kv"], s.longest
    k, v = k[:, :, :longest], v[:, :, :longest]
    key = torch.arange(longest, device="cuda")
    # Positions past a sequence's end hold other sequences' bytes: no part of its sums.
    v = torch.where(key[:, None] < (s.past + s.new)[:, None, None, None], v, 0.0)
    q = torch.zeros(n, s.most_new, c["kv"], group, c["hd"], device="cuda")
    q[s.rows, s.step] = s.q.view(-1, c["kv"], group, c["hd"]) / math.sqrt(c["hd"])
    q = q.permute(0, 2, 1, 3, 4).reshape(n, c["kv"], s.most_new * group, c["hd"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(n, c["kv"], s.most_new, group, longest)
    last = s.past[:, None] + torch.arange(s.most_new, device="cuda")
    scores.masked_fill_((key > last[:, :, None])[:, None, :, None, :], -math.inf)
    scores = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(n, c["kv"], -1, longest), v).view(n, c["kv"], s.most_new, group, c["hd"]) / total
    return out.permute(0, 2, 1, 3, 4)[s.rows, s.step].reshape(-1, c["heads"], c["hd"])


def _plain_edit(s, c):
    rows, vocab = c["rows"], c["vocab"]
    count = torch.bincount(s.history_row * vocab + s.history, minlength=rows * vocab).view(rows, vocab).float()
    x = s.logits
    y = torch.where(x > 0, x / s.repeat[:, None], x * s.repeat[:, None]) - (s.presence[:, None] + s.frequency[:, None] * count)
    y = torch.where(count > 0, y, x)
    y = y.index_put((s.bias_row, s.bias_tokens), s.bias, accumulate=True)
    token = torch.arange(vocab, device="cuda")
    allowed = (s.masks[:, token // 32] >> (token % 32).int() & 1).bool() | (s.mask_of == NO_MASK)[:, None]
    return torch.where(allowed, y, -math.inf)


_OWN = dict(store=_own_store, load=_own_load, attend=_own_attend, edit=_own_edit)
_PLAIN = dict(store=_plain_store, load=_plain_load, attend=_plain_attend, edit=_plain_edit)


# --- the definitions in float64 ---------------------------------------------------------

def exact(case: dict, seed: int):
    if case["kind"] == "edit":
        return _exact_edit(case, seed)
    d = _dense(case, seed)
    if case["kind"] == "load":
        n = d.past[0]
        return [_value(d.k)[:n], _value(d.v)[:n]]
    return _exact_store(case, seed, d) if case["kind"] == "store" else _exact_attend(case, d)


def _value(quantised) -> torch.Tensor:
    values, scale = quantised
    return values.to(F64) if scale is None else values.to(F64) * scale.to(F64)[..., None]


def _exact_store(case, seed, d):
    """Every new element put at its offset among the bytes that were there, as the values that the bytes stand for."""
    per_page, hd, kv, fmt = case["page"] // GROUP, case["hd"], case["kv"], case["fmt"]
    pages, total = _pages(case, [p + n for p, n in zip(d.past, d.new)], seed)
    before = _fill(case, seed, total * per_page).view(total, per_page, kv, -1).transpose(1, 2).reshape(-1, _block_bytes(case))
    size = 2 if fmt == "f16" else 1
    per, m = 16 // size, 4 // size
    kind = dict(f16=torch.float16, i8=torch.int8, f8=torch.float8_e4m3fn)[fmt]
    elements = before[:, :2 * GROUP * hd * size].contiguous().view(kind).to(F64)
    scales = None if fmt == "f16" else before[:, 2 * GROUP * hd:].contiguous().view(torch.float32).to(F64)
    block, slot = [], []
    for p, n, table in zip(d.past, d.new, pages):
        for at in range(p, p + n):
            block.append(table[at // case["page"]] * kv * per_page + at % case["page"] // GROUP)
            slot.append(at % GROUP)
    block = torch.tensor(block, device="cuda")[:, None] + torch.arange(kv, device="cuda") * per_page  # [token, head]
    i = torch.tensor(slot, device="cuda")[:, None, None]
    e = torch.arange(hd, device="cuda")
    offsets = ((e // per * GROUP + i) * per + e % per,
               GROUP * hd + (((e // (16 * m) * 4 + i // 4) * 16 + e % 16) * m + e // 16 % m) * 4 + i % 4)
    for part, (x, offset) in enumerate(zip((d.k_new, d.v_new), offsets)):
        x = x.to(F64)
        if fmt == "f16":
            y = x.half().to(F64)
        else:
            # (The scale is a float32 of the cache: the quotient is taken with it.)
            scale = (x.abs().amax(-1) / TOP[fmt]).clamp(SMALLEST, LARGEST).float()
            scales[block, GROUP * part + i[:, :, 0]] = scale.to(F64)
            y = (x / scale.to(F64)[..., None]).clamp(-TOP[fmt], TOP[fmt])
            y = y.round() if fmt == "i8" else y.float().to(torch.float8_e4m3fn).to(F64)
        elements[block[:, :, None], offset.expand(-1, kv, -1)] = y
    lead = (total, kv, per_page)
    out = [elements[:, :GROUP * hd].reshape(*lead, hd // per, GROUP, per),
           elements[:, GROUP * hd:].reshape(*lead, hd // (16 * m), 4, 16, m, 4)]
    if fmt == "i8":
        out = [x.to(torch.int8) for x in out]
    return out if scales is None else out + [scales.view(*lead, 2, GROUP)]


def _exact_attend(case, d):
    kv, group = case["kv"], case["heads"] // case["kv"]
    if sum(n * (p + n) for p, n in zip(d.past, d.new)) * case["heads"] * case["hd"] > 4e12:
        return None
    out, row = torch.empty(sum(d.new), case["heads"], case["hd"], dtype=F64, device="cuda"), 0
    for p, n, at in zip(d.past, d.new, d.begins):
        k = _value((d.k[0][at:at + p + n], None if d.k[1] is None else d.k[1][at:at + p + n]))
        v = _value((d.v[0][at:at + p + n], None if d.v[1] is None else d.v[1][at:at + p + n]))
        seen = torch.arange(p + n, device="cuda")[None] <= p + torch.arange(n, device="cuda")[:, None]
        for h in range(case["heads"]):
            a = d.q[row:row + n, h].to(F64) @ k[:, h // group].T.contiguous() / math.sqrt(case["hd"])
            out[row:row + n, h] = torch.softmax(a.masked_fill(~seen, -math.inf), 1) @ v[:, h // group].contiguous()
        row += n
    return out


def _exact_edit(case, seed):
    d = _edit_inputs(case, seed)
    x, hat, bat = d.logits.to(F64), 0, 0
    for r in range(case["rows"]):
        tokens, count = torch.unique(d.history[hat:hat + d.history_len[r]], return_counts=True)
        hat += d.history_len[r]
        rho, alpha, beta = (float(t[r]) for t in (d.repeat, d.presence, d.frequency))
        y = x[r, tokens]
        x[r, tokens] = torch.where(y > 0, y / rho, y * rho) - alpha - beta * count
        for token, value in zip(d.bias_tokens[bat:bat + d.bias_len[r]].tolist(), d.bias[bat:bat + d.bias_len[r]].tolist()):
            x[r, token] += value
        bat += d.bias_len[r]
        if r % 4 != 3:
            x[r, ~d.allowed[r]] = -math.inf
    return x

"""Operators of a serving step with drafted tokens: rotary positions of a ragged batch, attention for trees of drafts over
the paged cache, the verdict on the drafts, and the cache's rows of those that stay.

A batch holds sequences with `past` positions in the cache and `new` tokens each.  The new tokens of a sequence are a
tree: token i follows token parents[i], or the past where it has none; its position is past + its depth.  Its row in the
cache is at past + i until the kept ones are moved together.

  rope    turns the pairs of each head of the queries and keys by angle = position · frequency, after an RMS norm of the head
  attend  softmax(q·k/√hd)·v over the past, the token's ancestors and itself
  verify  walks down each tree: with p the target's probabilities at the current token (softmax of logits / temperature) and
          q what its children were drawn from, child x is kept where u·q(x) < p(x), else p becomes the normalised positive
          part of p − q and the next child is looked at; where no child stays the next token is drawn from what p has become
  keep    moves the kept tokens' rows of every layer's cache to the positions behind the past

`listed()` names the fixed cases, `draw()` gives others of the same ranges.  With `own` false an operator runs in its plain
form (elementary torch operations), with `own` true through the library's entry points.  `exact()` restates a case in
float64 from the operator's definition.

The cache.  A page holds `page` positions of every KV head.  Per head and per 16 positions it has a block: the 16 keys,
the 16 values and, in the 8-bit formats, the 16 + 16 float32 scales of the rows.  Within a block element d of key i lies at
((d // E)·16 + i)·E + d % E, E elements filling 16 bytes; element d of value i, d = 16M·D + 16m + l with M = 4 (8 bits) or
2 (f16), at (((D·4 + i // 4)·16 + l)·M + m)·4 + i % 4.
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
NOTHING = 0xFFFFFFFF          # no token
IN_FLIGHT = 3                 # recordings that a serving loop has queued at most


# --- the cases ----------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # The next token of one user, normalised heads: what a decode step runs in every layer.
        dict(name="rope_token", kind="rope", heads=32, kv=8, hd=64, rot=64, layout="halves", scaling="none", factor=1.0,
             theta=1e6, norm=True, seqs=1, new=1, width=1, past=600),
        # Trees of drafts of 24 users, a quarter of each head turned, queries beside their gates.
        dict(name="rope_trees", kind="rope", heads=8, kv=2, hd=256, rot=64, layout="halves", scaling="none", factor=1.0,
             theta=1e7, norm=True, seqs=24, new=24, width=4, past=30000),
        # Prompts deep in contexts eight times as long as those of training, interleaved pairs.
        dict(name="rope_prompts", kind="rope", heads=32, kv=8, hd=128, rot=128, layout="pairs", scaling="parts", factor=8.0,
             theta=5e5, norm=False, seqs=4, new=2048, width=1, past=120000),
        # One user's eight drafts.
        dict(name="attend_tree", kind="attend", fmt="i8", heads=32, kv=8, hd=64, page=16, seqs=1, new=8, width=3, past=600),
        # Trees of 32 users with ragged contexts.
        dict(name="attend_trees", kind="attend", fmt="i8", heads=32, kv=8, hd=64, page=64, seqs=32, new=24, width=4, past=8192),
        # Large trees over unquantised caches of wider heads.
        dict(name="attend_wide", kind="attend", fmt="f16", heads=32, kv=8, hd=128, page=32, seqs=8, new=64, width=6, past=12000),
        # Few heads of 256.
        dict(name="attend_f8", kind="attend", fmt="f8", heads=8, kv=2, hd=256, page=16, seqs=12, new=12, width=3, past=4096),
        # A chain of four drafts of one user.
        dict(name="verify_chain", kind="verify", vocab=65536, seqs=1, new=5, width=1, draft="drawn"),
        # Chains of 48 users with a large vocabulary.
        dict(name="verify_chains", kind="verify", vocab=151936, seqs=48, new=6, width=1, draft="drawn"),
        # Trees of the likeliest tokens of 16 users.
        dict(name="verify_trees", kind="verify", vocab=65536, seqs=16, new=32, width=4, draft="chosen"),
        # What one user keeps of eight drafts, in all attention layers.
        dict(name="keep_path", kind="keep", fmt="f16", kv=8, hd=64, page=16, seqs=1, new=9, width=3, past=200, layers=8),
        # What 64 users keep.
        dict(name="keep_paths", kind="keep", fmt="i8", kv=8, hd=64, page=64, seqs=64, new=24, width=4, past=300, layers=8),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng) -> dict:
    kind = rng.choice(["rope", "attend", "attend", "verify", "keep"])
    if kind == "verify":
        seqs, width = _log_int(rng, 1, 48), rng.choice([1, 1, 2, 3, 5])
        new = rng.randint(2, 9) if width == 1 else _log_int(rng, 4, 64)
        vocab = _log_int(rng, 1000, max(1001, min(151936, 40_000_000 // (seqs * new))))
        return dict(kind=kind, vocab=vocab, seqs=seqs, new=new, width=width,
                    draft=rng.choice(["drawn", "chosen"] if width == 1 else ["drawn", "distinct", "chosen", "chosen"]))
    hd, kv = rng.choice([64, 64, 128, 256]), rng.choice([1, 2, 4, 8])
    width = rng.choice([1, 2, 3, 4, 6])
    if kind == "rope":
        scaling = rng.choice(["none", "none", "linear", "parts"])
        seqs, group = _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8])
        most = 35_000_000 // (kv * (group + 1) * hd * seqs)  # tokens of a sequence
        return dict(kind=kind, heads=kv * group, kv=kv, hd=hd,
                    rot=rng.choice([hd, hd, hd // 2, hd // 4, 2 * rng.randint(1, hd // 2)]),
                    layout=rng.choice(["halves", "pairs"]), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
                    theta=rng.choice([1e4, 5e5, 1e6, 1e7]), norm=rng.random() < 0.5, seqs=seqs,
                    new=_log_int(rng, 1, min(most, 2048 if width == 1 else 64)), width=width, past=_log_int(rng, 1, 120000))
    case = dict(kind=kind, fmt=rng.choice(["f16", "i8", "f8"]), kv=kv, hd=hd, page=rng.choice([16, 16, 32, 48, 64, 128]))
    if kind == "keep":
        return dict(case, seqs=_log_int(rng, 1, 64), new=_log_int(rng, 3, 48), width=rng.randint(2, 6), past=_log_int(rng, 1, 300),
                    layers=rng.randint(1, 8))
    past = _log_int(rng, 1, 16384)
    heads, new = kv * rng.choice([1, 2, 3, 4, 6, 8]), _log_int(rng, 2, 64)
    most = min(32, 200_000_000 // (past * _position_bytes(case)), 30_000_000_000 // (2 * heads * hd * new * past))
    return dict(case, heads=heads, seqs=_log_int(rng, 1, max(1, most)), new=new, width=width, past=past)


def _position_bytes(case: dict) -> int:
    return case["kv"] * 2 * (2 * case["hd"] if case["fmt"] == "f16" else case["hd"] + 4)


def _rng(case: dict) -> random.Random:
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _trees(case: dict):
    """(past positions, each sequence's tokens' parents, -1 for none): the first sequence as the case says, others up to it."""
    rng, past, trees = _rng(case), [], []
    for i in range(case["seqs"]):
        most = case.get("past", 0)
        past.append(most if i == 0 else rng.randint(most // 8, most))
        n = case["new"] if i == 0 else rng.randint((case["new"] + 1) // 2, case["new"])
        parents, depth, children = [-1], [0], [0]
        for j in range(1, n):
            open_ = [a for a in range(j) if children[a] < case["width"] and (case["width"] == 1 or depth[a] < 7)]
            at = open_[min(rng.randrange(len(open_)), rng.randrange(len(open_)))]  # earlier tokens have more children
            children[at] += 1
            parents.append(at)
            depth.append(depth[at] + 1)
            children.append(0)
        trees.append(parents)
    return past, trees


def _depths(parents: list[int]) -> list[int]:
    depth = []
    for a in parents:
        depth.append(depth[a] + 1 if a >= 0 else 0)
    return depth


def _path(parents: list[int], at: int) -> list[int]:
    path = [at]
    while parents[path[0]] >= 0:
        path.insert(0, parents[path[0]])
    return path


def _kept(case: dict, seed: int) -> list[list[int]]:
    """A path of each sequence's tree from its root down that the step keeps.  (Of those whose rows lie behind all places
    that the path moves to, or in place, so that a second pass over the same cache moves the same bytes.)"""
    rng, kept = random.Random(seed), []
    for parents in _trees(case)[1]:
        paths = sorted((_path(parents, i) for i in range(len(parents))), key=len)
        kept.append(rng.choice([p for p in paths if all(a == j or a >= len(p) for j, a in enumerate(p))][-6:]))
    return kept


def work(case: dict) -> dict:
    past, trees = _trees(case)
    tokens = sum(map(len, trees))
    if case["kind"] == "rope":
        elements = tokens * (case["heads"] + case["kv"]) * case["hd"]
        return dict(bytes=8 * elements, flops=(10 if case["norm"] else 6) * elements)
    if case["kind"] == "verify":
        # (Every token's logits, and of the drafts' probabilities those of one token of each sequence.)
        rows = tokens + (case["seqs"] if case["draft"] != "chosen" else 0)
        return dict(bytes=4 * rows * case["vocab"] + 20 * tokens, flops=4 * rows * case["vocab"])
    position = _position_bytes(case)
    if case["kind"] == "keep":
        moved = sum(a != j for p in _kept(case, 1) for j, a in enumerate(p)) * case["layers"]
        return dict(bytes=2 * position * max(1, moved), flops=0)
    seen = sum(len(t) * p + sum(_depths(t)) + len(t) for p, t in zip(past, trees))
    return dict(bytes=position * (sum(past) + tokens) + 8 * tokens * case["heads"] * case["hd"],
                flops=4 * seen * case["heads"] * case["hd"])


# --- inputs -----------------------------------------------------------------------

def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


class State:
    """What a program keeps between calls."""


def _rows(gen, positions: int, kv: int, hd: int) -> torch.Tensor:
    """Rows of keys or values: normal, of a magnitude of its own per position and head."""
    size = torch.exp(0.4 * torch.randn(positions, kv, 1, generator=gen, device="cuda"))
    return torch.randn(positions, kv, hd, generator=gen, device="cuda").mul_(size)


def _quantise(x: torch.Tensor, fmt: str):
    """(values in the cache's type, scales or None) of rows x [..., hd]."""
    if fmt == "f16":
        return x.half(), None
    scale = (x.abs().amax(-1) / TOP[fmt]).clamp(2.0 ** -40, 2.0 ** 60)
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


def _pages(case: dict, lengths: list[int], seed: int):
    """Each sequence's pages out of a pool that other sequences use too: (lists, pages of the pool)."""
    need = [-(-n // case["page"]) for n in lengths]
    total = sum(need) + 1 + sum(need) // 8
    order = np.random.default_rng(seed).permutation(total)[:sum(need)]
    return [a.tolist() for a in np.split(order, np.cumsum(need)[:-1])], total


def _fill(case: dict, seed: int, blocks: int) -> torch.Tensor:
    """Bytes of blocks that belong to other sequences: finite in every format."""
    return torch.randint(0, 0x40, (blocks, case["kv"], _block_bytes(case)), generator=_generator(seed + 1), device="cuda",
                         dtype=torch.uint8)


def _attend_inputs(case: dict, seed: int):
    """Quantised keys and values of all positions (each sequence padded to whole blocks), where each sequence's begin among
    them, and the queries."""
    past, trees = _trees(case)
    gen, s = _generator(seed), State()
    lengths = [p + len(t) for p, t in zip(past, trees)]
    s.begins = (GROUP * np.cumsum([0] + [-(-n // GROUP) for n in lengths])).tolist()
    s.q = 1.5 * torch.randn(sum(map(len, trees)), case["heads"], case["hd"], generator=gen, device="cuda")
    s.k = _quantise(_rows(gen, s.begins[-1], case["kv"], case["hd"]), case["fmt"])
    s.v = _quantise(_rows(gen, s.begins[-1], case["kv"], case["hd"]), case["fmt"])
    return s


def _rope_inputs(case: dict, seed: int):
    """A batch's rows of queries (each head's beside its gate where heads are of 256), keys and values, as one projection
    leaves them."""
    past, trees = _trees(case)
    gen, s = _generator(seed), State()
    s.apart = case["hd"] * (2 if case["hd"] == 256 else 1)  # from one query head to the next
    s.k_at = case["heads"] * s.apart
    s.rows = 2 * torch.randn(sum(map(len, trees)), s.k_at + 2 * case["kv"] * case["hd"], generator=gen, device="cuda")
    s.q_norm = 1 + 0.2 * torch.randn(case["hd"], generator=gen, device="cuda")
    s.k_norm = 1 + 0.2 * torch.randn(case["hd"], generator=gen, device="cuda")
    return s


EPS = 1e-5
ORIGINAL, SLOW, FAST = 16384, 1.0, 32.0  # positions of the training, and the turns over them that "parts" goes by


def _magnitude(case: dict) -> float:
    return 0.1 * math.log(case["factor"]) + 1 if case["scaling"] == "parts" else 1.0


def _verify_inputs(case: dict, seed: int):
    """The target's logits, what each token's children were drawn from (the target's probabilities, disturbed), the drafted
    tokens, the random numbers and the temperatures; every fourth sequence takes the likeliest token, every eighth token's
    logits leave out most of the vocabulary."""
    _, trees = _trees(case)
    gen, s = _generator(seed), State()
    rows, vocab, kids = sum(map(len, trees)), case["vocab"], max(1, case["width"])
    s.logits = 2.5 * torch.randn(rows, vocab, generator=gen, device="cuda")
    some = torch.rand(rows, vocab, generator=gen, device="cuda") < 0.02
    some[:, 0] = True
    few = torch.arange(rows, device="cuda")[:, None] % 8 == 5
    s.logits = torch.where(few & ~some, -math.inf, s.logits)
    s.logits += torch.where(torch.rand(rows, vocab, generator=gen, device="cuda") < 8 / vocab, 9.0, 0.0)  # a few likely ones
    s.temperature = 0.3 + 0.9 * torch.rand(case["seqs"], generator=gen, device="cuda")
    s.temperature[3::4] = 0.0
    s.u = torch.rand(rows, generator=gen, device="cuda")
    each = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor([len(t) for t in trees])).cuda()
    heat = torch.where(s.temperature > 0, s.temperature, torch.ones_like(s.temperature))[each, None]
    near = s.logits / heat + 0.7 * torch.randn(rows, vocab, generator=gen, device="cuda")
    q = torch.exp(near - near.amax(-1, keepdim=True))
    q = q / q.sum(-1, keepdim=True)
    if case["draft"] == "drawn":
        picks = torch.multinomial(q, kids, replacement=True, generator=gen)
    elif case["draft"] == "distinct":
        picks = torch.multinomial(q, kids, generator=gen)
    else:
        picks = torch.topk(near, kids).indices
    s.q = None if case["draft"] == "chosen" else q
    # Child number i of token a is pick i of a's.
    parent, slot, at = [], [], 0
    for t in trees:
        count = [0] * len(t)
        for a in t:
            parent.append(max(a, 0) + at)
            slot.append(count[a] if a >= 0 else 0)
            if a >= 0:
                count[a] += 1
        at += len(t)
    s.tokens = picks[torch.tensor(parent, device="cuda"), torch.tensor(slot, device="cuda")]
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
    past, trees = _trees(case)
    s = dict(rope=_prepare_rope, attend=_prepare_attend, verify=_prepare_verify, keep=_prepare_keep)[case["kind"]](
        case, seed, past, trees)
    s.case = case
    torch.cuda.synchronize()
    return s


def _parents(trees):
    """The trees as the library takes them: a list of parents for each sequence, None for a chain."""
    return [None if t == list(range(-1, len(t) - 1)) else [NOTHING if a < 0 else a for a in t] for t in trees]


def _plan(s, case, past, trees, pages, total, heads):
    s.plan = _hip().kv_plan(case.get("fmt", "f16"), case.get("kv", 1), case.get("hd", 64), case.get("page", 512), total, heads)
    s.plan.set(past, [len(t) for t in trees], pages, parents=_parents(trees))


def _prepare_rope(case, seed, past, trees):
    d, s = _rope_inputs(case, seed), State()
    s.__dict__.update(d.__dict__)
    s.position = torch.tensor([p + n for p, t in zip(past, trees) for n in _depths(t)], device="cuda")
    if own:
        from bobcat_amd.backend import NormSpec, RopeRows
        pages, total = _pages(dict(case, page=512), [p + len(t) for p, t in zip(past, trees)], seed)
        _plan(s, case, past, trees, pages, total, case["heads"])
        s.rope = _hip().rope(case["rot"], case["theta"], layout=case["layout"], scaling=case["scaling"], factor=case["factor"],
                             n_original=ORIGINAL, slow=SLOW, fast=FAST, magnitude=_magnitude(case))
        at_rows, s.rows = _place(s.rows)
        at_qn, s.q_norm = _place(s.q_norm)
        at_kn, s.k_norm = _place(s.k_norm)
        n = s.rows.shape[0]
        at_q, s.q_out = _place(torch.zeros(n, case["heads"], case["hd"], device="cuda"))
        at_k, s.k_out = _place(torch.zeros(n, case["kv"], case["hd"], device="cuda"))
        norm = (lambda at: NormSpec(at, EPS)) if case["norm"] else (lambda at: None)
        s.at_q = RopeRows(at_rows, s.rows.shape[1], at_q, case["heads"] * case["hd"], case["heads"], head_stride=s.apart,
                          norm=norm(at_qn))
        s.at_k = RopeRows(at_rows.buffer.floats(s.k_at), s.rows.shape[1], at_k, case["kv"] * case["hd"], case["kv"],
                          norm=norm(at_kn))
    return s


def _prepare_attend(case, seed, past, trees):
    d, s = _attend_inputs(case, seed), State()
    per_page = case["page"] // GROUP
    lengths = [p + len(t) for p, t in zip(past, trees)]
    pages, total = _pages(case, lengths, seed)
    s.pool = _fill(case, seed, total * per_page)
    # Block g of a sequence is block g % per_page of its page g // per_page.
    where = [np.asarray(pg, np.int64)[g // per_page] * per_page + g % per_page
             for pg, n in zip(pages, lengths) for g in [np.arange(-(-n // GROUP))]]
    s.pool[torch.from_numpy(np.concatenate(where)).cuda()] = _pack(d.k, d.v, case)
    s.pool = s.pool.view(total, per_page, case["kv"], -1).transpose(1, 2).contiguous()  # [page, head, block of 16, bytes]
    widest = max(len(pg) for pg in pages)
    s.table = torch.tensor([pg + [0] * (widest - len(pg)) for pg in pages], device="cuda")
    new = [len(t) for t in trees]
    s.past, s.new = torch.tensor(past, device="cuda"), torch.tensor(new, device="cuda")
    s.rows = torch.repeat_interleave(torch.arange(len(new), device="cuda"), s.new)  # the sequence of each new token
    s.step = torch.arange(sum(new), device="cuda") - (torch.cumsum(s.new, 0) - s.new)[s.rows]
    s.most_new, s.longest = max(new), max(lengths)
    above = np.zeros((len(new), s.most_new, s.most_new), bool)  # [sequence, token, its ancestors and itself]
    for i, t in enumerate(trees):
        for j, a in enumerate(t):
            if a >= 0:
                above[i, j] = above[i, a]
            above[i, j, j] = True
    s.above = torch.from_numpy(above).cuda()
    s.q = d.q
    if own:
        _plan(s, case, past, trees, pages, total, case["heads"])
        s.at_pool, s.pool = _place(s.pool)
        s.at_q, s.q = _place(s.q)
        s.at_out, s.out = _place(torch.zeros_like(s.q))
    return s


def _prepare_verify(case, seed, past, trees):
    s = _verify_inputs(case, seed)
    n, starts = case["seqs"], np.cumsum([0] + [len(t) for t in trees])[:-1]
    kids = np.full((sum(map(len, trees)), max(1, case["width"])), -1, np.int64)  # a token's children's rows, in their order
    for at, t in zip(starts, trees):
        for j, a in enumerate(t):
            if a >= 0:
                kids[at + a, (kids[at + a] >= 0).sum()] = at + j
    s.kids, s.first = torch.from_numpy(kids).cuda(), torch.from_numpy(starts).cuda()
    s.deepest = max(max(_depths(t)) for t in trees)
    if own:
        pages, total = _pages(dict(case, page=512), [len(t) for t in trees], seed)
        _plan(s, case, past, trees, pages, total, 1)
        s.at_logits, s.logits = _place(s.logits)
        s.at_draft = None
        if s.q is not None:
            s.at_draft, s.q = _place(s.q)
        s.at_tokens, s.tokens = _place(s.tokens.int())
        s.at_u, s.u = _place(s.u)
        s.at_heat, s.temperature = _place(s.temperature)
        s.at_kept, s.kept = _place(torch.zeros(n, dtype=torch.int32, device="cuda"))
        s.at_path, s.path = _place(torch.zeros(len(kids), dtype=torch.int32, device="cuda"))
        s.at_next, s.next = _place(torch.zeros(n, dtype=torch.int32, device="cuda"))
        s.at_chances, s.chances = _place(torch.zeros(len(kids), device="cuda"))
    return s


def _keep_pool(case, seed, total):
    raw = _fill(case, seed, case["layers"] * total * (case["page"] // GROUP))
    return raw.view(case["layers"], total, case["page"] // GROUP, case["kv"], -1).transpose(2, 3).contiguous()


def _prepare_keep(case, seed, past, trees):
    s, kept = State(), _kept(case, seed)
    pages, total = _pages(case, [p + len(t) for p, t in zip(past, trees)], seed)
    s.pool = _keep_pool(case, seed, total)  # [layer, page, head, block of 16, bytes]
    s.kept = torch.tensor([len(p) for p in kept], dtype=torch.int32, device="cuda")
    s.path = torch.tensor([a for p, t in zip(kept, trees) for a in p + [-1] * (len(t) - len(p))], dtype=torch.int32, device="cuda")
    widest = max(len(pg) for pg in pages)
    s.table = torch.tensor([pg + [0] * (widest - len(pg)) for pg in pages], device="cuda")
    new = torch.tensor([len(t) for t in trees], device="cuda")
    s.past = torch.tensor(past, device="cuda")
    s.rows = torch.repeat_interleave(torch.arange(len(trees), device="cuda"), new)
    s.step = torch.arange(s.rows.numel(), device="cuda") - (torch.cumsum(new, 0) - new)[s.rows]
    if own:
        _plan(s, case, past, trees, pages, total, case["kv"])
        s.at_pool, s.pool = _place(s.pool)
        s.at_kept, s.kept = _place(s.kept)
        s.at_path, s.path = _place(s.path)
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


def _own_rope(hip, s, c):
    hip.rope_paged(s.rope, s.plan, s.at_q, s.at_k)
    return [s.q_out, s.k_out]


def _own_attend(hip, s, c):
    hip.attention_paged(s.plan, s.at_pool, s.at_q, c["heads"] * c["hd"], s.at_out, c["heads"] * c["hd"])
    return s.out


def _own_verify(hip, s, c):
    hip.verify_drafts(s.plan, 0, c["seqs"], c["vocab"], s.at_logits, s.at_tokens, s.at_u, s.at_heat, s.at_kept, s.at_path,
                      s.at_next, chances=s.at_chances, draft=s.at_draft, distinct=c["draft"] == "distinct")
    return [s.kept, s.path, s.next, s.chances]


def _own_keep(hip, s, c):
    hip.kv_keep(s.plan, 0, c["seqs"], s.at_pool, c["layers"], s.pool[0].numel(), s.at_kept, s.at_path)
    return _stored(s.pool, c)


def _stored(pool, c):
    """The cache as the values that it holds, with the rows' scales."""
    k, v, scales = _parts(pool, c)
    return [_elements(k, c["fmt"]), _elements(v, c["fmt"])] + ([] if scales is None else [scales])


def _plain_rope(s, c):
    j = torch.arange(c["rot"] // 2, dtype=F64, device="cuda")
    f = c["theta"] ** (-2 * j / c["rot"])
    if c["scaling"] == "linear":
        f = f / c["factor"]
    elif c["scaling"] == "parts":
        w = ((ORIGINAL * f / (2 * math.pi) - SLOW) / (FAST - SLOW)).clamp(0, 1)
        f = f * (w + (1 - w) / c["factor"])
    angle = s.position.to(F64)[:, None, None] * f  # far positions' angles need more than 32 bits
    cos, sin = (_magnitude(c) * torch.cos(angle)).float(), (_magnitude(c) * torch.sin(angle)).float()

    def turn(x, weight):
        if c["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        x, rest = x[..., :c["rot"]], x[..., c["rot"]:]
        a, b = (x[..., 0::2], x[..., 1::2]) if c["layout"] == "pairs" else x.chunk(2, -1)
        a, b = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack([a, b], -1).flatten(-2) if c["layout"] == "pairs" else torch.cat([a, b], -1)
        return torch.cat([turned, rest], -1)

    q = s.rows[:, :s.k_at].unflatten(-1, (c["heads"], s.apart))[..., :c["hd"]]
    k = s.rows[:, s.k_at:s.k_at + c["kv"] * c["hd"]].unflatten(-1, (c["kv"], c["hd"]))
    return [turn(q, s.q_norm), turn(k, s.k_norm)]


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


def _plain_attend(s, c):
    k, v = _gathered(s, c)
    n, group, longest = s.past.numel(), c["heads"] // c["kv"], s.longest
    k, v = k[:, :, :longest], v[:, :, :longest]
    key = torch.arange(longest, device="cuda")
    # Positions past a sequence's end hold other sequences' bytes: no part of its sums.
    v = torch.where(key[:, None] < (s.past + s.new)[:, None, None, None], v, 0.0)
    behind = (key - s.past[:, None])[:, None].expand(-1, s.most_new, -1)  # of the past: the new tokens' keys
    seen = (behind < 0) | (torch.gather(s.above, 2, behind.clamp(0, s.most_new - 1)) & (behind < s.most_new))
    q = torch.zeros(n, s.most_new, c["kv"], group, c["hd"], device="cuda")
    q[s.rows, s.step] = s.q.view(-1, c["kv"], group, c["hd"]) / math.sqrt(c["hd"])
    q = q.permute(0, 2, 1, 3, 4).reshape(n, c["kv"], s.most_new * group, c["hd"])
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(n, c["kv"], s.most_new, group, longest)
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(n, c["kv"], -1, longest), v).view(n, c["kv"], s.most_new, group, c["hd"]) / total
    return out.permute(0, 2, 1, 3, 4)[s.rows, s.step].reshape(-1, c["heads"], c["hd"])


def _plain_verify(s, c):
    # (Probabilities are added up and compared: in 64 bits.)
    rows, seqs, vocab = s.logits.shape[0], s.first.numel(), c["vocab"]
    new = torch.diff(s.first, append=torch.tensor([rows], device="cuda"))
    each = torch.repeat_interleave(torch.arange(seqs, device="cuda"), new)
    heat, every = s.temperature.to(F64), torch.arange(seqs, device="cuda")
    greedy = heat <= 0
    p = s.logits.to(F64) / torch.where(greedy, 1.0, heat)[each, None]
    p = torch.exp_(p.sub_(p.amax(-1, keepdim=True)))
    p /= p.sum(-1, keepdim=True)
    best = s.logits.argmax(-1)
    only = torch.zeros_like(p).scatter_(1, best[:, None], 1.0)
    p = torch.where(greedy[each, None], only, p)
    token, u = s.tokens.long(), s.u.to(F64)
    # The target's probability of each drafted token, after its parent.
    parent = torch.arange(rows, device="cuda").index_put(
        (s.kids[s.kids >= 0],), torch.arange(rows, device="cuda")[:, None].expand_as(s.kids)[s.kids >= 0])
    chances = p[parent, token]
    at, walking = s.first, torch.ones_like(greedy)
    path = torch.full((rows + 1,), -1, device="cuda")  # (the last place takes what is not kept)
    path[s.first] = 0
    kept = torch.ones_like(s.first)
    r = p[at]
    for _ in range(s.deepest):
        here, moved = at, torch.zeros_like(walking)
        left = torch.ones_like(heat)  # what the tokens that were not kept leave of q
        for slot in range(s.kids.shape[1]):
            child = s.kids[here, slot]
            trying, child = walking & ~moved & (child >= 0), child.clamp(min=0)
            x = token[child]
            point = torch.zeros(seqs, vocab, dtype=F64, device="cuda").scatter_(1, x[:, None], 1.0)
            q = point if s.q is None else torch.where(greedy[:, None], point, s.q[here].to(F64) / left[:, None])
            stays = trying & (u[child] * q[every, x] < r[every, x])
            falls = trying & ~stays
            rest = (r - q).clamp(min=0)
            total = rest.sum(-1, keepdim=True)
            r = torch.where(falls[:, None], torch.where(total > 0, rest / total, 0.0), r)
            if s.q is not None and c["draft"] == "distinct":
                left = torch.where(falls, left - s.q[here, x].to(F64), left)
            at = torch.where(stays, child, at)
            path[torch.where(stays, s.first + kept, rows)] = child - s.first
            kept = kept + stays
            moved = moved | stays
            r = torch.where(stays[:, None], p[at], r)
        walking = walking & moved
    r = torch.where((r.sum(-1, keepdim=True) > 0), r, p[at])
    up = torch.cumsum(r, -1)
    goal = u[s.first] * up[:, -1]
    next_ = torch.searchsorted(up, goal[:, None], right=True)[:, 0].clamp(max=vocab - 1)
    chances[s.first] = p[at, next_]
    return [kept.int(), path[:-1].int(), next_.int(), chances.float()]


def _plain_keep(s, c):
    k, v, scales = _parts(s.pool, c)
    stays = (s.step < s.kept[s.rows]) & (s.path >= 0)
    seq, to, of = s.rows[stays], (s.past[s.rows] + s.step)[stays], (s.past[s.rows] + s.path)[stays]
    page, block, i = s.table[seq, to // c["page"]], to % c["page"] // GROUP, to % GROUP
    page0, block0, i0 = s.table[seq, of // c["page"]], of % c["page"] // GROUP, of % GROUP
    k[:, page, :, block, :, i, :] = k[:, page0, :, block0, :, i0, :].clone()
    v[:, page, :, block, :, i // 4, :, :, i % 4] = v[:, page0, :, block0, :, i0 // 4, :, :, i0 % 4].clone()
    if scales is not None:
        scales[:, page, :, block, :, i] = scales[:, page0, :, block0, :, i0].clone()
    return _stored(s.pool, c)


_OWN = dict(rope=_own_rope, attend=_own_attend, verify=_own_verify, keep=_own_keep)
_PLAIN = dict(rope=_plain_rope, attend=_plain_attend, verify=_plain_verify, keep=_plain_keep)


# --- the definitions in float64 ---------------------------------------------------------

def exact(case: dict, seed: int):
    past, trees = _trees(case)
    return dict(rope=_exact_rope, attend=_exact_attend, verify=_exact_verify, keep=_exact_keep)[case["kind"]](
        case, seed, past, trees)


def _exact_rope(case, seed, past, trees):
    d = _rope_inputs(case, seed)
    position = torch.tensor([p + n for p, t in zip(past, trees) for n in _depths(t)], dtype=F64, device="cuda")
    out = []
    for at, apart, heads, weight in ((0, d.apart, case["heads"], d.q_norm), (d.k_at, case["hd"], case["kv"], d.k_norm)):
        x = torch.stack([d.rows[:, at + h * apart:at + h * apart + case["hd"]] for h in range(heads)], 1).to(F64)
        if case["norm"]:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * weight.to(F64)
        y = x.clone()
        for j in range(case["rot"] // 2):
            f = case["theta"] ** (-2 * j / case["rot"])
            if case["scaling"] == "linear":
                f /= case["factor"]
            if case["scaling"] == "parts":
                w = min(1.0, max(0.0, (ORIGINAL * f / (2 * math.pi) - SLOW) / (FAST - SLOW)))
                f = w * f + (1 - w) * f / case["factor"]
            a, b = (2 * j, 2 * j + 1) if case["layout"] == "pairs" else (j, j + case["rot"] // 2)
            z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(position, _magnitude(case)), position * f)[:, None]
            y[..., a], y[..., b] = z.real, z.imag
        out.append(y)
    return out


def _value(quantised, at, n) -> torch.Tensor:
    values, scale = quantised
    values = values[at:at + n].to(F64)
    return values if scale is None else values * scale[at:at + n].to(F64)[..., None]


def _exact_attend(case, seed, past, trees):
    d, group = _attend_inputs(case, seed), case["heads"] // case["kv"]
    if sum(len(t) * (p + len(t)) for p, t in zip(past, trees)) * case["heads"] * case["hd"] > 4e12:
        return None
    out, row = torch.empty(d.q.shape, dtype=F64, device="cuda"), 0
    for p, t, at in zip(past, trees, d.begins):
        n = len(t)
        k, v = _value(d.k, at, p + n), _value(d.v, at, p + n)
        seen = torch.zeros(n, p + n, dtype=torch.bool)
        seen[:, :p] = True
        for i in range(n):
            seen[i, [p + a for a in _path(t, i)]] = True
        for h in range(case["heads"]):
            a = d.q[row:row + n, h].to(F64) @ k[:, h // group].T.contiguous() / math.sqrt(case["hd"])
            out[row:row + n, h] = torch.softmax(a.masked_fill(~seen.cuda(), -math.inf), 1) @ v[:, h // group].contiguous()
        row += n
    return out


def _exact_verify(case, seed, past, trees):
    """The walk with what is left of p as (p − c·q)+ / total: a rejection adds total / (what is left of q) to c."""
    d = _verify_inputs(case, seed)
    kept, paths, nexts, chances, row = [], [], [], [], 0
    tokens, uniform = d.tokens.tolist(), d.u.double().tolist()
    for i, t in enumerate(trees):
        heat = float(d.temperature[i])

        def target(j):
            x = d.logits[row + j].to(F64)
            if heat > 0:
                return torch.softmax(x / heat, 0)
            return (torch.arange(x.numel(), device="cuda") == int(x.argmax())).to(F64)

        for j, a in enumerate(t):
            chances.append(float(target(a)[tokens[row + j]]) if a >= 0 else 0.0)
        path, settled = [0], False
        while not settled:
            p, settled = target(path[-1]), True
            q = None if d.q is None or heat <= 0 else d.q[row + path[-1]].to(F64)
            rest, total, c, left = p, 1.0, 0.0, 1.0
            for j in [j for j, a in enumerate(t) if a == path[-1]]:
                x = tokens[row + j]
                if uniform[row + j] * (1.0 if q is None else float(q[x]) / left) * total < float(rest[x]):
                    path.append(j)
                    settled = False
                    break
                if q is None:
                    rest = rest.clone()
                    rest[x] = 0
                else:
                    c += total / left
                    rest = (p - c * q).clamp(min=0)
                    left -= float(q[x]) if case["draft"] == "distinct" else 0
                total = float(rest.sum())
        up = torch.cumsum(rest if total > 0 else p, 0)
        pick = int((up > uniform[row] * up[-1]).nonzero()[0])
        chances[row] = float(p[pick])
        kept.append(len(path))
        paths += path + [-1] * (len(t) - len(path))
        nexts.append(pick)
        row += len(t)
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return [whole(kept), whole(paths), whole(nexts), torch.tensor(chances, dtype=F64, device="cuda")]


def _exact_keep(case, seed, past, trees):
    """Every element of a kept row put at its new offset among the bytes that were there, as the values they stand for."""
    hd, fmt = case["hd"], case["fmt"]
    pages, total = _pages(case, [p + len(t) for p, t in zip(past, trees)], seed)
    pool = _keep_pool(case, seed, total)
    size = 2 if fmt == "f16" else 1
    per, m, n = 16 // size, 4 // size, GROUP * hd * size
    kind = dict(f16=torch.float16, i8=torch.int8, f8=torch.float8_e4m3fn)[fmt]
    elements = pool[..., :2 * n].contiguous().view(kind).to(F64)
    scales = None if fmt == "f16" else pool[..., 2 * n:].contiguous().view(torch.float32).to(F64)
    e = torch.arange(hd, device="cuda")

    def slots(i):
        return torch.cat([(e // per * GROUP + i) * per + e % per,
                          GROUP * hd + (((e // (16 * m) * 4 + i // 4) * 16 + e % 16) * m + e // 16 % m) * 4 + i % 4])

    for p, table, path in zip(past, pages, _kept(case, seed)):
        for j, a in enumerate(path):
            (pt, bt, it), (pf, bf, i) = [(table[x // case["page"]], x % case["page"] // GROUP, x % GROUP) for x in (p + j, p + a)]
            elements[:, pt, :, bt, slots(it)] = elements[:, pf, :, bf, slots(i)]
            if scales is not None:
                scales[:, pt, :, bt, [it, GROUP + it]] = scales[:, pf, :, bf, [i, GROUP + i]]
    lead = tuple(pool.shape[:-1])
    out = [elements[..., :GROUP * hd].reshape(*lead, hd // per, GROUP, per),
           elements[..., GROUP * hd:].reshape(*lead, hd // (16 * m), 4, 16, m, 4)]
    if fmt == "i8":
        out = [x.to(torch.int8) for x in out]
    return out if scales is None else out + [scales.view(*lead, 2, GROUP)]

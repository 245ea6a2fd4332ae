"""GPU parity of the paged cache (bch_kv_store, bch_kv_load,
bch_attention_paged) against the plain restatements of tests/_paged.py: stored
bytes equal the definition's, attention is inside the bound that
`attention_bound` derives.  Free places of the caches hold NaN in every
format, so a read of one shows."""
from __future__ import annotations

import numpy as np
import pytest

from _paged import Batch, Pool, attention, attention_bound, dequantise, quantise, random_rows
from bobcat_amd import BobcatError
from bobcat_amd._lib import STATUS, Sampling
from bobcat_amd.backend import LOGIT_ROW, NO_MASK, Format, Hip, kv_page_bytes

pytestmark = pytest.mark.gpu

FORMATS = ["f16", "i8", "f8"]


def run(hip, fn):
    hip.begin()
    fn()
    hip.end()


def say(*what):
    print(*what, flush=True)


def plan_of(hip, pool, batch, heads):
    plan = hip.kv_plan(pool.fmt, pool.kv, pool.hd, pool.page, pool.n_pages, heads)
    assert kv_page_bytes(plan.shape) * pool.n_pages == pool.bytes.nbytes
    plan.set(batch.past, batch.new, batch.pages)
    return plan


def strided(rows, extra, fill=np.nan):
    """Rows [n, width] with `extra` floats behind each."""
    out = np.full((rows.shape[0], rows.shape[1] + extra), fill, np.float32)
    out[:, :rows.shape[1]] = rows
    return out


# --- store and load ---------------------------------------------------------------

STORES = [([(0, 1)], 16), ([(15, 1), (16, 1), (0, 16)], 16), ([(3, 40), (0, 0), (47, 1), (5, 11), (32, 16)], 48),
          ([(250, 300), (7, 2)], 256), ([(0, 33), (64, 0), (31, 2)], 32)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kv,hd", [(1, 64), (3, 128), (2, 256)])
@pytest.mark.parametrize("seqs,page", STORES)
def test_store_matches_the_definition(hip, fmt, kv, hd, seqs, page):
    say("kv_store", fmt, kv, hd, seqs, page)
    rng = np.random.default_rng(hd + page)
    batch = Batch(rng, seqs, page)
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    pool.bytes[:] = rng.integers(0, 256, pool.bytes.shape, np.uint8)  # every other byte keeps its value
    cache = hip.buffer_from(pool.bytes)
    plan = plan_of(hip, pool, batch, kv)
    rows = np.stack([random_rows(rng, kv, hd) for _ in range(batch.tokens)])
    k, v = rows[:, 0], rows[:, 1]
    kb, vb = hip.buffer_from(strided(k.reshape(-1, kv * hd), 4)), hip.buffer_from(strided(v.reshape(-1, kv * hd), 12))
    run(hip, lambda: hip.kv_store(plan, cache.at(0), kb.at(0), kv * hd + 4, vb.at(0), kv * hd + 12))
    batch.put(pool, k, v)
    assert np.array_equal(hip.read(cache.at(0), np.empty_like(pool.bytes)), pool.bytes)
    # And what was stored reads back as the definition's values (one f32 product).
    for s, (past, new) in enumerate(seqs):
        if new:
            kb, vb = hip.new_buffer(new * kv * hd * 4), hip.new_buffer(new * kv * hd * 4)
            run(hip, lambda: hip.kv_load(plan, cache.at(0), s, past, new, kb.at(0), vb.at(0)))
            at = [i for i, (t, _) in enumerate(batch.rows) if t == s]
            for buffer, x in ((kb, k), (vb, v)):
                bits, scale = quantise(x[at], fmt)
                want = dequantise(bits, scale, fmt).astype(np.float32)
                assert np.array_equal(hip.read(buffer.at(0), np.empty_like(want)), want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_store_of_rows_at_the_ends_of_the_range(hip, fmt):
    """Zeros, rows below and above the scales' range, ties between two integers, infinities and NaN."""
    kv, hd, page = 1, 64, 16
    rng = np.random.default_rng(5)
    x = rng.standard_normal((16, kv, hd)).astype(np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2] *= 1e-30
    x[3] *= np.float32(1e30)
    x[4] = np.arange(-32, 32, dtype=np.float32)[None] + 0.5
    x[4, 0, 0] = 127.0  # scale 1: every other element a tie
    x[5, 0, 7] = np.inf
    x[6, 0, 9] = -np.inf
    x[7, 0, 3] = np.nan
    x[8] = np.finfo(np.float32).max
    x[9] = np.finfo(np.float32).tiny
    x[10] = 1e-42
    x[11] = 65520.0  # rounds past f16's end
    x[12, 0, 0] = 448.0
    x[12, 0, 1:] = np.linspace(-30, 30, 63)
    batch = Batch(rng, [(0, 16)], page)
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    cache = hip.buffer_from(pool.bytes)
    plan = plan_of(hip, pool, batch, 1)
    xb = hip.buffer_from(x)
    run(hip, lambda: hip.kv_store(plan, cache.at(0), xb.at(0), hd, xb.at(0), hd))
    batch.put(pool, x, x)
    got = hip.read(cache.at(0), np.empty_like(pool.bytes))
    part = 16 * hd * (2 if fmt == "f16" else 1)
    if fmt == "f16":  # (a NaN's bits may differ)
        a, b = (t.reshape(-1).view(np.float16) for t in (got, pool.bytes))
        assert np.array_equal(a, b, equal_nan=True)
        return
    assert np.array_equal(got[..., :2 * part], pool.bytes[..., :2 * part])
    a, b = (np.ascontiguousarray(t[..., 2 * part:]).view(np.float32) for t in (got, pool.bytes))
    assert np.array_equal(a, b, equal_nan=True)
    out = [hip.new_buffer(x.nbytes) for _ in range(2)]
    run(hip, lambda: hip.kv_load(plan, cache.at(0), 0, 0, 16, out[0].at(0), out[1].at(0)))
    for buffer in out:
        back = hip.read(buffer.at(0), np.empty_like(x))
        assert np.isnan(back[[5, 6, 7]]).all() and np.isfinite(np.delete(back, [5, 6, 7], 0)).all()


@pytest.mark.parametrize("fmt,hd", [("f16", 64), ("i8", 128), ("f8", 256)])
def test_load_ranges(hip, fmt, hd):
    """Parts of a sequence from any position, and nothing outside them."""
    rng = np.random.default_rng(11)
    kv, page = 2, 48
    batch = Batch(rng, [(20, 0), (131, 4)], page)
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    batch.fill(rng, pool)
    batch.put(pool, *np.stack([random_rows(rng, kv, hd) for _ in range(4)], 1))
    cache, plan = hip.buffer_from(pool.bytes), plan_of(hip, pool, batch, kv)
    for seq, first, n in [(0, 0, 20), (1, 0, 135), (1, 1, 1), (1, 15, 2), (1, 47, 50), (1, 134, 1), (1, 7, 0), (1, 135, 0)]:
        keys, values = batch.gather(pool, seq)
        guard = np.full((n + 1) * kv * hd, 7.0, np.float32)
        kb, vb = hip.buffer_from(guard), hip.buffer_from(guard)
        run(hip, lambda: hip.kv_load(plan, cache.at(0), seq, first, n, kb.at(0), vb.at(0)))
        for buffer, want in ((kb, keys), (vb, values)):
            got = hip.read(buffer.at(0), np.empty_like(guard))
            assert np.array_equal(got[:n * kv * hd], want[first:first + n].astype(np.float32).reshape(-1)), (seq, first, n)
            assert (got[n * kv * hd:] == 7.0).all()


# --- attention ---------------------------------------------------------------------

def attend(hip, pool, batch, heads, q, plan=None, extra=(0, 0)):
    cache = hip.buffer_from(pool.bytes)
    plan = plan or plan_of(hip, pool, batch, heads)
    width = heads * pool.hd
    qb = hip.buffer_from(strided(q.reshape(-1, width), extra[0]))
    out = hip.buffer_from(np.full((batch.tokens + 1, width + extra[1]), 7.0, np.float32))
    run(hip, lambda: hip.attention_paged(plan, cache.at(0), qb.at(0), width + extra[0], out.at(0), width + extra[1]))
    got = hip.read(out.at(0), np.empty((batch.tokens + 1, width + extra[1]), np.float32))
    assert (got[-1] == 7.0).all() and (got[:, width:] == 7.0).all()  # nothing behind the rows
    return got[:-1, :width].reshape(batch.tokens, heads, pool.hd)


def check_attention(hip, pool, batch, heads, q, **kw):
    got = attend(hip, pool, batch, heads, q, **kw)
    row = 0
    for s, (past, new) in enumerate(zip(batch.past, batch.new)):
        if new:
            k, v = batch.gather(pool, s)
            want = attention(q[row:row + new], k, v, past)
            worst = np.abs(got[row:row + new] - want).max()
            assert worst <= attention_bound(q[row:row + new], k, v), (s, past, new, worst)
        row += new
    return got


def case(rng, fmt, heads, kv, hd, page, seqs, scale=1.0):
    batch = Batch(rng, seqs, page)
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    batch.fill(rng, pool, scale)
    batch.put(pool, *np.stack([random_rows(rng, kv, hd, scale) for _ in range(batch.tokens)], 1))
    q = (1.5 * rng.standard_normal((batch.tokens, heads, hd))).astype(np.float32)
    return pool, batch, q


TOKENS = [([(0, 1)], 16), ([(0, 1), (600, 1), (15, 1), (16, 1), (31, 1)], 16), ([(130, 1), (0, 0), (700, 1)], 48),
          ([(1029, 1)], 256)]
CHUNKS = [([(0, 2)], 16), ([(5, 17), (0, 33), (40, 1), (3, 0)], 32), ([(100, 5), (33, 5), (290, 3)], 16),
          ([(61, 130)], 64), ([(0, 150), (500, 70)], 48)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 64), (4, 4, 128), (8, 1, 256), (6, 2, 64)])
@pytest.mark.parametrize("seqs,page", TOKENS + CHUNKS)
def test_attention_matches_float64(hip, fmt, heads, kv, hd, seqs, page):
    say("attention_paged", fmt, heads, kv, hd, seqs, page)
    rng = np.random.default_rng(heads * hd + page + len(seqs))
    check_attention(hip, *case_args(rng, fmt, heads, kv, hd, page, seqs))


def case_args(rng, fmt, heads, kv, hd, page, seqs, scale=1.0):
    pool, batch, q = case(rng, fmt, heads, kv, hd, page, seqs, scale)
    return pool, batch, heads, q


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (5, 1), (16, 1), (32, 1), (16, 8), (34, 2)])
@pytest.mark.parametrize("fmt,seqs", [("i8", [(77, 1), (200, 1)]), ("f16", [(77, 9), (0, 20)]), ("f8", [(30, 3)])])
def test_attention_groups(hip, heads, kv, fmt, seqs):
    say("attention_paged groups", heads, kv, fmt, seqs)
    check_attention(hip, *case_args(np.random.default_rng(heads), fmt, heads, kv, 64, 16, seqs))


# (past, new) with 4 heads a KV head: 8 and 9, 16 and 17, 32 and 33, 96 and 97, 128 and 129 rows and the like, alone and
# beside others; a wide tile with each number of rows in its last wave; many pieces of many tiles.
ROWS = [[(40, 2)], [(40, 3), (7, 2)], [(40, 4), (9, 5)], [(300, 8), (20, 9)], [(100, 24)], [(100, 25)], [(60, 32)],
        [(60, 33)], [(33, 41), (5, 9), (90, 1), (70, 3)], [(0, 64)], [(2000, 33), (3000, 20)], [(700, 100), (900, 1)] * 3]


@pytest.mark.parametrize("fmt,hd", [("f16", 64), ("i8", 64), ("f8", 128), ("f16", 128), ("i8", 256)])
@pytest.mark.parametrize("seqs", ROWS)
def test_attention_tiles(hip, fmt, hd, seqs):
    say("attention_paged tiles", fmt, hd, seqs)
    check_attention(hip, *case_args(np.random.default_rng(len(seqs)), fmt, 4, 1, hd, 48, seqs))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 40])
def test_attention_strides(hip, fmt, new):
    rng = np.random.default_rng(3)
    pool, batch, heads, q = case_args(rng, fmt, 4, 2, 64, 16, [(90, new), (20, new)])
    plain = check_attention(hip, pool, batch, heads, q)
    assert np.array_equal(plain, attend(hip, pool, batch, heads, q, extra=(8, 20)))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale", [1e-6, 1e4])
@pytest.mark.parametrize("new", [1, 36])
def test_attention_scales(hip, fmt, scale, new):
    """Keys and values far from 1 (the queries the other way, so that the softmax stays a mixture), with rows a
    thousand times their neighbours among them."""
    if fmt == "f16":  # (inside f16's range)
        scale = min(max(scale, 1e-2), 500.0)
    rng = np.random.default_rng(8)
    pool, batch, heads, q = case_args(rng, fmt, 4, 2, 64, 16, [(150, new)], scale)
    for at in (3, 40, 41, 100):
        rows = random_rows(rng, pool.kv, pool.hd, scale)
        pool.put(batch.pages[0][at // 16], at % 16, rows[0], rows[1] * (1000 if fmt != "f16" else 10))
    check_attention(hip, pool, batch, heads, (q / scale).astype(np.float32))


@pytest.mark.parametrize("size", [1e-8, 1e6, 1e20])
@pytest.mark.parametrize("new", [1, 36])
def test_attention_of_large_and_small_queries(hip, size, new):
    """Queries past f16's range: a large one picks its best key."""
    rng = np.random.default_rng(9)
    pool, batch, heads, q = case_args(rng, "i8", 4, 2, 64, 16, [(100, new)])
    got = attend(hip, pool, batch, heads, (q * np.float32(size)))
    k, v = batch.gather(pool, 0)
    want = attention(q * np.float32(size), k, v, batch.past[0])
    # (At 1e6 scores differ by thousands, so a probability is 0 or 1 unless two keys tie; the bound on scores says nothing.)
    worst = np.abs(got - want).max()
    assert worst <= (attention_bound(q * size, k, v) if size < 1 else np.abs(v).max() * 2.0 ** -20), worst


@pytest.mark.parametrize("fmt", ["i8", "f8"])
@pytest.mark.parametrize("scale", [1e5, 1e8, 1e15])
@pytest.mark.parametrize("new", [1, 36])
def test_attention_of_small_queries_and_large_keys(hip, fmt, scale, new):
    """Queries below f16's numbers, whose scores are ordinary ones; between them rows of zeros and of ordinary size
    (whose softmax picks one key, or two that tie)."""
    say("attention_paged small queries", fmt, scale, new)
    rng = np.random.default_rng(10)
    pool, batch, heads, q = case_args(rng, fmt, 4, 2, 64, 16, [(150, new)], scale)
    q = (q / scale).astype(np.float32)
    q[:, 1] = 0.0
    q[::3, 2] *= np.float32(scale)
    got = attend(hip, pool, batch, heads, q)
    k, v = batch.gather(pool, 0)
    want = attention(q, k, v, batch.past[0])
    small = np.ones(q.shape[:2], bool)
    small[::3, 2] = False
    bound = attention_bound(np.where(small[..., None], q, 0), k, v)
    assert np.abs(got - want)[small].max() <= bound
    assert np.abs(got - want)[~small].max() <= np.abs(v).max() * 2.0 ** -20


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e6, 3e7, 1e9, 1e15])
@pytest.mark.parametrize("new", [1, 36])
def test_attention_of_large_scores_and_values(hip, fmt, size, new):
    """Scores whose last place in f32 is more than the room that the probabilities have, with values far above 1: each
    query picks its best key (the next is millions below)."""
    say("attention_paged large scores", fmt, size, new)
    rng = np.random.default_rng(13)
    pool, batch, heads, q = case_args(rng, fmt, 4, 2, 64, 16, [(150, new)], 100.0)
    q *= np.float32(size)
    got = attend(hip, pool, batch, heads, q)
    k, v = batch.gather(pool, 0)
    assert np.abs(got - attention(q, k, v, batch.past[0])).max() <= np.abs(v).max() * 2.0 ** -20


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("seqs", [[(20, 40)], [(100, 1), (37, 1)], [(0, 5), (64, 3)], [(10, 140)]])
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_attention_leaves_out_what_a_query_does_not_see(hip, fmt, seqs, what):
    """Rows that are not finite: queries before them keep their bits, queries that see them become NaN."""
    rng = np.random.default_rng(21)
    heads, kv, hd, page = 4, 2, 64, 32
    pool, batch, q = case(rng, fmt, heads, kv, hd, page, seqs)
    before = check_attention(hip, pool, batch, heads, q)
    marks, row = {}, 0
    for s, (past, new) in enumerate(seqs):
        bad = new // 2  # token of the sequence whose rows are spoilt (of a single token's sequence: a position behind its end)
        at = past + bad if new > 1 else past + 1
        if at < len(batch.pages[s]) * page:
            k, v = random_rows(rng, kv, hd)
            k[:, 5] = v[:, 9] = np.nan if what == "nan" else np.inf
            pool.put(batch.pages[s][at // page], at % page, k, v)
        marks[s] = (row, row + (bad if new > 1 else new), row + new)
        row += new
    after = attend(hip, pool, batch, heads, q)
    for first, spoilt, end in marks.values():
        assert np.array_equal(after[first:spoilt], before[first:spoilt])
        assert np.isnan(after[spoilt:end, :, 9]).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("new", [1, 3, 130])
def test_attention_probabilities(hip, fmt, new):
    """Key i has 64 in element i alone and value i has 1 there, so that an output is the softmax of 8·q itself and shows
    every query element's rounding.  A score s is off by s·(2^-22 + 8·2^-24): the query's two parts and seven f32
    roundings (its scaling, the constant's, the key's scale, the reference's twice, the product's and the sum's); a
    probability by twice the largest of that (its own and the sum's), 2^-22 for its parts, 64·2^-24 for the sum and as
    many as 16 roundings more.  Besides, a part below f16's normal range is a multiple of 2^-24, off by 2^-25 at most,
    where the row's largest is 2^8 or more: 2^-33 of the sum."""
    rng = np.random.default_rng(77)
    heads, kv, hd, page, n = 8, 2, 64, 32, 24 if new < 100 else 2
    batch = Batch(rng, [(64, new)] * n, page)
    for pages in batch.pages:
        pages[:2] = batch.pages[0][:2]
    pool = Pool(fmt, kv, hd, page, batch.n_pages)
    eye = np.eye(64, dtype=np.float32)
    for i in range(64):
        pool.put(batch.pages[0][i // page], i % page, np.tile(64 * eye[i], (kv, 1)), np.tile(eye[i], (kv, 1)))
    batch.put(pool, np.zeros((batch.tokens, kv, hd), np.float32), np.zeros((batch.tokens, kv, hd), np.float32))
    q = rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32)
    got, row = attend(hip, pool, batch, heads, q), 0
    size = 8 * np.abs(q).max()
    bound = 2 * size * (2.0 ** -22 + 8 * 2.0 ** -24) + 2.0 ** -22 + (64 + 16) * 2.0 ** -24
    for s in range(n):
        k, v = batch.gather(pool, s)
        want = attention(q[row:row + new], k, v, 64)
        assert (np.abs(got[row:row + new] - want) <= bound * want + 2.0 ** -33).all(), s
        row += new


@pytest.mark.parametrize("fmt,hd", [("i8", 64), ("f16", 128), ("f8", 256)])
@pytest.mark.parametrize("many", ["tokens", "chunks"])
def test_attention_of_many_sequences(hip, fmt, hd, many):
    """More tiles than workgroups run at once: a workgroup has several, and pieces of some."""
    say("attention_paged many", fmt, hd, many)
    rng = np.random.default_rng(14)
    if many == "tokens":
        seqs = [(int(n), 1) for n in rng.integers(0, 40, 260)] + [(1500, 1)]
        pool, batch, heads, q = case_args(rng, fmt, 16, 8, hd, 16, seqs)
    else:
        seqs = [(int(n), 17) for n in rng.integers(0, 60, 66)] + [(900, 20)]
        pool, batch, heads, q = case_args(rng, fmt, 64, 8, hd, 32, seqs)
    check_attention(hip, pool, batch, heads, q)


@pytest.mark.parametrize("seqs", [[], [(0, 0)], [(40, 0), (0, 0), (16, 0)]])
def test_batches_without_tokens(hip, seqs):
    rng = np.random.default_rng(15)
    batch = Batch(rng, seqs, 16)
    pool = Pool("i8", 2, 64, 16, batch.n_pages)
    batch.fill(rng, pool)
    cache, plan, b = hip.buffer_from(pool.bytes), plan_of(hip, pool, batch, 4), hip.buffer_from(np.full(1024, 7.0, np.float32))

    def step():
        hip.kv_store(plan, cache.at(0), b.at(0), 128, b.at(0), 128)
        hip.attention_paged(plan, cache.at(0), b.at(0), 256, b.at(2048), 256)

    run(hip, step)
    assert np.array_equal(hip.read(cache.at(0), np.empty_like(pool.bytes)), pool.bytes)
    assert (hip.read(b.at(0), np.empty(1024, np.float32)) == 7.0).all()


def test_attention_shared_prefix_and_changed_batches(hip):
    """Sequences that share pages, a plan that is given another batch, and batches without tokens."""
    rng = np.random.default_rng(13)
    heads, kv, hd, page = 4, 2, 64, 16
    pool, batch, q = case(rng, "i8", heads, kv, hd, page, [(64, 3), (64, 1), (10, 20)])
    batch.pages[1][:4] = batch.pages[0][:4]
    plan = plan_of(hip, pool, batch, heads)
    check_attention(hip, pool, batch, heads, q, plan=plan)
    other_pool, other, other_q = case(rng, "i8", heads, kv, hd, page, [(333, 1)] * 5)
    plan2 = plan_of(hip, other_pool, other, heads)
    plan2.set([], [], [])
    check_empty(hip, plan2, other_pool, other, heads)
    plan2.set([3, 0], [0, 0], [[1], []])
    check_empty(hip, plan2, other_pool, other, heads)
    plan2.set(other.past, other.new, other.pages)
    check_attention(hip, other_pool, other, heads, other_q, plan=plan2)
    check_attention(hip, pool, batch, heads, q, plan=plan)


def check_empty(hip, plan, pool, batch, heads):
    cache, b = hip.buffer_from(pool.bytes), hip.new_buffer(1 << 16)
    width = heads * pool.hd
    run(hip, lambda: (hip.kv_store(plan, cache.at(0), b.at(0), width, b.at(0), width),
                      hip.attention_paged(plan, cache.at(0), b.at(0), width, b.at(1 << 15), width)))
    assert np.array_equal(hip.read(cache.at(0), np.empty_like(pool.bytes)), pool.bytes)
    assert not hip.read(b.at(0), np.empty(1 << 16, np.uint8)).any()


@pytest.mark.parametrize("new", [1, 50])
def test_attention_far_into_a_large_cache(hip, new):
    """Pages past the first 4 GiB."""
    rng = np.random.default_rng(2)
    heads, kv, hd, page, n_pages = 8, 8, 256, 512, 1100
    small_pool, batch, q = case(rng, "f16", heads, kv, hd, page, [(300, new)])
    plan = hip.kv_plan("f16", kv, hd, page, n_pages, heads)
    size = kv_page_bytes(plan.shape)
    assert size * n_pages > 2 ** 32 + size
    cache = hip.new_buffer(size * n_pages)
    try:
        far = n_pages - 1 - np.arange(len(batch.pages[0]))
        for near, page_no in zip(batch.pages[0], far):
            hip.write(cache.at(int(page_no) * size), small_pool.bytes[near])
        plan.set(batch.past, batch.new, [far.tolist()])
        qb, out = hip.buffer_from(q), hip.new_buffer(q.nbytes)
        run(hip, lambda: hip.attention_paged(plan, cache.at(0), qb.at(0), heads * hd, out.at(0), heads * hd))
        got = hip.read(out.at(0), np.empty_like(q))
        k, v = batch.gather(small_pool, 0)
        assert np.abs(got - attention(q, k, v, 300)).max() <= attention_bound(q, k, v)
        # And the store puts its rows there.
        rows = np.stack([random_rows(rng, kv, hd) for _ in range(new)], 1)
        kb, vb = hip.buffer_from(rows[0]), hip.buffer_from(rows[1])
        run(hip, lambda: hip.kv_store(plan, cache.at(0), kb.at(0), kv * hd, vb.at(0), kv * hd))
        batch.put(small_pool, rows[0], rows[1])
        for near, page_no in zip(batch.pages[0], far):
            assert np.array_equal(hip.read(cache.at(int(page_no) * size), np.empty_like(small_pool.bytes[near])),
                                  small_pool.bytes[near])
    finally:
        cache.free()


@pytest.mark.parametrize("fmt", FORMATS)
def test_store_then_attend_over_steps(hip, fmt):
    """A prompt in two chunks, then single tokens, each step's rows stored before they are attended to."""
    rng = np.random.default_rng(31)
    heads, kv, hd, page = 8, 2, 64, 16
    total = [70, 45]
    pages = [list(range(5)), [9, 8, 7]]
    pool = Pool(fmt, kv, hd, page, 10)
    cache = hip.buffer_from(pool.bytes)
    plan = hip.kv_plan(fmt, kv, hd, page, 10, heads)
    past = [0, 0]
    for new in ([40, 0], [25, 43], [1, 1], [4, 1]):
        batch = Batch(rng, list(zip(past, new)), page)
        batch.pages = [p[:-(-(a + n) // page)] for p, a, n in zip(pages, past, new)]
        rows = np.stack([random_rows(rng, kv, hd) for _ in range(batch.tokens)], 1)
        q = rng.standard_normal((batch.tokens, heads, hd)).astype(np.float32)
        kb, vb, qb, out = (hip.buffer_from(x) for x in (rows[0], rows[1], q, np.empty_like(q)))
        plan.set(past, new, batch.pages)
        run(hip, lambda: (hip.kv_store(plan, cache.at(0), kb.at(0), kv * hd, vb.at(0), kv * hd),
                          hip.attention_paged(plan, cache.at(0), qb.at(0), heads * hd, out.at(0), heads * hd)))
        batch.put(pool, rows[0], rows[1])
        got, row = hip.read(out.at(0), np.empty_like(q)), 0
        for s in range(2):
            if new[s]:
                k, v = batch.gather(pool, s)
                want = attention(q[row:row + new[s]], k, v, past[s])
                assert np.abs(got[row:row + new[s]] - want).max() <= attention_bound(q[row:row + new[s]], k, v)
            row += new[s]
        past = [a + n for a, n in zip(past, new)]
    assert past == total
    assert np.array_equal(hip.read(cache.at(0), np.empty_like(pool.bytes)), pool.bytes)


def test_a_serving_step(hip):
    """Two sequences' step in one recording: rows stored, attended to, projected to logits, ruled and sampled greedily."""
    rng = np.random.default_rng(41)
    heads, kv, hd, page, vocab = 4, 2, 64, 16, 1000
    pool, batch, q = case(rng, "i8", heads, kv, hd, page, [(50, 1), (7, 1)])
    rows = np.stack([random_rows(rng, kv, hd) for _ in range(2)], 1)
    head = (rng.standard_normal((vocab, heads * hd)) / 16).astype(np.float32)
    cache, plan = hip.buffer_from(pool.bytes), plan_of(hip, pool, batch, heads)
    kb, vb, qb, wb = (hip.buffer_from(x) for x in (rows[0], rows[1], q, head))
    out, logits, tokens = hip.new_buffer(q.nbytes), hip.new_buffer(2 * vocab * 4), hip.new_buffer(8)
    state = hip.buffer_from(np.zeros(1, np.uint64))
    batch.put(pool, rows[0], rows[1])
    attended = [attention(q[s:s + 1], *batch.gather(pool, s), batch.past[s]).reshape(-1) for s in range(2)]
    want = np.stack(attended) @ head.astype(np.float64).T
    best = want.argmax(1)
    # The first row's best token is forbidden, the second's is in its history.
    mask = np.full((vocab + 31) // 32, 0xFFFFFFFF, np.uint32)
    mask[best[0] // 32] &= ~np.uint32(1 << int(best[0] % 32))
    table = np.zeros(2, LOGIT_ROW)
    table["mask"], table["repeat"], table["history_len"] = [0, NO_MASK], 1.0, [0, 1]
    table["presence"] = 100.0
    tb, hb, mb = hip.buffer_from(table), hip.buffer_from(best[1:].astype(np.uint32)), hip.buffer_from(mask)

    def step():
        hip.kv_store(plan, cache.at(0), kb.at(0), kv * hd, vb.at(0), kv * hd)
        hip.attention_paged(plan, cache.at(0), qb.at(0), heads * hd, out.at(0), heads * hd)
        for s in range(2):
            hip.matvec(Format.F32, wb.at(0), vocab, heads * hd, out.at(4 * s * heads * hd), logits.at(4 * s * vocab))
        hip.logits_edit(logits.at(0), logits.at(0), 2, vocab, tb.at(0), history=hb.at(0), n_history=1, masks=mb.at(0),
                        n_masks=1)
        for s in range(2):
            hip.sample(logits.at(4 * s * vocab), vocab, hb.at(0), 0, Sampling(0.0, 0, 1.0, 0.0, 1.0), state.at(0),
                       tokens.at(4 * s))

    run(hip, step)
    assert np.array_equal(hip.read(cache.at(0), np.empty_like(pool.bytes)), pool.bytes)
    want[[0, 1], best] = -np.inf
    got = hip.read(tokens.at(0), np.empty(2, np.uint32))
    gap = np.sort(want, axis=1)
    assert (gap[:, -1] - gap[:, -2]).min() > 1e-3  # (the choice is not one of rounding)
    assert got.tolist() == want.argmax(1).tolist()


# --- refusals -------------------------------------------------------------------------

def test_refusals(hip):
    rng = np.random.default_rng(1)
    heads, kv, hd, page = 4, 2, 64, 16
    pool, batch, q = case(rng, "i8", heads, kv, hd, page, [(20, 3)])
    cache, b, plan = hip.buffer_from(pool.bytes), hip.new_buffer(1 << 20), plan_of(hip, pool, batch, heads)
    fresh = hip.kv_plan("i8", kv, hd, page, 4, heads)
    w, o = heads * hd, 1 << 19

    def refused(status, fn):
        hip.begin()
        with pytest.raises(BobcatError) as e:
            fn()
        hip.discard()
        assert e.value.status == STATUS[status], str(e.value)

    refused("Argument", lambda: hip.attention_paged(fresh, cache.at(0), b.at(0), w, b.at(o), w))
    refused("OutOfBounds", lambda: hip.attention_paged(plan, cache.at(16), b.at(0), w, b.at(o), w))
    refused("OutOfBounds", lambda: hip.attention_paged(plan, cache.at(0), b.at((1 << 20) - 64), w, b.at(0), w))
    refused("Argument", lambda: hip.attention_paged(plan, cache.at(0), b.at(4), w, b.at(o), w))
    refused("Argument", lambda: hip.attention_paged(plan, cache.at(0), b.at(0), w - 4, b.at(o), w))
    refused("Argument", lambda: hip.attention_paged(plan, cache.at(0), b.at(0), w + 2, b.at(o), w))
    refused("Argument", lambda: hip.attention_paged(plan, cache.at(0), b.at(0), w, b.at(16), w))
    refused("Argument", lambda: hip.attention_paged(plan, cache.at(0), b.at(0), w, b.at(0), w))
    refused("Argument", lambda: hip.kv_store(plan, cache.at(0), cache.at(0), kv * hd, b.at(0), kv * hd))
    refused("Argument", lambda: hip.kv_store(plan, cache.at(0), b.at(8), kv * hd, b.at(0), kv * hd))
    refused("Argument", lambda: hip.kv_load(plan, cache.at(0), 1, 0, 1, b.at(0), b.at(o)))
    refused("OutOfBounds", lambda: hip.kv_load(plan, cache.at(0), 0, 20, 4, b.at(0), b.at(o)))
    refused("OutOfBounds", lambda: hip.kv_load(plan, cache.at(0), 0, 0xFFFFFFFF, 2, b.at(0), b.at(o)))
    refused("Argument", lambda: hip.kv_load(plan, cache.at(0), 0, 0, 4, b.at(0), b.at(16)))
    with pytest.raises(BobcatError) as e:
        hip.attention_paged(plan, cache.at(0), b.at(0), w, b.at(o), w)
    assert e.value.status == STATUS["NotRecording"]
    # Side by side in one buffer's rows, queries and outputs are apart.
    qo = hip.new_buffer(3 * 2 * w * 4)
    run(hip, lambda: hip.attention_paged(plan, cache.at(0), qo.at(0), 2 * w, qo.at(4 * w), 2 * w))
    run(hip, lambda: hip.attention_paged(plan, cache.at(0), qo.at(4 * w), 2 * w, qo.at(0), 2 * w))


def test_plans_of_other_contexts_and_busy_plans(hip):
    rng = np.random.default_rng(1)
    pool, batch, q = case(rng, "i8", 4, 2, 64, 16, [(20, 3)])
    cache, b, plan = hip.buffer_from(pool.bytes), hip.new_buffer(1 << 16), plan_of(hip, pool, batch, 4)
    other = Hip()
    try:
        foreign = other.kv_plan("i8", 2, 64, 16, pool.n_pages, 4)
        foreign.set(batch.past, batch.new, batch.pages)
        hip.begin()
        with pytest.raises(BobcatError) as e:
            hip.attention_paged(foreign, cache.at(0), b.at(0), 256, b.at(1 << 15), 256)
        assert e.value.status == STATUS["ForeignBuffer"]
        plan.set(batch.past, batch.new, batch.pages)  # nothing that uses it has been recorded
        hip.attention_paged(plan, cache.at(0), b.at(0), 256, b.at(1 << 15), 256)
        with pytest.raises(BobcatError) as e:
            plan.set(batch.past, batch.new, batch.pages)
        assert e.value.status == STATUS["Busy"]
        ticket = hip.commit()
        plan_of(hip, pool, batch, 4)  # another plan is free
        with pytest.raises(BobcatError) as e:
            plan.set(batch.past, batch.new, batch.pages)
        assert e.value.status == STATUS["Busy"]
        hip.wait(ticket)
        # A batch that is refused leaves the one before.
        with pytest.raises(BobcatError):
            plan.set(batch.past, batch.new, [[99] * 2])
        check_attention(hip, pool, batch, 4, q, plan=plan)
        # A discarded recording's launches run on; its plan can be set again.
        hip.begin()
        hip.attention_paged(plan, cache.at(0), b.at(0), 256, b.at(1 << 15), 256)
        hip.discard()
        plan.set(batch.past, batch.new, batch.pages)
        check_attention(hip, pool, batch, 4, q, plan=plan)
    finally:
        other.close()

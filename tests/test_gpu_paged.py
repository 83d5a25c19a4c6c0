"""Paged KV cache, attention over it and reordering, against statements of them in 64 bits.

Tolerances:
* rotated q and k: computed in double and rounded once, so 1 ulp of fp32 (sine and cosine of two libraries); a BF16
  cache rounds that value to nearest: half a step, 2^-8 of it.
* attention: every score and every output is a sum of products in fp32, half an ulp (2^-24 of the largest score, 2^-24
  of the largest output) per term at most: (dim + 32) 2^-23 of the largest output counts the dim roundings of a score
  twice, in the weights and in their sum, and 32 more for scale, exponential, sums and the division.
* everything else moves data: exact.
"""
import math

import numpy as np
import pytest

from quicknn_amd import hip
from tests.conftest import bf16_to_f32, normwise_rel_err

pytestmark = pytest.mark.gpu

F32, BF16 = hip.DT_F32, hip.DT_BF16
THETA = 1e6


def up(ctx, a):
    return ctx.UploadRaw(np.ascontiguousarray(a).view(np.float32).reshape(-1))


def words(ctx, a):
    return up(ctx, np.asarray(a, np.int32))


def tol(dim):
    return (dim + 32) * 2.0 ** -23


def to_bf16(x):
    """Nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


class Store:
    """Pages on the host: values [page][2][kv][page_size][dim] and their packed words."""

    def __init__(self, rng, dtype, pages, page, kv, dim, fill=1.0):
        self.dtype, self.page, self.kv, self.dim, self.count = dtype, page, kv, dim, pages
        x = (fill * rng.standard_normal((pages, 2, kv, page, dim))).astype(np.float32)
        self.x = x if dtype == F32 else bf16_to_f32(to_bf16(x))

    def pack(self):
        x, (n, _, kv, page, dim) = self.x, self.x.shape
        e = 4 if self.dtype == F32 else 8
        k = x[:, 0].reshape(n, kv, page // 16, 16, dim // e, e).transpose(0, 1, 2, 4, 3, 5).reshape(n, 1, kv, page * dim)
        if self.dtype == F32:
            v = x[:, 1].reshape(n, kv, page // 16, 4, 4, dim).transpose(0, 1, 2, 3, 5, 4)
        else:
            v = x[:, 1].reshape(n, kv, page // 32, 2, 4, 4, dim).transpose(0, 1, 2, 4, 6, 3, 5)
        flat = np.concatenate([k, v.reshape(n, 1, kv, page * dim)], 1).reshape(-1)
        return flat if self.dtype == F32 else to_bf16(flat)

    def unpack(self, w):
        n, kv, page, dim = self.count, self.kv, self.page, self.dim
        x = w.view(np.float32) if self.dtype == F32 else bf16_to_f32(w.view(np.uint16))
        x = x.reshape(n, 2, kv, page * dim)
        e = 4 if self.dtype == F32 else 8
        k = x[:, 0].reshape(n, kv, page // 16, dim // e, 16, e).transpose(0, 1, 2, 4, 3, 5).reshape(n, kv, page, dim)
        if self.dtype == F32:
            v = x[:, 1].reshape(n, kv, page // 16, 4, dim, 4).transpose(0, 1, 2, 3, 5, 4)
        else:
            v = x[:, 1].reshape(n, kv, page // 32, 4, dim, 2, 4).transpose(0, 1, 2, 5, 3, 6, 4)
        return np.stack([k, v.reshape(n, kv, page, dim)], 1)

    def put(self, ctx):
        t = up(ctx, self.pack())
        assert t.count == hip.PagedCache.words(self.dtype, self.count, self.page, self.kv, self.dim)
        return hip.PagedCache(t, self.dtype, self.count, self.page, self.kv, self.dim)

    def get(self, ctx, cache):
        return self.unpack(ctx.Download(cache.pages))

    def keys(self, table, n):
        """[2][kv][n][dim] of the first n tokens of a row of page ids."""
        p = -(-n // self.page)
        x = self.x[np.asarray(table[:p], int)].transpose(1, 2, 0, 3, 4).reshape(2, self.kv, p * self.page, self.dim)
        return x[:, :, :n]


class Batch:
    """Sequences with `n` rows and `own` keys each, groups of `share` with `prefix` keys."""

    def __init__(self, rng, page, n, own, prefix=None, share=1, spare_rows=0, extra_pages=1):
        self.n, self.own, self.share, self.page = list(n), list(own), share, page
        self.prefix = [0] * (len(n) // share) if prefix is None else list(prefix)
        self.has_prefix = prefix is not None
        width = max(1, -(-max(own) // page)) + extra_pages
        pwidth = max(1, -(-max(self.prefix) // page))
        self.pages = len(n) * width + len(self.prefix) * pwidth + 2
        ids = rng.permutation(self.pages).astype(np.int32)
        self.tables = ids[:len(n) * width].reshape(len(n), width)
        self.prefix_tables = ids[len(n) * width:len(n) * width + len(self.prefix) * pwidth].reshape(-1, pwidth)
        self.starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + spare_rows

    def put(self, ctx, lengths=None, starts=None, force_starts=False):
        kw = {}
        if self.has_prefix:
            kw = dict(prefix_tables=words(ctx, self.prefix_tables), prefix_lengths=words(ctx, self.prefix),
                      prefix_pages=self.prefix_tables.shape[1])
        plain = starts is None and not force_starts and all(x == 1 for x in self.n) and self.rows == len(self.n)
        return hip.PagedBatch(words(ctx, self.tables), words(ctx, self.own if lengths is None else lengths), len(self.n),
                              self.rows, self.tables.shape[1], share=self.share,
                              starts=None if plain else words(ctx, self.starts if starts is None else starts), **kw)

    def each(self):
        """(sequence, row, own position, absolute position) of every row."""
        for s, n in enumerate(self.n):
            for i in range(n):
                at = self.own[s] - n + i
                yield s, int(self.starts[s]) + i, at, at + self.prefix[s // self.share]


def free(ctx, *things):
    for t in things:
        if isinstance(t, hip.Tensor):
            ctx.Recycle(t)
        elif isinstance(t, hip.PagedCache):
            ctx.Recycle(t.pages)
        elif isinstance(t, hip.PagedBatch):
            for x in (t.tables, t.lengths, t.starts, t.prefix_tables, t.prefix_lengths):
                if x is not None:
                    ctx.Recycle(x)


def rotate(x, at, theta):
    half = x.shape[-1] // 2
    a = at * float(np.float32(theta)) ** (-2.0 * np.arange(half) / (2 * half))
    lo, hi = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), lo * np.sin(a) + hi * np.cos(a)], -1)


def attention(store, batch, q, heads, window=0, softcap=0.0, scale=0.0):
    """Every row in 64 bits; q [rows][heads][dim].  Rows behind the last sequence are NaN."""
    dim, g = store.dim, heads // store.kv
    out = np.full((batch.rows, heads, dim), np.nan)
    mul = scale or 1 / math.sqrt(dim)
    cached = {}
    for s, row, at, absolute in batch.each():
        p = batch.prefix[s // batch.share]
        if s not in cached:
            cached = {s: np.concatenate([store.keys(batch.prefix_tables[s // batch.share], p),
                                         store.keys(batch.tables[s], batch.own[s])], 2).astype(np.float64)}
        low = max(0, absolute - window + 1) if window else 0
        kv = cached[s][:, :, low:max(absolute + 1, low)]
        for h in range(heads):
            if kv.shape[2] == 0:
                out[row, h] = 0
                continue
            with np.errstate(all="ignore"):
                sc = kv[0, h // g] @ q[row, h].astype(np.float64) * mul
                if softcap:
                    sc = softcap * np.tanh(np.clip(sc / softcap, -20, 20))
                w = np.exp(sc - sc.max())
                out[row, h] = w @ kv[1, h // g] / w.sum()
    return out


def run_attention(ctx, store, batch, q, heads, window=0, softcap=0.0, scale=0.0, **put):
    cache, b, tq = store.put(ctx), batch.put(ctx, **put), up(ctx, q)
    dst = up(ctx, np.full(q.size, 7.5, np.float32))
    ctx.PagedAttention(dst, tq, cache, b, heads, window, softcap, scale)
    got = ctx.Download(dst).reshape(batch.rows, heads, store.dim)
    free(ctx, cache, b, tq, dst)
    return got


def check_attention(ctx, rng, dtype, page, kv, heads, dim, batch, window=0, softcap=0.0, scale=0.0, spread=1.0, **put):
    store = Store(rng, dtype, batch.pages, page, kv, dim)
    q = (spread * rng.standard_normal((batch.rows, heads, dim))).astype(np.float32)
    got = run_attention(ctx, store, batch, q, heads, window, softcap, scale, **put)
    want = attention(store, batch, q, heads, window, softcap, scale)
    rows = int(batch.starts[-1])
    assert np.all(got[rows:] == 7.5)  # rows behind the last sequence
    assert np.all(np.isfinite(got[:rows]))
    for s, n in enumerate(batch.n):
        r = slice(int(batch.starts[s]), int(batch.starts[s]) + n)
        if n and np.any(want[r]):
            assert normwise_rel_err(got[r], want[r]) <= tol(dim) * max(1.0, spread), s
        elif n:
            assert not np.any(got[r]), s


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,kv,heads,dim,n,own,prefix,share", [
    (32, 1, 1, 16, [1], [1], None, 1),
    (64, 8, 32, 128, [1, 1, 1], [64, 65, 1], None, 1),
    (64, 2, 6, 80, [5, 0, 70, 1], [5, 9, 200, 33], [17, 0], 2),
    (128, 4, 28, 256, [130, 1], [131, 256], [1000], 2),
    (256, 3, 3, 48, [33, 40], [300, 40], None, 1),
    (32, 2, 2, 64, [97, 64], [100, 64], None, 1)])
def test_append(ctx, rng, dtype, page, kv, heads, dim, n, own, prefix, share):
    batch = Batch(rng, page, n, own, prefix, share, spare_rows=2)
    store = Store(rng, dtype, batch.pages, page, kv, dim)
    q, k, v = (rng.standard_normal((batch.rows, h, dim)).astype(np.float32) for h in (heads, kv, kv))
    for theta in (THETA, 0.0):
        cache, b = store.put(ctx), batch.put(ctx)
        tq, tk, tv = (up(ctx, x) for x in (q, k, v))
        out = up(ctx, np.full(q.size, 7.5, np.float32))
        ctx.PagedAppend(cache, b, tk, tv, tq, out, heads, theta)
        got, gq = store.get(ctx, cache), ctx.Download(out).reshape(q.shape)
        want, wq = store.x.astype(np.float64), np.full(q.shape, 7.5)
        written = np.zeros(want.shape, bool)
        for s, row, at, absolute in batch.each():
            page_id, t = batch.tables[s][at // page], at % page
            wq[row] = rotate(q[row], absolute, theta) if theta else q[row]
            want[page_id, 0, :, t] = rotate(k[row], absolute, theta) if theta else k[row]
            want[page_id, 1, :, t] = v[row]
            written[page_id, :, :, t] = True
        assert np.array_equal(got[~written], store.x[~written])
        assert np.max(np.abs(gq - wq) / np.maximum(np.abs(wq), 1e-3)) <= 2.0 ** -23
        step = 2.0 ** -23 if dtype == F32 else 2.0 ** -8 + 2.0 ** -23
        assert np.all(np.abs(got - want)[written] <= step * np.maximum(np.abs(want[written]), 1e-3))
        # In place, and without q: the same bits.
        cache2 = store.put(ctx)
        ctx.PagedAppend(cache2, b, tk, tv, tq, tq, heads, theta)
        rows = int(batch.starts[-1])
        assert np.array_equal(ctx.Download(tq).reshape(q.shape)[:rows], gq[:rows])
        cache3 = store.put(ctx)
        ctx.PagedAppend(cache3, b, tk, tv, None, None, 0, theta)
        assert np.array_equal(store.get(ctx, cache2), got) and np.array_equal(store.get(ctx, cache3), got)
        free(ctx, cache, cache2, cache3, b, tq, tk, tv, out)


def test_append_equals_the_dense_cache_ops(ctx, rng):
    """One sequence in F32 holds what GO_LLM_ROPE and GO_LLM_CACHE_WRITE make, to the bit."""
    rows, kv, dim, page = 37, 4, 128, 32
    batch = Batch(rng, page, [rows], [rows])
    store = Store(rng, F32, batch.pages, page, kv, dim)
    cache, b = store.put(ctx), batch.put(ctx)
    k, v = (up(ctx, rng.standard_normal(rows * kv * dim).astype(np.float32)) for _ in range(2))
    turned, dense = ctx.NewTensor(k.count), ctx.NewTensor(2 * rows * kv * dim)
    ctx.Kernel(hip.GO_LLM_ROPE, k.count // 2, turned, k, None, None, [kv, dim, 0, hip.float_bits(THETA)])
    ctx.Kernel(hip.GO_LLM_CACHE_WRITE, k.count, dense, turned, v, None, [rows, kv, dim, rows, 0])
    ctx.PagedAppend(cache, b, k, v, theta=THETA)
    got = Store(rng, F32, batch.pages, page, kv, dim)
    got.x = store.get(ctx, cache)
    got = got.keys(batch.tables[0], rows)
    d = ctx.Download(dense)
    assert np.array_equal(got[0], d[:kv * dim * rows].reshape(kv, dim, rows).transpose(0, 2, 1))
    assert np.array_equal(got[1], d[kv * dim * rows:].reshape(kv, rows, dim))
    free(ctx, cache, b, k, v, turned, dense)


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,kv,heads,dim,own", [
    (32, 1, 1, 16, [1]), (64, 8, 32, 128, [4001]), (64, 2, 2, 64, [31, 32, 33, 63, 64, 65, 1]),
    (128, 4, 28, 128, [1000, 17]), (256, 1, 8, 256, [700]), (32, 3, 15, 80, [95, 96, 97]), (64, 1, 40, 96, [130, 5]),
    (64, 2, 2, 240, [333]), (32, 1, 71, 32, [40]), (64, 8, 64, 128, [2, 3000, 1, 513])])
def test_attention_of_single_tokens(ctx, rng, dtype, page, kv, heads, dim, own):
    check_attention(ctx, rng, dtype, page, kv, heads, dim, Batch(rng, page, [1] * len(own), own))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,kv,heads,dim,n,own,window,softcap", [
    (32, 1, 1, 16, [2], [2], 0, 0.0),
    (64, 2, 8, 128, [130, 1, 0, 9], [130, 700, 4, 100], 0, 0.0),
    (64, 2, 14, 64, [40, 3], [200, 3], 50, 0.0),
    (32, 4, 8, 256, [65, 70], [65, 300], 33, 20.0),
    (128, 1, 5, 80, [300], [301], 1, 0.0),
    (64, 2, 4, 112, [20, 100], [1000, 100], 0, 5.0),
    (32, 1, 3, 144, [77], [500], 0, 0.0), (64, 2, 12, 208, [33, 1, 12], [64, 3, 70], 40, 0.0),
    (128, 1, 16, 240, [9, 30], [300, 30], 0, 9.0), (64, 1, 6, 176, [25], [129], 0, 0.0)])
def test_attention_of_prompts(ctx, rng, dtype, page, kv, heads, dim, n, own, window, softcap):
    check_attention(ctx, rng, dtype, page, kv, heads, dim, Batch(rng, page, n, own, spare_rows=3), window, softcap)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,kv,heads,dim,n,own,prefix,share,window,softcap", [
    (64, 2, 8, 128, [1] * 8, [20, 1, 64, 65, 200, 3, 4, 5], [500, 0], 4, 0, 0.0),
    (32, 1, 4, 64, [1] * 6, [7] * 6, [1], 6, 0, 0.0),
    (64, 8, 32, 128, [1] * 16, list(range(1, 17)), [1000, 37], 8, 0, 0.0),
    (64, 2, 14, 80, [3, 0, 40, 1], [10, 2, 41, 9], [333, 64], 2, 0, 30.0),
    (128, 1, 8, 256, [1, 1, 1], [30, 40, 50], [700], 3, 45, 0.0),
    (32, 2, 6, 48, [9, 1], [9, 1], [100, 200], 1, 60, 0.0),
    (64, 1, 7, 128, [2] * 24, [2] * 24, [129], 24, 0, 0.0)])
def test_attention_with_a_shared_prefix(ctx, rng, dtype, page, kv, heads, dim, n, own, prefix, share, window, softcap):
    check_attention(ctx, rng, dtype, page, kv, heads, dim, Batch(rng, page, n, own, prefix, share, spare_rows=1), window,
                    softcap)


@pytest.mark.parametrize("count", [64, 65, 100, 300])
def test_attention_of_many_sequences(ctx, rng, count):
    """More sequences than a wave has lanes, and than a workgroup has threads; empty and idle ones among them."""
    own = [int(x) for x in rng.integers(0, 90, count)]
    check_attention(ctx, rng, BF16, 32, 2, 8, 32, Batch(rng, 32, [1] * count, own))
    n = [min(o, int(x)) for o, x in zip(own, rng.integers(0, 12, count))]
    check_attention(ctx, rng, BF16, 32, 2, 10, 32, Batch(rng, 32, n, own, spare_rows=5), window=20)
    if count % 20 == 0:
        check_attention(ctx, rng, F32, 32, 1, 4, 32, Batch(rng, 32, n, own, [int(x) for x in rng.integers(0, 99, count // 20)],
                                                           20))


def test_attention_of_thousands_of_sequences(ctx, rng):
    """5000 sequences over a few pages that they share (single tokens, and ragged rows behind a prefix)."""
    count, page, kv, heads, dim = 5000, 32, 1, 2, 16
    store = Store(rng, BF16, 40, page, kv, dim)
    for n, prefix in ((np.ones(count, int), None), (rng.integers(0, 3, count), [50])):
        batch = Batch.__new__(Batch)
        batch.n, batch.own, batch.share, batch.page = n.tolist(), rng.integers(2, 60, count).tolist(), 1, page
        batch.tables = rng.integers(0, 40, (count, 2)).astype(np.int32)
        batch.has_prefix, batch.share = prefix is not None, count if prefix else 1
        batch.prefix = prefix or [0] * count
        batch.prefix_tables = rng.integers(0, 40, (len(batch.prefix), 2)).astype(np.int32)
        batch.starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        batch.rows = int(batch.starts[-1])
        q = rng.standard_normal((batch.rows, heads, dim)).astype(np.float32)
        got, want = run_attention(ctx, store, batch, q, heads), attention(store, batch, q, heads)
        assert np.max(np.abs(got - want)) <= tol(dim) * np.max(np.abs(want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_rows_without_keys(ctx, rng, dtype):
    """Rows in front of all own keys: zeros without a prefix, the prefix up to their position with one."""
    check_attention(ctx, rng, dtype, 64, 2, 4, 64, Batch(rng, 64, [1, 1, 3], [0, 5, 1]))
    check_attention(ctx, rng, dtype, 64, 2, 4, 64, Batch(rng, 64, [1, 2, 1, 1], [0, 0, 70, 0], [100, 0], 2))
    check_attention(ctx, rng, dtype, 64, 2, 4, 64, Batch(rng, 64, [40, 40], [0, 3], [20], 2))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_scale_and_large_scores(ctx, rng, dtype):
    """Scores in the hundreds (their roundings grow with them) and an explicit scale."""
    check_attention(ctx, rng, dtype, 64, 2, 8, 128, Batch(rng, 64, [1, 1], [700, 90]), scale=0.31, spread=8.0)
    check_attention(ctx, rng, dtype, 64, 2, 8, 128, Batch(rng, 64, [50], [300]), scale=0.31, spread=8.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,share,prefix", [([1, 1], 1, None), ([40, 3], 1, None), ([1] * 24, 24, [200])])
def test_hidden_keys_reach_nothing(ctx, rng, dtype, n, share, prefix):
    """Infinities and NaN behind a sequence's last key, in keys of later rows, outside the window and in other pages
    leave a row's result as it is."""
    page, kv, heads, dim, window = 64, 2, 8, 128, 30
    own = [90 + i for i in range(len(n))]
    batch = Batch(rng, page, n, own, prefix, share)
    store = Store(rng, dtype, batch.pages, page, kv, dim)
    q = rng.standard_normal((batch.rows, heads, dim)).astype(np.float32)
    clean = run_attention(ctx, store, batch, q, heads, window)
    used = np.zeros(store.x.shape[0] * page, bool)
    for s, row, at, absolute in batch.each():
        for t in range(max(0, absolute - window + 1), absolute + 1):
            p = batch.prefix[s // share]
            table, o = (batch.prefix_tables[s // share], t) if t < p else (batch.tables[s], t - p)
            used[table[o // page] * page + o % page] = True
    hidden = ~used.reshape(-1, page)
    for bad in (np.nan, np.inf, -np.inf):
        x = store.x.copy()
        x.transpose(0, 3, 1, 2, 4)[hidden] = bad
        dirty = Store(rng, dtype, batch.pages, page, kv, dim)
        dirty.x = x
        differ = int(np.sum(run_attention(ctx, dirty, batch, q, heads, window) != clean))
        assert differ == 0, bad
    # A key that only the last rows see reaches those alone.
    if n[0] > 1:
        x = store.x.copy()
        t = own[0] - 5
        x[batch.tables[0][t // page], :, :, t % page, 3] = np.nan
        dirty = Store(rng, dtype, batch.pages, page, kv, dim)
        dirty.x = x
        got = run_attention(ctx, dirty, batch, q, heads, 0)
        plain = run_attention(ctx, store, batch, q, heads, 0)
        first = n[0] - 5
        assert np.all(np.isnan(got[first:n[0]]).any(-1)) and not np.any(np.isnan(got[:first]))
        want = attention(store, batch, q, heads, 0)
        assert normwise_rel_err(got[:first], want[:first]) <= tol(dim)
        assert np.array_equal(got[n[0]:], plain[n[0]:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,own,prefix,share", [([1, 1], [90, 40], None, 1), ([40], [70], None, 1), ([1] * 20, [9] * 20,
                                                                                                    [300], 20)])
def test_visible_infinities(ctx, rng, dtype, n, own, prefix, share):
    """An infinite or NaN key, value or query gives what the formula gives in 64 bits."""
    page, kv, heads, dim = 64, 2, 4, 64
    batch = Batch(rng, page, n, own, prefix, share)
    for what, bad in (("v", np.inf), ("v", -np.inf), ("v", np.nan), ("k", np.nan), ("q", np.nan), ("k", np.inf),
                      ("k", -np.inf)):
        store = Store(rng, dtype, batch.pages, page, kv, dim)
        q = rng.standard_normal((batch.rows, heads, dim)).astype(np.float32)
        t = 3
        place = (batch.prefix_tables if prefix else batch.tables)[0][t // page], 0 if what == "k" else 1, 1, t % page, 5
        if what == "q":
            q[0, 1, 2] = bad
        else:
            store.x[place] = bad
        got = run_attention(ctx, store, batch, q, heads)
        want = attention(store, batch, q, heads)
        nans, infs, finite = np.isnan(want), np.isinf(want), np.isfinite(want)
        same = int(np.sum(np.isnan(got) != nans)), int(np.sum(got[infs] != want[infs]))
        assert same == (0, 0), (what, bad)
        assert np.max(np.abs(got[finite] - want[finite])) <= tol(dim) * np.max(np.abs(want[finite])), (what, bad)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,own,prefix,share", [([1, 1], [90, 40], None, 1), ([1], [3000], None, 1), ([40], [70], None, 1),
                                                ([1] * 20, [9] * 20, [300], 20)])
def test_scores_that_are_all_minus_infinity(ctx, rng, dtype, n, own, prefix, share):
    """Zeros; with one finite score, that key's value."""
    page, kv, heads, dim = 64, 2, 4, 64
    batch = Batch(rng, page, n, own, prefix, share)
    store = Store(rng, dtype, batch.pages, page, kv, dim)
    store.x[:, 0, :, :, 5] = -np.inf
    q = np.abs(rng.standard_normal((batch.rows, heads, dim))).astype(np.float32)
    assert not np.any(run_attention(ctx, store, batch, q, heads))
    table = (batch.prefix_tables if prefix else batch.tables)[0]
    store.x[table[0], 0, 1, 3, 5] = 1.0
    want = np.zeros_like(q)
    rows = batch.rows if prefix else n[0]
    at = own[0] - n[0] + np.arange(rows)
    seen = np.arange(rows) if prefix else np.arange(rows)[at >= 3]
    want[seen, heads // 2:] = store.x[table[0], 1, 1, 3]
    assert np.array_equal(run_attention(ctx, store, batch, q, heads), want)


def test_attention_repeats_and_ignores_the_batch(ctx, rng):
    """The same call gives the same bits; so do explicit row starts for one row per sequence."""
    batch = Batch(rng, 64, [1] * 5, [700, 3, 64, 1000, 129])
    store = Store(rng, BF16, batch.pages, 64, 8, 128)
    q = rng.standard_normal((batch.rows, 32, 128)).astype(np.float32)
    a = run_attention(ctx, store, batch, q, 32)
    assert np.array_equal(a, run_attention(ctx, store, batch, q, 32))
    assert np.array_equal(a, run_attention(ctx, store, batch, q, 32, force_starts=True))


def test_attention_of_a_large_group_with_a_window(ctx, rng):
    """A window over a prefix that many sequences share hides keys; it shall not cost a look at the whole group for every
    row and head.  At 2000 sequences that was more than twenty times the time without a window."""
    count, page, kv, heads, dim = 2000, 32, 2, 8, 64
    n = [int(x) for x in rng.integers(0, 3, count)]
    store = Store(rng, BF16, 60, page, kv, dim)
    batch = Batch.__new__(Batch)
    batch.n, batch.own, batch.share, batch.page = n, [x + int(y) for x, y in zip(n, rng.integers(0, 50, count))], count, page
    batch.tables, batch.prefix_tables = (rng.integers(0, 60, s).astype(np.int32) for s in ((count, 2), (1, 20)))
    batch.has_prefix, batch.prefix = True, [600]
    batch.starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    batch.rows = int(batch.starts[-1])
    q = rng.standard_normal((batch.rows, heads, dim)).astype(np.float32)
    cache, b, tq, dst, times = store.put(ctx), batch.put(ctx), up(ctx, q), ctx.NewTensor(q.size), {}
    for window in (0, 300):
        want, took = attention(store, batch, q, heads, window), []
        for _ in range(6):
            ctx.EventRecord(0)
            ctx.PagedAttention(dst, tq, cache, b, heads, window)
            ctx.EventRecord(1)
            ctx.Flush()
            took.append(ctx.EventElapsedMs(0, 1))
        times[window] = min(took)
        assert np.max(np.abs(ctx.Download(dst).reshape(q.shape) - want)) <= tol(dim) * np.max(np.abs(want))
    assert times[300] <= 4 * times[0], times
    free(ctx, cache, b, tq, dst)


@pytest.mark.parametrize("n,own,prefix,share", [([1] * 5, [700, 3, 64, 1000, 129], None, 1),
                                                ([40, 1, 9], [200, 50, 9], None, 1),
                                                ([1] * 6, [20, 90, 7, 33, 8, 64], [300, 41], 3)])
def test_attention_of_a_sequence_among_others(ctx, rng, n, own, prefix, share):
    """What the other sequences' keys, values and queries are makes no difference to a sequence, to the bit."""
    page, kv, heads, dim = 64, 2, 8, 128
    batch = Batch(rng, page, n, own, prefix, share)
    store, other = (Store(rng, BF16, batch.pages, page, kv, dim) for _ in range(2))
    q, q2 = (rng.standard_normal((batch.rows, heads, dim)).astype(np.float32) for _ in range(2))
    mine = np.concatenate([batch.tables[0]] + ([batch.prefix_tables[0]] if prefix else []))
    other.x[mine] = store.x[mine]
    q2[:n[0]] = q[:n[0]]
    a, b = run_attention(ctx, store, batch, q, heads), run_attention(ctx, other, batch, q2, heads)
    assert np.array_equal(a[:n[0]], b[:n[0]]) and not np.any(np.all(a[n[0]:] == b[n[0]:], axis=(1, 2)))


def test_attention_in_a_cache_past_32_bit_offsets(ctx, rng):
    """Pages whose byte offsets pass 2^32 (a tensor holds up to 2^31 words)."""
    page, kv, heads, dim = 256, 8, 16, 256
    pages = 4000  # 8.4 GB of BF16
    batch = Batch(rng, page, [1, 70], [300, 270])
    small = Store(rng, BF16, batch.pages, page, kv, dim)
    q, k, v = (rng.standard_normal((batch.rows, h, dim)).astype(np.float32) for h in (heads, kv, kv))
    want = run_attention(ctx, small, batch, q, heads)
    big = hip.PagedCache(ctx.NewTensor(hip.PagedCache.words(BF16, pages, page, kv, dim)), BF16, pages, page, kv, dim)
    old, packed = batch.tables, up(ctx, small.pack())
    per = packed.count // batch.pages
    batch.tables = (pages - batch.pages + old).astype(np.int32)
    assert (pages - batch.pages) * per * 4 > 2 ** 32
    ctx.Copy(big.pages, packed, packed.count, (pages - batch.pages) * per)
    b, tq, dst, tk, tv = batch.put(ctx), up(ctx, q), ctx.NewTensor(q.size), up(ctx, k), up(ctx, v)
    ctx.PagedAttention(dst, tq, big, b, heads)
    assert np.array_equal(ctx.Download(dst).reshape(q.shape), want)
    ctx.PagedAppend(big, b, tk, tv, theta=THETA)
    ctx.Copy(packed, big.pages, packed.count, 0, (pages - batch.pages) * per)
    got = small.unpack(ctx.Download(packed))
    batch.tables = old
    cache, b2 = small.put(ctx), batch.put(ctx)
    ctx.PagedAppend(cache, b2, tk, tv, theta=THETA)
    assert np.array_equal(got, small.get(ctx, cache))
    free(ctx, big, b, b2, cache, tq, dst, tk, tv, packed)


# ---------------------------------------------------------------- advance, gather
def test_advance(ctx, rng):
    batch = Batch(rng, 64, [3, 0, 1], [3, 9, 64])
    b = batch.put(ctx)
    ctx.PagedAdvance(b, 64)
    ctx.PagedAdvance(b, 64)
    assert ctx.Download(b.lengths, dtype=np.int32).tolist() == [9, 9, 66]
    one = Batch(rng, 32, [1] * 300, list(range(300)))
    b1 = one.put(ctx)
    ctx.PagedAdvance(b1, 32)
    assert ctx.Download(b1.lengths, dtype=np.int32).tolist() == list(range(1, 301))
    free(ctx, b, b1)


@pytest.mark.parametrize("rows,cols,src_rows", [(1, 1, 1), (7, 5, 3), (64, 1000, 64), (3, 70001, 5)])
def test_gather_rows(ctx, rng, rows, cols, src_rows):
    src = rng.integers(0, 1 << 31, (src_rows, cols), dtype=np.int32)
    idx = rng.integers(0, src_rows, rows, dtype=np.int32)
    t, i, dst = words(ctx, src), words(ctx, idx), ctx.NewTensor(rows * cols)
    ctx.GatherRows(dst, t, i, rows, cols)
    assert np.array_equal(ctx.Download(dst, dtype=np.int32).reshape(rows, cols), src[idx])
    free(ctx, t, i, dst)


def test_gather_of_more_rows_than_workgroups(ctx, rng):
    rows = (1 << 24) + 5
    src, idx = rng.integers(0, 1 << 31, 1000, dtype=np.int32), rng.integers(0, 1000, rows, dtype=np.int32)
    t, i, dst = words(ctx, src), words(ctx, idx), ctx.NewTensor(rows)
    ctx.GatherRows(dst, t, i, rows, 1)
    assert np.array_equal(ctx.Download(dst, dtype=np.int32), src[idx])
    free(ctx, t, i, dst)


def test_gather_of_a_row_that_fills_a_tensor(ctx, rng):
    """One row of nearly 2^31 words, the most that a tensor holds: copied to its end, and nothing behind it."""
    pattern = rng.integers(0, 1 << 31, (7, 1000), dtype=np.int32)
    rows = (2 ** 31 - 1) // 1000
    kinds = (np.arange(rows) * 5 // 3 % 7).astype(np.int32)
    t, i, src, dst = words(ctx, pattern), words(ctx, kinds), ctx.NewTensor(2 ** 31 - 1), ctx.NewTensor(2 ** 31 - 1)
    ctx.GatherRows(src, t, i, rows, 1000)  # 2147483 rows
    zero, tail = words(ctx, np.zeros(647, np.int32)), ctx.NewTensor(647)
    ctx.Copy(dst, zero, 647, rows * 1000)
    only = words(ctx, [0])
    for width in ((rows - 1) * 1000, rows * 1000):  # less than a step of the loop, and of a workgroup, below 2^31
        ctx.GatherRows(dst, src, only, 1, width, 1)
    look = np.array([0, 1, 16383, rows // 2, rows - 17, rows - 2, rows - 1], np.int32)
    at, out = words(ctx, look), ctx.NewTensor(look.size * 1000)
    ctx.GatherRows(out, dst, at, look.size, 1000)
    assert np.array_equal(ctx.Download(out, dtype=np.int32).reshape(-1, 1000), pattern[kinds[look]])
    ctx.Copy(tail, dst, 647, 0, rows * 1000)
    assert not np.any(ctx.Download(tail, dtype=np.int32))
    free(ctx, t, i, src, dst, zero, tail, only, at, out)


# ---------------------------------------------------------------- reorder
def reorder_plan(tables, length, parents, share, page):
    """New tables and (from page, to page) copies, by the documented rule."""
    full, rest = divmod(length, page)
    new, copies = tables.copy(), []
    for g in range(0, len(tables), share):
        p = [x - g for x in parents[g:g + share]]
        spare = [i for i in range(share) if i not in p]
        for i in range(share):
            new[g + i, :full] = tables[g + p[i], :full]
            if rest:
                if p[i] in p[:i]:
                    take = spare.pop(0)
                    copies.append((tables[g + p[i], full], tables[g + take, full]))
                else:
                    take = p[i]
                new[g + i, full] = tables[g + take, full]
    return new, copies


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page,kv,dim,share,groups,length,layers", [
    (64, 2, 64, 4, 1, 41, 1), (32, 1, 16, 1, 3, 5, 2), (64, 8, 128, 8, 4, 200, 3), (32, 2, 80, 5, 2, 96, 2),
    (128, 1, 48, 64, 2, 130, 1), (64, 1, 32, 2, 1, 0, 1), (32, 1, 16, 3, 2, 33, 100), (32, 1, 16, 1, 3, 40, 1)])
def test_reorder(ctx, rng, dtype, page, kv, dim, share, groups, length, layers):
    n = share * groups
    batch = Batch(rng, page, [1] * n, [length] * n, share=share)
    stores = [Store(rng, dtype, batch.pages, page, kv, dim) for _ in range(layers)]
    caches, b = [s.put(ctx) for s in stores], batch.put(ctx)
    for kind in ("random", "one", "same"):
        parents = {"random": [g * share + int(x) for g in range(groups) for x in rng.integers(0, share, share)],
                   "one": [g * share + share - 1 for g in range(groups) for _ in range(share)],
                   "same": list(range(n))}[kind]
        new, copies = reorder_plan(batch.tables, length, parents, share, page)
        tp, tn = words(ctx, parents), ctx.NewTensor(batch.tables.size)
        for _ in range(2):  # again: the same
            ctx.PagedReorder(b, tn, tp, caches)
            assert np.array_equal(ctx.Download(tn, dtype=np.int32).reshape(new.shape), new)
        used = -(-(length % page) // 32) * 32
        for s, c in zip(stores, caches):
            want = s.x.copy()
            for a, z in copies:
                want[z, :, :, :used] = s.x[a, :, :, :used]
            for i in range(n):  # every sequence holds its parent's keys
                a, z = Store.__new__(Store), Store.__new__(Store)
                a.__dict__.update(s.__dict__)
                z.__dict__.update(s.__dict__, x=want)
                assert np.array_equal(z.keys(new[i], length), a.keys(batch.tables[parents[i]], length))
            assert np.array_equal(s.get(ctx, c), want)
            s.x = want
        partial = new[:, length // page]
        assert len(set(partial.tolist())) == n  # what is written next belongs to one sequence
        free(ctx, tp, tn)
    free(ctx, b, *caches)


# ---------------------------------------------------------------- refusals
def test_refusals(ctx, rng):
    batch = Batch(rng, 64, [1] * 4, [70] * 4, [30, 40], 2)
    store = Store(rng, BF16, batch.pages, 64, 2, 64)
    c, b = store.put(ctx), batch.put(ctx)
    q, k, v, out, big = (ctx.NewTensor(n) for n in (4 * 4 * 64, 4 * 2 * 64, 4 * 2 * 64, 4 * 4 * 64, 1 << 16))
    tables, parents = ctx.NewTensor(batch.tables.size), ctx.NewTensor(4)

    def cache(**kw):
        a = dict(pages=c.pages, dtype=BF16, page_count=batch.pages, page_size=64, kv_heads=2, dim=64)
        return hip.PagedCache(**{**a, **kw})

    def bat(**kw):
        a = dict(tables=b.tables, lengths=b.lengths, sequences=4, rows=4, table_pages=b.table_pages,
                 prefix_tables=b.prefix_tables, prefix_lengths=b.prefix_lengths, prefix_pages=b.prefix_pages, share=2)
        return hip.PagedBatch(**{**a, **kw})

    def att(cc=c, bb=b, **kw):
        a = dict(dst=out, q=q, heads=4, window=0, softcap=0.0, scale=0.0)
        a.update(kw)
        ctx.PagedAttention(a["dst"], a["q"], cc, bb, a["heads"], a["window"], a["softcap"], a["scale"])

    def app(cc=c, bb=b, **kw):
        a = dict(k=k, v=v, q=q, q_out=out, heads=4, theta=1e4)
        a.update(kw)
        ctx.PagedAppend(cc, bb, a["k"], a["v"], a["q"], a["q_out"], a["heads"], a["theta"])

    att(), app()
    small = ctx.NewTensor(3)
    gone = hip.Tensor(ctx, ctx.NewTensor(4096).handle)
    ctx.Recycle(gone)
    for kw, err in ((dict(dtype=hip.DT_F16), hip.ENotSupportedException), (dict(page_size=16), hip.ENotSupportedException),
                    (dict(page_size=96), hip.ENotSupportedException), (dict(dim=40), hip.ENotSupportedException),
                    (dict(dim=272), hip.ENotSupportedException), (dict(dim=0), hip.ENotSupportedException),
                    (dict(kv_heads=0), hip.EArgumentException), (dict(page_count=0), hip.EArgumentException),
                    (dict(page_count=batch.pages + 1), hip.EArgumentException),
                    (dict(page_count=1 << 30), hip.ERangeError), (dict(pages=None), hip.EArgumentException),
                    (dict(pages=gone), hip.EArgumentException)):
        for f in (att, app):
            with pytest.raises(err):
                f(cc=cache(**kw))
        with pytest.raises(err):
            ctx.PagedReorder(b, tables, parents, [c, cache(**kw)] if err is hip.EArgumentException else [cache(**kw)])
    for kw in (dict(sequences=0), dict(sequences=5, rows=5), dict(rows=0), dict(rows=3), dict(rows=65536), dict(share=0),
               dict(share=3), dict(table_pages=0), dict(table_pages=b.table_pages + 1), dict(table_pages=1 << 25),
               dict(prefix_tables=None), dict(prefix_lengths=None), dict(prefix_pages=0), dict(prefix_pages=1000),
               dict(tables=None), dict(lengths=None), dict(lengths=small), dict(starts=small)):
        for f in (att, app):
            with pytest.raises(hip.EArgumentException):
                f(bb=bat(**kw))
        with pytest.raises(hip.EArgumentException):
            ctx.PagedReorder(bat(**kw), tables, parents, [c])
        with pytest.raises(hip.EArgumentException):
            ctx.PagedAdvance(bat(**kw), 64)
    for kw in (dict(heads=3), dict(heads=0), dict(heads=8), dict(window=-1), dict(softcap=-1.0), dict(softcap=math.nan),
               dict(softcap=math.inf), dict(scale=-1.0), dict(scale=math.nan), dict(dst=q), dict(dst=c.pages), dict(q=small),
               dict(dst=small), dict(dst=None), dict(q=None)):
        with pytest.raises(hip.EArgumentException):
            att(**kw)
    for kw in (dict(k=small), dict(v=None), dict(q=None), dict(q_out=None), dict(heads=0), dict(heads=8), dict(theta=-1.0),
               dict(theta=math.nan), dict(theta=math.inf), dict(q_out=k), dict(q_out=c.pages), dict(k=c.pages)):
        with pytest.raises(hip.EArgumentException):
            app(**kw)
    with pytest.raises(hip.ERangeError):  # 4000 sequences with room for 2^20 keys each, 3 KV heads
        ctx.PagedAttention(ctx.Scratch(2, 4000 * 48), ctx.Scratch(0, 4000 * 48), hip.PagedCache(c.pages, BF16, 1, 32, 3, 16),
                           hip.PagedBatch(ctx.Scratch(1, 1 << 27), big, 4000, 4000, 32000), 3)
    wide = hip.PagedBatch(big, big, 65, 65, 1, share=65)
    with pytest.raises(hip.ENotSupportedException):
        ctx.PagedReorder(wide, big, big, [c])
    for a in ((b, tables, parents, []), (b, b.tables, parents, [c]), (b, small, parents, [c]), (b, tables, small, [c]),
              (b, tables, tables, [c]), (b, tables, parents, [c, c])):
        with pytest.raises(hip.EArgumentException):
            ctx.PagedReorder(*a)
    with pytest.raises(hip.ENotSupportedException):
        ctx.PagedAdvance(b, 100)
    for a in ((out, q, parents, 0, 4), (out, q, parents, 4, 0), (q, q, parents, 4, 4), (out, q, small, 4, 4),
              (small, q, parents, 4, 4), (out, q, parents, 4, 4, 1000)):
        with pytest.raises(hip.EArgumentException):
            ctx.GatherRows(*a)
    ctx.Flush()
    free(ctx, c, b, q, k, v, out, big, tables, parents, small)


def test_bad_device_data_is_reported(ctx, rng):
    """Lengths, starts, page ids, parents and indices outside their range: no access out of range, an error at the next
    Download, and the context goes on."""
    page, kv, heads, dim = 64, 2, 4, 64
    batch = Batch(rng, page, [1, 70], [70, 80], [30, 40], 1)
    store = Store(rng, BF16, batch.pages, page, kv, dim)
    q, k, v = (up(ctx, rng.standard_normal(batch.rows * h * dim).astype(np.float32)) for h in (heads, kv, kv))
    out = ctx.NewTensor(q.count)
    good = (batch.tables.copy(), batch.prefix_tables.copy(), list(batch.prefix))
    for bad in ("page", "negative page", "huge page", "length", "negative length", "prefix", "prefix page", "starts past",
                "starts falling", "starts negative"):
        batch.tables, batch.prefix_tables, batch.prefix = good[0].copy(), good[1].copy(), list(good[2])
        lengths, starts = list(batch.own), batch.starts.copy()
        if bad.endswith("page") and bad != "prefix page":
            batch.tables[1, 1] = {"page": batch.pages, "negative page": -1, "huge page": 0x7FFFFFFF}[bad]
        elif bad.endswith("length"):
            lengths[1] = 100000 if bad == "length" else -5
        elif bad == "prefix":
            batch.prefix[1] = 1 << 30
        elif bad == "prefix page":
            batch.prefix_tables[0, 0] = -7
        else:
            starts = np.array({"starts past": [0, 1, 1 << 30], "starts falling": [0, 71, 3],
                               "starts negative": [-9, 1, 71]}[bad], np.int32)
        cache, b = store.put(ctx), batch.put(ctx, lengths=lengths, starts=starts)
        ctx.PagedAttention(out, q, cache, b, heads)
        with pytest.raises(hip.EInvalidOp, match="outside its range"):
            ctx.Download(out)
        if not bad.startswith("prefix p"):
            ctx.PagedAppend(cache, b, k, v, q, out, heads, THETA)
            with pytest.raises(hip.EInvalidOp, match="outside its range"):
                ctx.Download(out)
        ctx.Download(out)  # reported once
        free(ctx, cache, b)
    batch.tables, batch.prefix_tables, batch.prefix = good
    # Groups whose row starts do not ascend: rows in front of their group's first.
    four = Batch(rng, page, [20, 15, 30, 6], [70, 80, 40, 9], [30, 40], 2)
    other = Store(rng, BF16, four.pages, page, kv, dim)
    cache, q4 = other.put(ctx), up(ctx, rng.standard_normal(four.rows * heads * dim).astype(np.float32))
    out4 = ctx.NewTensor(q4.count)
    for starts in ([0, 50, 20, 71, 10], [71, 0, 71, 0, 71], [60, 71, 0, 30, 71]):
        b = four.put(ctx, starts=np.array(starts, np.int32))
        ctx.PagedAttention(out4, q4, cache, b, heads)
        with pytest.raises(hip.EInvalidOp, match="outside its range"):
            ctx.Download(out4)
        free(ctx, b)
    free(ctx, cache, q4, out4)
    cache, b = store.put(ctx), batch.put(ctx)
    few = batch.put(ctx, lengths=[0, 80])  # more rows than keys to append
    ctx.PagedAppend(cache, few, k, v)
    with pytest.raises(hip.EInvalidOp, match="outside its range"):
        ctx.Download(out)
    free(ctx, few)
    full = batch.put(ctx, lengths=[batch.tables.shape[1] * page, 1])
    ctx.PagedAdvance(full, page)
    with pytest.raises(hip.EInvalidOp, match="outside its range"):
        ctx.Download(out)
    free(ctx, full, b)
    beams = Batch(rng, page, [1] * 4, [70] * 4, share=2)
    wide = Store(rng, BF16, beams.pages, page, kv, dim)
    c2, new = wide.put(ctx), ctx.NewTensor(beams.tables.size)
    for parents, lengths in (([0, 2, 2, 3], None), ([0, -1, 2, 3], None), ([0, 0, 2, 2], [70, 71, 70, 70])):
        b2, tp = beams.put(ctx, lengths=lengths), words(ctx, parents)
        ctx.PagedReorder(b2, new, tp, [c2])
        with pytest.raises(hip.EInvalidOp, match="outside its range"):
            ctx.Download(new)
        free(ctx, b2, tp)
    src, idx, dst = words(ctx, range(12)), words(ctx, [0, 3, -1]), ctx.NewTensor(12)
    ctx.GatherRows(dst, src, idx, 3, 4, 3)
    with pytest.raises(hip.EInvalidOp, match="outside its range"):
        ctx.Download(dst)
    assert ctx.Download(dst, dtype=np.int32).tolist() == [0, 1, 2, 3] + [0] * 8
    free(ctx, cache, c2, new, src, idx, dst, q, k, v, out)


@pytest.mark.parametrize("starts,own,prefix", [
    ([0, 100, 5, 200], [256, 256, 256], None),  # groups of 32 tokens: the second sequence is behind no row and no group
    ([0, 64, 0, 128], [256, 256, 256], None),
    ([0, 3, 1, 4], [9, 9, 9], None),  # workgroups per row
    ([0, 2, 2, 1, 2], [9, 9, 9, 9], None),
    ([0, 2, 100], [9, 9], None),  # a last range wholly behind the rows
    ([0, 1, 1, 2], [9, 1 << 20, 9], None),  # lengths of sequences without rows
    ([0, 1, 1, 2], [9, -1, 9], None),
    ([0, 70, 70], [90, 1 << 20], None),
    ([0, 1, 1], [9, 9], [5, 1 << 20])])
def test_append_reports_what_no_row_leads_to(ctx, rng, starts, own, prefix):
    """Row starts and lengths outside their range are reported wherever they stand in the batch."""
    page, kv, heads, dim = 64, 1, 2, 32
    batch = Batch(rng, page, [1] * len(own), [256] * len(own), None if prefix is None else [64] * len(own))
    store = Store(rng, BF16, batch.pages, page, kv, dim)
    batch.rows, batch.prefix = min(starts[-1], 2) if starts[-1] == 100 else starts[-1], prefix or batch.prefix
    cache, b = store.put(ctx), batch.put(ctx, lengths=own, starts=starts)
    q, k, v = (up(ctx, rng.standard_normal(batch.rows * h * dim).astype(np.float32)) for h in (heads, kv, kv))
    ctx.PagedAppend(cache, b, k, v, q, q, heads, THETA)
    with pytest.raises(hip.EInvalidOp, match="outside its range"):
        ctx.Download(q)
    ctx.Download(q)
    free(ctx, cache, b, q, k, v)

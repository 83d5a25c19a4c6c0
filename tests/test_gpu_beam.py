"""Beam selection against its definition in 64 bits, and beam searches over the paged cache.

Parents and tokens have to be equal.  Scores: one rounding to fp32 (2^-24 of the score) and the sum of exponentials, whose
terms are fp32 (2 ulp each, and 2^-24 of a difference of up to 20): 2e-6 absolute covers both.
"""
import numpy as np
import pytest

from quicknn_amd import hip
from tests.test_gpu_paged import BF16, F32, Store, free, up, words

pytestmark = pytest.mark.gpu


def select(logits, scores, done, groups, beams, vocab, k, end):
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        cand = scores.astype(np.float64)[:, None] + (x - top - np.log(np.exp(x - top).sum(1, keepdims=True)))
    for b in range(groups * beams):
        if not np.isfinite(scores[b]):
            cand[b] = -np.inf
        elif done is not None and done[b]:
            cand[b] = -np.inf
            cand[b, end] = scores[b]
        elif not np.isfinite(top[b, 0]):
            cand[b] = -np.inf
    flat = cand.reshape(groups, beams * vocab)
    order = np.argsort(-flat, axis=1, kind="stable")[:, :k]
    return order // vocab + np.arange(groups)[:, None] * beams, order % vocab, np.take_along_axis(flat, order, 1)


def run_select(ctx, logits, scores, done, groups, beams, vocab, k, end=0):
    tl, ts, td = up(ctx, logits), up(ctx, scores), None if done is None else words(ctx, done)
    p, t, s = (ctx.NewTensor(groups * k) for _ in range(3))
    ctx.BeamSelect(p, t, s, tl, ts, td, groups, beams, vocab, k, end)
    got = [ctx.Download(x, dtype=d).reshape(groups, k) for x, d in ((p, np.int32), (t, np.int32), (s, np.float32))]
    free(ctx, tl, ts, p, t, s, *([] if td is None else [td]))
    return got


def check_select(ctx, logits, scores, done, groups, beams, vocab, k, end=0):
    got = run_select(ctx, logits, scores, done, groups, beams, vocab, k, end)
    want = select(logits, scores, done, groups, beams, vocab, k, end)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    finite = np.isfinite(want[2])
    assert np.all(got[2][~finite] == -np.inf)
    a, w = got[2][finite], want[2][finite]
    assert np.all(np.abs(a - w) <= 2e-6 + 2.0 ** -23 * np.abs(w))


@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (1, 4, 32000, 4), (2, 8, 151936, 16), (3, 5, 1001, 10), (1, 64, 5000, 64), (7, 2, 4096, 3),
    (1, 2, 4097, 64), (2, 3, 7, 21), (1, 1, 200000, 64), (5, 16, 130, 32), (1, 3, 500001, 6), (300, 2, 50, 4),
    (1, 64, 70000, 64), (1, 1, 65, 65 - 1), (3, 1, 1024, 1)])
def test_select(ctx, rng, groups, beams, vocab, k):
    n = groups * beams
    logits = (3 * rng.standard_normal((n, vocab))).astype(np.float32)
    scores = (-5 * rng.random(n)).astype(np.float32)
    check_select(ctx, logits, scores, None, groups, beams, vocab, k)
    done = (rng.random(n) < 0.3).astype(np.int32)
    check_select(ctx, logits, scores, done, groups, beams, vocab, k, vocab // 2)
    first = np.where(np.arange(n) % beams == 0, np.float32(0), np.float32(-np.inf))  # a search's first step
    check_select(ctx, logits, first, None, groups, beams, vocab, k)


def test_select_ties(ctx, rng):
    """Equal candidates: the lower beam, then the lower token."""
    groups, beams, vocab, k = 2, 4, 9001, 20
    row = rng.integers(-3, 4, vocab).astype(np.float32)
    logits = np.broadcast_to(row, (groups * beams, vocab)).copy()
    check_select(ctx, logits, np.zeros(groups * beams, np.float32), None, groups, beams, vocab, k)
    flat = np.zeros((groups * beams, vocab), np.float32)
    flat[:, ::2] = -0.0
    check_select(ctx, flat, np.zeros(groups * beams, np.float32), None, groups, beams, vocab, 64)
    check_select(ctx, flat, np.zeros(groups * beams, np.float32), np.ones(groups * beams, np.int32), groups, beams, vocab, 64,
                 7)


def test_select_of_odd_values(ctx, rng):
    """Masked tokens, beams without a distribution or score, and lists that end in minus infinities."""
    groups, beams, vocab, k = 1, 8, 6000, 40
    logits = rng.standard_normal((beams, vocab)).astype(np.float32)
    scores = (-rng.random(beams)).astype(np.float32)
    logits[0, rng.random(vocab) < 0.9] = -np.inf
    logits[1, 17] = np.nan
    logits[2, 5000] = np.inf
    logits[3] = -np.inf
    logits[4, 1:] = -np.inf
    logits[5] = -3e38
    logits[5, 3] = 3e38
    scores[6], scores[7] = np.nan, np.inf
    check_select(ctx, logits, scores, None, groups, beams, vocab, k)
    done = np.array([0, 1, 0, 1, 0, 0, 1, 1], np.int32)
    check_select(ctx, logits, scores, done, groups, beams, vocab, k, 5999)
    check_select(ctx, logits[1:4], scores[1:4], None, 1, 3, vocab, 64)  # nothing but minus infinities
    check_select(ctx, logits[3:5], scores[3:5], None, 1, 2, vocab, 64)
    check_select(ctx, logits[[4, 3, 4]], scores[:3], np.array([1, 0, 0], np.int32), 1, 3, vocab, 64, 2)


def test_select_of_finitely_masked_logits(ctx, rng):
    """Constrained decoding masks with a large negative value: with fewer allowed tokens than ranks nearly every token
    ties.  The selection is the defined one, and costs a further pass over the logits, not one per rank: more than a
    hundred times an unmasked call (20 us) would be a pass per rank (11 ms)."""
    groups, beams, vocab, k = 8, 8, 151936, 16
    n = groups * beams
    free_logits = (3 * rng.standard_normal((n, vocab))).astype(np.float32)
    scores = (-5 * rng.random(n)).astype(np.float32)
    forced, few, low = (np.full((n, vocab), m, np.float32) for m in (-1e9, -1e9, -3.4028235e38))
    forced[np.arange(n), rng.integers(0, vocab, n)] = 1.5
    few[:, 5000:5003] = rng.standard_normal((n, 3))
    low[:, 77] = 0.25
    took = {}
    for name, x in (("free", free_logits), ("forced", forced), ("few", few), ("lowest", low), ("flat", np.zeros_like(low))):
        check_select(ctx, x, scores, None, groups, beams, vocab, k)
        tl, ts, found = up(ctx, x), up(ctx, scores), [ctx.NewTensor(groups * k) for _ in range(3)]
        times = []
        for _ in range(6):
            ctx.EventRecord(0)
            ctx.BeamSelect(*found, tl, ts, None, groups, beams, vocab, k)
            ctx.EventRecord(1)
            ctx.Flush()
            times.append(ctx.EventElapsedMs(0, 1))
        took[name] = min(times)
        free(ctx, tl, ts, *found)
    assert all(t <= 100 * took["free"] for t in took.values()), took


def test_select_of_thousands_above_the_bound(ctx, rng):
    """Lists of candidates too long to be ranked at once: distinct, in ascending order, and with ended beams among ties."""
    for groups, beams, vocab, k in ((1, 64, 2000, 64), (2, 3, 1500, 64), (1, 2, 40000, 33)):
        n = groups * beams
        for logits in (rng.standard_normal((n, vocab)), np.broadcast_to(np.arange(vocab) / 64, (n, vocab)),
                       rng.integers(0, 2, (n, vocab)), np.full((n, vocab), -1e9)):
            scores = np.where(np.arange(n) % beams == beams - 1, np.float32(0), np.float32(-np.inf))
            check_select(ctx, logits.astype(np.float32), scores, None, groups, beams, vocab, k)  # one live beam
            done = (np.arange(n) % 2).astype(np.int32)
            check_select(ctx, logits.astype(np.float32), np.full(n, -1.5, np.float32), done, groups, beams, vocab, k, 9)


def test_select_of_a_vocabulary_that_fills_a_tensor(ctx, rng):
    """One beam of nearly 2^31 tokens: the last ones count, in the sum and among the selected."""
    pattern, k = rng.standard_normal((5, 1000)).astype(np.float32), 6
    rows = (2 ** 31 - 1) // 1000
    vocab = rows * 1000
    kinds = (np.arange(rows) % 5).astype(np.int32)
    t, i, logits = up(ctx, pattern), words(ctx, kinds), ctx.NewTensor(vocab)
    ctx.GatherRows(logits, t, i, rows, 1000)
    places = [vocab - 1, 3, vocab - 700, vocab - 1100, vocab // 2, 1 << 30]
    values = [9.0, 9.0, 8.5, 8.0, 7.5, 7.0]
    total = np.bincount(kinds) @ np.exp(pattern.astype(np.float64)).sum(1)
    for p, v in zip(places, values):
        one = up(ctx, np.array([v], np.float32))
        ctx.Copy(logits, one, 1, p)
        ctx.Recycle(one)
        total += np.exp(v) - np.exp(np.float64(pattern[kinds[p // 1000], p % 1000]))
    scores, found = up(ctx, np.array([-1.5], np.float32)), [ctx.NewTensor(k) for _ in range(3)]
    ctx.BeamSelect(*found, logits, scores, None, 1, 1, vocab, k)
    assert ctx.Download(found[0], dtype=np.int32).tolist() == [0] * k
    assert ctx.Download(found[1], dtype=np.int32).tolist() == [places[j] for j in (1, 0, 2, 3, 4, 5)]
    want = -1.5 + np.array(values) - np.log(total)
    assert np.all(np.abs(ctx.Download(found[2]) - want) <= 2e-6 + 2.0 ** -23 * np.abs(want))
    free(ctx, t, i, logits, scores, *found)


def test_select_refusals(ctx):
    n = 8 * 100
    logits, scores, done, p, t, s, small = (ctx.NewTensor(x) for x in (n, 8, 8, 16, 16, 16, 7))
    ok = dict(parents=p, tokens=t, best=s, logits=logits, scores=scores, done=done, groups=2, beams=4, vocab=100, select=8,
              end_token=3)
    ctx.Kernel(hip.GO_FILL, n, logits, None, None, None, [0])
    ctx.Kernel(hip.GO_FILL, 8, scores, None, None, None, [0])
    ctx.Kernel(hip.GO_FILL, 8, done, None, None, None, [0])
    ctx.BeamSelect(**ok)
    for kw in (dict(groups=0), dict(beams=0), dict(beams=65, groups=1), dict(vocab=0), dict(select=0), dict(select=65),
               dict(vocab=101), dict(groups=3), dict(select=9), dict(end_token=-1), dict(end_token=100), dict(logits=small),
               dict(scores=small), dict(done=small), dict(parents=small), dict(best=logits), dict(tokens=p), dict(best=scores),
               dict(parents=done), dict(logits=None), dict(tokens=None), dict(groups=1, beams=1, vocab=2, select=3)):
        with pytest.raises(hip.EArgumentException):
            ctx.BeamSelect(**{**ok, **kw})
    ctx.BeamSelect(**{**ok, "done": None, "end_token": -1})
    ctx.Flush()
    free(ctx, logits, scores, done, p, t, s, small)


# ---------------------------------------------------------------- searches
class Model:
    """Two decoder layers of F32 weights: norm-free attention blocks with residuals, and an output head."""

    def __init__(self, rng, hidden=64, heads=4, kv=2, dim=32, vocab=211, layers=2):
        self.hidden, self.heads, self.kv, self.dim, self.vocab, self.layers = hidden, heads, kv, dim, vocab, layers
        w = lambda n, k, s: (s * rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)  # noqa: E731
        self.embed = w(vocab, hidden, 8.0)
        self.blocks = [dict(q=w(heads * dim, hidden, 1.0), k=w(kv * dim, hidden, 1.0), v=w(kv * dim, hidden, 1.0),
                            o=w(hidden, heads * dim, 1.0)) for _ in range(layers)]
        self.head = w(vocab, hidden, 2.0)
        self.m = {id(x): hip.MemoryBlock.matrix(x) for x in [self.embed, self.head] + [y for b in self.blocks
                                                                                    for y in b.values()]}

    def logits(self, tokens):
        """The last token's logits in 64 bits, everything computed anew."""
        x = self.embed[tokens].astype(np.float64)
        n, g = len(tokens), self.heads // self.kv
        half = self.dim // 2
        a = np.arange(n)[:, None] * 1e4 ** (-np.arange(half) / half)
        co, si = np.cos(a)[:, None], np.sin(a)[:, None]
        turn = lambda y: np.concatenate([y[..., :half] * co - y[..., half:] * si,  # noqa: E731
                                         y[..., :half] * si + y[..., half:] * co], -1)
        for b in self.blocks:
            q, k, v = (x @ b[w].T.astype(np.float64) for w in "qkv")
            q, k, v = (y.reshape(n, -1, self.dim) for y in (q, k, v))
            q, k = turn(q), turn(k)
            out = np.empty_like(q)
            for h in range(self.heads):
                sc = q[:, h] @ k[:, h // g].T / np.sqrt(self.dim)
                sc[np.triu_indices(n, 1)] = -np.inf
                w = np.exp(sc - sc.max(1, keepdims=True))
                out[:, h] = w / w.sum(1, keepdims=True) @ v[:, h // g]
            x = x + out.reshape(n, -1) @ b["o"].T.astype(np.float64)
        return x[-1] @ self.head.T.astype(np.float64)

    def forward(self, ctx, t, batch, caches, ids, rows):
        """Logits of every row, as recorded on the context; t holds its tensors."""
        h, qd, kd = self.hidden, self.heads * self.dim, self.kv * self.dim
        ctx.Gather(t["x"], ids, self.m[id(self.embed)], None, rows, h, self.vocab)
        for b, c in zip(self.blocks, caches):
            for name, n in (("q", qd), ("k", kd), ("v", kd)):
                ctx.Linear(t[name], t["x"], self.m[id(b[name])], None, None, rows, h, n)
            ctx.PagedAppend(c, batch, t["k"], t["v"], t["q"], t["q"], self.heads, 1e4)
            ctx.PagedAttention(t["a"], t["q"], c, batch, self.heads)
            ctx.Linear(t["o"], t["a"], self.m[id(b["o"])], None, None, rows, qd, h)
            ctx.Kernel(hip.GO_ADD, rows * h, t["x"], t["o"], None, None, [h, h, hip.float_bits(1.0), 0, 0])
        ctx.Linear(t["logits"], t["x"], self.m[id(self.head)], None, None, rows, h, self.vocab)

    def tensors(self, ctx, rows):
        sizes = dict(x=self.hidden, q=self.heads * self.dim, k=self.kv * self.dim, v=self.kv * self.dim,
                     a=self.heads * self.dim, o=self.hidden, logits=self.vocab)
        return {n: ctx.NewTensor(rows * s) for n, s in sizes.items()}


@pytest.mark.parametrize("graph", [False, True])
def test_beam_search(ctx, rng, graph):
    """Prompts prefilled as one ragged batch become the prefixes of their beams; every step's selection equals the one
    that a search without any cache makes.  With `graph` two steps (one for each table) are captured once and replayed."""
    m, page, beams, steps, prompts = Model(rng), 32, 4, 80, [[int(x) for x in rng.integers(0, 211, n)] for n in (37, 5, 64)]
    groups, width, pwidth = len(prompts), 4, 2
    n = groups * beams
    pages = n * width + groups * pwidth
    order = rng.permutation(pages).astype(np.int32)
    stores = [Store(rng, F32, pages, page, m.kv, m.dim) for _ in range(m.layers)]
    for s in stores:
        s.x[:] = np.nan  # nothing but what is appended may be read
    caches = [s.put(ctx) for s in stores]
    # The prompts: one ragged batch.
    total = sum(map(len, prompts))
    lengths = [len(p) for p in prompts]
    ptables, plengths = words(ctx, order[n * width:]), words(ctx, lengths)
    prefill = hip.PagedBatch(ptables, plengths, groups, total, pwidth, starts=words(ctx, np.cumsum([0] + lengths)))
    t = m.tensors(ctx, total)
    ids = words(ctx, sum(prompts, []))
    m.forward(ctx, t, prefill, caches, ids, total)
    last = np.cumsum(lengths) - 1
    start = ctx.Download(t["logits"]).reshape(total, -1)[last]
    for g in range(groups):
        want = m.logits(prompts[g])
        assert np.max(np.abs(start[g] - want)) <= 1e-4 * np.max(np.abs(want))
    # The beams.
    t2 = m.tensors(ctx, n)
    view = np.repeat(start, beams, 0).astype(np.float32)
    tab = [words(ctx, order[:n * width]), ctx.NewTensor(n * width)]
    blen = words(ctx, [0] * n)
    common = dict(prefix_tables=ptables, prefix_lengths=plengths, prefix_pages=pwidth, share=beams)
    batches = [hip.PagedBatch(x, blen, n, n, width, **common) for x in tab]
    scores = up(ctx, np.where(np.arange(n) % beams == 0, np.float32(0), np.float32(-np.inf)))
    best, parents, tokens = (ctx.NewTensor(n) for _ in range(3))
    history = [words(ctx, np.zeros((n, steps), np.int32)), ctx.NewTensor(n * steps)]
    logits = up(ctx, view)
    ctx.Copy(t2["logits"], logits, n * m.vocab)

    def step(i):
        old, new = i % 2, (i + 1) % 2
        ctx.BeamSelect(parents, tokens, best, t2["logits"], scores, None, groups, beams, m.vocab, beams)
        ctx.Copy(scores, best, n)
        ctx.PagedReorder(batches[old], tab[new], parents, caches)
        ctx.GatherRows(history[new], history[old], parents, n, steps)
        ctx.PagedAdvance(batches[new], page)
        m.forward(ctx, t2, batches[new], caches, tokens, n)

    texts = [[list(p) for _ in range(beams)] for p in prompts]
    sums = [[0.0] + [-np.inf] * (beams - 1) for _ in prompts]
    g0 = None
    for i in range(0, steps, 2):
        results = []
        if graph and i == 2:
            ctx.GraphBegin()
            step(0), step(1)
            g0 = ctx.GraphEnd()
        if graph and i >= 2:
            ctx.GraphLaunch(g0)
            results.append((1, [ctx.Download(x, dtype=d) for x, d in ((parents, np.int32), (tokens, np.int32),
                                                                       (best, np.float32))]))
        else:
            for j in (0, 1):
                step(j)
                results.append((j, [ctx.Download(x, dtype=d) for x, d in ((parents, np.int32), (tokens, np.int32),
                                                                           (best, np.float32))]))
        if i % 10 and i < steps - 2 and not graph:  # the statement without a cache is slow: follow, and check some
            for _, (p, tk, sc) in results:
                for g in range(groups):
                    texts[g] = [texts[g][int(a) - g * beams] + [int(b)] for a, b in zip(p[g * beams:(g + 1) * beams],
                                                                                     tk[g * beams:(g + 1) * beams])]
                    sums[g] = [float(x) for x in sc[g * beams:(g + 1) * beams]]
            continue
        for j in (0, 1):
            for g in range(groups):
                if i == 0 and j == 0:
                    x = np.repeat(m.logits(prompts[g])[None], beams, 0)
                else:
                    x = np.stack([m.logits(text) for text in texts[g]])
                x -= x.max(1, keepdims=True)
                cand = (np.array(sums[g])[:, None] + x - np.log(np.exp(x).sum(1, keepdims=True))).reshape(-1)
                top = np.argsort(-cand, kind="stable")[:beams]
                texts[g] = [texts[g][o // m.vocab] + [int(o % m.vocab)] for o in top]
                sums[g] = [float(cand[o]) for o in top]
                got = [r for k, r in results if k == j]
                if got:
                    p, tk, sc = (y[g * beams:(g + 1) * beams] for y in got[0])
                    assert (p - g * beams).tolist() == (top // m.vocab).tolist(), (i, j, g)
                    assert tk.tolist() == (top % m.vocab).tolist(), (i, j, g)
                    assert np.max(np.abs(sc - cand[top])) <= 1e-4 * max(1.0, np.max(np.abs(cand[top])))
    assert ctx.Download(blen, dtype=np.int32).tolist() == [steps] * n
    ctx.Flush()
    free(ctx, ptables, plengths, ids, blen, scores, best, parents, tokens, logits, *tab, *history, *caches, *t.values(),
         *t2.values())


def test_beam_search_with_ends(ctx, rng):
    """Beams that end stay on the device too: the next step's `done` is a gather of a table with a one at the end token, by
    the selected tokens.  Every step equals a search without any cache, in which an ended beam is carried on as it is."""
    m, page, beams, steps, prompts, end = Model(rng), 32, 4, 14, [[int(x) for x in rng.integers(0, 211, n)] for n in (9, 21)], 45
    groups, width, pwidth = len(prompts), 1, 1
    n = groups * beams
    order = rng.permutation(n * width + groups * pwidth).astype(np.int32)
    caches = [Store(rng, F32, order.size, page, m.kv, m.dim).put(ctx) for _ in range(m.layers)]
    total, lengths = sum(map(len, prompts)), [len(p) for p in prompts]
    ptables, plengths = words(ctx, order[n * width:]), words(ctx, lengths)
    starts = words(ctx, np.cumsum([0] + lengths))
    prefill = hip.PagedBatch(ptables, plengths, groups, total, pwidth, starts=starts)
    t, ids = m.tensors(ctx, total), words(ctx, sum(prompts, []))
    m.forward(ctx, t, prefill, caches, ids, total)
    start = ctx.Download(t["logits"]).reshape(total, -1)[np.cumsum(lengths) - 1]
    t2, logits = m.tensors(ctx, n), up(ctx, np.repeat(start, beams, 0).astype(np.float32))
    ctx.Copy(t2["logits"], logits, n * m.vocab)
    tab, blen = [words(ctx, order[:n * width]), ctx.NewTensor(n * width)], words(ctx, [0] * n)
    batches = [hip.PagedBatch(x, blen, n, n, width, prefix_tables=ptables, prefix_lengths=plengths, prefix_pages=pwidth,
                              share=beams) for x in tab]
    scores = up(ctx, np.where(np.arange(n) % beams == 0, np.float32(0), np.float32(-np.inf)))
    best, parents, tokens = (ctx.NewTensor(n) for _ in range(3))
    ends, done = words(ctx, np.arange(m.vocab) == end), words(ctx, [0] * n)
    texts = [[list(p) for _ in range(beams)] for p in prompts]
    sums = [[0.0] + [-np.inf] * (beams - 1) for _ in prompts]
    over = [[False] * beams for _ in prompts]
    for i in range(steps):
        ctx.BeamSelect(parents, tokens, best, t2["logits"], scores, done, groups, beams, m.vocab, beams, end)
        ctx.Copy(scores, best, n)
        ctx.GatherRows(done, ends, tokens, n, 1)
        ctx.PagedReorder(batches[i % 2], tab[(i + 1) % 2], parents, caches)
        ctx.PagedAdvance(batches[(i + 1) % 2], page)
        m.forward(ctx, t2, batches[(i + 1) % 2], caches, tokens, n)
        got = [ctx.Download(x, dtype=d).reshape(groups, beams) for x, d in ((parents, np.int32), (tokens, np.int32),
                                                                            (best, np.float32), (done, np.int32))]
        for g in range(groups):
            top, value = ended_step(m, texts[g], sums[g], over[g], end)
            texts[g] = [texts[g][o // m.vocab] + [int(o % m.vocab)] for o in top]
            sums[g], over[g] = value.tolist(), [int(o % m.vocab) == end for o in top]
            assert (got[0][g] - g * beams).tolist() == (top // m.vocab).tolist(), (i, g)
            assert got[1][g].tolist() == (top % m.vocab).tolist(), (i, g)
            assert np.max(np.abs(got[2][g] - value)) <= 1e-4 * max(1.0, np.max(np.abs(value)))
            assert got[3][g].tolist() == [int(x) for x in over[g]]
    assert any(map(any, over)) and not all(map(all, over))
    free(ctx, ptables, plengths, starts, ids, blen, scores, best, parents, tokens, logits, ends, done, *tab, *caches,
         *t.values(), *t2.values())


def ended_step(m, texts, sums, over, end):
    """One group's step in 64 bits: candidates in order and their scores; an ended beam only offers `end` at its score."""
    x = np.stack([m.logits(text) for text in texts])
    x -= x.max(1, keepdims=True)
    cand = np.array(sums)[:, None] + x - np.log(np.exp(x).sum(1, keepdims=True))
    for b, o in enumerate(over):
        if o:
            cand[b] = -np.inf
            cand[b, end] = sums[b]
    top = np.argsort(-cand.reshape(-1), kind="stable")[:len(texts)]
    return top, cand.reshape(-1)[top]


def test_two_graphs_and_a_larger_call(ctx, rng):
    """Two captured graphs share the context's workspace; a larger eager call between their replays outgrows it."""
    from tests.test_gpu_paged import Batch

    page, kv, heads, dim = 64, 1, 4, 64
    runs = []
    for n, own, prefix, share in ((5, 300, [500], 5), (3, 900, None, 1)):
        batch = Batch(rng, page, [1] * n, [own] * n, prefix, share)
        store = Store(rng, F32, batch.pages, page, kv, dim)
        q = up(ctx, rng.standard_normal(n * heads * dim).astype(np.float32))
        runs.append((store.put(ctx), batch.put(ctx), q, ctx.NewTensor(q.count)))
    logits = up(ctx, rng.standard_normal((8, 3000)).astype(np.float32))
    scores, found = up(ctx, np.zeros(8, np.float32)), [ctx.NewTensor(16) for _ in range(3)]

    def attend(r):
        ctx.PagedAttention(r[3], r[2], r[0], r[1], heads)

    def choose():
        ctx.BeamSelect(*found, logits, scores, None, 2, 4, 3000, 8)

    want = []
    for r in runs:
        attend(r)
        want.append(ctx.Download(r[3]))
    choose()
    want.append(ctx.Download(found[1], dtype=np.int32))
    graphs = []
    for r in runs:
        ctx.GraphBegin()
        attend(r)
        choose()
        graphs.append(ctx.GraphEnd())
    big = Batch(rng, page, [700, 400], [2000, 400], [300, 200])
    big_store = Store(rng, F32, big.pages, page, kv, dim)
    bc, bb, bq = big_store.put(ctx), big.put(ctx), up(ctx, rng.standard_normal(1100 * heads * dim).astype(np.float32))
    bo = ctx.NewTensor(bq.count)
    for i in range(4):
        for g, r, w in zip(graphs, runs, want):
            ctx.Kernel(hip.GO_FILL, r[3].count, r[3], None, None, None, [0])
            ctx.Kernel(hip.GO_FILL, 16, found[1], None, None, None, [0])
            ctx.GraphLaunch(g)
            assert np.array_equal(ctx.Download(r[3]), w), i
            assert np.array_equal(ctx.Download(found[1], dtype=np.int32), want[2]), i
            if i == 1:
                ctx.PagedAttention(bo, bq, bc, bb, heads)
    free(ctx, bc, bb, bq, bo, logits, scores, *found, *(x for r in runs for x in r))


def test_captured_step_against_eager(ctx, rng):
    """Append, attention and advance captured once: replays with lengths that grow on the device equal eager calls, with
    larger eager work (which needs a larger workspace) and synchronisations between the replays."""
    from tests.test_gpu_paged import Batch

    page, kv, heads, dim, n = 64, 2, 8, 128, 6
    batch = Batch(rng, page, [1] * n, [60 + i for i in range(n)], [200], n, extra_pages=2)
    store = Store(rng, BF16, batch.pages, page, kv, dim)
    big = Batch(rng, page, [90, 300], [2000, 300])
    big_store = Store(rng, BF16, big.pages, page, kv, dim)
    big_cache, bb, bq = big_store.put(ctx), big.put(ctx), up(ctx, rng.standard_normal(390 * heads * dim).astype(np.float32))
    bout = ctx.NewTensor(bq.count)
    runs = []
    k, v, q = (up(ctx, rng.standard_normal(n * h * dim).astype(np.float32)) for h in (kv, kv, heads))
    for captured in (False, True):
        cache, b, qr, out = store.put(ctx), batch.put(ctx), ctx.NewTensor(q.count), ctx.NewTensor(q.count)

        def step():
            ctx.PagedAdvance(b, page)
            ctx.PagedAppend(cache, b, k, v, q, qr, heads, 1e4)
            ctx.PagedAttention(out, qr, cache, b, heads)

        got = []
        step()
        got.append(ctx.Download(out))
        if captured:
            ctx.GraphBegin()
            step()
            g = ctx.GraphEnd()
        for i in range(5):
            ctx.GraphLaunch(g) if captured else step()
            got.append(ctx.Download(out))
            if i % 2:
                ctx.PagedAttention(bout, bq, big_cache, bb, heads)
                ctx.Flush()
        runs.append(got)
        free(ctx, cache, b, qr, out)
    assert all(np.array_equal(a, c) for a, c in zip(*runs))
    free(ctx, big_cache, bb, bq, bout, k, v, q)

"""Serving several sequences over one paged KV cache, and beam search, as cases that can be timed and compared.

Four families, each one call (or two that always go together) of ``quicknn_amd.hip``:

* ``append``     rotary embedding of q and k, keys and values appended to the pages of their sequences
* ``attention``  attention of a ragged batch over the pages; consecutive sequences may share a prefix
* ``select``     the best continuations of every group of beams over beams and vocabulary
* ``reorder``    page tables, partial pages of every layer and the token histories follow the selected parents

With ``own`` false a pass computes the same in elementary torch operations.

The pages (as ``include/qnn_hip.h`` documents them): a page holds, for each KV head, page_size keys, then for each KV
head as many values, in pieces of 16 bytes, E elements.  Keys: blocks of 16 tokens, [dim / E][16 tokens][E channels].
Values: in BF16 groups of 32 tokens, [4][dim][8 tokens], token 16 a + 4 g + b of the group at [g][.][4 a + b]; in F32
blocks of 16 tokens, [4][dim][4 tokens].
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
THETA = 1000000.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One decoded token of one sequence: latency.
        dict(name="append_token", family="append", dtype="bf16", sequences=1, share=1, prefix=0, longest=4001, ragged=0.0,
             rows=1, heads=32, kv=8, dim=128, page=64),
        # Prompts of several users prefilled together, of all lengths, one of five sequences idle.
        dict(name="append_prompts", family="append", dtype="bf16", sequences=9, share=1, prefix=0, longest=1500,
             ragged=0.8, rows=700, heads=32, kv=8, dim=128, page=64),
        # One decoded token of one sequence at a 4k context: latency.
        dict(name="attention_token", family="attention", dtype="bf16", sequences=1, share=1, prefix=0, longest=4001,
             ragged=0.0, rows=1, heads=32, kv=8, dim=128, page=64, window=0, softcap=0.0),
        # A serving step: forty sequences of all lengths up to 8k, one token each.
        dict(name="attention_batch", family="attention", dtype="bf16", sequences=40, share=1, prefix=0, longest=8191,
             ragged=0.95, rows=1, heads=32, kv=8, dim=128, page=64, window=0, softcap=0.0),
        # Two long contexts in full precision, odd group of heads.
        dict(name="attention_long_f32", family="attention", dtype="f32", sequences=2, share=1, prefix=0, longest=32749,
             ragged=0.3, rows=1, heads=28, kv=4, dim=128, page=128, window=0, softcap=0.0),
        # A beam search step: four prompts of up to 12k tokens, eight beams each, 200 tokens into the answers.
        dict(name="attention_beams", family="attention", dtype="bf16", sequences=32, share=8, prefix=12000, longest=201,
             ragged=0.0, rows=1, heads=32, kv=8, dim=128, page=64, window=0, softcap=0.0),
        # One system prompt under a whole batch.
        dict(name="attention_prefix", family="attention", dtype="bf16", sequences=48, share=48, prefix=16384, longest=400,
             ragged=0.9, rows=1, heads=32, kv=8, dim=128, page=64, window=0, softcap=0.0),
        # Prompt chunks of several users over what they have in the cache, windowed and capped, wide heads.
        dict(name="attention_prompts", family="attention", dtype="bf16", sequences=4, share=1, prefix=0, longest=4000,
             ragged=0.7, rows=512, heads=16, kv=8, dim=256, page=32, window=2048, softcap=50.0),
        # Four beams over a small vocabulary.
        dict(name="select_small", family="select", groups=1, beams=4, vocab=32000, select=4),
        # Eight prompts, eight beams each, twice as many candidates for those that end.
        dict(name="select_batch", family="select", groups=8, beams=8, vocab=151936, select=16),
        # One prompt's four beams over a few layers.
        dict(name="reorder_small", family="reorder", dtype="bf16", sequences=4, share=4, longest=41, layers=4, kv=8, dim=128,
             page=64, history=64),
        # Four prompts, eight beams each, a dozen layers.
        dict(name="reorder_batch", family="reorder", dtype="bf16", sequences=32, share=8, longest=200, layers=12, kv=8,
             dim=128, page=64, history=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= most[1]:
            return c


def _draw(rng):
    family = rng.choice(["append", "attention", "attention", "attention", "select", "reorder"])
    if family == "select":
        beams = _log(rng, 1, 32)
        vocab = _log(rng, 1000, 200000)
        return dict(family="select", groups=_log(rng, 1, 16), beams=beams, vocab=vocab,
                    select=min(64, rng.choice([beams, 2 * beams, beams + 1])))
    kv = rng.choice([1, 2, 4, 8])
    shape = dict(dtype=rng.choice(["bf16", "bf16", "f32"]), kv=kv, dim=rng.choice([64, 80, 96, 128, 128, 256]),
                 page=rng.choice([32, 64, 64, 128, 256]))
    if family == "reorder":
        share = _log(rng, 2, 16)
        return dict(family="reorder", sequences=share * _log(rng, 1, 6), share=share, longest=_log(rng, 1, 300),
                    layers=_log(rng, 1, 12), history=_log(rng, 16, 2000), **shape)
    share = rng.choice([1, 1, _log(rng, 2, 32)])
    sequences = share * _log(rng, 1, max(1, 64 // share))
    rows = _log(rng, 2, 1000) if rng.random() < 0.4 else 1
    longest = rows - 1 + _log(rng, 1, 16000)
    c = dict(family=family, sequences=sequences, share=share, prefix=_log(rng, 1, 20000) if share > 1 else 0,
             longest=longest, ragged=rng.choice([0.0, 0.5, 0.95]), rows=rows, heads=kv * rng.choice([1, 2, 4, 5, 7, 8]),
             **shape)
    if family == "append":
        c["longest"] = min(longest, rows + 600)  # the cache before the call does not matter to it
        c["prefix"] = min(c["prefix"], 600)
        return c
    return dict(c, window=rng.choice([0, 0, 1 + longest // 3]), softcap=rng.choice([0.0, 0.0, 30.0]))


# ---------------------------------------------------------------------------------------------------------------
# Sizes of a batch: plain functions of the case
# ---------------------------------------------------------------------------------------------------------------
def _part(i, ragged):
    return 1 - ragged * ((0.6180339887 * i) % 1.0)


def _batch(c):
    """Rows and own keys of every sequence, keys of every group's prefix."""
    n, own_keys = [], []
    for i in range(c["sequences"]):
        keys = max(1, round(c["longest"] * _part(i, c["ragged"])))
        rows = min(keys, max(1, round(c["rows"] * _part(3 * i + 1, c["ragged"]))))
        n.append(0 if c["rows"] > 1 and i % 5 == 4 else rows)
        own_keys.append(keys)
    return n, own_keys, [round(c["prefix"] * _part(g, c["ragged"])) for g in range(c["sequences"] // c["share"])]


def _visible(c, absolute):
    """Keys that a row at this absolute position sees."""
    return min(absolute + 1, c.get("window") or absolute + 1)


def work(case):
    c, f = case, case["family"]
    if f == "select":
        beams = c["groups"] * c["beams"]
        return {"bytes": 4.0 * beams * (c["vocab"] + 2) + 12.0 * c["groups"] * c["select"],
                "flops": 4.0 * beams * c["vocab"]}
    size = 4 if c["dtype"] == "f32" else 2
    token = 2.0 * c["kv"] * c["dim"] * size
    if f == "reorder":
        extra = sum(_extra_children(c, g) for g in range(c["sequences"] // c["share"]))
        blocks = -(-(c["longest"] % c["page"]) // 32) * 32
        cols = -(-c["longest"] // c["page"])
        return {"bytes": 2 * extra * blocks * token * c["layers"] + 8.0 * c["sequences"] * (cols + c["history"]),
                "flops": 1.0 * c["sequences"] * (cols + c["history"])}
    n, keys, prefix = _batch(c)
    rows = sum(n)
    if f == "append":
        return {"bytes": 4.0 * rows * (2 * c["heads"] + 2 * c["kv"]) * c["dim"] + rows * token,
                "flops": 3.0 * rows * (c["heads"] + c["kv"]) * c["dim"]}
    seen, read = 0, 0
    for g, p in enumerate(prefix):
        first = None
        for s in range(g * c["share"], (g + 1) * c["share"]):
            if not n[s]:
                continue
            at = [p + keys[s] - n[s] + i for i in range(n[s])]
            seen += sum(_visible(c, a) for a in at)
            low = at[0] + 1 - _visible(c, at[0])
            first = low if first is None else min(first, low)
            read += keys[s] - max(0, low - p)
        if first is not None:
            read += max(0, p - first)
    return {"bytes": read * token + 8.0 * rows * c["heads"] * c["dim"], "flops": 4.0 * seen * c["heads"] * c["dim"]}


def _parents(c, g):
    """Parents within a group as a beam search has them: a few beams survive, the best ones more than once."""
    share = c["share"]
    return [min(share - 1, int(share * ((0.6180339887 * (i + g)) % 1.0) ** 2)) for i in range(share)]


def _extra_children(c, g):
    return c["share"] - len(set(_parents(c, g)))


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------
class Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device=DEV, dtype=torch.float32) * std

    def pages(self, c, count):
        """Flat storage of `count` pages holding values of any layer's scale."""
        return self.normal(count * 2 * c["kv"] * c["page"] * c["dim"]).to(DTYPES[c["dtype"]])

    def order(self, count):
        return torch.randperm(count, generator=self.g, device=DEV).int()


def _words(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tables(c, g, need, width, order, used):
    """Page tables [len(need)][width]: the first pages of each row from `order`, the rest unused (page 0)."""
    table = torch.zeros(len(need), width, dtype=torch.int32)
    for i, pages in enumerate(need):
        table[i, :pages] = order[used:used + pages]
        used += pages
    return table.to(DEV), used


def inputs(c, seed):
    g, f = Gen(seed), c["family"]
    if f == "select":
        beams = c["groups"] * c["beams"]
        logits = g.normal(beams, c["vocab"], std=2.5)
        logits[:, :: max(1, c["vocab"] // 50)] += 6.0  # a few likely words
        scores = -4.0 * g.normal(beams).abs()
        done = (torch.rand(beams, generator=g.g, device=DEV) < 0.15).int()
        return dict(logits=logits, scores=scores, done=done)
    page = c["page"]
    if f == "reorder":
        width = -(-c["longest"] // page) + 1
        count = c["sequences"] * width
        tables = g.order(count).view(c["sequences"], width).contiguous()
        parents = _words([g_ * c["share"] + p for g_ in range(c["sequences"] // c["share"]) for p in _parents(c, g_)])
        return dict(tables=tables, lengths=_words([c["longest"]] * c["sequences"]), parents=parents,
                    history=torch.randint(0, 150000, (c["sequences"], c["history"]), generator=g.g, device=DEV,
                                          dtype=torch.int32),
                    caches=[g.pages(c, count) for _ in range(c["layers"])])
    n, keys, prefix = _batch(c)
    rows = sum(n)
    need = [-(-k // page) for k in keys]
    need_prefix = [-(-p // page) for p in prefix]
    count = sum(need) + sum(need_prefix) + 3
    order = g.order(count).cpu()
    tables, used = _tables(c, g, need, max(need), order, 0)
    out = dict(tables=tables, lengths=_words(keys), cache=g.pages(c, count), rows=rows, n=n, keys=keys, prefix=prefix,
               starts=_words([sum(n[:i]) for i in range(len(n) + 1)]), prefix_tables=None, prefix_lengths=None)
    if c["prefix"]:
        out["prefix_tables"], _ = _tables(c, g, need_prefix, max(1, max(need_prefix)), order, used)
        out["prefix_lengths"] = _words(prefix)
    out["q"] = g.normal(rows, c["heads"], c["dim"])
    if f == "append":
        out["k"], out["v"] = g.normal(rows, c["kv"], c["dim"]), g.normal(rows, c["kv"], c["dim"])
    return out


# ---------------------------------------------------------------------------------------------------------------
# The framework's context and what a state holds in it
# ---------------------------------------------------------------------------------------------------------------
_ctx = None


def context():
    """One context per process, as the engine has one."""
    global _ctx
    if _ctx is None:
        from quicknn_amd import hip

        _ctx = hip.GPUContext(0)
    return _ctx


class View:
    """Device memory of a context tensor, for torch."""

    def __init__(self, tensor, typestr):
        self.__cuda_array_interface__ = dict(shape=(tensor.count,), typestr=typestr, data=(tensor.device_ptr, False),
                                             version=2)


def view(tensor, *shape, dtype=torch.float32):
    words = torch.as_tensor(View(tensor, "<f4"), device=DEV)
    return words.view(dtype).view(*shape)


class State:
    """A plain state holds torch tensors, an own one context tensors of the same words."""

    def __init__(self, case):
        self.case, self.tensors = case, []

    def new(self, words):
        t = context().NewTensor(int(words))
        self.tensors.append(t)
        return t

    def put(self, values):
        words = values.contiguous().view(-1).view(torch.float32)
        t = self.new(words.numel())
        view(t, -1).copy_(words)
        return t

    def __del__(self):
        try:
            torch.cuda.synchronize()
            for t in self.tensors:
                context().Recycle(t)
        except Exception:  # the context has gone first
            pass


def prepare(case, seed):
    c, s, i = case, State(case), inputs(case, seed)
    s.i = i
    if not own:
        return s
    from quicknn_amd import hip

    f = c["family"]
    if f == "select":
        s.logits, s.scores, s.done = s.put(i["logits"]), s.put(i["scores"]), s.put(i["done"])
        found = c["groups"] * c["select"]
        s.parents, s.tokens, s.best = s.new(found), s.new(found), s.new(found)
        s.i = None
    else:
        dtype = hip.DT_F32 if c["dtype"] == "f32" else hip.DT_BF16
        make = lambda pages: hip.PagedCache(s.put(pages), dtype, pages.numel() // (2 * c["kv"] * c["page"] * c["dim"]),  # noqa: E731
                                            c["page"], c["kv"], c["dim"])
        tables, lengths = s.put(i["tables"]), s.put(i["lengths"])
        if f == "reorder":
            s.caches = [make(p) for p in i["caches"]]
            s.batch = hip.PagedBatch(tables, lengths, c["sequences"], c["sequences"], i["tables"].shape[1],
                                     share=c["share"])
            s.parents, s.tables, s.history = s.put(i["parents"]), s.new(i["tables"].numel()), s.put(i["history"])
            s.new_history = s.new(i["history"].numel())
            s.i = None
        else:
            s.cache = make(i["cache"])
            prefix = {}
            if i["prefix_tables"] is not None:
                prefix = dict(prefix_tables=s.put(i["prefix_tables"]), prefix_lengths=s.put(i["prefix_lengths"]),
                              prefix_pages=i["prefix_tables"].shape[1])
            starts = None if c["rows"] == 1 else s.put(i["starts"])
            s.batch = hip.PagedBatch(tables, lengths, c["sequences"], i["rows"], i["tables"].shape[1], starts=starts,
                                     share=c["share"], **prefix)
            s.q, s.out = s.put(i["q"]), s.new(i["q"].numel())
            if f == "append":
                s.k, s.v = s.put(i["k"]), s.put(i["v"])
            s.i = dict(rows=i["rows"])
    torch.cuda.synchronize()
    context().Flush()
    return s


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    c, f = s.case, s.case["family"]
    if not own:
        return dict(append=plain_append, attention=plain_attention, select=plain_select, reorder=plain_reorder)[f](c, s.i)
    ctx = context()
    if f == "select":
        ctx.BeamSelect(s.parents, s.tokens, s.best, s.logits, s.scores, s.done, c["groups"], c["beams"], c["vocab"],
                       c["select"], 2)
        shape = (c["groups"], c["select"])
        return {"parents": view(s.parents, *shape, dtype=torch.int32), "tokens": view(s.tokens, *shape, dtype=torch.int32),
                "scores": view(s.best, *shape)}
    if f == "reorder":
        ctx.PagedReorder(s.batch, s.tables, s.parents, s.caches)
        ctx.GatherRows(s.new_history, s.history, s.parents, c["sequences"], c["history"])
        return {"tables": view(s.tables, c["sequences"], -1, dtype=torch.int32),
                "history": view(s.new_history, c["sequences"], -1, dtype=torch.int32),
                "caches": [view(p.pages, -1, dtype=DTYPES[c["dtype"]]) for p in s.caches]}
    if f == "append":
        ctx.PagedAppend(s.cache, s.batch, s.k, s.v, s.q, s.out, c["heads"], THETA)
        return {"q": view(s.out, -1, c["heads"], c["dim"]), "cache": view(s.cache.pages, -1, dtype=DTYPES[c["dtype"]])}
    ctx.PagedAttention(s.out, s.q, s.cache, s.batch, c["heads"], c["window"], c["softcap"])
    return {"out": view(s.out, -1, c["heads"], c["dim"])}


# ---- plain forms ------------------------------------------------------------------------------------------------
def key_view(c, pages):
    """[pages][blocks of 16][16][kv][dim / E][E] of flat pages, the keys."""
    e = 4 if c["dtype"] == "f32" else 8
    x = pages.view(-1, 2, c["kv"], c["page"] // 16, c["dim"] // e, 16, e)[:, 0]
    return x.permute(0, 2, 4, 1, 3, 5)


def value_view(c, pages):
    """[pages][groups][.. tokens of a group ..][kv][dim] of flat pages, the values."""
    if c["dtype"] == "f32":
        return pages.view(-1, 2, c["kv"], c["page"] // 16, 4, c["dim"], 4)[:, 1].permute(0, 2, 3, 5, 1, 4)
    return pages.view(-1, 2, c["kv"], c["page"] // 32, 4, c["dim"], 2, 4)[:, 1].permute(0, 2, 5, 3, 6, 1, 4)


def read(c, pages, table, count):
    """Keys and values [kv][count][dim] in 32 bits of the first `count` tokens of a row of page ids."""
    ids = table[:-(-count // c["page"])].long()
    return [w(c, pages)[ids].float().reshape(-1, c["kv"], c["dim"])[:count].transpose(0, 1)
            for w in (key_view, value_view)]


def spread(per_sequence, n):
    """A value per row of a value per sequence."""
    return torch.repeat_interleave(per_sequence, _words(n).long())


def positions(c, i):
    """Own and absolute position of every row."""
    n = _words(i["n"])
    at = torch.arange(i["rows"], device=DEV) - spread(i["starts"][:-1] - i["lengths"] + n, i["n"])
    if i["prefix_lengths"] is None:
        return at, at
    return at, at + spread(i["prefix_lengths"].repeat_interleave(c["share"]), i["n"])


def rotate(x, at):
    half = x.shape[-1] // 2
    turn = THETA ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    angle = (at.double()[:, None] * turn)[:, None]
    a, b, co, si = x[..., :half].double(), x[..., half:].double(), torch.cos(angle), torch.sin(angle)
    return torch.cat([a * co - b * si, a * si + b * co], -1).float()


def plain_append(c, i):
    at, absolute = positions(c, i)
    row = torch.arange(len(i["n"]), device=DEV).repeat_interleave(_words(i["n"]).long())
    page, t = i["tables"][row, at // c["page"]].long(), at % c["page"]
    k, v = rotate(i["k"], absolute).to(i["cache"].dtype), i["v"].to(i["cache"].dtype)
    key_view(c, i["cache"])[page, t // 16, t % 16] = k.view(*k.shape[:2], -1, 16 // k.element_size())
    if c["dtype"] == "f32":
        value_view(c, i["cache"])[page, t // 16, t % 16 // 4, t % 4] = v
    else:
        value_view(c, i["cache"])[page, t // 32, t % 32 // 16, t % 16 // 4, t % 4] = v
    return {"q": rotate(i["q"], absolute), "cache": i["cache"]}


def part(c, q, k, v, visible):
    """Running maximum, sum and weighted values [kv][rows x group](.. [dim]) of these keys; visible [rows][keys]."""
    kv, rows, group, dim = q.shape
    sc = (q.reshape(kv, rows * group, dim) @ k.transpose(1, 2).contiguous()) / math.sqrt(dim)
    if c["softcap"]:
        sc = c["softcap"] * torch.tanh((sc / c["softcap"]).clamp(-20, 20))
    sc = sc.view(kv, rows, group, -1).masked_fill_(~visible[None, :, None], -math.inf).view(kv, rows * group, -1)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - m.clamp_min(-3e38))
    return m, p.sum(-1, keepdim=True), p @ v.contiguous()


def plain_attention(c, i):
    own_at, absolute = positions(c, i)
    kv, dim, rows = c["kv"], c["dim"], i["rows"]
    q = i["q"].view(rows, kv, c["heads"] // kv, dim).transpose(0, 1)
    out = torch.zeros(rows, kv, c["heads"] // kv, dim, device=DEV)
    window = c["window"] or 1 << 30
    start = 0
    for g, prefix in enumerate(i["prefix"]):
        first = start
        group_rows = slice(first, first + sum(i["n"][g * c["share"]:(g + 1) * c["share"]]))
        a = absolute[group_rows, None]
        if group_rows.stop == first:
            continue
        shared = None
        if prefix:
            k, v = read(c, i["cache"], i["prefix_tables"][g], prefix)
            shared = part(c, q[:, group_rows], k, v, torch.arange(prefix, device=DEV)[None] > a - window)
        for s in range(g * c["share"], (g + 1) * c["share"]):
            n = i["n"][s]
            if not n:
                continue
            r = slice(start, start + n)
            k, v = read(c, i["cache"], i["tables"][s], i["keys"][s])
            key, o = torch.arange(i["keys"][s], device=DEV)[None], own_at[r, None]
            m, l, x = part(c, q[:, r], k, v, (key <= o) & (key > o - window))
            if shared is not None:
                w = q.shape[2]
                m2, l2, x2 = (y[:, (start - first) * w:(start - first + n) * w] for y in shared)
                top = torch.maximum(m, m2).clamp_min(-3e38)
                w1, w2 = torch.exp(m - top), torch.exp(m2 - top)
                l, x = l * w1 + l2 * w2, x * w1 + x2 * w2
            out[r] = (x / l).view(kv, n, -1, dim).transpose(0, 1)
            start += n
    return {"out": out.view(rows, c["heads"], dim)}


def plain_select(c, i, end=2):
    logits = i["logits"].double()
    top = logits.amax(-1, keepdim=True)
    cand = i["scores"].double()[:, None] + logits - (top + torch.log(torch.exp(logits - top).sum(-1, keepdim=True)))
    ended = torch.full_like(cand, -math.inf)
    ended[:, end] = i["scores"].double()
    cand = torch.where(i["done"][:, None] != 0, ended, cand).view(c["groups"], -1)
    values, order = torch.sort(cand, dim=1, descending=True, stable=True)
    order = order[:, :c["select"]]
    first = torch.arange(c["groups"], device=DEV)[:, None] * c["beams"]
    return {"parents": (first + order // c["vocab"]).int(), "tokens": (order % c["vocab"]).int(),
            "scores": values[:, :c["select"]].float()}


def plain_reorder(c, i):
    full, rest = divmod(c["longest"], c["page"])
    parents = i["parents"].long()
    tables = i["tables"].clone()
    tables[:, :full] = i["tables"][parents][:, :full]
    if rest:
        p = parents.view(-1, c["share"])
        slots = torch.arange(c["sequences"], device=DEV).view(-1, c["share"])
        same = p[:, :, None] == p[:, None]
        again = (same & torch.ones(c["share"], c["share"], dtype=torch.bool, device=DEV).tril(-1)).any(-1)
        free = ~(slots[:, :, None] == p[:, None]).any(-1)
        pages = i["tables"][:, full]
        source, target = parents.view(-1)[again.view(-1)], slots[free]
        tables[:, full] = pages[parents]
        tables[slots[again], full] = pages[target]
        tokens = -(-rest // 32) * 32
        block = c["dim"] * tokens
        for cache in i["caches"]:
            v = cache.view(-1, 2 * c["kv"], c["page"] * c["dim"])
            v[pages[target].long(), :, :block] = v[pages[source].long(), :, :block]
    return {"tables": tables, "history": i["history"][parents], "caches": i["caches"]}


# ---------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def place(c, kind, head, t, d):
    """Element within a page of token t, channel d (keys: kind 0, values: kind 1)."""
    base = (kind * c["kv"] + head) * c["page"] * c["dim"]
    if kind == 0:
        e = 4 if c["dtype"] == "f32" else 8
        return base + t // 16 * 16 * c["dim"] + (d // e * 16 + t % 16) * e + d % e
    if c["dtype"] == "f32":
        return base + t // 16 * 16 * c["dim"] + (t % 16 // 4 * c["dim"] + d) * 4 + t % 4
    return base + t // 32 * 32 * c["dim"] + (t % 16 // 4 * c["dim"] + d) * 8 + t % 32 // 16 * 4 + t % 4


def places(c, kind, head, table, tokens):
    """Elements of the whole storage of these tokens, [tokens][dim]."""
    d = torch.arange(c["dim"], device=DEV)[None]
    page = table[tokens // c["page"]].long()[:, None] * (2 * c["kv"] * c["page"] * c["dim"])
    return page + place(c, kind, head, (tokens % c["page"])[:, None], d)


def exact(case, seed):
    c, f = case, case["family"]
    if f == "reorder":
        return None  # copies only
    i = inputs(c, seed)
    if f == "select":
        x = i["logits"].double()
        cand = i["scores"].double()[:, None] + torch.log_softmax(x, -1)
        for b in torch.nonzero(i["done"])[:, 0].tolist():
            cand[b] = -math.inf
            cand[b, 2] = i["scores"][b].double()
        parents, tokens, scores = [], [], []
        for g in range(c["groups"]):
            flat = cand[g * c["beams"]:(g + 1) * c["beams"]].reshape(-1).cpu().numpy()
            order = (-flat).argsort(kind="stable")[:c["select"]]
            parents.append([g * c["beams"] + int(o) // c["vocab"] for o in order])
            tokens.append([int(o) % c["vocab"] for o in order])
            scores.append([float(flat[o]) for o in order])
        return {"parents": _words(parents), "tokens": _words(tokens),
                "scores": torch.tensor(scores, dtype=torch.float64, device=DEV)}
    cache = i["cache"].double()
    if f == "append":
        q = torch.empty_like(i["q"], dtype=torch.float64)
        j = torch.arange(c["dim"] // 2, device=DEV, dtype=torch.float64)
        row = 0
        for s, n in enumerate(i["n"]):
            if not n:
                continue
            own_at = torch.arange(i["keys"][s] - n, i["keys"][s], device=DEV)
            z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                            (own_at + i["prefix"][s // c["share"]]).double()[:, None] * THETA ** (-2 * j / c["dim"]))
            turned = []
            for x in (i["q"], i["k"]):
                lo, hi = x[row:row + n].double().chunk(2, -1)
                y = torch.complex(lo.contiguous(), hi.contiguous()) * z[:, None]
                turned.append(torch.cat([y.real, y.imag], -1))
            q[row:row + n] = turned[0]
            for h in range(c["kv"]):
                cache[places(c, 0, h, i["tables"][s], own_at)] = turned[1][:, h]
                cache[places(c, 1, h, i["tables"][s], own_at)] = i["v"][row:row + n, h].double()
            row += n
        return {"q": q, "cache": cache}
    out = torch.empty(i["rows"], c["heads"], c["dim"], dtype=torch.float64, device=DEV)
    group, row = c["heads"] // c["kv"], 0
    for s, n in enumerate(i["n"]):
        if not n:
            continue
        prefix, keys = i["prefix"][s // c["share"]], i["keys"][s]
        at = prefix + keys - n + torch.arange(n, device=DEV)[:, None]
        key = torch.arange(prefix + keys, device=DEV)[None]
        hidden = key > at
        if c["window"]:
            hidden |= key <= at - c["window"]
        for h in range(c["kv"]):
            kv = []
            for kind in (0, 1):
                where = [places(c, kind, h, i["tables"][s], torch.arange(keys, device=DEV))]
                if prefix:
                    where.insert(0, places(c, kind, h, i["prefix_tables"][s // c["share"]],
                                           torch.arange(prefix, device=DEV)))
                kv.append(cache[torch.cat(where)])
            for x in range(h * group, (h + 1) * group):
                sc = i["q"][row:row + n, x].double() @ kv[0].T.contiguous() / math.sqrt(c["dim"])
                if c["softcap"]:
                    sc = c["softcap"] * torch.tanh(sc / c["softcap"])
                out[row:row + n, x] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ kv[1]
        row += n
    return {"out": out}

"""The library's host side on a machine without a GPU: its calls run against a stand-in for the HIP runtime
(hip_recorder.cpp), which keeps device memory in host memory, counts kernels instead of running them, and can make an
allocation fail.  Each test is a process of its own, so that the library resolves to the stand-in."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PRELUDE = """
import ctypes, sys
import numpy as np
rec = ctypes.CDLL({stub!r}, ctypes.RTLD_GLOBAL)
for n in ("allocations", "live_bytes", "largest"):
    getattr(rec, "rec_" + n).restype = ctypes.c_uint64
rec.rec_fail_at.argtypes = [ctypes.c_int64]
rec.rec_launched.restype = ctypes.c_char_p
from quicknn_amd import hip

def raises(kind, f, *a, **kw):
    try:
        f(*a, **kw)
    except kind as e:
        return str(e)
    raise AssertionError((kind, a, kw))

ctx = hip.GPUContext(0)
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """host(code): runs it with `hip`, a context `ctx` and the stand-in `rec`."""
    stub = str(tmp_path_factory.mktemp("rec") / "libhip_recorder.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(ROOT, "tests", "hip_recorder.cpp"), "-o",
                    stub], check=True)

    def run(code):
        r = subprocess.run([sys.executable, "-c", PRELUDE.format(stub=stub) + code], cwd=ROOT, capture_output=True, text=True,
                           timeout=120)
        assert r.returncode == 0, r.stdout + r.stderr

    return run


GROW = """
def int4(n, k):
    w = hip.MemoryBlock.int4(np.zeros((n, (k + 31) // 32 * 20), np.uint8))
    ctx.RetainWeight(w, n, w.shape[1])
    return w

def linear(w, k, n):
    ctx.Int4Linear(y, x, w, 1, k, n)

small, large = int4(64, 4096), int4(4096, 9728)
x, y = ctx.NewTensor(9728), ctx.NewTensor(4096)
linear(small, 4096, 64)
ctx.Flush()
"""


def test_an_error_is_reported_once(host):
    """A failed allocation is that call's error, not the next launch's too."""
    host(GROW + """
logits, scores, found = ctx.NewTensor(8000), ctx.NewTensor(4), [ctx.NewTensor(4) for _ in range(3)]
rec.rec_fail_at(0)
assert "out of memory" in raises(hip.EInvalidOp, ctx.BeamSelect, *found, logits, scores, None, 1, 4, 2000, 4)
rec.rec_forget_launched()
linear(small, 4096, 64)
ctx.BeamSelect(*found, logits, scores, None, 1, 4, 2000, 4)
ctx.Flush()
assert rec.rec_launched().count(b"k_beam") == 2 and rec.rec_launched().count(b"\\n") == 3
""")


@pytest.mark.parametrize("which", [0, 1])
def test_a_failed_workspace_leaves_none_behind(host, which):
    """When one of the split-K workspace's two allocations fails, the next call makes a workspace of its own instead of
    taking the one that is gone for there, and the other allocation is not lost."""
    host(GROW + f"""
rec.rec_fail_at({which})
assert "out of memory" in raises(hip.EInvalidOp, linear, large, 9728, 4096)
before = rec.rec_allocations()
linear(small, 4096, 64)
assert rec.rec_allocations() == before + 2
linear(large, 9728, 4096)
ctx.close()
assert rec.rec_live_bytes() == 0
""")


@pytest.mark.parametrize("count,share,heads,kv,dim,rows", [
    (4096, 32, 32, 8, 128, 1), (1000, 1000, 32, 8, 128, 1), (20000, 20000, 32, 8, 128, 1), (512, 8, 64, 2, 128, 1),
    (300, 300, 16, 2, 256, 3), (2000, 50, 8, 8, 64, 2), (8, 8, 32, 8, 128, 700)])
def test_attention_workspace_behind_prefixes(host, count, share, heads, kv, dim, rows):
    """With prefixes the workspace holds, for every column, one part of its own keys and one of its prefix, what each
    of the 512 workgroups of either kind of tile leaves of split items (two parts, of 32 and 128 columns), and tables."""
    host(f"""
n, rows = {count}, {count * rows}
cache = hip.PagedCache(ctx.NewTensor(hip.PagedCache.words(hip.DT_BF16, 4, 64, {kv}, {dim})), hip.DT_BF16, 4, 64, {kv}, {dim})
starts = None if rows == n else ctx.NewTensor(n + 1)
batch = hip.PagedBatch(ctx.NewTensor(n), ctx.NewTensor(n), n, rows, 1, starts=starts,
                       prefix_tables=ctx.NewTensor(n // {share} * 200), prefix_lengths=ctx.NewTensor(n // {share}),
                       prefix_pages=200, share={share})
q, out = ctx.NewTensor(rows * {heads * dim}), ctx.NewTensor(rows * {heads * dim})
rec.rec_forget_largest()
before = rec.rec_allocations()
ctx.PagedAttention(out, q, cache, batch, {heads})
assert rec.rec_allocations() == before + 1
column = 4 * ({dim} + 4)
assert rec.rec_largest() <= (2 * rows * {heads} + 2 * 512 * (32 + 128)) * column + (1 << 20), rec.rec_largest()
""")


def test_results_over_the_batchs_own_data_are_refused(host):
    """Kernels read tables, lengths and starts many times in a call: a result over them would change them meanwhile."""
    host("""
B = hip.DT_BF16
words = hip.PagedCache.words(B, 8, 64, 2, 64)
big = dict(tables=8, lengths=4, starts=5, prefix_tables=4, prefix_lengths=2)
t = {n: ctx.NewTensor(words) for n in big}
cache = hip.PagedCache(ctx.NewTensor(words), B, 8, 64, 2, 64)
q, k, v, out, parents = (ctx.NewTensor(4 * 4 * 64) for _ in range(5))

def batch(**kw):
    return hip.PagedBatch(**{**dict(t, sequences=4, rows=4, table_pages=2, prefix_pages=2, share=2), **kw})

b = batch()
ctx.PagedAttention(out, q, cache, b, 4)
ctx.PagedAppend(cache, b, k, v, q, out, 4, 1e4)
ctx.PagedAdvance(b, 64)
ctx.PagedReorder(b, out, parents, [cache])
A = hip.EArgumentException
for name, x in t.items():
    raises(A, ctx.PagedAttention, x, q, cache, b, 4)
    raises(A, ctx.PagedAppend, cache, b, k, v, q, x, 4, 1e4)
    raises(A, ctx.PagedReorder, b, x, parents, [cache])
    if name != "lengths":
        raises(A, ctx.PagedAdvance, batch(lengths=x), 64)
    inside = hip.PagedCache(x, B, 8, 64, 2, 64)
    raises(A, ctx.PagedAppend, inside, b, k, v, q, out, 4, 1e4)
    raises(A, ctx.PagedReorder, b, out, parents, [cache, inside])
ctx.Flush()
""")


def test_selection_of_the_largest_vocabulary(host):
    """The workspace of a vocabulary within a tile of 2^31 tokens: 8 bytes per 1024."""
    host("""
vocab = 2 ** 31 - 1
logits, scores, found = ctx.NewTensor(vocab), ctx.NewTensor(1), [ctx.NewTensor(4) for _ in range(3)]
rec.rec_forget_largest()
ctx.BeamSelect(*found, logits, scores, None, 1, 1, vocab, 4)
assert rec.rec_largest() == 2 ** 21 * 8, rec.rec_largest()
""")


@pytest.mark.parametrize("rows,cols", [(1 << 24, 1), (2 ** 31 - 1, 1), (20_000_003, 100), (1, 2 ** 31 - 1)])
def test_gather_of_many_rows(host, rows, cols):
    """As many rows as tensors hold, in one launch."""
    host(f"""
dst, src, indices = ctx.NewTensor({rows * cols}), ctx.NewTensor({cols}), ctx.NewTensor({rows})
ctx.GatherRows(dst, src, indices, {rows}, {cols})
ctx.Flush()
assert rec.rec_launched().count(b"k_gather_rows") == 1
""")


def test_reorder_of_tables_past_32_bits_is_refused(host):
    """64 sequences with 2^25 - 1 pages each: the copy of their tables steps past 2^31."""
    host("""
pages = 2 ** 25 - 1
cache = hip.PagedCache(ctx.NewTensor(hip.PagedCache.words(hip.DT_BF16, 1, 32, 1, 16)), hip.DT_BF16, 1, 32, 1, 16)
tables, new, lengths, parents = (ctx.NewTensor(n) for n in (64 * pages, 64 * pages, 64, 64))
raises(hip.ERangeError, ctx.PagedReorder, hip.PagedBatch(tables, lengths, 64, 64, pages, share=64), new, parents, [cache])
ctx.PagedReorder(hip.PagedBatch(tables, lengths, 64, 64, 2 ** 24, share=64), new, parents, [cache])
ctx.Flush()
""")


def test_descriptors_follow_their_attributes(host):
    """What is set on a cache's or batch's description after its making is what the next call takes."""
    host("""
a, b, q, out = (ctx.NewTensor(n) for n in (8 * 64 * 64, 8, 4 * 64, 4 * 64))
cache = hip.PagedCache(a, hip.DT_F32, 4, 64, 1, 64)
batch = hip.PagedBatch(b, b, 4, 4, 1)
ctx.PagedAttention(out, q, cache, batch, 1)
batch.rows = 3
raises(hip.EArgumentException, ctx.PagedAttention, out, q, cache, batch, 1)
batch.starts = b
ctx.PagedAttention(out, q, cache, batch, 1)
batch.starts, batch.rows, batch.tables = None, 4, None
raises(hip.EArgumentException, ctx.PagedAttention, out, q, cache, batch, 1)
batch.tables = b
ctx.PagedAttention(out, q, cache, batch, 1)
cache.page_count = 5
raises(hip.EArgumentException, ctx.PagedAttention, out, q, cache, batch, 1)
raises(AttributeError, setattr, batch, "length", b)
assert (batch.rows, batch.tables, cache.page_count) == (4, b, 5)
import copy
other = copy.copy(cache)
other.page_count = 4
assert cache._c.page_count == 5
ctx.PagedAttention(out, q, other, batch, 1)
ctx.Flush()
""")


def test_outgrown_workspaces_that_no_graph_uses_are_freed(host):
    """A workspace outlives its growth only if a graph was captured with it, not because there is a graph."""
    host(GROW + """
logits, scores, found = ctx.NewTensor(64 << 20), ctx.NewTensor(1), [ctx.NewTensor(4) for _ in range(3)]
def select(vocab):
    ctx.BeamSelect(*found, logits, scores, None, 1, 1, vocab, 4)
select(1 << 20)
before = rec.rec_live_bytes()
ctx.GraphBegin()
select(1 << 20)
graph = ctx.GraphEnd()
for i in range(2, 64):
    select(i << 20)
grown = 63 << 13
assert rec.rec_live_bytes() == before + grown, (rec.rec_live_bytes() - before, grown)  # the graph's, and the last
ctx.GraphLaunch(graph)
before = rec.rec_live_bytes()
linear(large, 9728, 4096)  # outgrows the split-K workspace, which no graph has
assert rec.rec_live_bytes() > before
ctx.GraphBegin()
linear(large, 9728, 4096)
ctx.GraphEnd()
kept = rec.rec_live_bytes()
larger = int4(9728, 9728)
y = ctx.NewTensor(9728)
middle = rec.rec_live_bytes()
linear(larger, 9728, 9728)
linear(small, 4096, 64)
assert rec.rec_live_bytes() > middle
ctx.Recycle(found[0])
ctx.close()
assert rec.rec_live_bytes() == 0
""")

"""Sparse decode on the GPU: the key index, the choice of pages and attention over listed pages, against
plain 64-bit implementations over the values that the pool holds (its bytes, decoded here).

Bounds and lists are whole numbers or one rounding from them: compared bit for bit. Attention: a score
is a sum of D rounded products, in log2 units with an error of about sqrt(D) 2^-24 S, S the largest sum of
their magnitudes (8 times that is allowed); p, its two fp16 parts and the sums of p add less than 2^-20. An
output is a mean of the values with weights off by that much: max |v| (8 sqrt(D) 2^-24 S + 2^-20)."""
import ctypes as C
import math
import os

import numpy as np
import pytest

import pyoracle as O
import velokv
from velokv import synth

pytestmark = pytest.mark.gpu
KVS = [O.F32, O.F16, O.I8_REF, O.I8_BLK]


class Cache:
    """A one-layer pool with the given contexts in scattered pages, and what it holds as fp64 values."""

    def __init__(self, ctx, kv, lens, n_kv_heads=2, head_dim=128, page=16, seed=1, spread=1.0):
        self.ctx, self.lens, self.page, self.hkv, self.hd = ctx, np.asarray(lens, np.int32), page, n_kv_heads, head_dim
        pages = [-(-int(n) // page) for n in lens]
        self.n_pages = sum(pages) + 5
        self.table = synth.scatter_block_tables(self.n_pages, pages, seed, stride=max(pages + [1]) + 1)
        self.pool = velokv.Pool(ctx, 1, self.n_pages, page, n_kv_heads, head_dim, kv)
        r = synth.rng(seed)
        for s, n in enumerate(lens):
            if n:
                topic = np.repeat(r.standard_normal((pages[s], n_kv_heads, head_dim)), page, 0)[:n]
                k = ((r.standard_normal((n, n_kv_heads, head_dim)) + topic) * spread).astype(np.float16)
                v = r.standard_normal(k.shape).astype(np.float16)
                self.append(s, np.arange(n), k, v)
        self.read()

    def append(self, s, pos, k, v):
        slots = synth.slots_for_positions(self.table, pos, self.page, np.full(len(pos), s))
        self.ctx.append(self.pool, 0, self.ctx.upload(k), self.ctx.upload(v), velokv.DT_F16, self.ctx.upload(slots), len(pos))
        self.ctx.sync()

    def read(self):
        """self.k, self.v: fp64 [tiles][heads][16][head_dim]; self.k32: the keys as fp32 holds them."""
        kv, got, w = self.pool.kv_type, self.pool.download_layer(0), 64 if self.hd <= 64 else 128
        t, h = self.n_pages * self.page // 16, self.hkv
        kind = {O.F32: np.float32, O.F16: np.float16}.get(kv, np.int8)
        k, v = got["k"].view(kind), got["v"].view(kind).reshape(t, h, 8, w, 2).transpose(0, 1, 2, 4, 3).reshape(t, h, 16, w)
        if kind == np.int8:
            k = k.reshape(t, h, 2, 16, w // 32, 16).transpose(0, 1, 3, 4, 2, 5)
        k = k.reshape(t, h, 16, w)
        out = []
        for x, name in ((k, "ks"), (v, "vs")):
            x = x.astype(np.float64)
            if kv == O.I8_BLK:
                x = x * got[name].view(np.float16).astype(np.float64).reshape(t, h, 1, 1)
            if kv == O.I8_REF:
                x = x * got[name].view(np.float32).astype(np.float64).reshape(t, h, 16, 1)
            out.append(x[..., :self.hd])
        self.k, self.v = out
        self.k32 = self.k.astype(np.float32)

    def tokens(self, x, s, pages, h):
        """Rows of x at places `pages` of sequence s, one KV head: [tokens][head_dim]."""
        per = self.page // 16
        tiles = (self.table[s, pages].astype(np.int64)[:, None] * per + np.arange(per)).reshape(-1)
        return x[tiles, h].reshape(-1, self.hd)

    def dev(self, rows=None, lens=None):
        lens = self.lens if lens is None else np.asarray(lens, np.int32)
        return dict(block_tables=self.ctx.upload(self.table), bt_stride=self.table.shape[1], context_lens=self.ctx.upload(lens),
                    n_seqs=len(lens), max_context_len=int(max(lens.max(initial=0), 0)),
                    seq_rows=None if rows is None else self.ctx.upload(np.asarray(rows, np.int32)))


def code_parts(x):
    """Scale and inverse of the largest magnitude of the last axis, in fp32."""
    top = np.abs(x).max(-1).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.float32(127) / top
    return top / np.float32(127), np.where(np.isfinite(inv), inv, 0).astype(np.float32)


def bounds(c, s, page, h, n_tok):
    """Codes of the lower and the upper bound, and the scale."""
    k = c.tokens(c.k32, s, [page], h)[:n_tok]
    lo, hi = k.min(0), k.max(0)
    scale, inv = code_parts(np.concatenate([lo, hi]))
    return np.rint(lo * inv), np.rint(hi * inv), scale


def read_index(c, index, pages):
    ctx, shape = c.ctx, (len(pages), c.hkv, c.hd)
    lower, upper = ctx.alloc(4 * int(np.prod(shape))), ctx.alloc(4 * int(np.prod(shape)))
    ctx.index_read(index, 0, ctx.upload(np.asarray(pages, np.int32)), len(pages), lower, upper)
    ctx.sync()
    return lower.download(shape, np.float32), upper.download(shape, np.float32)


def check_index(c, index, lens=None):
    for s, n in enumerate(c.lens if lens is None else lens):
        for p in range(-(-int(n) // c.page)):
            lower, upper = read_index(c, index, [c.table[s, p]])
            for h in range(c.hkv):
                lo, hi, scale = bounds(c, s, p, h, min(c.page, int(n) - p * c.page))
                assert np.array_equal(lower[0, h], (lo * scale).astype(np.float32)), (s, p, h)
                assert np.array_equal(upper[0, h], (hi * scale).astype(np.float32)), (s, p, h)


@pytest.mark.parametrize("head_dim,page", [(128, 16), (96, 48), (64, 32), (40, 16)])
@pytest.mark.parametrize("kv", KVS)
def test_index_update(ctx, kv, head_dim, page):
    """Whole contexts, the last page partly filled; then three more tokens a sequence, brought up to date alone."""
    c = Cache(ctx, kv, [1, page, 2 * page + 7, 0, 5 * page - 1], head_dim=head_dim, page=page, seed=3)
    index = velokv.KeyIndex(ctx, c.pool)
    assert index.nbytes >= c.n_pages * 2 * (2 * head_dim + 4)
    ctx.index_update(index, 0, **c.dev())
    ctx.sync()
    check_index(c, index)
    shorter = np.maximum(c.lens - 3, 0)
    fresh = velokv.KeyIndex(ctx, c.pool)
    d = c.dev()
    ctx.index_update(fresh, 0, **c.dev(lens=shorter))
    ctx.sync()
    check_index(c, fresh, shorter)
    ctx.index_update(fresh, 0, first_tokens=ctx.upload(shorter.astype(np.int32)), max_tokens=3, **d)
    ctx.sync()
    check_index(c, fresh)


@pytest.mark.parametrize("kv", [O.F32, O.F16])
def test_index_of_special_keys(ctx, kv):
    """Zero keys, keys below fp32's inverse, infinities and NaN; what lies past the context does not count."""
    c = Cache(ctx, kv, [16 * 6 - 4], seed=5)
    k = np.ones((16 * 6, c.hkv, c.hd), np.float16)
    k[:16] = 0
    k[20, 0, 3], k[37, 1, 5] = np.inf, np.nan
    k[48:64] = 6e-8  # one fp16 step
    k[16 * 6 - 4:] = np.nan
    c.append(0, np.arange(16 * 6), k, k)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    lower, upper = read_index(c, index, c.table[0, :6])
    assert np.all(lower[0] == 0) and np.all(upper[0] == 0)
    for page, h in ((1, 0), (2, 1)):
        assert np.all(lower[page, h] == -np.inf) and np.all(upper[page, h] == np.inf)
        assert np.all(lower[page, 1 - h] == 1) and np.all(upper[page, 1 - h] == 1)
    step = np.float32(np.float16(6e-8))
    assert np.all(lower[3] == np.float32(127) * (step / np.float32(127))) and np.all(lower[4:] == 1) and np.all(upper[4:] == 1)


def choose(c, q, lens, rows, n_list, n_first, n_last):
    """Lists [S][Hkv][n_list] from the pool's keys and q."""
    known = {}  # a page's bounds, by what they depend on
    out = np.full((len(lens), c.hkv, n_list), -1, np.int32)
    g = q.shape[1] // c.hkv
    q_scale, q_inv = code_parts(q.astype(np.float32))
    code = np.rint(q.astype(np.float32) * q_inv[..., None]).astype(np.int64)
    for s, n in enumerate(lens):
        pages = -(-int(n) // c.page)
        if pages <= n_list:
            out[s, :, :pages] = np.arange(pages)
            continue
        for h in range(c.hkv):
            score = np.zeros(pages, np.float32)
            for p in range(pages):
                at = (rows[s], p, h, min(c.page, int(n) - p * c.page))
                if at not in known:
                    known[at] = bounds(c, *at)
                lo, hi, scale = known[at]
                x = code[s, h * g:(h + 1) * g]
                dot = np.where(x < 0, x * lo.astype(np.int64), x * hi.astype(np.int64)).sum(-1)
                score[p] = ((dot.astype(np.float32) * scale) * q_scale[s, h * g:(h + 1) * g]).max()
            score[:n_first] = np.inf
            score[pages - n_last:] = np.inf if n_last else score[pages - n_last:]
            out[s, h] = np.sort(np.lexsort((np.arange(pages), -score))[:n_list])
    return out


def queries(c, n, heads, q_dtype, seed=9):
    return synth.rng(seed).standard_normal((n, heads, c.hd)).astype(q_dtype)


def dt(q):
    return velokv.DT_F32 if q.dtype == np.float32 else velokv.DT_F16


def select(c, index, q, lens, rows, n_list, n_first=1, n_last=1, **kw):
    pages = c.ctx.upload(np.full((len(lens), c.hkv, n_list), 77, np.int32))
    c.ctx.select_pages(index, 0, c.ctx.upload(q), dt(q), pages, n_list, n_heads=q.shape[1], n_first=n_first, n_last=n_last,
                       **c.dev(rows, lens), **kw)
    c.ctx.sync()
    return pages.download((len(lens), c.hkv, n_list), np.int32)


@pytest.mark.parametrize("group,head_dim,page,kv", [(1, 128, 16, O.F16), (4, 128, 16, O.I8_BLK), (7, 64, 32, O.I8_REF),
                                                    (20, 128, 16, O.F32), (32, 40, 16, O.F16), (16, 96, 48, O.I8_BLK)])
@pytest.mark.parametrize("q_dtype", [np.float16, np.float32])
def test_select_pages(ctx, group, head_dim, page, kv, q_dtype):
    """Contexts from none to 75 pages, one table row queried at several lengths, lists of several lengths."""
    c = Cache(ctx, kv, [0, 1, 40 * page + 3, 75 * page, 12 * page - 1], head_dim=head_dim, page=page, seed=group)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    rows, lens = [0, 1, 2, 3, 4, 3, 3], [int(n) for n in c.lens] + [75 * page, 20 * page]  # (whole pages: the index's bounds hold)
    q = queries(c, len(rows), 2 * group, q_dtype)
    for n_list, n_first, n_last in ((1, 0, 0), (5, 1, 1), (12, 3, 4), (33, 0, 1), (80, 1, 1)):
        got = select(c, index, q, lens, rows, n_list, n_first, n_last)
        ref = choose(c, q, lens, rows, n_list, n_first, n_last)
        assert np.array_equal(got, ref), (n_list, n_first, n_last)


@pytest.mark.parametrize("group,head_dim,page,kv", [(1, 128, 16, O.I8_BLK), (8, 64, 16, O.F16), (20, 96, 32, O.I8_REF), (24, 40, 16, O.F32)])
def test_select_pages_of_many_rows(ctx, group, head_dim, page, kv):
    """As many (row, KV head)s as CUs and more: the loads take another order. Queries of one table row at many
    lengths among them (whole pages: the index's bounds hold)."""
    c = Cache(ctx, kv, [70 * page, 9 * page + 1], head_dim=head_dim, page=page, seed=31)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    rows = [0] * 160 + [1] * 3
    lens = [page * (1 + i % 70) for i in range(160)] + [int(c.lens[1])] * 3
    q = queries(c, len(rows), 2 * group, np.float16)
    for n_list in (7, 30):
        assert np.array_equal(select(c, index, q, lens, rows, n_list), choose(c, q, lens, rows, n_list, 1, 1))


def test_select_long_contexts_of_some(ctx):
    """40 (row, KV head)s of up to 2500 pages: several turns of a wave, one launch."""
    c = Cache(ctx, O.F16, [16 * 2500 - 5], n_kv_heads=2, head_dim=64, seed=32)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    lens = [16 * 2500 - 5] + [16 * (100 * i + 70) for i in range(1, 20)]
    q = queries(c, 20, 4, np.float32)
    assert np.array_equal(select(c, index, q, lens, [0] * 20, 100), choose(c, q, lens, [0] * 20, 100, 1, 1))


def test_select_ties_and_special_scores(ctx):
    """Equal pages: the lowest are listed. Pages that are not finite come first; a query that is not finite scores all alike."""
    c = Cache(ctx, O.F16, [16 * 300], seed=2)
    one = np.ones((16 * 300, c.hkv, c.hd), np.float16)
    c.append(0, np.arange(16 * 300), one, one)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    q = queries(c, 1, 4, np.float16)
    assert np.array_equal(select(c, index, q, c.lens, [0], 40, 0, 0), np.broadcast_to(np.arange(40), (1, 2, 40)))
    k = one[:16].copy()
    k[3] = np.inf
    for p in (211, 17):
        c.append(0, np.arange(16 * p, 16 * p + 16), k, one[:16])
    ctx.index_update(index, 0, **c.dev())
    assert np.array_equal(select(c, index, q, c.lens, [0], 4, 1, 0)[0, 0], [0, 1, 17, 211])
    q[:] = np.nan
    assert np.array_equal(select(c, index, q, c.lens, [0], 4, 0, 0)[0, 0], [0, 1, 17, 211])
    q[:] = 0
    assert np.array_equal(select(c, index, q, c.lens, [0], 4, 0, 1)[0, 0], [0, 17, 211, 299])


def test_select_long_context(ctx):
    """More pages than a workgroup's threads many times over, and a list of 700."""
    c = Cache(ctx, O.I8_BLK, [16 * 5000 - 3], n_kv_heads=1, head_dim=64, seed=8)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    q = queries(c, 1, 4, np.float16)
    assert np.array_equal(select(c, index, q, c.lens, [0], 700), choose(c, q, c.lens, [0], 700, 1, 1))


def attend(c, q, lists, lens, rows, scale=None):
    """fp64 outputs and the bound on their error."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape[:2] + (1,))
    g, scale = q.shape[1] // c.hkv, scale or 1 / math.sqrt(c.hd)
    for s, n in enumerate(lens):
        for h in range(c.hkv):
            at = [p for p in lists[s, h].tolist() if 0 <= p and p * c.page < n]
            if not at:
                continue
            at = np.array(at)
            ok = ((at[:, None] * c.page + np.arange(c.page)) < n).reshape(-1)
            k, v = c.tokens(c.k, rows[s], at, h)[ok], c.tokens(c.v, rows[s], at, h)[ok]
            x = q[s, h * g:(h + 1) * g].astype(np.float64)
            sc = x @ k.T * scale
            p = np.exp(sc - sc.max(-1, keepdims=True))
            out[s, h * g:(h + 1) * g] = p @ v / p.sum(-1, keepdims=True)
            big = (np.abs(x) @ np.abs(k).T).max() * scale * math.log2(math.e)
            tol[s, h * g:(h + 1) * g] = np.abs(v).max() * (8 * math.sqrt(c.hd) * 2.0 ** -24 * big + 2.0 ** -20)
    return out, tol


def sparse(c, q, lists, lens, rows, **kw):
    ctx = c.ctx
    out = ctx.upload(np.full(q.shape, np.nan, np.float32))
    ctx.sparse_decode(c.pool, 0, ctx.upload(q), dt(q), out, ctx.upload(np.ascontiguousarray(lists, np.int32)), lists.shape[2],
                      n_heads=q.shape[1], **c.dev(rows, lens), **kw)
    ctx.sync()
    return out.download(q.shape, np.float32)


def close(got, want):
    ref, tol = want
    err = np.abs(got - ref)
    assert np.all(err <= tol), f"max err {err.max():.3g}, allowed there {np.broadcast_to(tol, err.shape).flat[err.argmax()]:.3g}"


def some_lists(c, lens, n, seed=4):
    """Random places, some past the context, some -1, some twice, in no order."""
    r, out = synth.rng(seed), np.full((len(lens), c.hkv, n), -1, np.int32)
    for s, length in enumerate(lens):
        for h in range(c.hkv):
            pages = -(-int(length) // c.page)
            x = r.integers(-1, pages + 2, n)
            x[r.random(n) < 0.1] = 2 ** 31 - 1
            if pages and n > 2:
                x[1] = pages - 1
            out[s, h] = x
    return out


@pytest.mark.parametrize("group,head_dim,page", [(1, 128, 16), (4, 128, 48), (7, 64, 16), (16, 96, 32), (20, 128, 16), (32, 40, 16)])
@pytest.mark.parametrize("q_dtype", [np.float16, np.float32])
@pytest.mark.parametrize("kv", KVS)
def test_sparse_decode(ctx, kv, q_dtype, group, head_dim, page):
    print(f"sparse decode kv={kv} q={np.dtype(q_dtype).name} group={group} head_dim={head_dim} page={page}", flush=True)
    c = Cache(ctx, kv, [0, 1, page, 30 * page + 5, 9 * page - 1], head_dim=head_dim, page=page, seed=20 + group, spread=1.5)
    rows, lens = [0, 1, 2, 3, 4, 3, 4], [int(n) for n in c.lens] + [7 * page + 2, 0]
    q = queries(c, len(rows), 2 * group, q_dtype)
    for n in (1, 6, 25):
        lists = some_lists(c, lens, n)
        got = sparse(c, q, lists, lens, rows)
        close(got, attend(c, q, lists, lens, rows))
        assert np.all(got[[0, 6]] == 0)  # no context
    lists[:] = -1
    assert np.all(sparse(c, q, lists, lens, rows) == 0)


@pytest.mark.parametrize("rows,group,head_dim", [(140, 4, 128), (270, 4, 128), (270, 3, 64)])
@pytest.mark.parametrize("kv", KVS)
def test_sparse_decode_many_rows(ctx, kv, rows, group, head_dim):
    """More (row, KV head)s than CUs, and more than twice as many: a list is one workgroup's, of eight waves or four."""
    c = Cache(ctx, kv, [16 * 20 + 3, 5], head_dim=head_dim, seed=33)
    at, lens = [i % 2 for i in range(rows)], [int(c.lens[0]) - i if i % 2 == 0 else 5 for i in range(rows)]
    q = queries(c, rows, 2 * group, np.float16)
    lists = some_lists(c, lens, 15)
    close(sparse(c, q, lists, lens, at), attend(c, q, lists, lens, at))


@pytest.mark.parametrize("kv", KVS)
def test_sparse_decode_long_lists(ctx, kv):
    """A list of 1100 entries (several parts of 512 at most) for one sequence, another of one token beside it."""
    c = Cache(ctx, kv, [16 * 1200 - 9, 1], seed=6)
    q = queries(c, 2, 8, np.float16)
    lists = np.full((2, 2, 1100), -1, np.int32)
    lists[0, 0], lists[0, 1] = np.arange(100, 1200), np.arange(1100)
    lists[1, :, 900] = 0
    close(sparse(c, q, lists, c.lens, [0, 1], scale=0.05), attend(c, q, lists, c.lens, [0, 1], 0.05))


def test_sparse_decode_value_scales(ctx):
    """int8 values of scales from 2^-14 to 100 in one context keep the precision of their own."""
    c = Cache(ctx, O.I8_BLK, [16 * 24], seed=7)
    r = synth.rng(1)
    k = r.standard_normal((16 * 24, c.hkv, c.hd)).astype(np.float16)
    size = np.repeat(2.0 ** r.integers(-7, 13, 24), 16)[:, None, None]
    c.append(0, np.arange(16 * 24), k, (r.standard_normal(k.shape) * size).astype(np.float16))
    c.read()
    q = queries(c, 1, 8, np.float16)
    lists = np.broadcast_to(np.arange(24, dtype=np.int32), (1, 2, 24))
    close(sparse(c, q, lists, c.lens, [0]), attend(c, q, lists, c.lens, [0]))
    small = np.nonzero(size[::16, 0, 0] < 1)[0].astype(np.int32)
    lists = np.broadcast_to(small, (1, 2, len(small)))
    close(sparse(c, q, lists, c.lens, [0]), attend(c, q, lists, c.lens, [0]))


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** -40])
@pytest.mark.parametrize("kv", KVS)
def test_sparse_decode_query_sizes(ctx, kv, size):
    """fp32 queries past fp16's largest value and far below its least, one row's heads apart by 2^8."""
    c = Cache(ctx, kv, [16 * 20 + 3], seed=35)
    q = (queries(c, 1, 8, np.float32) * (size * 2.0 ** np.arange(0, -8, -1))[None, :, None]).astype(np.float32)
    lists = some_lists(c, c.lens, 15)
    scale = 1 / (size * math.sqrt(c.hd))
    close(sparse(c, q, lists, c.lens, [0], scale=scale), attend(c, q, lists, c.lens, [0], scale))


@pytest.mark.parametrize("kv", KVS)
def test_what_lies_past_the_context(ctx, kv):
    """Infinite and NaN rows in the last page past the context do not reach the result."""
    c = Cache(ctx, kv, [16 * 3 + 5], seed=11)
    bad = np.full((11, c.hkv, c.hd), np.nan, np.float16)
    bad[::2] = np.inf
    if kv != O.I8_BLK:  # there a block's scale is its rows' own
        c.append(0, np.arange(16 * 3 + 5, 16 * 4), bad, bad)
    c.read()
    q = queries(c, 1, 8, np.float32)
    lists = np.broadcast_to(np.arange(4, dtype=np.int32), (1, 2, 4))
    close(sparse(c, q, lists, c.lens, [0]), attend(c, q, lists, c.lens, [0]))


def test_bad_page_ids_are_reported(ctx):
    """Ids outside the pool: read clamped and reported; the index skips them."""
    c = Cache(ctx, O.F16, [16 * 8], seed=12)
    index = velokv.KeyIndex(ctx, c.pool)
    c.table[0, 3], c.table[0, 5] = -4, c.n_pages
    lists = np.broadcast_to(np.arange(8, dtype=np.int32), (1, 2, 8))
    q = queries(c, 1, 8, np.float16)
    for call in (lambda: ctx.index_update(index, 0, **c.dev()), lambda: select(c, index, q, c.lens, [0], 4),
                 lambda: sparse(c, q, lists, c.lens, [0]), lambda: read_index(c, index, [0, c.n_pages])):
        flags = 0
        try:
            call()
        except velokv.VkError as e:
            assert e.code == velokv.ERR_BAD_ARG
            flags = velokv.MISUSE_PAGE_OUT_OF_POOL
        assert (flags | ctx.check_misuse()) == velokv.MISUSE_PAGE_OUT_OF_POOL
    c.table[0, 3] = 0
    lists = np.full((1, 2, 8), 0, np.int32)  # the other bad page is not listed
    assert np.all(np.isfinite(sparse(c, q, lists, c.lens, [0])))


@pytest.mark.parametrize("kv,page", [(O.F16, 16), (O.I8_BLK, 64)])
def test_select_decode(ctx, kv, page):
    """The call of both equals its parts; a list that holds the whole context equals the dense decode."""
    c = Cache(ctx, kv, [page * 40 + 1, 17, page * 33], n_kv_heads=2, page=page, seed=13)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    q = queries(c, 3, 8, np.float16)
    for n_list in (9, 50):
        pages, out = ctx.alloc(3 * 2 * n_list * 4), ctx.alloc(q.size * 4)
        ctx.select_decode(index, 0, ctx.upload(q), velokv.DT_F16, out, pages, n_list, n_heads=8, **c.dev())
        ctx.sync()
        lists = select(c, index, q, c.lens, [0, 1, 2], n_list)
        assert np.array_equal(pages.download(lists.shape, np.int32), lists)
        got = out.download(q.shape, np.float32)
        assert np.array_equal(got, sparse(c, q, lists, c.lens, [0, 1, 2]))
        close(got, attend(c, q, lists, c.lens, [0, 1, 2]))
    dense = ctx.alloc(q.size * 4)
    ctx.paged_decode(c.pool, 0, ctx.upload(q), velokv.DT_F16, dense, n_heads=8, **c.dev())
    ctx.sync()
    dense = dense.download(q.shape, np.float32)
    assert np.all(np.abs(got - dense) <= 2e-3 + 1e-2 * np.abs(dense))  # the dense decode's own tolerance


def test_decode_steps_together(ctx):
    """Prompts, then decode steps as a program runs them: rope and append, the index, selection and attention,
    logits from the outputs, the next token's log probability. Each step against 64 bits."""
    page, hkv, heads, hd, vocab, n_list = 16, 2, 8, 128, 1000, 6
    lens0 = np.array([150, 31, 16], np.int32)
    c = Cache(ctx, O.I8_BLK, lens0 + 6, n_kv_heads=hkv, page=page, seed=14)  # room for six more tokens
    r = synth.rng(15)
    rope = ctx.upload(velokv.rope_table(256, hd, 10000.0))
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev(lens=lens0))
    w_out = r.standard_normal((heads * hd, vocab)) / 32
    stream = velokv.Stream(ctx)
    for step in range(6):
        lens = lens0 + step + 1
        pos = (lens - 1).astype(np.int32)
        d = c.dev(lens=lens)
        q = ctx.upload(queries(c, 3, heads, np.float16, seed=100 + step))
        k, v = (ctx.upload(r.standard_normal((3, hkv, hd)).astype(np.float16)) for _ in range(2))
        slots = ctx.upload(synth.slots_for_positions(c.table, pos.astype(np.int64), page))
        pages, out, at = ctx.alloc(3 * hkv * n_list * 4), ctx.alloc(3 * heads * hd * 4), ctx.upload(pos)
        ctx.sync()
        ctx.append_rope(c.pool, 0, k, v, velokv.DT_F16, at, slots, 3, rope, 256, velokv.ROPE_HALF, q=q, n_heads=heads, stream=stream)
        ctx.index_update(index, 0, first_tokens=at, max_tokens=1, stream=stream, **d)
        ctx.select_decode(index, 0, q, velokv.DT_F16, out, pages, n_list, n_heads=heads, stream=stream, **d)
        stream.sync()
        c.read()
        q = q.download((3, heads, hd), np.float16)
        lists = pages.download((3, hkv, n_list), np.int32)
        assert np.array_equal(lists, choose(c, q, lens, [0, 1, 2], n_list, 1, 1))
        got = out.download(q.shape, np.float32)
        close(got, attend(c, q, lists, lens, [0, 1, 2]))
        logits = (got.reshape(3, -1) @ w_out).astype(np.float32)
        ids, top = ctx.alloc(3 * 4), ctx.alloc(3 * 4)
        ctx.token_logprobs(ctx.upload(logits), velokv.DT_F32, 3, vocab, top_ids=ids, top_logprobs=top, n_top=1)
        ctx.sync()
        x = logits.astype(np.float64)
        x -= x.max(-1, keepdims=True) + np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True))
        assert np.array_equal(ids.download((3,), np.int32), logits.argmax(-1))
        assert np.all(np.abs(top.download((3,), np.float32) - x.max(-1)) <= 2e-6 * (1 + np.abs(x.max(-1))))


class Graph:
    """Launches captured from a stream (the HIP runtime that the library is linked to)."""

    def __init__(self, stream):
        self.hip, self.stream = C.CDLL(os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "libamdhip64.so")), stream
        self.graph, self.exec = C.c_void_p(), C.c_void_p()

    def __enter__(self):
        assert self.hip.hipStreamBeginCapture(self.stream.h, 1) == 0
        return self

    def __exit__(self, *exc):
        rc = self.hip.hipStreamEndCapture(self.stream.h, C.byref(self.graph))
        if exc[0] is None:
            assert rc == 0
            assert self.hip.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, C.c_size_t(0)) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream.h) == 0
        self.stream.sync()

    def close(self):
        self.hip.hipGraphExecDestroy(self.exec)
        self.hip.hipGraphDestroy(self.graph)


def test_captured_steps_replay(ctx):
    """index_update and select_decode in a captured graph, replayed as the inputs change, beside eager calls of
    other shapes; the capture has a workspace of its own, and without one that is at hand it is refused."""
    c = Cache(ctx, O.F16, [16 * 900, 16 * 50], seed=16)
    index = velokv.KeyIndex(ctx, c.pool)
    d = c.dev()
    host_lens = np.array([16 * 880, 16 * 40], np.int32)
    ctx.index_update(index, 0, **d)
    lens = d["context_lens"] = ctx.upload(host_lens)
    q, pages, out = ctx.upload(queries(c, 2, 8, np.float16)), ctx.alloc(2 * 2 * 32 * 4), ctx.alloc(2 * 8 * 128 * 4)
    fresh = velokv.Context(0)  # holds no scratch yet
    pool2 = velokv.Pool(fresh, 1, 64, 16, 2, 128, O.F16)
    index2 = velokv.KeyIndex(fresh, pool2)
    need = ctx.sparse_workspace_bytes(c.pool, 2, 8, d["max_context_len"], 32, bt_stride=d["bt_stride"])
    ws, stream = ctx.alloc(need), velokv.Stream(ctx)
    ctx.sync()
    with Graph(stream) as graph:
        ctx.index_update(index, 0, stream=stream, **d)
        ctx.select_decode(index, 0, q, velokv.DT_F16, out, pages, 32, n_heads=8, workspace=ws, workspace_bytes=need, stream=stream, **d)
        with pytest.raises(velokv.VkError) as e:
            fresh.select_decode(index2, 0, q, velokv.DT_F16, out, pages, 700, stream=stream, n_heads=8, context_lens=lens, n_seqs=2,
                                max_context_len=640, block_tables=d["block_tables"], bt_stride=40)
        assert "workspace" in str(e.value)
    for step in range(4):
        host_lens = host_lens + 48 + step
        host_q = queries(c, 2, 8, np.float16, seed=50 + step)
        lens.upload(host_lens.astype(np.int32))
        q.upload(host_q)
        graph.replay()
        lists = pages.download((2, 2, 32), np.int32)
        close(out.download(host_q.shape, np.float32), attend(c, host_q, lists, host_lens, [0, 1]))
        ctx.select_pages(index, 0, q, velokv.DT_F16, pages, 32, n_heads=8, **d)
        ctx.sync()
        assert np.array_equal(lists, pages.download(lists.shape, np.int32)), step
        sparse(c, queries(c, 1, 4, np.float16, seed=step), np.zeros((1, 2, 700), np.int32), [16 * 50], [1])  # another shape
    graph.close()
    index2.close()
    pool2.close()
    fresh.close()


def test_refusals(ctx):
    c = Cache(ctx, O.F16, [64], seed=17)
    index = velokv.KeyIndex(ctx, c.pool)
    d, q = c.dev(), ctx.upload(queries(c, 1, 8, np.float16))
    pages, out = ctx.alloc(1024), ctx.alloc(8 * 128 * 4)
    good = dict(d, q=q, q_dtype=velokv.DT_F16, pages=pages, n_pages=2, n_heads=8)
    for bad, code in ((dict(n_heads=7), velokv.ERR_BAD_ARG), (dict(n_heads=2 * 33), velokv.ERR_UNSUPPORTED),
                      (dict(n_pages=0), velokv.ERR_BAD_ARG), (dict(n_first=2), velokv.ERR_BAD_ARG),
                      (dict(n_last=-1), velokv.ERR_BAD_ARG), (dict(q_dtype=5), velokv.ERR_BAD_ARG),
                      (dict(max_context_len=10 ** 6), velokv.ERR_BAD_ARG), (dict(q=None), velokv.ERR_BAD_ARG),
                      (dict(pages=None), velokv.ERR_BAD_ARG), (dict(context_lens=None), velokv.ERR_BAD_ARG),
                      (dict(block_tables=None), velokv.ERR_BAD_ARG), (dict(bt_stride=0), velokv.ERR_BAD_ARG),
                      (dict(n_seqs=-1), velokv.ERR_BAD_ARG)):
        with pytest.raises(velokv.VkError) as e:
            ctx.select_pages(index, 0, **{**good, **bad})
        assert e.value.code == code, bad
        if not {"n_first", "n_last"} & set(bad):
            with pytest.raises(velokv.VkError) as e:
                ctx.sparse_decode(c.pool, 0, out=out, **{**good, **bad})
            assert e.value.code == code, bad
    for call in (lambda: ctx.select_pages(index, 1, **good), lambda: ctx.sparse_decode(c.pool, 0, out=None, **good),
                 lambda: ctx.index_update(index, 0, **dict(d, max_tokens=-1)), lambda: ctx.index_update(index, -1, **d),
                 lambda: ctx.index_update(index, 0, **dict(d, context_lens=None)),
                 lambda: ctx.index_read(index, 0, pages, 1, out.ptr + 4, out),
                 lambda: ctx.index_read(index, 0, pages, -1, out, out),
                 lambda: ctx.sparse_decode(c.pool, 0, out=out, workspace=pages, workspace_bytes=4, **dict(good, n_pages=700))):
        with pytest.raises(velokv.VkError) as e:
            call()
        assert e.value.code == velokv.ERR_BAD_ARG
    ctx.select_pages(index, 0, **dict(good, n_seqs=0))
    ctx.index_read(index, 0, None, 0, None, None)
    ctx.sync()

"""Sparse decode and log probabilities at the ends of what their arguments may be."""
import numpy as np
import pytest

import velokv
from test_gpu_logprobs import run
from velokv import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(2, 100), (3, 20000), (2, 70000)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_extreme_scales(ctx, dtype, rows, vocab):
    """The largest scale leaves the row's largest logits alone, equally likely; the least makes all logits equal.
    log n is one fp32 logarithm and product from what is returned: 2^-22 relative is four roundings."""
    x = np.zeros((rows, vocab), dtype)
    x[:, 1::2] = 1
    x[:, 50] = -np.inf
    tokens = np.tile(np.array([0, 1, 50], np.int32), (rows, 1))
    for scale, n, first in ((2.35e38, vocab // 2, -np.inf), (1e-45, vocab - 1, -np.log(vocab - 1))):
        got = run(ctx, x, tokens, 2, scale=scale)
        want = np.array([first, -np.log(n), -np.inf])
        with np.errstate(invalid="ignore"):
            assert np.all((got["token_logprobs"] == want) | (np.abs(got["token_logprobs"] - want) <= 2.0 ** -22 * np.abs(want)))
        assert np.all(np.abs(got["entropy"] - np.log(n)) <= 2.0 ** -22 * np.log(n))
        assert np.array_equal(got["top_ids"], np.tile([1, 3], (rows, 1)))


def test_longest_context(ctx):
    """2^31 - 1 tokens: a table row of 2^27 entries that name page 0 over and over, the page of the largest score
    at `places`, and pages of their own at the end, which are brought up to date by themselves."""
    n, page, hd, last = 2 ** 31 - 1, 16, 64, 2 ** 27 - 1
    pool = velokv.Pool(ctx, 1, 8, page, 1, hd, velokv.KV_F16)
    r = synth.rng(1)
    k = (0.5 + r.random((8 * page, 1, hd))).astype(np.float16)
    k[3 * page:4 * page] *= 4
    k[4 * page:7 * page] *= 0.5
    v = r.standard_normal(k.shape).astype(np.float16)
    ctx.append(pool, 0, ctx.upload(k), ctx.upload(v), velokv.DT_F16, ctx.upload(np.arange(8 * page)), 8 * page)
    index = velokv.KeyIndex(ctx, pool)
    few = dict(block_tables=ctx.upload(np.arange(8, dtype=np.int32)), bt_stride=8)
    ctx.index_update(index, 0, ctx.upload(np.array([8 * page], np.int32)), 1, 8 * page, **few)
    places, table = [5, 77_000_000, 2 ** 27 - 70], np.zeros(2 ** 27, np.int32)
    table[places] = 3
    table[last - 2:] = [4, 5, 6]
    lens = ctx.upload(np.array([n], np.int32))
    d = dict(block_tables=ctx.upload(table), bt_stride=2 ** 27, context_lens=lens, n_seqs=1, max_context_len=n)
    del table
    # the last 40 tokens, the last of the last page left out
    ctx.index_update(index, 0, first_tokens=ctx.upload(np.array([n - 40], np.int32)), max_tokens=40, **d)
    lower, upper = ctx.alloc(8 * hd * 4), ctx.alloc(8 * hd * 4)
    ctx.index_read(index, 0, ctx.upload(np.arange(8, dtype=np.int32)), 8, lower, upper)
    ctx.sync()
    lower, upper = lower.download((8, hd), np.float32), upper.download((8, hd), np.float32)
    for p in range(8):
        x = k[p * page:p * page + (15 if p == 6 else 16), 0].astype(np.float32)
        step = x.max() / np.float32(127)
        assert np.all(np.abs(lower[p] - x.min(0)) <= step * 0.5001) and np.all(np.abs(upper[p] - x.max(0)) <= step * 0.5001)
    q = np.ones((1, 2, hd), np.float16)
    pages, out = ctx.upload(np.full(6, 77, np.int32)), ctx.alloc(2 * hd * 4)
    need = ctx.sparse_workspace_bytes(pool, 1, 2, n, 6, bt_stride=2 ** 27)
    assert need >= 4 * 2 ** 27
    ctx.select_decode(index, 0, ctx.upload(q), velokv.DT_F16, out, pages, 6, n_heads=2, workspace=ctx.alloc(need), workspace_bytes=need, **d)
    ctx.sync()
    want = [0, 1] + places + [last]
    assert pages.download((6,), np.int32).tolist() == want
    held = np.r_[0:16, 0:16, np.tile(np.arange(48, 64), 3), 96:111]
    x = k[held, 0].astype(np.float64).sum(-1) / 8
    p = np.exp(x - x.max())
    # scores to 8 sqrt(D) 2^-24 of their size in log2 units, p and its parts to 2^-20 (as in test_gpu_sparse)
    tol = np.abs(v).max() * (8 * 8 * 2.0 ** -24 * x.max() * 1.4427 + 2.0 ** -20)
    assert np.all(np.abs(out.download((2, hd), np.float32) - p @ v[held, 0].astype(np.float64) / p.sum()) <= tol)

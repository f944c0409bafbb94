"""Log probabilities, entropy and alternatives on the GPU against 64-bit sums.

Ids are compared exactly. With m the row's largest logit, x - m is one rounding off, e^(x - m) a few, the
sums of at most 2^17 terms in a tree about 2^-20 relative: log Z is off by less than 2^-19 (1 + |log Z|),
a log probability by that and the rounding of x - m, the entropy by that and the same part of its second
term."""
import numpy as np
import pytest

import velokv
from test_gpu_sparse import Graph
from velokv import synth

pytestmark = pytest.mark.gpu


def reference(x, scale=1.0):
    """fp64 log probabilities and entropy of rows x."""
    x = x.astype(np.float64) * np.float64(np.float32(scale))
    m = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.exp(x - m)
        z = e.sum(-1, keepdims=True)
        lp = x - m - np.log(z)
        entropy = np.where(e > 0, -e / z * lp, 0).sum(-1)
    return lp, entropy


def order(x, n):
    """Ids of the n largest, ties to the lower; NaN counts as -inf."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    return np.stack([np.lexsort((np.arange(x.shape[1]), -row))[:n] for row in x]).astype(np.int32)


def run(ctx, x, tokens, n_top, scale=0.0, stride=0, offset=0, entropy=True, **kw):
    rows, vocab = x.shape
    stride = stride or vocab
    buf = np.full(offset + rows * stride, np.nan, x.dtype)
    for r in range(rows):
        buf[offset + r * stride:offset + r * stride + vocab] = x[r]
    d = ctx.upload(buf)
    outs = {"token_logprobs": np.float32, "top_ids": np.int32, "top_logprobs": np.float32}
    shapes = {"token_logprobs": (rows, tokens.shape[1]), "top_ids": (rows, n_top), "top_logprobs": (rows, n_top)}
    bufs = {k: ctx.upload(np.full(shapes[k], -7, t)) for k, t in outs.items()}
    ent = ctx.upload(np.full(rows, -7, np.float32)) if entropy else None
    ctx.token_logprobs(d.ptr + offset * x.itemsize, velokv.DT_F32 if x.dtype == np.float32 else velokv.DT_F16, rows, vocab,
                       tokens=ctx.upload(tokens), n_tokens=tokens.shape[1], entropy=ent, n_top=n_top, row_stride=stride,
                       scale=scale, **bufs, **kw)
    ctx.sync()
    got = {k: bufs[k].download(shapes[k], t) for k, t in outs.items()}
    got["entropy"] = ent.download((rows,), np.float32) if entropy else None
    return got


def check(got, x, tokens, n_top, scale=1.0):
    lp, entropy = reference(x, scale)
    finite = np.where(np.isfinite(lp), lp, 0)
    tol = 2.0 ** -19 * (2 + np.abs(finite))
    ids = order(x, n_top)
    assert np.array_equal(got["top_ids"], ids)
    for have, at in ((got["token_logprobs"], tokens), (got["top_logprobs"], ids)):
        want, t = np.take_along_axis(lp, at, 1), np.take_along_axis(tol, at, 1)
        same = (have == want) | (np.isnan(have) & np.isnan(want))
        with np.errstate(invalid="ignore"):
            assert np.all(same | (np.abs(have - want) <= t))
    if got["entropy"] is not None:
        same = np.isnan(got["entropy"]) & np.isnan(entropy)
        with np.errstate(invalid="ignore"):
            assert np.all(same | (np.abs(got["entropy"] - entropy) <= 2.0 ** -18 * (2 + np.abs(entropy))))


def some(rows, vocab, dtype, seed=1, n_tokens=3):
    r = synth.rng(seed)
    return (2.5 * r.standard_normal((rows, vocab))).astype(dtype), r.integers(0, vocab, (rows, n_tokens)).astype(np.int32)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 64), (300, 100), (5, 2049), (2, 8191), (2, 8193), (1, 32000),
                                        (1100, 1025), (3, 50001), (1, 131072)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_sizes(ctx, dtype, rows, vocab):
    x, tokens = some(rows, vocab, dtype)
    for n_top in {0, 1, min(5, vocab), min(32, vocab)}:
        check(run(ctx, x, tokens, n_top), x, tokens, n_top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_strides_and_alignment(ctx, dtype):
    """Rows that start anywhere, with NaN between and around them."""
    for vocab, stride, offset in ((1000, 1003, 1), (9000, 9001, 3), (17, 17, 5), (8192, 8200, 0)):
        x, tokens = some(4, vocab, dtype, seed=vocab)
        check(run(ctx, x, tokens, 7, stride=stride, offset=offset), x, tokens, 7)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_special_rows(ctx, dtype):
    """Masks of -inf and of the type's lowest value, rows of nothing else, equal, rising and falling rows, one
    token far above, zeros of both signs, NaN and +inf."""
    vocab = 20011
    x, tokens = some(14, vocab, dtype, seed=3)
    low = np.finfo(dtype).min
    r = synth.rng(5)
    x[0][r.random(vocab) < 0.999] = -np.inf
    x[1][r.random(vocab) < 0.999] = low
    x[2] = -np.inf
    x[3] = low
    x[4] = 1.5
    x[5] = np.linspace(-8, 8, vocab).astype(dtype)
    x[6] = x[5][::-1]
    x[7] = -np.inf
    x[7, vocab - 1] = -3
    x[8, 777] = 500
    x[9] = np.where(np.arange(vocab) % 2, 0.0, -0.0).astype(dtype)
    x[10, 4000] = np.nan
    x[11, 9000] = np.inf
    x[12] = np.nan
    x[13, :15000], x[13, 15000] = low, 10
    for n_top in (1, 20, 32):
        got = run(ctx, x, tokens, n_top)
        assert np.array_equal(got["top_ids"], order(x, n_top))
        usual = [0, 1, 3, 4, 5, 6, 7, 8, 9, 13]
        check({k: v[usual] for k, v in got.items()}, x[usual], tokens[usual], n_top)
        assert np.all(got["top_logprobs"][2] == -np.inf) and np.all(got["token_logprobs"][2] == -np.inf) and got["entropy"][2] == 0
        for row in (10, 11, 12):
            assert np.isnan(got["entropy"][row])
            assert np.all(np.isnan(got["top_logprobs"][row]) | (got["top_logprobs"][row] == -np.inf))
        assert np.isnan(got["token_logprobs"][10]).all()


def test_scale_and_tokens_outside(ctx):
    x, tokens = some(6, 3000, np.float32, seed=8)
    for scale in (0.3, 1.0, 7.0):
        check(run(ctx, x, tokens, 10, scale=scale), x, tokens, 10, scale)
    tokens[0, 0], tokens[1, 1], tokens[2, 2] = -1, 3000, 2 ** 31 - 1
    got = run(ctx, x, tokens, 0)["token_logprobs"]
    assert got[0, 0] == got[1, 1] == got[2, 2] == -np.inf and np.isfinite(got).sum() == got.size - 3


def test_many_tokens_and_no_entropy(ctx):
    x, _ = some(2, 9000, np.float16, seed=9)
    tokens = synth.rng(2).integers(0, 9000, (2, 700)).astype(np.int32)
    check(run(ctx, x, tokens, 2, entropy=False), x, tokens, 2)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("parts", [5, 9, 32])
def test_alternatives_of_uneven_parts(ctx, dtype, parts):
    """Rows of several parts whose largest values lie in one part, in the last few values, in order, or are equal."""
    vocab, r = 8192 * parts - 8190, synth.rng(parts)  # the last part: two values
    x = r.standard_normal((8, vocab)).astype(dtype)
    x[0, 8192:16384] += dtype(8)
    x[1, -3:] = 20
    x[2] = np.sort(x[2])
    x[3] = np.sort(x[3])[::-1]
    x[4] = 1
    x[5] = r.integers(0, 2, vocab)
    x[6] = -np.inf
    x[6, [5, 9000, vocab - 1]] = [1, 2, 3]
    x[7] = r.integers(0, 40, vocab)
    tokens = r.integers(0, vocab, (8, 1)).astype(np.int32)
    for n_top in (1, 2, 7, 20, 31, 32):
        check(run(ctx, x, tokens, n_top), x, tokens, n_top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("vocab", [70, 2001, 20003])
def test_rows_without_a_bound(ctx, dtype, vocab):
    """Masks that leave few tokens (-infinity, the type's lowest value, zero), NaN in masked places, values in
    order and steps; as many rows as make a row one workgroup's."""
    r, rows = synth.rng(vocab), 1100
    x = np.broadcast_to(r.standard_normal(vocab).astype(dtype), (rows, vocab)).copy()
    for i, masked in enumerate((-np.inf, np.finfo(dtype).min, 0, np.nan)):
        for j, left in enumerate((0.0, 0.01, 0.5)):
            x[3 * i + j] = np.where(r.random(vocab) < left, r.standard_normal(vocab), masked).astype(dtype)
    x[9:12] = np.where(np.isnan(x[9:12]), np.where(r.random((3, vocab)) < 0.5, np.nan, -np.inf), x[9:12])
    x[12], x[13] = np.sort(x[12]), np.sort(x[13])[::-1]
    x[14] = (np.arange(vocab) // 40).astype(dtype)
    x[15] = -(np.arange(vocab) // 700).astype(dtype)
    x[16] = -np.inf
    x[16, -1] = 0
    at, nothing = np.r_[0:18, 1099], np.r_[0, 9:12]  # rows of -infinity alone and rows with NaN: ids alone
    usual = np.setdiff1d(at, nothing)
    tokens = r.integers(0, vocab, (rows, 1)).astype(np.int32)
    for n_top in (1, 5, 20, 32):
        got = run(ctx, x, tokens, n_top)
        assert np.array_equal(got["top_ids"][at], order(x[at], n_top))
        check({k: v[usual] for k, v in got.items()}, x[usual], tokens[usual], n_top)


def test_captured_calls_replay(ctx):
    """A call in parts with a workspace of its own, replayed as the logits change, beside eager calls."""
    rows, vocab, n_top = 3, 100000, 5
    need = ctx.token_logprobs_workspace_bytes(rows, vocab, n_top)
    x, tokens = some(rows, vocab, np.float16, seed=11)
    dx, dt, ws, stream = ctx.upload(x), ctx.upload(tokens), ctx.alloc(need), velokv.Stream(ctx)
    outs = dict(token_logprobs=ctx.alloc(tokens.size * 4), top_ids=ctx.alloc(rows * n_top * 4),
                top_logprobs=ctx.alloc(rows * n_top * 4), entropy=ctx.alloc(rows * 4))
    shapes = dict(token_logprobs=tokens.shape, top_ids=(rows, n_top), top_logprobs=(rows, n_top), entropy=(rows,))
    ctx.sync()
    with Graph(stream) as graph:
        ctx.token_logprobs(dx, velokv.DT_F16, rows, vocab, tokens=dt, n_tokens=tokens.shape[1], n_top=n_top, workspace=ws,
                           workspace_bytes=need, stream=stream, **outs)
    for step in range(4):
        x, tokens = some(rows, vocab, np.float16, seed=20 + step)
        dx.upload(x)
        dt.upload(tokens)
        graph.replay()
        check({k: o.download(shapes[k], np.int32 if k == "top_ids" else np.float32) for k, o in outs.items()}, x, tokens, n_top)
        y, given = some(2, 50000, np.float32, seed=40 + step)
        check(run(ctx, y, given, 3), y, given, 3)
    graph.close()


def test_workspace_and_streams(ctx):
    """Two streams at once, each with its own workspace; one too small is refused."""
    a, b = (some(4, 100000, np.float16, seed=s) for s in (1, 2))
    need = ctx.token_logprobs_workspace_bytes(4, 100000, 20)
    assert need > 0 and ctx.token_logprobs_workspace_bytes(4, 100, 20) == 0
    streams, got = [velokv.Stream(ctx), velokv.Stream(ctx)], []
    for (x, tokens), s in zip((a, b), streams):
        outs = dict(token_logprobs=ctx.alloc(4 * 3 * 4), top_ids=ctx.alloc(4 * 20 * 4), top_logprobs=ctx.alloc(4 * 20 * 4), entropy=ctx.alloc(16))
        got.append((x, tokens, outs, ctx.upload(x), ctx.upload(tokens), ctx.alloc(need), s))
    for x, tokens, outs, dx, dt, ws, s in got:
        ctx.token_logprobs(dx, velokv.DT_F16, 4, 100000, tokens=dt, n_tokens=3, n_top=20, workspace=ws, workspace_bytes=need, stream=s, **outs)
    for x, tokens, outs, dx, dt, ws, s in got:
        s.sync()
        shapes = dict(token_logprobs=(4, 3), top_ids=(4, 20), top_logprobs=(4, 20), entropy=(4,))
        check({k: o.download(shapes[k], np.int32 if k == "top_ids" else np.float32) for k, o in outs.items()}, x, tokens, 20)
    with pytest.raises(velokv.VkError) as e:
        ctx.token_logprobs(got[0][3], velokv.DT_F16, 4, 100000, tokens=got[0][4], n_tokens=3, n_top=20, workspace=got[0][5],
                           workspace_bytes=need - 1, **got[0][2])
    assert e.value.code == velokv.ERR_BAD_ARG


def test_refusals(ctx):
    b = ctx.alloc(4096)
    good = dict(logits=b, dtype=velokv.DT_F32, n_rows=1, vocab=100, tokens=b, n_tokens=1, token_logprobs=b, top_ids=b, top_logprobs=b, n_top=2)
    for bad, code in ((dict(dtype=9), velokv.ERR_BAD_ARG), (dict(vocab=0), velokv.ERR_BAD_ARG), (dict(n_rows=-1), velokv.ERR_BAD_ARG),
                      (dict(n_top=33), velokv.ERR_UNSUPPORTED), (dict(vocab=1, n_top=2), velokv.ERR_BAD_ARG),
                      (dict(n_top=-1), velokv.ERR_BAD_ARG), (dict(row_stride=99), velokv.ERR_BAD_ARG), (dict(logits=None), velokv.ERR_BAD_ARG),
                      (dict(tokens=None), velokv.ERR_BAD_ARG), (dict(token_logprobs=None), velokv.ERR_BAD_ARG),
                      (dict(top_ids=None), velokv.ERR_BAD_ARG), (dict(scale=-1.0), velokv.ERR_BAD_ARG),
                      (dict(scale=float("nan")), velokv.ERR_BAD_ARG), (dict(scale=float("inf")), velokv.ERR_BAD_ARG),
                      (dict(vocab=2 ** 28 + 1), velokv.ERR_UNSUPPORTED), (dict(logits=b.ptr + 2), velokv.ERR_BAD_ARG)):
        with pytest.raises(velokv.VkError) as e:
            ctx.token_logprobs(**{**good, **bad})
        assert e.value.code == code, bad
    ctx.token_logprobs(**dict(good, n_rows=0))
    ctx.sync()


def test_tree_verification(ctx):
    """SpeculativeTree.verify_logits: the accepted path follows the target's most probable tokens."""
    tree = velokv.branching_tree([2, 2, 2])
    n, vocab = len(tree.nodes), 500
    x, _ = some(n, vocab, np.float16, seed=4)
    want = [0, 2, 5, 12]  # a root path of the breadth-first tree, as its parents say
    path = tree.path_nodes(want[-1])
    for node, nxt in zip(path, path[1:]):
        x[node, tree.nodes[nxt].token] = 30
    got = tree.verify_logits(ctx, ctx.upload(x), velokv.DT_F16, vocab)
    assert got.expected == x.astype(np.float64).argmax(-1).tolist()
    lp, _ = reference(x)
    assert np.all(np.abs(np.array(got.logprobs) - lp.max(-1)) <= 2.0 ** -19 * (2 + np.abs(lp.max(-1))))
    assert tree.best_path_nodes(got) == path
    assert tree.find_best_path(got)[0] == tree.get_path(path[-1])

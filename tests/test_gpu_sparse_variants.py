"""Every kernel that a plan of sparse decode or of the log probabilities may take, at sizes that take it: long
contexts in several turns of a workgroup and in two launches, lists in more parts than a merge takes in a
turn, the pool's slot table, rows of logits of several steps a part. References in 64 bits as in
test_gpu_sparse and test_gpu_logprobs."""
import threading

import numpy as np
import pytest

import pyoracle as O
import velokv
from test_gpu_logprobs import check, reference, run, some
from test_gpu_sparse import KVS, Cache, Graph, attend, close, code_parts, dt, queries, select, some_lists, sparse
from velokv import synth

pytestmark = pytest.mark.gpu
PAGES = 8300  # more than one launch's scores fit LDS


@pytest.fixture(scope="module", params=[128, 64])
def long(request, ctx):
    """A context of PAGES pages (the last one short), its index, and its bounds: codes [pages][dim] and scales."""
    c = Cache(ctx, O.F16, [16 * PAGES - 5], n_kv_heads=1, head_dim=request.param, seed=41)
    index = velokv.KeyIndex(ctx, c.pool)
    ctx.index_update(index, 0, **c.dev())
    ctx.sync()
    k = c.tokens(c.k32, 0, np.arange(PAGES), 0).reshape(PAGES, 16, -1)
    k[-1, 11:] = k[-1, 10]
    lo, hi = k.min(1), k.max(1)
    scale, inv = code_parts(np.concatenate([lo, hi], 1))
    yield c, index, np.rint(lo * inv[:, None]).astype(np.float64), np.rint(hi * inv[:, None]).astype(np.float64), scale
    index.close()


def chosen(long, q, pages, n_list):
    """Lists [S][1][n_list]; row s sees pages[s] pages. Sums of codes are whole numbers, exact in fp64."""
    _, _, lo, hi, scale = long
    q_scale, inv = code_parts(q.astype(np.float32))
    code = np.rint(q.astype(np.float32) * inv[..., None]).astype(np.float64)
    out = np.full((len(pages), 1, n_list), -1, np.int32)
    for s, n in enumerate(pages):
        if n <= n_list:
            out[s, 0, :n] = np.arange(n)
            continue
        dot = np.minimum(code[s], 0) @ lo[:n].T + np.maximum(code[s], 0) @ hi[:n].T
        score = ((dot.astype(np.float32) * scale[:n]) * q_scale[s][:, None]).max(0)
        score[[0, -1]] = np.inf
        out[s, 0] = np.sort(np.lexsort((np.arange(n), -score))[:n_list])
    return out


# rows (one KV head), longest context in pages: two launches with one turn a wave, with three turns, with
# seventeen (a workgroup a row); one launch by rows, with up to five turns, and in the operands' order
@pytest.mark.parametrize("rows,longest", [(1, 2600), (32, 2600), (70, PAGES), (600, PAGES), (40, 2500), (1, 1500), (260, 3000), (300, 520)])
@pytest.mark.parametrize("group", [3, 20])
@pytest.mark.parametrize("q_dtype", [np.float16, np.float32])
def test_select_variants(ctx, long, q_dtype, group, rows, longest):
    c, index = long[:2]
    print(f"select dim={c.hd} group={group} q={np.dtype(q_dtype).name} rows={rows} longest={longest}", flush=True)
    r = synth.rng(rows)
    pages = np.r_[longest, np.minimum(longest, np.exp(r.uniform(0, np.log(longest + 0.5), rows - 1)).astype(int) + 1)].astype(int)
    lens = [min(16 * int(n), int(c.lens[0])) for n in pages]
    q = queries(c, rows, group, q_dtype)
    for n_list in (33, 700):
        assert np.array_equal(select(c, index, q, lens, [0] * rows, n_list), chosen(long, q, pages, n_list)), n_list


def test_captured_selection_in_two_launches(ctx, long):
    """Replayed as the queries and the length change, beside eager calls of another shape."""
    c, index = long[:2]
    lens, q = ctx.upload(np.array([16 * 4000], np.int32)), ctx.upload(queries(c, 1, 4, np.float16))
    d = dict(c.dev(), context_lens=lens)
    need = ctx.sparse_workspace_bytes(c.pool, 1, 4, d["max_context_len"], 50, bt_stride=d["bt_stride"])
    ws, pages, stream = ctx.alloc(need), ctx.alloc(50 * 4), velokv.Stream(ctx)
    ctx.sync()
    with Graph(stream) as graph:
        ctx.select_pages(index, 0, q, velokv.DT_F16, pages, 50, n_heads=4, workspace=ws, workspace_bytes=need, stream=stream, **d)
    for step in range(4):
        n, host_q = 2300 + 2000 * step, queries(c, 1, 4, np.float16, seed=60 + step)
        lens.upload(np.array([min(16 * n, int(c.lens[0]))], np.int32))
        q.upload(host_q)
        graph.replay()
        assert np.array_equal(pages.download((1, 1, 50), np.int32), chosen(long, host_q, [n], 50)), step
        other = queries(c, 3, 4, np.float32, seed=step)
        assert np.array_equal(select(c, index, other, [16 * 3000] * 3, [0] * 3, 20), chosen(long, other, [3000] * 3, 20))
    graph.close()


@pytest.mark.parametrize("head_dim,group", [(128, 4), (40, 20)])
@pytest.mark.parametrize("kv", KVS)
def test_lists_in_many_parts(ctx, kv, head_dim, group):
    """One (row, KV head): 237 parts of a list of 2600 entries, most of them of pages listed before."""
    c = Cache(ctx, kv, [16 * 300 - 3], n_kv_heads=1, head_dim=head_dim, seed=42)
    q = queries(c, 1, group, np.float16)
    for n in (2600, 700):
        lists = some_lists(c, c.lens, n)
        close(sparse(c, q, lists, c.lens, [0]), attend(c, q, lists, c.lens, [0]))


@pytest.mark.parametrize("kv,page", [(O.F16, 16), (O.I8_BLK, 48), (O.I8_REF, 16), (O.F32, 32)])
def test_slot_table(ctx, kv, page):
    """The pool's own table gives what the same table of the caller's gives; rows past it are its last."""
    pages, slots = 30, 3
    pool = velokv.Pool(ctx, 1, slots * pages, page, 2, 128, kv, max_slots=slots, max_pages_per_slot=pages)
    index, other = velokv.KeyIndex(ctx, pool), velokv.KeyIndex(ctx, pool)
    r = synth.rng(43)
    table = r.permutation(slots * pages).astype(np.int32).reshape(slots, pages)
    for s in range(slots):
        pool.bind_slot(s, table[s])
    n = slots * pages * page
    k, v = (r.standard_normal((n, 2, 128)).astype(np.float16) for _ in range(2))
    ctx.append(pool, 0, ctx.upload(k), ctx.upload(v), velokv.DT_F16, ctx.upload(np.arange(n)), n)
    lens, rows = np.array([page * 29 + 3, 17, page * 30, 5 * page], np.int32), np.array([1, 0, 2, 2], np.int32)
    q = ctx.upload(r.standard_normal((4, 8, 128)).astype(np.float16))

    def both(index, rows, **tables):
        d = dict(tables, context_lens=ctx.upload(lens), seq_rows=ctx.upload(rows), n_seqs=4, max_context_len=page * 30)
        lists, out = ctx.upload(np.full((4, 2, 9), 77, np.int32)), ctx.alloc(4 * 8 * 128 * 4)
        ctx.index_update(index, 0, **d)
        ctx.select_decode(index, 0, q, velokv.DT_F16, out, lists, 9, n_heads=8, **d)
        ctx.sync()
        return lists.download((4, 2, 9), np.int32), out.download((4, 8, 128), np.float32)

    want = both(index, rows, block_tables=ctx.upload(table), bt_stride=pages)
    for given in (rows, np.where(rows == 2, 2 ** 31 - 1, rows).astype(np.int32)):
        got = both(other, given)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    with pytest.raises(velokv.VkError) as e:
        ctx.index_update(other, 0, ctx.upload(lens), 4, page * 30 + 1)
    assert e.value.code == velokv.ERR_BAD_ARG


@pytest.mark.parametrize("page,head_dim,group", [(256, 8, 2), (144, 120, 5), (16, 72, 17)])
@pytest.mark.parametrize("q_dtype", [np.float16, np.float32])
@pytest.mark.parametrize("kv", KVS)
def test_a_layer_among_others(ctx, kv, q_dtype, page, head_dim, group):
    """Layer 2 of 3, three KV heads, the longest pages and the least head_dim, queries and results that start one
    element into their buffers, and table entries past a context that name nothing."""
    c = Cache(ctx, kv, [page * 12 + 5, 3, page * 7], n_kv_heads=3, head_dim=head_dim, page=page, seed=44)
    pool = velokv.Pool(ctx, 3, c.n_pages, page, 3, head_dim, kv)
    pool.upload_layer(2, c.pool.download_layer(0))
    for s, n in enumerate(c.lens):
        c.table[s, -(-int(n) // page):] = 2 ** 31 - 1
    one, index, q = velokv.KeyIndex(ctx, c.pool), velokv.KeyIndex(ctx, pool), queries(c, 3, 3 * group, q_dtype)
    ctx.index_update(one, 0, **c.dev())
    for layer in (2, 1):  # the layer beside it, of zeros, is not its own
        ctx.index_update(index, layer, **c.dev())
    shifted, out = ctx.upload(np.r_[q.reshape(-1)[:1], q.reshape(-1)]), ctx.upload(np.full(q.size + 2, np.nan, np.float32))
    lists = ctx.upload(np.full((3, 3, 4), 77, np.int32))
    ctx.select_decode(index, 2, shifted.ptr + q.itemsize, dt(q), out.ptr + 4, lists, 4, n_heads=q.shape[1], **c.dev())
    ctx.sync()  # and no page is reported
    lists, out = lists.download((3, 3, 4), np.int32), out.download()
    assert np.array_equal(lists, select(c, one, q, c.lens, [0, 1, 2], 4))
    assert np.isnan(out[0]) and np.isnan(out[-1])
    got = out[1:-1].reshape(q.shape)
    assert np.array_equal(got, sparse(c, q, lists, c.lens, [0, 1, 2]))
    close(got, attend(c, q, lists, c.lens, [0, 1, 2]))


@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** -66])
def test_small_value_scales(ctx, size):
    """int8 values of fp32 scales down to 2^-74 keep their precision."""
    c = Cache(ctx, O.I8_REF, [16 * 24], seed=45)
    r = synth.rng(46)
    k = r.standard_normal((16 * 24, c.hkv, c.hd)).astype(np.float32)
    v = (r.standard_normal(k.shape) * size).astype(np.float32)
    slots = synth.slots_for_positions(c.table, np.arange(16 * 24), 16, np.zeros(16 * 24, int))
    ctx.append(c.pool, 0, ctx.upload(k), ctx.upload(v), velokv.DT_F32, ctx.upload(slots), len(k))
    c.read()
    lists = np.broadcast_to(np.arange(24, dtype=np.int32), (1, 2, 24))
    q = queries(c, 1, 8, np.float16)
    close(sparse(c, q, lists, c.lens, [0]), attend(c, q, lists, c.lens, [0]))


def test_subnormal_keys_and_values(ctx):
    """fp16 keys and values below 2^-14 keep the bits they have."""
    c = Cache(ctx, O.F16, [16 * 24 - 3], seed=47)
    r = synth.rng(48)
    k, v = ((r.standard_normal((16 * 24 - 3, c.hkv, c.hd)) * 2.0 ** -17).astype(np.float16) for _ in range(2))
    c.append(0, np.arange(len(k)), k, v)
    c.read()
    lists = np.broadcast_to(np.arange(24, dtype=np.int32), (1, 2, 24))
    for q_dtype in (np.float16, np.float32):
        q = queries(c, 1, 8, q_dtype)
        close(sparse(c, q, lists, c.lens, [0], scale=2.0 ** 14), attend(c, q, lists, c.lens, [0], 2.0 ** 14))


def test_index_of_a_closed_pool(ctx):
    """The pool's close closes its indexes; calls on them are refused."""
    pool = velokv.Pool(ctx, 1, 4, 16, 1, 64, velokv.KV_F16)
    index = velokv.KeyIndex(ctx, pool)
    pool.close()
    with pytest.raises(velokv.VkError) as e:
        ctx.index_update(index, 0, None, 0, 0)
    assert e.value.code == velokv.ERR_NOT_WIRED
    index.close()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("vocab", [262145, 300001, 700003])
def test_rows_of_several_steps_a_part(ctx, dtype, vocab):
    """More than 32 parts of a step: ordinary, sorted, equal and masked rows. A thread adds up to 96 values one
    after the other: at most 96 2^-24 of the sum, within check()'s 2^-19 (2 + 7) at the least |log p| of 7 here."""
    x, tokens = some(6, vocab, dtype, seed=7)
    x[1], x[2], x[3] = np.sort(x[1]), np.sort(x[2])[::-1], 2
    x[4, synth.rng(3).random(vocab) < 0.9999] = np.finfo(dtype).min
    x[5] = -np.inf
    x[5, [3, vocab // 2, vocab - 1]] = [1, 5, 2]
    for n_top in (1, 5, 32):
        check(run(ctx, x, tokens, n_top), x, tokens, n_top)


def test_trees_verified_at_once(ctx):
    """Two host threads, a stream and a tree each, rows of several parts: nothing is shared."""
    tree, vocab = velokv.branching_tree([2, 2, 2]), 100000
    x = [some(len(tree.nodes), vocab, np.float16, seed=70 + i)[0] for i in range(2)]
    dev, streams, got = [ctx.upload(y) for y in x], [velokv.Stream(ctx), velokv.Stream(ctx)], [[], []]
    ctx.sync()

    def work(i):
        for _ in range(20):
            got[i].append(tree.verify_logits(ctx, dev[i], velokv.DT_F16, vocab, stream=streams[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        best = reference(x[i])[0].max(-1)
        assert len(got[i]) == 20
        for g in got[i]:
            assert g.expected == x[i].astype(np.float64).argmax(-1).tolist()
            assert np.all(np.abs(np.array(g.logprobs) - best) <= 2.0 ** -19 * (2 + np.abs(best)))

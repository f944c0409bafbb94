"""Operators of long-context decoding: what a serving program calls beside the dense decode step.

Five kinds of work, each through velokv's public entry points where `own` is true, and as elementary
torch operations where it is false:

  index     the key index (per page and KV head the lower and upper bound of the keys, in 8 bits)
            brought up to date, after a prompt or after a decode step's token, and the touched pages'
            bounds read back (Context.index_update, index_read)
  select    the pages that each sequence's query attends to, chosen by their bounds (Context.select_pages)
  attend    decode attention over listed pages (Context.sparse_decode)
  both      selection and attention of a decode step in one call (Context.select_decode)
  logprobs  log probabilities of given tokens, entropy and the most probable tokens
            (Context.token_logprobs)

listed() names twelve, draw() gives others of the same ranges. Lengths follow from a case's sizes,
everything else from the seed. A cache of n pages is held as [n * page / 16][KV heads][16][dim] tiles:
fp32 or fp16 values, or int8 codes with a scale per tile ("int8blk") or per token ("int8").
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

TILE = 16  # tokens of a storage tile
CODE_BYTES = {"fp32": 4, "fp16": 2, "int8": 1, "int8blk": 1}
TYPES = {"fp32": torch.float32, "fp16": torch.float16}


def listed():
    return [
        # one token a sequence after a decode step of a full batch: the last page's bounds
        _index("index_step_64x8192_fp16", 64, 7000, 8192, 8, 128, "fp16", 16, 1),
        # a batch of prompts into the compressed cache
        _index("index_prompt_4x1500-2500_int8blk", 4, 1500, 2500, 8, 128, "int8blk", 16, 0),
        # one user, a chat of ordinary length: launches and latency
        _select("select_1x6000_fp16", 1, 6000, 6000, 32, 8, 128, "fp16", 16, 64),
        # a full batch of the benchmark's shape, an eighth of the cache kept
        _select("select_64x8192_fp16", 64, 8192, 8192, 32, 8, 128, "fp16", 16, 64),
        # a small model: 64-dim heads, 7 query heads per KV head, fp32 queries, ragged, larger pages
        _select("select_24x900-30000_d64", 24, 900, 30000, 14, 2, 64, "int8", 32, 48),
        # one user, 1024 tokens attended
        _attend("attend_1x6000_fp16", 1, 6000, 6000, 32, 8, 128, "fp16", "fp16", 16, 64),
        # the default cache type with fp32 queries, odd lengths, some contexts shorter than the list
        _attend("attend_8x100-2500_fp32", 8, 100, 2500, 32, 8, 128, "fp32", "fp32", 16, 50),
        # a full batch over an fp16 cache
        _attend("attend_64x8192_fp16", 64, 8192, 8192, 32, 8, 128, "fp16", "fp16", 16, 64),
        # one GPU's share of a long-context batch, compressed cache, 8 query heads per KV head
        _both("both_32x32768_int8blk_gqa8", 32, 32768, 32768, 64, 8, 128, "int8blk", "fp16", 16, 128),
        # one sequence's next token: 32,000 logits, a few alternatives
        _logprobs("logprobs_1x32000_fp32", 1, 32000, "fp32", 1, 5),
        # a decode batch over a large vocabulary
        _logprobs("logprobs_64x128000_fp16", 64, 128000, "fp16", 1, 20),
        # a scored prompt: every position's given token, no alternatives but the best, an odd vocabulary
        _logprobs("logprobs_1500x50001_fp16", 1500, 50001, "fp16", 1, 1),
    ]


def _cache(name, kind, seqs, lo, hi, heads, kv_heads, dim, kv, act, page, pick):
    return dict(name=name, kind=kind, seqs=seqs, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, dim=dim, kv=kv, act=act,
                page=page, pick=pick)


def _index(name, seqs, lo, hi, kv_heads, dim, kv, page, new):
    return dict(_cache(name, "index", seqs, lo, hi, kv_heads, kv_heads, dim, kv, "fp16", page, 1), new=new)


def _select(name, seqs, lo, hi, heads, kv_heads, dim, kv, page, pick):
    return _cache(name, "select", seqs, lo, hi, heads, kv_heads, dim, kv, "fp32" if kv in ("fp32", "int8") else "fp16", page, pick)


def _attend(name, *rest):
    return _cache(name, "attend", *rest)


def _both(name, *rest):
    return _cache(name, "both", *rest)


def _logprobs(name, rows, vocab, act, given, top):
    return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, act=act, given=given, top=top)


def draw(rng):
    def log_uniform(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))

    kind = rng.choice(["index", "select", "attend", "attend", "both", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = log_uniform(100, 160000)
        rows = log_uniform(1, min(1500, max(1, 75_000_000 // vocab)))
        c = _logprobs("", rows, vocab, rng.choice(["fp16", "fp32"]), rng.choice([0, 1, 1, 3]), min(vocab, rng.choice([0, 1, 5, 20, 32])))
        if c["given"] + c["top"] == 0:
            c["given"] = 1
    else:
        kv = rng.choice(["fp16", "int8blk", "int8blk", "fp32", "int8"])
        kv_heads, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([128, 128, 128, 64, 96])
        heads, page = kv_heads * rng.choice([1, 2, 4, 4, 7, 8, 16]), rng.choice([16, 16, 32, 48, 64, 128])
        row = kv_heads * dim * 2 * CODE_BYTES[kv]
        seqs, hi = log_uniform(1, 64), log_uniform(64, 32768)
        hi = min(hi, max(64, 1_200_000_000 // (row * seqs)))
        lo = hi if rng.random() < 0.3 else max(1, int(hi * rng.uniform(0.1, 0.9)))
        pick = log_uniform(3, max(3, 2048 // page))
        act = "fp32" if kv in ("fp32", "int8") else rng.choice(["fp16", "fp16", "fp32"])
        c = _cache("", kind, seqs, lo, hi, heads, kv_heads, dim, kv, act, page, pick)
        if kind == "index":
            c.update(heads=kv_heads, act="fp16", pick=1, new=rng.choice([0, 1, 5]))
    del c["name"]
    return c


# ---- sizes -----------------------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths, the same for every seed."""
    r = np.random.Generator(np.random.PCG64(case["seqs"] * 1_000_003 + case["lo"] * 101 + case["hi"]))
    return r.integers(case["lo"], case["hi"] + 1, case["seqs"]).astype(np.int64)


def _ceil(a, b):
    return -(-a // b)


def _touched(case, lens):
    """First and last-but-one page that the new tokens of each sequence are in (new = 0: every page)."""
    first = np.maximum(lens - case["new"], 0) if case["new"] else 0 * lens
    return first // case["page"], _ceil(lens, case["page"])


def work(case):
    if case["kind"] == "logprobs":
        n, act = case["rows"] * case["vocab"], 4 if case["act"] == "fp32" else 2
        return {"bytes": n * act + case["rows"] * (8 * case["given"] + 8 * case["top"] + 4), "flops": 5 * n}
    lens, page, hkv, hq, dim = _lengths(case), case["page"], case["kv_heads"], case["heads"], case["dim"]
    act, esz = 4 if case["act"] == "fp32" else 2, CODE_BYTES[case["kv"]]
    token = hkv * dim * esz  # K (or V) codes of a token
    scales = {"int8blk": 2 * hkv / TILE, "int8": 4 * hkv}.get(case["kv"], 0)
    pages = _ceil(lens, page)
    if case["kind"] == "index":
        a, b = _touched(case, lens)
        tokens, n = int((lens - a * page).sum()), int((b - a).sum())
        return {"bytes": tokens * (token + scales) + n * (4 + hkv * (2 * dim + 4) + hkv * dim * 8), "flops": 2 * tokens * hkv * dim}
    q = case["seqs"] * hq * dim * act
    lists = case["seqs"] * hkv * case["pick"] * 4
    n = int(pages.sum())
    select = {"bytes": n * (hkv * (2 * dim + 4) + 4) + q + lists, "flops": 4 * n * hq * dim}
    kept = np.minimum(lens, case["pick"] * page)  # at most: the last page may be short
    attend = {"bytes": 2 * int(kept.sum() * (token + scales)) + q + lists + case["seqs"] * hq * dim * 4,
              "flops": 4 * hq * dim * int(kept.sum())}
    if case["kind"] == "select":
        return select
    if case["kind"] == "attend":
        return attend
    return {"bytes": select["bytes"] + attend["bytes"] - q - lists, "flops": select["flops"] + attend["flops"]}


# ---- inputs ----------------------------------------------------------------------------------------

def _tables(n_pages, counts, seed):
    """Block tables: a random scatter of the pool's pages over the sequences."""
    perm = np.random.Generator(np.random.PCG64(seed)).permutation(n_pages).astype(np.int32)
    table = np.zeros((len(counts), int(max(counts))), np.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = perm[at:at + n]
        at += n
    return table


def _quantized(x, kv):
    """int8 codes and scales of tiles x: a scale per tile and head (fp16), or per token and head (fp32)."""
    if kv == "int8blk":
        scale = (x.abs().amax((2, 3)).float() / 127).half()
        return (x / scale[:, :, None, None]).round_().clamp_(-127, 127).to(torch.int8), scale
    scale = x.abs().amax(3).float() / 127
    return (x / scale[:, :, :, None].half()).round_().clamp_(-127, 127).to(torch.int8), scale


def _inputs(case, seed):
    """The tensors of a case: a cache's tiles and scales, table, lengths and queries, or logits and tokens."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    act = TYPES[case["act"]]
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab), generator=g, device="cuda", dtype=act).mul_(2.5)
        few = torch.rand((rows, vocab), generator=g, device="cuda", dtype=torch.float16) < 0.99
        few[:, 0] = False
        x[1::8].masked_fill_(few[1::8], -math.inf)  # rows that a grammar leaves few tokens
        tokens = torch.randint(0, vocab, (rows, case["given"]), generator=g, device="cuda", dtype=torch.int32)
        return {"x": x, "tokens": tokens}
    lens, page, hkv, dim, kv = _lengths(case), case["page"], case["kv_heads"], case["dim"], case["kv"]
    counts = _ceil(lens, page)
    n_pages = int(counts.sum()) * 9 // 8 + 4
    tiles = n_pages * page // TILE
    shape = (tiles, hkv, TILE, dim)
    kind = torch.float32 if kv == "fp32" else torch.float16
    topic = torch.randn((tiles, hkv, 1, dim), generator=g, device="cuda", dtype=kind).mul_(0.7)  # what a tile is about
    k = torch.randn(shape, generator=g, device="cuda", dtype=kind).add_(topic)
    st = {"lens": torch.from_numpy(lens.astype(np.int32)).cuda(), "table": torch.from_numpy(_tables(n_pages, counts, seed)).cuda()}
    st["k"], st["ks"] = _quantized(k, kv) if kv.startswith("int8") else (k, None)
    del k, topic
    if case["kind"] != "index":
        if case["kind"] != "select":
            v = torch.randn(shape, generator=g, device="cuda", dtype=kind)
            st["v"], st["vs"] = _quantized(v, kv) if kv.startswith("int8") else (v, None)
            del v
        st["q"] = torch.randn((case["seqs"], case["heads"], dim), generator=g, device="cuda", dtype=act)
    if case["kind"] == "attend":  # a list in hand: random pages, the first and the last among them
        n = int(counts.max())
        r = torch.rand((case["seqs"], hkv, n), generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        count = torch.from_numpy(counts).cuda()[:, None, None]
        r.masked_fill_((at == 0) | (at == count - 1), 2.0).masked_fill_(at >= count, -1.0)
        best = r.sort(-1, descending=True)
        pick = torch.where(best.values >= 0, best.indices, n)[..., :case["pick"]].sort(-1).values
        pick = torch.where(pick < n, pick, -1).to(torch.int32)
        st["pages"] = torch.nn.functional.pad(pick, (0, case["pick"] - pick.shape[-1]), value=-1).contiguous()
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if case["kind"] == "logprobs":
        return _own_logprobs(st) if own else st
    if case["kind"] == "index":
        a, b = _touched(case, _lengths(case))
        cols = np.concatenate([np.arange(x, y) for x, y in zip(a, b)])
        rows = np.repeat(np.arange(len(a)), b - a)
        st["touched_row"], st["touched_col"] = torch.from_numpy(rows).cuda(), torch.from_numpy(cols).cuda()
        st["touched"] = st["table"][st["touched_row"], st["touched_col"]].contiguous()
    if own:
        return _own_cache(st)
    if case["kind"] in ("select", "both"):  # the index that earlier steps left
        rows = torch.arange(case["seqs"], device="cuda")[:, None].expand_as(st["table"])
        cols = torch.arange(st["table"].shape[1], device="cuda")[None].expand_as(st["table"])
        has = cols * case["page"] < st["lens"][:, None]
        at = st["table"][has]
        lower, upper, scale = _bounds(st, at, rows[has], cols[has])
        n_pages = st["k"].shape[0] * TILE // case["page"]
        st["codes"] = torch.zeros((n_pages, case["kv_heads"], 2, case["dim"]), dtype=torch.int8, device="cuda")
        st["scale"] = torch.zeros((n_pages, case["kv_heads"]), device="cuda")
        st["codes"][at], st["scale"][at] = torch.stack([lower, upper], 2), scale
    return st


def run(st):
    kind = st["case"]["kind"]
    if own:
        return st["own"](st)
    if kind == "logprobs":
        return _plain_logprobs(st)
    if kind == "index":
        lower, upper, scale = _bounds(st, st["touched"], st["touched_row"], st["touched_col"])
        return [lower.float() * scale[..., None], upper.float() * scale[..., None]]
    if kind == "select":
        return _plain_select(st)
    if kind == "attend":
        return _plain_attend(st, st["pages"])
    pages = _plain_select(st)
    return [pages, _plain_attend(st, pages)]


# ---- plain forms -----------------------------------------------------------------------------------

def _tiles(st, name, tiles, heads):
    """Tiles of the K or V cache in 32 bits: [..., 16, dim]."""
    x, scale = st[name][tiles, heads].float(), st[name + "s"]
    if scale is None:
        return x
    scale = scale[tiles, heads].float()
    return x * (scale[..., None, None] if scale.dim() == tiles.dim() else scale[..., None])


def _bounds(st, pages, rows, cols):
    """int8 codes of the keys' lower and upper bound, and their scale, of pages that are column `cols` of
    table row `rows`; tokens past the sequence's length do not count."""
    case = st["case"]
    per, hkv = case["page"] // TILE, case["kv_heads"]
    tiles = pages.long()[:, None, None] * per + torch.arange(per, device="cuda")[None, None]
    k = _tiles(st, "k", tiles.expand(-1, hkv, -1), torch.arange(hkv, device="cuda")[None, :, None])
    k = k.reshape(len(pages), hkv, case["page"], case["dim"])
    pos = cols[:, None] * case["page"] + torch.arange(case["page"], device="cuda")
    out = (pos >= st["lens"].long()[rows][:, None])[:, None, :, None]
    lower, upper = k.masked_fill(out, math.inf).amin(2), k.masked_fill(out, -math.inf).amax(2)
    top = torch.maximum(lower.abs(), upper.abs()).amax(-1)
    scale = torch.div(top, torch.full_like(top, 127))
    inv = torch.where(top > 0, torch.div(torch.full_like(top, 127), top), 0)[..., None]
    return (lower * inv).round().to(torch.int8), (upper * inv).round().to(torch.int8), scale


def _plain_select(st):
    case = st["case"]
    s, hkv, dim, pick = case["seqs"], case["kv_heads"], case["dim"], case["pick"]
    q = st["q"].float().reshape(s, hkv, -1, dim)
    top = q.abs().amax(-1)
    q_scale = torch.div(top, torch.full_like(top, 127))
    q = (q * torch.where(top > 0, torch.div(torch.full_like(top, 127), top), 0)[..., None]).round()
    q = torch.cat([q.clamp(max=0), q.clamp(min=0)], -1)
    at = st["table"].long()
    codes = st["codes"][at].permute(0, 2, 3, 4, 1).reshape(s, hkv, 2 * dim, -1).float()
    dot = torch.matmul(q, codes)  # whole numbers below 2^24: exact in any order
    score = (dot * st["scale"][at].permute(0, 2, 1)[:, :, None, :] * q_scale[..., None]).amax(2)
    n = at.shape[1]
    page = torch.arange(n, device="cuda")
    count = ((st["lens"].long() + case["page"] - 1) // case["page"])[:, None, None]
    score = score.masked_fill((page == 0) | (page == count - 1), math.inf).masked_fill(page >= count, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :pick]
    best = torch.where(best < count, best, n).sort(-1).values
    best = torch.where(best < n, best, -1).to(torch.int32)
    return torch.nn.functional.pad(best, (0, pick - best.shape[-1]), value=-1)


def _plain_attend(st, pages):
    case = st["case"]
    s, hkv, dim, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    at = pages.long()
    held = torch.gather(st["table"].long()[:, None].expand(-1, hkv, -1), 2, at.clamp(min=0))
    tiles = (held[..., None] * (page // TILE) + torch.arange(page // TILE, device="cuda")).reshape(s, hkv, -1)
    heads = torch.arange(hkv, device="cuda")[None, :, None]
    k = _tiles(st, "k", tiles, heads).reshape(s, hkv, -1, dim)
    q = st["q"].float().reshape(s, hkv, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    del k
    pos = at[..., None] * page + torch.arange(page, device="cuda")
    out = ((at < 0)[..., None] | (pos >= st["lens"].long()[:, None, None, None])).reshape(s, hkv, 1, -1)
    score = score.masked_fill(out, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - top.masked_fill(top == -math.inf, 0)).exp()
    total = p.sum(-1, keepdim=True)
    v = _tiles(st, "v", tiles, heads).reshape(s, hkv, -1, dim)
    return (torch.matmul(p, v) / total.masked_fill(total == 0, 1)).reshape(s, -1, dim)


def _plain_logprobs(st):
    x, case = st["x"].float(), st["case"]
    top = x.amax(-1, keepdim=True)
    d = x - top
    e = d.exp()
    z = e.sum(-1, dtype=torch.float64, keepdim=True)
    t = (e * d.masked_fill(e == 0, 0)).sum(-1, dtype=torch.float64, keepdim=True)
    lse = top + z.log()
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)  # ordered as the values are
    place = torch.arange(case["vocab"], device="cuda")
    ids = (order * 2 ** 20 - place).topk(case["top"], -1).indices  # of equal values the first
    return {"token": (x.gather(1, st["tokens"].long()) - lse).float(), "entropy": (z.log() - t / z)[:, 0].float(),
            "top_ids": ids.int(), "top": (x.gather(1, ids) - lse).float()}


# ---- the framework's calls -------------------------------------------------------------------------

@functools.lru_cache(None)
def _context():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "velo-core_amd"))
    import velokv
    return velokv, velokv.Context(0)


class _Raw:
    """Device memory of a pool as a torch tensor writes it; keeps the pool."""

    def __init__(self, pool, ptr, shape, kind):
        self.pool = pool
        self.__cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (ptr, False), "version": 2}


def _fill(pool, name, codes, scale):
    """Writes tiles into layer 0 of a pool, in the pool's layout (include/velokv.h)."""
    view = pool.layer_view(0)
    tiles, hkv, _, dim = codes.shape
    width = 64 if dim <= 64 else 128
    codes = torch.nn.functional.pad(codes, (0, width - dim))
    if name == "v":
        codes = codes.reshape(tiles, hkv, 8, 2, width).transpose(3, 4)
    elif codes.dtype == torch.int8:
        codes = codes.reshape(tiles, hkv, TILE, width // 32, 2, 16).permute(0, 1, 4, 2, 3, 5)
    kind = {torch.int8: "|i1", torch.float16: "<f2", torch.float32: "<f4"}[codes.dtype]
    raw = _Raw(pool, getattr(view, name + "_codes"), tuple(codes.shape), kind)
    torch.as_tensor(raw, device="cuda").copy_(codes)
    if scale is None:
        return
    if scale.dtype == torch.float32:
        torch.as_tensor(_Raw(pool, getattr(view, name + "_scales"), tuple(scale.shape), "<f4"), device="cuda").copy_(scale)
    else:  # one word holds a tile's K and V scale
        pair = torch.as_tensor(_Raw(pool, view.k_scales, tuple(scale.shape) + (2,), "<f2"), device="cuda")
        pair[..., 0 if name == "k" else 1] = scale


def _own_cache(st):
    velokv, ctx = _context()
    case = st["case"]
    kinds = {"fp32": velokv.KV_F32, "fp16": velokv.KV_F16, "int8": velokv.KV_I8_REF, "int8blk": velokv.KV_I8_BLK}
    pool = velokv.Pool(ctx, 1, st["k"].shape[0] * TILE // case["page"], case["page"], case["kv_heads"], case["dim"], kinds[case["kv"]])
    _fill(pool, "k", st.pop("k"), st.pop("ks"))
    if "v" in st:
        _fill(pool, "v", st.pop("v"), st.pop("vs"))
    torch.cuda.synchronize()
    longest = int(_lengths(case).max())
    rows = dict(block_tables=st["table"].data_ptr(), bt_stride=st["table"].shape[1], context_lens=st["lens"].data_ptr(),
                n_seqs=case["seqs"], max_context_len=longest)
    st.update(ctx=ctx, pool=pool)
    if case["kind"] != "attend":
        st["index"] = velokv.KeyIndex(ctx, pool)
    if case["kind"] in ("select", "both"):  # the index that earlier steps left
        ctx.index_update(st["index"], 0, **rows)
        torch.cuda.synchronize()
    if case["kind"] == "index":  # no bounds yet: what the case reads back is what its update wrote
        n = len(st["touched"])
        st["lower"] = torch.empty((n, case["kv_heads"], case["dim"]), device="cuda")
        st["upper"] = torch.empty_like(st["lower"])
        if case["new"]:
            st["first"] = (st["lens"] - case["new"]).clamp(min=0)
            rows.update(first_tokens=st["first"].data_ptr(), max_tokens=case["new"])
        st.update(own=_own_index, rows=rows)
        return st
    st["list"] = st["pages"] if "pages" in st else torch.empty((case["seqs"], case["kv_heads"], case["pick"]), dtype=torch.int32, device="cuda")
    st["out"] = torch.empty((case["seqs"], case["heads"], case["dim"]), device="cuda")
    st["rows"] = dict(rows, q=st["q"].data_ptr(), q_dtype=velokv.DT_F32 if case["act"] == "fp32" else velokv.DT_F16,
                      n_heads=case["heads"], pages=st["list"].data_ptr(), n_pages=case["pick"])
    st["own"] = {"select": _own_select, "attend": _own_attend, "both": _own_both}[case["kind"]]
    return st


def _own_index(st):
    st["ctx"].index_update(st["index"], 0, **st["rows"])
    st["ctx"].index_read(st["index"], 0, st["touched"].data_ptr(), len(st["touched"]), st["lower"].data_ptr(), st["upper"].data_ptr())
    return [st["lower"], st["upper"]]


def _own_select(st):
    st["ctx"].select_pages(st["index"], 0, **st["rows"])
    return st["list"]


def _own_attend(st):
    st["ctx"].sparse_decode(st["pool"], 0, out=st["out"].data_ptr(), **st["rows"])
    return st["out"]


def _own_both(st):
    st["ctx"].select_decode(st["index"], 0, out=st["out"].data_ptr(), **st["rows"])
    return [st["list"], st["out"]]


def _own_logprobs(st):
    velokv, ctx = _context()
    case = st["case"]
    rows = case["rows"]
    st["answer"] = {"token": torch.empty((rows, case["given"]), device="cuda"), "entropy": torch.empty(rows, device="cuda"),
                    "top_ids": torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda"),
                    "top": torch.empty((rows, case["top"]), device="cuda")}
    got = st["answer"]
    st.update(ctx=ctx, own=_own_run_logprobs,
              call=dict(logits=st["x"].data_ptr(), dtype=velokv.DT_F32 if case["act"] == "fp32" else velokv.DT_F16,
                        n_rows=rows, vocab=case["vocab"], tokens=st["tokens"].data_ptr(), n_tokens=case["given"],
                        token_logprobs=got["token"].data_ptr(), entropy=got["entropy"].data_ptr(),
                        top_ids=got["top_ids"].data_ptr(), top_logprobs=got["top"].data_ptr(), n_top=case["top"]))
    return st


def _own_run_logprobs(st):
    st["ctx"].token_logprobs(**st["call"])
    return st["answer"]


# ---- the definitions in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    st = _inputs(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(st["x"], st["tokens"], case["top"])
    lens, table = _lengths(case), st["table"].cpu().numpy()
    per, dim, hkv = case["page"] // TILE, case["dim"], case["kv_heads"]

    def rows(name, s, pages, h):
        """Tokens of the s-th sequence's pages, one KV head: [tokens, dim] in 64 bits."""
        held = torch.from_numpy(table[s, pages].astype(np.int64)).cuda()
        tiles = (held[:, None] * per + torch.arange(per, device="cuda")).reshape(-1)
        x, scale = st[name][tiles, h].double(), st[name + "s"]
        if scale is not None:
            x = x * scale[tiles, h].double().reshape(len(tiles), -1, 1)
        return x.reshape(-1, dim)

    def bounds(s, page, h, tokens):
        """lower, upper codes and the scale; the inverse and each product are rounded to 32 bits, as defined."""
        k = rows("k", s, [page], h)[:tokens].float().double()
        lower, upper = k.amin(0), k.amax(0)
        top = torch.maximum(lower.abs(), upper.abs()).amax()
        inv = (127 / top).float().double() if top > 0 else top
        return (lower * inv).float().round().double(), (upper * inv).float().round().double(), (top / 127).float().double()

    if case["kind"] == "index":
        got = [[], []]
        a, b = _touched(case, lens)
        if int((b - a).sum()) * hkv > 4096:
            return None
        for s in range(case["seqs"]):
            for page in range(a[s], b[s]):
                both = [bounds(s, page, h, min(case["page"], int(lens[s]) - page * case["page"])) for h in range(hkv)]
                for i in (0, 1):
                    got[i].append(torch.stack([x[i] * x[2] for x in both]))
        return [torch.stack(g) for g in got]
    if case["kind"] == "select":
        return None
    group = case["heads"] // hkv

    def chosen(s, h):
        """The pages of the s-th sequence that KV head h attends to: whole numbers, each rounding as defined."""
        count = int(_ceil(lens[s], case["page"]))
        if count <= case["pick"]:
            return np.arange(count)
        k = rows("k", s, np.arange(count), h).float().double()
        k[int(lens[s]):] = k[int(lens[s]) - 1]
        k = k.reshape(count, case["page"], dim)
        lower, upper = k.amin(1), k.amax(1)
        top = torch.maximum(lower.abs(), upper.abs()).amax(1, keepdim=True)
        inv = torch.where(top > 0, 127 / top, 0).float().double()
        lower, upper = (lower * inv).float().round().double(), (upper * inv).float().round().double()
        q = st["q"][s, h * group:(h + 1) * group].double()
        q_top = q.abs().amax(1, keepdim=True)
        q = (q * (127 / q_top).float().double()).float().round().double()
        dot = torch.where(q[:, None] < 0, q[:, None] * lower, q[:, None] * upper).sum(-1)
        score = ((dot * (top / 127).float().double().T).float().double() * (q_top / 127).float().double()).float().amax(0)
        score = score.cpu().numpy().astype(np.float64)
        score[[0, -1]] = np.inf
        return np.sort(np.lexsort((np.arange(count), -score))[:case["pick"]])

    out = torch.zeros((case["seqs"], case["heads"], dim), dtype=torch.float64, device="cuda")
    lists = st["pages"].cpu().numpy().astype(np.int64) if case["kind"] == "attend" else None
    for s in range(case["seqs"]):
        for h in range(hkv):
            listed_pages = chosen(s, h) if lists is None else lists[s, h][lists[s, h] >= 0]
            if not len(listed_pages):
                continue
            pos = (listed_pages[:, None] * case["page"] + np.arange(case["page"])).reshape(-1)
            there = torch.from_numpy(pos < lens[s]).cuda()
            k, v = rows("k", s, listed_pages, h)[there], rows("v", s, listed_pages, h)[there]
            score = st["q"][s, h * group:(h + 1) * group].double() @ k.T / math.sqrt(dim)
            out[s, h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out if case["kind"] == "attend" else [None, out]


def _exact_logprobs(x, tokens, n):
    got = {"token": [], "entropy": [], "top_ids": None, "top": []}
    for lo in range(0, len(x), 128):
        y = x[lo:lo + 128].double()
        lse = torch.logsumexp(y, -1, keepdim=True)
        p = (y - lse).exp()
        got["token"].append(y.gather(1, tokens[lo:lo + 128].long()) - lse)
        got["entropy"].append(torch.where(p > 0, p * (lse - y), 0).sum(-1))
        got["top"].append(y.topk(n, -1).values - lse)
    return {k: v if v is None else torch.cat(v) for k, v in got.items()}

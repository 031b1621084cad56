"""Page numbers outside of the pool in 4-bit attention of runs of tokens: their tokens are left out, whichever kernel a sequence goes through and
whatever else the call holds.  Tolerances are those of tests/test_gpu_kv_q4.py."""
import numpy as np
import pytest

from tests import helpers as H
from tests import test_gpu_kv_q4 as T

pytestmark = pytest.mark.gpu
env = T.env
BAD = [-1, 2 ** 31 - 1, -2 ** 31, 10 ** 6, -5]


def attention(q, k, v, scale, there):
    """As oracle.kv_q4.attention, over the keys that are there; rows that see none are zeros."""
    n, hq, hd = q.shape
    hkv, ctx, _ = k.shape
    out, size = np.zeros((n, hq, hd)), 0.0
    sees = there[None] & (np.arange(ctx)[None] <= ctx - n + np.arange(n)[:, None])
    some = sees.any(-1)
    for h in range(hq):
        kk, vv = k[h // (hq // hkv)], v[h // (hq // hkv)]
        s = np.where(sees, q[:, h] @ kk.T * scale, -np.inf)
        size = max(size, float((np.abs(q[:, h]) @ np.abs(kk).T * scale).max()))
        w = np.exp(s[some] - s[some].max(-1, keepdims=True))
        out[some, h] = w @ vv / w.sum(-1, keepdims=True)
    return out, size


def run(env, cache, tables, cu, lengths, q, hq, hkv, hd, page):
    ctx, K = env
    out = ctx.buf(np.full(q.shape, 0x7FC1, np.uint16))
    K.paged_attn_prefill_q4(ctx, ctx.buf(T.as_bf16(q)), cache.pool, cache.pages, ctx.buf(tables), cache.max_blocks, cu, lengths, hq, hkv, hd, page, hd ** -0.5, out)
    ctx.sync()
    return H.bf16_to_f32_np(out.download())


@pytest.mark.parametrize("where", ["first", "among the cached", "under the queries", "last", "every other", "all"])
@pytest.mark.parametrize("seqs, hq, hkv, hd, page", [
    ([(2, 500), (2, 400)], 32, 8, 128, 16),           # few columns
    ([(300, 500), (300, 400), (40, 7)], 8, 2, 128, 16),  # tensor cores, whole segments
    ([(200, 300), (1, 90)], 32, 8, 128, 48),          # pages that end inside a tile
    ([(100, 6000)], 8, 1, 128, 128),                  # keys split over blocks, pages of whole tiles
    ([(300, 2500), (129, 60)], 4, 2, 64, 64),
    ([(600, 0)], 12, 2, 64, 32),
])
def test_pages_outside_of_the_pool_are_left_out(env, where, seqs, hq, hkv, hd, page):
    lengths = [a + b for a, b in seqs]
    cache = T.Cache(env, hq + len(seqs), lengths, hkv, hd, page)
    cu = np.concatenate([[0], np.cumsum([a for a, _ in seqs])]).astype(np.int32)
    q = T.queries(hq, int(cu[-1]), hq, hd)
    tables = cache.tables.copy()
    blocks, cached = -(-lengths[0] // page), seqs[0][1] // page
    gone = {"first": [0], "among the cached": range(cached // 2, cached // 2 + 3), "under the queries": [blocks - 1 - (blocks - cached) // 2], "last": [blocks - 1],
            "every other": range(0, blocks, 2), "all": range(blocks)}[where]
    gone = [b for b in gone if b < blocks]
    tables[0, gone] = [(BAD + [cache.pages])[i % 6] for i in range(len(gone))]  # of the first sequence
    there = np.ones(blocks * page, bool)
    for b in gone:
        there[b * page:(b + 1) * page] = False
    got = run(env, cache, tables, cu, lengths, q, hq, hkv, hd, page)
    for i, n in enumerate(lengths):
        rows = slice(cu[i], cu[i + 1])
        ref, size = attention(q[rows], cache.k[i], cache.v[i], hd ** -0.5, there[:n] if i == 0 else np.ones(n, bool))
        tol = T.tolerance(ref, size, np.abs(cache.v[i]).max(), n, many=True)
        assert (np.abs(got[rows] - ref) <= tol).all(), (i, np.nanmax(np.abs(got[rows] - ref) - tol))
    if where == "all":
        assert (got[:cu[1]] == 0).all()


def test_neighbours_do_not_decide_what_a_bad_page_means(env):
    """The same sequence alone, where its few columns stream the records, and next to one that takes the call through the tensor cores."""
    hq, hkv, hd, page = 32, 8, 128, 16
    cache = T.Cache(env, 4, [406, 900], hkv, hd, page)
    q = T.queries(4, 906, hq, hd)
    tables = cache.tables.copy()
    tables[0, 3:9] = -1
    alone = run(env, cache, tables[:1], [0, 6], [406], q[:6], hq, hkv, hd, page)
    beside = run(env, cache, tables, [0, 6, 906], [406, 900], q, hq, hkv, hd, page)[:6]
    there = np.ones(406, bool)
    there[48:144] = False
    ref, size = attention(q[:6], cache.k[0], cache.v[0], hd ** -0.5, there)
    for got in (alone, beside):
        assert (np.abs(got - ref) <= T.tolerance(ref, size, np.abs(cache.v[0]).max(), 406, many=True)).all()

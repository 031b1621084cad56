"""4-bit attention of long contexts, with queries that each look for one key: a record that is left out, or a causal mask that is off by one, changes
rows by the size of the values, where the rounding of the weights allows a hundredth of it.

Tolerance: that of tests/test_gpu_kv_q4.py with 2^-8 sum(w |v|) / sum(w) of each element in the place of its bound by the largest value.  That it tells
such mistakes apart is shown on the CPU, by planting them in the reference."""
import numpy as np
import pytest

from oracle import kv_q4 as O
from tests import helpers as H
from tests import test_gpu_kv_q4 as T

env = T.env
CASES = [
    # new, cached, hq, hkv, hd, page
    (100, 6000, 8, 1, 128, 16),   # keys split over blocks at uneven tiles
    (300, 5001, 4, 2, 64, 64),
    (48, 3000, 16, 2, 128, 64),
    (700, 1300, 6, 2, 128, 48),   # whole segments
    (517, 0, 5, 1, 64, 16),
    (6, 4000, 64, 1, 128, 16),    # few columns: the other kernel
]


class Host:
    @staticmethod
    def buf(a):
        return a


def inputs(seed, new, cached, hq, hkv, hd, page, ctx=Host):
    """A cache and queries: of six rows of a kv head one looks for the first key that it does not see, one for the last that it sees, and the others
    for the records one after the other."""
    n = new + cached
    cache = T.Cache((ctx, None), seed, [n], hkv, hd, page)
    rng = np.random.default_rng(seed)
    q, group = np.zeros((new, hq, hd)), hq // hkv
    wanted = np.zeros((new, hq), np.int64)
    for h in range(hq):
        for r in range(new):
            last = cached + r
            i = r * group + h % group
            t = (last + 1, last)[i % 6] if i % 6 < 2 else ((i // 6 * 4 + i % 6 - 2) * 16 + rng.integers(16)) % (last + 1)
            wanted[r, h] = t
            q[r, h] = 2.5 * cache.k[0][h // group][min(t, n - 1)]
    return cache, O.bf16(q), wanted


def attention(q, k, v, scale, late=0, without=None):
    """Result, tolerance.  Mistakes to plant: every query sees `late` keys more; a record is missing."""
    n, hq, hd = q.shape
    hkv, ctx, _ = k.shape
    out, weighed, size = np.zeros((n, hq, hd)), np.zeros((n, hq, hd)), 0.0
    hidden = np.arange(ctx)[None] > ctx - n + late + np.arange(n)[:, None]
    if without is not None:
        hidden |= (np.arange(ctx)[None] // 16) == without
    for h in range(hq):
        kk, vv = k[h // (hq // hkv)], v[h // (hq // hkv)]
        s = np.where(hidden, -np.inf, q[:, h] @ kk.T * scale)
        size = max(size, float((np.abs(q[:, h]) @ np.abs(kk).T * scale).max()))
        with np.errstate(invalid="ignore"):  # (a row that a mistake leaves without keys)
            w = np.exp(s - s.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        out[:, h], weighed[:, h] = w @ vv, w @ np.abs(vv)
    return out, 2.0 ** -8 * weighed + T.tolerance(out, size, np.abs(v).max(), ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_each_query_finds_its_key(env, case):
    ctx, K = env
    new, cached, hq, hkv, hd, page = case
    cache, q, _ = inputs(40 + new, *case, ctx=ctx)
    out = ctx.empty(q.shape, np.uint16)
    K.paged_attn_prefill_q4(ctx, ctx.buf(T.as_bf16(q)), cache.pool, cache.pages, cache.dev_tables, cache.max_blocks, [0, new], [new + cached], hq, hkv, hd, page,
                            hd ** -0.5, out)
    ctx.sync()
    ref, tol = attention(q, cache.k[0], cache.v[0], hd ** -0.5)
    off = np.abs(H.bf16_to_f32_np(out.download()) - ref)
    assert (off <= tol).all(), (np.argwhere(~(off <= tol))[:4], np.nanmax(off - tol))


@pytest.mark.parametrize("case", CASES)
def test_the_tolerance_tells_mistakes_apart(case):
    new, cached, hq, hkv, hd, page = case
    cache, q, wanted = inputs(40 + new, *case)
    k, v = cache.k[0], cache.v[0]
    ref, tol = attention(q, k, v, hd ** -0.5)
    off = lambda **mistake: (np.abs(attention(q, k, v, hd ** -0.5, **mistake)[0] - ref) > tol).any(-1)  # a row with an element that is off
    rows = np.arange(new)[:, None] + cached
    # A query for the first hidden key sees it; the last row has none behind it.
    assert off(late=1)[(wanted == rows + 1) & (rows + 1 < new + cached)].mean() > 0.5
    if cached:
        assert off(late=-1)[wanted == rows].mean() > 0.5
    for record in np.random.default_rng(1).permutation(max(cached // 16, 6))[:6]:  # every record of the cached tokens is looked for
        looks = (wanted // 16 == record) & (rows >= 16 * record + 15)
        assert off(without=record)[looks].any()
    assert set(range(cached // 16)) <= set((wanted // 16).reshape(-1).tolist())

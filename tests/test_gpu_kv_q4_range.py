"""The 4-bit cache at the ends of what its numbers reach: large and small groups, and tokens that hold no numbers.

What the append stores is compared bit for bit with the statement in 64 bits, so nothing here has a tolerance but the attention, whose tolerance is
that of tests/test_gpu_kv_q4.py."""
import numpy as np
import pytest

from oracle import kv_q4 as O
from tests import helpers as H
from tests import test_gpu_kv_q4 as T

pytestmark = pytest.mark.gpu
env = T.env


def stored(pool, page, hkv, hd, slot, kvh, is_v):
    """Codes, scales and biases of a token's head, as the header of the C ABI describes the record."""
    base = ((slot // page * hkv + kvh) * (page // 16) + slot % page // 16) * O.record_bytes(hd)
    t, rec = slot % 16, pool.reshape(-1)[base:base + O.record_bytes(hd)]
    if not is_v:
        raw = rec[t * hd // 2:(t + 1) * hd // 2]
    else:
        words = [((t // 8 * 8 + d // (hd // 8)) * 4 + t % 8 // 2) * (hd // 32) + d % (hd // 8) // 4 for d in range(0, hd, 4)]
        raw = np.concatenate([rec[8 * hd + 4 * w + t % 2 * 2:][:2] for w in words])
    codes = np.stack([raw & 15, raw >> 4], -1).reshape(-1)
    sb = np.array([rec[16 * hd + ((hd // 64 if is_v else 0) + g) * 64 + 4 * t:][:4].copy().view(np.uint32)[0] for g in range(hd // 64)])
    as_float = lambda x: (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return codes, as_float(sb & 0xffff), as_float(sb >> 16)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [-133, -131, -129, -128, -127, -126, -120, -100, -64, 50, 58, 59, 60, 61, 62, 63, 64, 70, 100, 120, 122, 123, 124, 125, 126])
def test_append_of_large_and_small_values(env, hd, power):
    """Normal numbers times 2^power, groups on one side of zero, and groups of equal values."""
    n, hq, hkv, page, pages = 24, 1, 1, 16, 2
    rng = np.random.default_rng(power + 500)
    x = np.clip(rng.standard_normal((n, hq + 2 * hkv, hd)), -3, 3)
    x[1::4] = np.sign(x[1::4]) * 2  # ends that are as far from zero as one another
    x[2::4] = 2 + np.abs(x[2::4]) / 4
    x[3::4] = x[3::4, :, :1]
    qkv = O.bf16(x * 2.0 ** power)
    pos, slots = np.zeros(n, np.int32), rng.permutation(pages * page)[:n].astype(np.int32)
    cos, sin = np.ones((1, hd // 2)), np.zeros((1, hd // 2))
    _, after, q, (k, v) = T.run_append(env, qkv, pos, slots, cos, sin, None, None, page, pages, hq, hkv, hd)
    assert np.array_equal(H.bf16_to_f32_np(q), qkv[:, :1])
    bad = 0
    for t in range(n):
        for is_v, rows, got in ((False, qkv[:, 1], k), (True, qkv[:, 2], v)):
            codes, scale, bias = O.quantize(rows[t])
            have = stored(after, page, hkv, hd, int(slots[t]), 0, is_v)
            assert np.array_equal(have[1], scale, equal_nan=True) and np.array_equal(have[2], bias) and np.array_equal(have[0], codes), (t, is_v)
            assert np.array_equal(H.bf16_to_f32_np(got[t, 0]), O.values(codes, scale, bias), equal_nan=True), (t, is_v)
            bad += np.isnan(scale).sum()
    assert (bad > 0) == (power >= 61)  # 2 / 8 2^power is 2^59 there
    assert bad < 2 * n * (hd // 64)  # (equal values are kept as they are, however large)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new, cached", [(1, 20), (3, 37), (400, 700)])
def test_attention_to_large_values(env, hd, new, cached):
    """Values up to the largest that are kept: finite sums, and the same numbers that the append gives back."""
    ctx, K = env
    n, hq, hkv, page = cached + new, 4, 1, 16
    pages = (n + page - 1) // page
    rng = np.random.default_rng(hd + new)
    qkv = rng.standard_normal((n, hq + 2, hd))
    qkv[:, hq + 1] *= 2.0 ** 60 / np.abs(qkv[:, hq + 1]).max()
    qkv = O.bf16(qkv)
    order = rng.permutation(pages).astype(np.int32)
    slots = (order[np.arange(n) // page] * page + np.arange(n) % page).astype(np.int32)
    cos, sin = np.ones((1, hd // 2)), np.zeros((1, hd // 2))
    _, pool, _, (k, v) = T.run_append(env, qkv, np.zeros(n, np.int32), slots, cos, sin, None, None, page, pages, hq, hkv, hd)
    cache = T.Cache.__new__(T.Cache)
    cache.k, cache.v = ([H.bf16_to_f32_np(x).astype(np.float64).transpose(1, 0, 2)] for x in (k, v))
    assert np.abs(cache.v[0]).max() > 2.0 ** 59
    q = qkv[-new:, :hq]
    out = ctx.empty(q.shape, np.uint16)
    K.paged_attn_prefill_q4(ctx, ctx.buf(T.as_bf16(q)), ctx.buf(pool), pages, ctx.buf(order[None]), pages, [0, new], [n], hq, hkv, hd, page, 0.1, out)
    ctx.sync()
    T.check_rows(out.download(), q, cache, 0, 0.1, many=new * hq > 32)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [2.0 ** 59, 2.0 ** 60, -2.0 ** 63, 2.0 ** 100])
@pytest.mark.parametrize("new, cached", [(3, 37), (60, 37), (400, 700), (900, 700)])
def test_prefill_keeps_a_scale_that_is_too_large_from_earlier_queries(env, hd, scale, new, cached):
    """A pool of another writer may hold a value's scale that attention cannot take: queries that do not see the token are as without it."""
    ctx, K = env
    hq, hkv, page = 4, 2, 16
    n = cached + new
    cache = T.Cache(env, 92, [n], hkv, hd, page)
    q = T.queries(92, new, hq, hd)
    bad = cached + new // 2
    pool = cache.pool.download()
    at = 16 * hd + 64 * (hd // 64) + (bad % 16) * 4
    pool[cache.tables[0, bad // page], 0, 0, at:at + 2] = O.bits([scale]).astype(np.uint16).view(np.uint8)  # of kv head 0, first group
    out = ctx.empty(q.shape, np.uint16)
    K.paged_attn_prefill_q4(ctx, ctx.buf(T.as_bf16(q)), ctx.buf(pool), cache.pages, cache.dev_tables, cache.max_blocks, [0, new], [n], hq, hkv, hd, page, 0.1, out)
    ctx.sync()
    got = out.download()
    before = new // 2
    assert np.isfinite(H.bf16_to_f32_np(got[:, 2:])).all()  # the other kv head
    cache.k[0], cache.v[0] = cache.k[0][:, :cached + before], cache.v[0][:, :cached + before]
    T.check_rows(got[:before], q[:before], cache, 0, 0.1, many=new * hq // hkv > 32)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new, cached", [(1, 20), (1, 3000), (3, 37), (400, 700), (100, 6000)])
def test_scores_far_below_zero(env, hd, new, cached):
    """All scores are the same number of some -2^113: the result is the mean of the values, not nothing.  Tolerance: equal weights are 1 each, which is
    exact, so what is left are sums in f32 of at most n terms and the result's rounding."""
    ctx, K = env
    n, hq, hkv, page = cached + new, 4, 1, 16
    pages = (n + page - 1) // page
    rng = np.random.default_rng(hd + n)
    qkv = rng.standard_normal((n, hq + 2, hd))
    qkv[:, :hq], qkv[:, hq] = 2.0 ** 90, -2.0 ** 20
    qkv = O.bf16(qkv)
    slots, order = np.arange(n, dtype=np.int32), np.arange(pages, dtype=np.int32)
    cos, sin = np.ones((1, hd // 2)), np.zeros((1, hd // 2))
    _, pool, _, (k, v) = T.run_append(env, qkv, np.zeros(n, np.int32), slots, cos, sin, None, None, page, pages, hq, hkv, hd)
    assert (H.bf16_to_f32_np(k) == -2.0 ** 20).all()
    v = H.bf16_to_f32_np(v).astype(np.float64)[:, 0]
    q, out = ctx.buf(T.as_bf16(qkv[-new:, :hq])), ctx.empty((new, hq, hd), np.uint16)
    K.paged_attn_prefill_q4(ctx, q, ctx.buf(pool), pages, ctx.buf(order[None]), pages, [0, new], [n], hq, hkv, hd, page, 0.125, out)
    ctx.sync()
    ref = (np.cumsum(v, 0) / np.arange(1, n + 1)[:, None])[-new:, None]
    tol = 2 * n * 2.0 ** -24 * np.abs(v).max() + 2.0 ** -8 * np.abs(ref)
    assert (np.abs(H.bf16_to_f32_np(out.download()) - ref) <= tol).all()
    if new == 1:
        K.paged_attn_decode_q4(ctx, q, ctx.buf(pool), pages, ctx.buf(order[None]), ctx.buf(np.array([n], np.int32)), 1, hq, hkv, hd, page, 0.125, out, pages)
        ctx.sync()
        assert (np.abs(H.bf16_to_f32_np(out.download()) - ref) <= tol).all()

"""Calls over a 4-bit cache next to what goes wrong elsewhere."""
import numpy as np
import pytest

from oracle import kv_q4 as O
from tests import helpers as H
from tests import test_gpu_kv_q4 as T

pytestmark = pytest.mark.gpu
env = T.env


def test_calls_behind_an_allocation_that_failed(env):
    """The error is the allocation's: the calls behind it run, and say so."""
    from mlx_llm_b200 import _lib

    ctx, K = env
    cache = T.Cache(env, 11, [40, 333], 2, 128, 16)
    q = T.queries(11, 2, 8, 128)
    dev, out, n = ctx.buf(T.as_bf16(q)), ctx.empty(q.shape, np.uint16), ctx.buf(np.array([40, 333], np.int32))
    for _ in range(2):
        with pytest.raises(_lib.B2Error):
            ctx.empty((1 << 44,), np.uint8)
        K.paged_attn_decode_q4(ctx, dev, cache.pool, cache.pages, cache.dev_tables, n, 2, 8, 2, 128, 16, 0.1, out, cache.max_blocks)
        ctx.sync()
        for i in range(2):
            T.check_rows(out.download()[i:i + 1], q[i:i + 1], cache, i, 0.1)


@pytest.mark.parametrize("tail", [11, 15, -5])
def test_decode_of_a_context_that_ends_just_below_2_31(env, tail):
    """One page, named again and again, and another one at the end whose last tokens lie behind the context and hold no numbers."""
    ctx, K = env
    hd, page = 64, 1 << 20
    length, records = 2 ** 31 - 32 + tail, page // 16
    rng = np.random.default_rng(tail + 9)
    pool = np.frombuffer(rng.bytes(2 * records * 1152), np.uint8).reshape(2, records, 1152).copy()
    words = pool[..., 1024:].view(np.uint32)  # [2, records, 16 of K and 16 of V]
    k_scale, k_bias, v_scale, v_bias = 2.0 ** -5, -0.234375, 2.0 ** -4, 1.0
    words[..., :16] = O.bits([k_scale])[0] | O.bits([k_bias])[0] << 16
    words[..., 16:] = O.bits([v_scale])[0] | O.bits([v_bias])[0] << 16
    rest = length - 2047 * page
    behind = np.arange(page).reshape(records, 16) >= rest
    words[1, :, :16][behind] = 0xFFFFFFFF
    words[1, :, 16:][behind] = 0xFFFFFFFF
    q = T.queries(tail + 9, 1, 1, hd)
    dev, out = ctx.buf(pool), ctx.empty((1, 1, hd), np.uint16)
    tables = np.zeros((1, 2048), np.int32)
    tables[0, -1] = 1
    K.paged_attn_decode_q4(ctx, ctx.buf(T.as_bf16(q)), dev, 2, ctx.buf(tables), ctx.buf(np.array([length], np.int32)), 1, 1, 1, hd, page, 0.125, out, 2048)
    ctx.sync()
    dev.free()
    got = H.bf16_to_f32_np(out.download())[0, 0]
    total, sums = 0.0, np.zeros(hd)
    for which, count, times in ((0, page, 2047), (1, rest, 1)):
        raw = pool[which, :, :512].reshape(page, hd // 2)
        keys = O.bf16(np.arange(16) * k_scale + k_bias)[np.stack([raw & 15, raw >> 4], -1).reshape(page, hd)[:count]].astype(np.float32)
        w = np.exp((keys @ q[0, 0].astype(np.float32)).astype(np.float64) * 0.125) * times
        # V: u32 [2 halves][8 blocks][4 pairs][2 words], a half word per token: its four dims
        raw = pool[which, :, 512:1024].reshape(records, 2, 8, 4, 2, 2, 2).transpose(0, 1, 3, 5, 2, 4, 6).reshape(page, hd // 2)
        vals = O.bf16(np.arange(16) * v_scale + v_bias)[np.stack([raw & 15, raw >> 4], -1).reshape(page, hd)[:count]].astype(np.float32)
        total += w.sum()
        sums += w @ vals
    # The f32 sums: a warp's run is 56 680 records of the 2^27, and a lane adds to its sum, or a product to its accumulator, at most four times a
    # record; what joins the warps' parts adds 2368 times at most.  Scores are below 64 * 0.24 * 4 / 8 = 8 (a weight is off by 264 2^-24 of that).
    steps = 4 * 56680 + 2368
    assert np.isfinite(got).all()
    assert (np.abs(got - sums / total) <= 2 * (steps * 2.0 ** -24 + 264 * 2.0 ** -24 * 8 + 2.0 ** -16) * 2 + 2.0 ** -8 * 2).all()

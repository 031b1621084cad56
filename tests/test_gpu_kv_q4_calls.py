"""Calls over a 4-bit cache next to what goes wrong elsewhere."""
import numpy as np
import pytest

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

"""The queries of the append into a 4-bit cache, whose head sizes take paths of their own through the norm: the same bits as the append into bf16 pages
gives, and each element against the statement in 64 bits.

Tolerance with norms.  The norm's f32 sum is off by less than 2^-16 relatively, so a normed element is the statement's bf16 number a or its neighbour:
2^-7 |a| at most.  Each product a c is rounded to bf16, here and there, half a step, 2^-8 of it, and so is their sum: in all
(2^-7 + 2 2^-8) (|a c| + |b s|) + 2 2^-8 |result|, and the products of these errors, which 2 % more cover."""
import numpy as np
import pytest

from oracle import kv_q4 as O
from tests import helpers as H
from tests import test_gpu_kv_q4 as T

pytestmark = pytest.mark.gpu
env = T.env


@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("hq, hkv", [(8, 2), (1, 1), (7, 1), (3, 3), (15, 5)])
@pytest.mark.parametrize("hd", [64, 128])
def test_queries(env, hd, hq, hkv, norms):
    ctx, K = env
    n, page, pages = 37, 16, 6
    rng, qkv, pos, slots, cos, sin = T.append_case(60 + hq, n, hq, hkv, hd, page, pages)
    qkv[3] *= 2.0 ** -20  # (where epsilon counts)
    qkv[5] *= 2.0 ** 20
    qn, kn = (O.bf16(1 + 0.2 * rng.standard_normal(hd)) if there else None for there in norms)
    _, _, q, _ = T.run_append(env, qkv, pos, slots, cos, sin, qn, kn, page, pages, hq, hkv, hd, values=False)
    wide = [ctx.buf(np.zeros((pages, hkv, page, hd), np.uint16)) for _ in range(2)]
    q16 = ctx.empty((n, hq, hd), np.uint16)
    norm = lambda w: None if w is None else ctx.buf(T.as_bf16(w))
    K.rope_kv_append(ctx, ctx.buf(T.as_bf16(qkv)), n, hq, hkv, hd, ctx.buf(pos), ctx.buf(slots), ctx.buf(T.as_bf16(cos)), ctx.buf(T.as_bf16(sin)), norm(qn),
                     norm(kn), 1e-6, page, wide[0], wide[1], q16)
    ctx.sync()
    assert np.array_equal(q, q16.download())
    x = qkv[:, :hq]
    a = x if qn is None else O.bf16(x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * qn)
    ref, got = T.rope_in_64(a, cos[pos], sin[pos]), H.bf16_to_f32_np(q)
    if qn is None:
        assert np.array_equal(got, ref)
        return
    c, s = (np.concatenate([np.abs(t[pos])[:, None]] * 2, -1) for t in (cos, sin))
    other = np.roll(np.abs(a), hd // 2, -1)
    tol = 1.02 * ((2.0 ** -7 + 2.0 ** -7) * (np.abs(a) * c + other * s) + 2.0 ** -7 * np.abs(ref))
    assert (np.abs(got - ref) <= tol).all()
    assert (got == ref).mean() > 0.99

"""What the entry points over a 4-bit cache and the rules on logits refuse, and sizes: nothing of it reaches a GPU."""
import ctypes as C

import numpy as np
import pytest

from oracle import kv_q4 as O

HERE = C.create_string_buffer(1 << 16)  # stands for a context and for device memory: a refusal comes before either is looked at


@pytest.fixture(scope="module")
def kernels():
    from mlx_llm_b200 import build, kernels

    build.build()
    return kernels


class FakeContext:
    h = C.c_void_p(C.addressof(HERE))


CTX = FakeContext()
AT = (C.addressof(HERE) + 255) & ~255


def refused(call, code):
    from mlx_llm_b200 import _lib

    with pytest.raises(_lib.B2Error) as e:
        call()
    assert e.value.code == code, str(e.value)
    assert "b2_" in str(e.value)


def append(K, ctx=CTX, qkv=AT, T=1, hq=4, hkv=2, hd=128, pos=AT, slots=AT, page=16, pool=AT, pages=4, q_out=AT, k_out=None):
    K.rope_kv_append_q4(ctx, qkv, T, hq, hkv, hd, pos, slots, AT, AT, None, None, 1e-6, page, pool, pages, q_out, k_out)


def decode(K, q=AT, pool=AT, pages=4, tables=AT, n=1, hq=4, hkv=2, hd=128, page=16, out=AT, blocks=4, scale=0.1):
    K.paged_attn_decode_q4(CTX, q, pool, pages, tables, AT, n, hq, hkv, hd, page, scale, out, blocks)


def prefill(K, q=AT, pool=AT, pages=4, blocks=4, cu=(0, 1), ctx=(1,), hq=4, hkv=2, hd=128, page=16, out=AT, scale=0.1):
    K.paged_attn_prefill_q4(CTX, q, pool, pages, AT, blocks, cu, ctx, hq, hkv, hd, page, scale, out)


@pytest.mark.parametrize("call", [append, decode, prefill])
@pytest.mark.parametrize("bad, code", [
    (dict(hd=96), -5), (dict(hd=256), -5), (dict(page=8), -5), (dict(page=0), -5), (dict(page=24), -5), (dict(hq=5), -7), (dict(hkv=0), -7),
    (dict(hq=0), -7), (dict(pages=0), -7), (dict(pages=1 << 28), -7), (dict(pool=AT + 8), -5), (dict(pool=None), -7),
])
def test_pool_and_heads(kernels, call, bad, code):
    refused(lambda: call(kernels, **bad), code)


@pytest.mark.parametrize("call, bad, code", [
    (append, dict(qkv=None), -7), (append, dict(pos=None), -7), (append, dict(slots=None), -7), (append, dict(q_out=None), -7), (append, dict(T=-1), -7),
    (append, dict(q_out=AT + 2), -5), (append, dict(k_out=AT + 2), -5), (append, dict(T=1 << 29), -5),
    (decode, dict(q=None), -7), (decode, dict(tables=None), -7), (decode, dict(n=-1), -7), (decode, dict(blocks=0), -7), (decode, dict(q=AT + 2), -5),
    (decode, dict(out=AT + 4), -5), (decode, dict(n=1 << 20, blocks=1 << 12), -5),
    (decode, dict(scale=0.0), -7), (decode, dict(scale=float("nan")), -7), (prefill, dict(scale=-1.0), -7), (prefill, dict(scale=float("inf")), -7),
    (prefill, dict(q=None), -7), (prefill, dict(cu=(0, 2)), -7), (prefill, dict(cu=(3, 1), ctx=(9,)), -7), (prefill, dict(cu=(-1, 1), ctx=(9,)), -7),
    (prefill, dict(ctx=(65,)), -7), (prefill, dict(out=AT + 8), -5), (prefill, dict(ctx=(0x7fffff01,), blocks=1 << 27), -5),
])
def test_arguments(kernels, call, bad, code):
    refused(lambda: call(kernels, **bad), code)


def test_calls_without_work(kernels):
    prefill(kernels, cu=(0,), ctx=())


@pytest.mark.parametrize("rules, kw, code", [
    ({}, dict(logits=None), -7), ({}, dict(argmax=None), -7), ({}, dict(vocab=0), -7), ({}, dict(rows=-1), -7), ({}, dict(ld=63), -7),
    (dict(history=AT), {}, -7), (dict(bias_id=AT, bias_off=AT), {}, -7), (dict(bias_id=AT, bias_value=AT), {}, -7),
    (dict(mask=AT, mask_words=1), {}, -7), ({}, dict(vocab=(1 << 30) + 1, ld=1 << 31), -5), ({}, dict(logits=AT + 1), -5), ({}, dict(logits=AT + 2, f32=True), -5), ({}, dict(out=AT + 1), -5),
])
def test_rules_on_logits(kernels, rules, kw, code):
    args = dict(dict(logits=AT, rows=1, vocab=64, argmax=AT), **kw)
    refused(lambda: kernels.logits_adjust(CTX, args.pop("logits"), args.pop("rows"), args.pop("vocab"), kernels.logit_rules(**rules), **args), code)


def test_pool_bytes(kernels):
    assert kernels.kv_q4_pool_bytes(10, 8, 128, 16) == 10 * 8 * 2304
    assert kernels.kv_q4_pool_bytes(10, 3, 64, 48) == 10 * 3 * 3 * 1152
    assert kernels.kv_q4_pool_bytes(1 << 25, 8, 128, 16) == (1 << 28) * 2304  # (past 32 bits)
    for bad in ((0, 8, 128, 16), (10, 0, 128, 16), (10, 8, 80, 16), (10, 8, 128, 20)):
        assert kernels.kv_q4_pool_bytes(*bad) == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_oracle_record_holds_every_nibble_once(hd):
    """The statement of the record that the GPU tests compare with: no two tokens share a byte, and none is left over."""
    pool = np.zeros(O.record_bytes(hd), np.uint8)
    for is_v in (False, True):
        for t in range(16):
            before = pool.copy()
            O.put(pool, 16, 1, hd, t, 0, is_v, np.full(hd, 15), np.full(hd // 64, -1.0), np.full(hd // 64, -1.0))
            assert np.count_nonzero(before != pool) == hd // 2 + 4 * (hd // 64) - np.count_nonzero(np.array([0xbf80bf80], np.uint32).view(np.uint8) == 0) * (hd // 64)
    assert pool[:16 * hd].min() == 255


def test_oracle_quantizes_to_half_a_step_and_ends_to_one():
    """Half a step inside the codes' range.  The range itself ends up to one step before the value opposite to the farthest one, e: with
    u = 15 |e| / span >= 7.5 and n = round(u) <= u + 1/2 the step is s = |e| / n, and span - 15 s = span (1 - u / n) <= span / 2n = 15 s / 2u <= s."""
    rng = np.random.default_rng(3)
    x = O.bf16(rng.standard_normal((200, 128)) * np.exp(rng.standard_normal((200, 1))) + rng.standard_normal((200, 1)))
    codes, scale, bias = O.quantize(x)
    step, c = np.repeat(np.abs(scale), 64, -1), np.asarray(codes)
    error = np.abs(O.values(codes, scale, bias) - x)
    # the rounding of the scale (2^-9 of 16 steps at most) and of the value (2^-8 of it) come on top
    rest = step * 16 * 2.0 ** -8 + np.abs(x) * 2.0 ** -7 + 1e-12
    assert (error <= step + rest).all()
    assert (error[c < 15] <= (step * 0.5 + rest)[c < 15]).all()
    assert np.array_equal(O.values(codes, scale, bias)[c == 0], np.repeat(bias, 64, -1)[c == 0])  # the farthest value is kept as it is

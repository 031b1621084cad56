"""What the Python side of the 4-bit cache and of the rules on logits checks before anything reaches the library."""
import numpy as np
import pytest

from tests.test_kv_q4_host import AT, CTX, append, decode, kernels, prefill, refused  # noqa: F401


@pytest.mark.parametrize("wrong", ["masks", "repetiton", "bias_ids", "history_dev", "h"])
def test_a_rule_that_is_not_there(kernels, wrong):
    with pytest.raises(TypeError, match=wrong):
        kernels.logit_rules(history=AT, history_off=AT, **{wrong: AT})


def test_rules_reach_their_fields(kernels):
    names = ["history", "history_off", "n_prompt", "repetition", "presence", "frequency", "bias_id", "bias_value", "bias_off", "mask", "mask_row"]
    rules = kernels.logit_rules(mask_words=5, **{n: 16 * (i + 1) for i, n in enumerate(names)})
    assert [getattr(rules, n) for n in names] == [16 * (i + 1) for i in range(len(names))] and rules.mask_words == 5
    assert kernels.logit_rules(mask=None).mask is None


@pytest.mark.parametrize("call", [decode, prefill])
@pytest.mark.parametrize("scale", [2.0 ** 62, 2.0 ** 63, 3e38, -2.0 ** 62])
def test_softmax_scales_that_attention_cannot_take(kernels, call, scale):
    refused(lambda: call(kernels, scale=scale), -7)


@pytest.mark.parametrize("call", [
    lambda K, a: decode(K, q=a), lambda K, a: decode(K, tables=a), lambda K, a: prefill(K, pool=a), lambda K, a: prefill(K, out=a), lambda K, a: append(K, pos=a),
    lambda K, a: K.logit_rules(mask=a), lambda K, a: K.logits_adjust(CTX, a, 1, 64, K.logit_rules(), argmax=AT),
    lambda K, a: K.logits_adjust(CTX, AT, 1, 64, K.logit_rules(), argmax=a),
])
def test_host_arrays_are_no_device_buffers(kernels, call):
    with pytest.raises(TypeError, match="host array"):
        call(kernels, np.zeros(64, np.int32))


@pytest.mark.parametrize("cu, ctx", [((0,), (1,)), ((0, 1), (1, 1)), ((), ()), ((0, 1, 2), (4,)), (((0, 1), (1, 2)), (4, 4, 4))])
def test_one_more_offset_than_sequences(kernels, cu, ctx):
    with pytest.raises(ValueError, match="cu_seqlens"):
        prefill(kernels, cu=cu, ctx=ctx)


def test_more_queries_than_a_plan_holds(kernels):
    """Refused before a list of them is made: memory that runs out would be an exception that no C caller can catch."""
    n = 0x7fffff00
    refused(lambda: prefill(kernels, cu=(0, n), ctx=(n,), blocks=1 << 27, hq=16, hkv=8), -5)
    refused(lambda: prefill(kernels, cu=(0, n), ctx=(n,), blocks=1 << 27, hq=1024, hkv=2), -5)
    refused(lambda: prefill(kernels, cu=(9, -(1 << 31)), ctx=(n,), blocks=1 << 27), -7)  # (a difference that 32 bits do not hold)


def test_numbers_of_numpy(kernels):
    """They go through to the library, whose refusal comes back; what is no number does not."""
    refused(lambda: decode(kernels, n=np.int64(-1)), -7)
    refused(lambda: decode(kernels, hd=np.int32(96)), -5)
    refused(lambda: append(kernels, T=np.int64(-1)), -7)
    refused(lambda: prefill(kernels, scale=np.float32(-1)), -7)
    refused(lambda: kernels.logits_adjust(CTX, AT, np.int64(-1), 64, kernels.logit_rules(mask_words=np.int64(4)), argmax=AT), -7)
    with pytest.raises(TypeError):
        decode(kernels, n=1.5)
    with pytest.raises(TypeError):
        decode(kernels, n="3")


def test_a_rule_that_is_not_there_set_by_hand(kernels):
    rules = kernels.logit_rules()
    with pytest.raises(AttributeError):
        rules.masks = AT

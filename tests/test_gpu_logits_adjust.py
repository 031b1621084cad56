"""Rules on logits and the greedy choice against their statement in f32 steps: equal bit for bit, since every step is one rounding."""
import numpy as np
import pytest

from oracle import kv_q4 as O
from tests import helpers as H

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    from mlx_llm_b200 import _lib, kernels

    ctx = _lib.Context(0)
    yield ctx, kernels
    ctx.close()


def offsets(lists):
    return np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)


def check(env, logits, f32, history=None, n_prompt=None, repetition=None, presence=None, frequency=None, bias=None, allowed=None, mask_row=None, pad=0,
          in_place=False, write=True, choose=True):
    """logits [rows, vocab]; history, bias (pairs) a list per row; allowed [masks, vocab]."""
    ctx, K = env
    rows, vocab = logits.shape
    kind = np.float32 if f32 else np.uint16
    held = np.full((rows, vocab + pad), np.nan, np.float32)
    held[:, :vocab] = logits if f32 else O.bf16(logits)
    raw = held.astype(np.float32) if f32 else H.f32_to_bf16_np(held)
    dev = ctx.buf(raw)
    rules, kw = {}, {}
    if history is not None:
        flat = np.concatenate([np.asarray(h, np.int32) for h in history] + [np.zeros(1, np.int32)])
        rules.update(history=ctx.buf(flat.astype(np.int32)), history_off=ctx.buf(offsets(history)))
    for name, x, t in (("n_prompt", n_prompt, np.int32), ("repetition", repetition, np.float32), ("presence", presence, np.float32), ("frequency", frequency, np.float32),
                       ("mask_row", mask_row, np.int32)):
        if x is not None:
            rules[name] = ctx.buf(np.asarray(x, t))
    if bias is not None:
        flat = [p for b in bias for p in b] + [(0, 0.0)]
        rules.update(bias_id=ctx.buf(np.array([p[0] for p in flat], np.int32)), bias_value=ctx.buf(np.array([p[1] for p in flat], np.float32)), bias_off=ctx.buf(offsets(bias)))
    if allowed is not None:
        words = (vocab + 31) // 32 + 1  # (a row of masks may be longer than the vocabulary)
        b = np.ones((len(allowed), words * 32), bool)
        b[:, :vocab] = allowed
        rules.update(mask=ctx.buf(np.packbits(b, axis=1, bitorder="little").view(np.uint32)), mask_words=words)
    out = dev if in_place else ctx.buf(np.full(raw.shape, 7, kind)) if write else None
    tokens = ctx.buf(np.full(rows + 1, -9, np.int32)) if choose else None
    K.logits_adjust(ctx, dev, rows, vocab, K.logit_rules(**rules), f32=f32, ld=vocab + pad, out=out, argmax=tokens)
    ctx.sync()
    got = out.download() if out is not None else None
    chosen = tokens.download() if choose else None
    if choose:
        assert chosen[rows] == -9
    if not in_place:
        assert dev.download().tobytes() == raw.tobytes()
    for i in range(rows):
        m = -1 if allowed is None else i if mask_row is None else mask_row[i]
        want, token = O.adjust(held[i, :vocab], history[i] if history is not None else (), n_prompt[i] if n_prompt is not None else 0,
                               repetition[i] if repetition is not None else 1.0, presence[i] if presence is not None else 0.0,
                               frequency[i] if frequency is not None else 0.0, bias[i] if bias is not None else (), allowed[m] if m >= 0 else None)
        if choose:
            assert chosen[i] == token, i
        if got is not None:
            row = got[i, :vocab] if f32 else H.bf16_to_f32_np(got[i, :vocab])
            want = want if f32 else np.where(np.isnan(want), want, O.bf16(want)).astype(np.float32)
            assert np.array_equal(row, want, equal_nan=True), i
            if pad:
                assert got[i, vocab:].tobytes() == (raw[i, vocab:] if in_place else np.full(pad, 7, kind)).tobytes()


def case(seed, rows, vocab, n_history, n_bias):
    rng = np.random.default_rng(seed)
    logits = 3 * rng.standard_normal((rows, vocab))
    history = [np.minimum((vocab * rng.random(rng.integers(0, 2 * n_history + 1)) ** 4).astype(np.int64), vocab - 1) for _ in range(rows)]
    bias = [[(int(i), float(b)) for i, b in zip(np.unique(rng.integers(0, vocab, rng.integers(0, 2 * n_bias + 1))), rng.normal(0, 4, vocab))] for _ in range(rows)]
    return rng, dict(logits=logits, history=history, n_prompt=[len(h) // 2 for h in history], repetition=rng.uniform(1, 1.5, rows).astype(np.float32),
                     presence=rng.uniform(0, 1, rows).astype(np.float32), frequency=rng.uniform(0, 1, rows).astype(np.float32), bias=bias)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows, vocab, history, bias", [(1, 1, 3, 1), (1, 7, 5, 2), (3, 33, 40, 5), (5, 1000, 100, 20), (2, 32001, 3000, 300), (9, 4096, 0, 0), (1, 128256, 600, 12)])
def test_all_rules(env, f32, rows, vocab, history, bias):
    rng, c = case(rows + vocab, rows, vocab, history, bias)
    check(env, f32=f32, allowed=rng.random((rows, vocab)) < rng.choice([0.02, 0.5, 0.98], (rows, 1)), **c)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows, vocab, history, bias", [(40, 4099, 300, 20), (40, 170001, 700, 20), (150, 1003, 60, 9), (150, 40000, 900, 30)])
def test_many_rows(env, f32, rows, vocab, history, bias):
    rng, c = case(rows + vocab, rows, vocab, history, bias)
    check(env, f32=f32, allowed=rng.random((rows, vocab)) < rng.choice([0.02, 0.5, 0.98], (rows, 1)), **c)


@pytest.mark.parametrize("f32", [False, True])
def test_vocabulary_of_several_rounds(env, f32):
    rng, c = case(5, 2, 420001, 5000, 400)
    check(env, f32=f32, allowed=rng.random((2, 420001)) < 0.5, **c)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rule", ["none", "repetition", "presence", "frequency", "bias", "mask"])
def test_each_rule_alone(env, f32, rule):
    rng, c = case(17, 4, 2500, 80, 30)
    kw = dict(logits=c["logits"])
    if rule in ("repetition", "presence", "frequency"):
        kw.update(history=c["history"])
        kw[rule] = c[rule]
    if rule == "bias":
        kw.update(bias=c["bias"])
    if rule == "mask":
        kw.update(allowed=rng.random((3, 2500)) < 0.3, mask_row=[2, -1, 0, 2])
    check(env, f32=f32, **kw)
    check(env, f32=f32, write=False, **kw)
    check(env, f32=f32, choose=False, **kw)
    check(env, f32=f32, in_place=True, **kw)


@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_apart(env, pad, in_place):
    rng, c = case(23, 5, 1003, 60, 9)
    check(env, f32=False, pad=pad, in_place=in_place, allowed=rng.random((5, 1003)) < 0.5, **c)
    check(env, f32=True, pad=pad, in_place=in_place, allowed=rng.random((5, 1003)) < 0.5, **c)


def test_nothing_allowed_and_values_that_are_no_numbers(env):
    vocab = 500
    logits = np.zeros((6, vocab))
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, :] = -np.inf
    logits[2, 7] = np.nan
    logits[3, 9] = np.inf
    logits[4] = -3.4e38  # the type's lowest values still count as allowed
    logits[5] = 1.0
    allowed = np.ones((6, vocab), bool)
    allowed[5] = False
    history = [[3], [3], [7], [9, 9], [1, 2], [0]]
    check(env, logits, True, history=history, repetition=[1.5] * 6, frequency=[0.5] * 6, allowed=allowed)


def test_ties_go_to_the_lowest_index(env):
    logits = np.zeros((4, 100000))
    logits[1, [99999, 50000, 12]] = 5
    logits[2, [70000, 70001]] = 5
    logits[3, 31] = 8.0
    check(env, logits, False, history=[[], [12], [], [31]], repetition=[2.0] * 4)
    check(env, logits, True)


def test_tokens_outside_of_the_vocabulary_and_repeats(env):
    logits = np.random.default_rng(2).standard_normal((2, 700))
    history = [[-1, 700, 5, 5, 5, 699, -2**31, 2**31 - 1, 0], [5] * 40000 + [6]]
    bias = [[(-4, 1.0), (0, 2.0), (5, 3.0), (5, 100.0), (699, -1.0), (700, 9.0)], []]
    check(env, logits, True, history=history, n_prompt=[4, 1], repetition=[1.2, 0.5], presence=[0.25, 0.0], frequency=[0.125, 0.001], bias=bias)


def test_same_as_argmax_without_rules(env):
    ctx, K = env
    logits = H.f32_to_bf16_np(np.random.default_rng(4).standard_normal((7, 5001)).astype(np.float32))
    dev, a, b = ctx.buf(logits), ctx.empty((7,), np.int32), ctx.empty((7,), np.int32)
    K.argmax(ctx, dev, 7, 5001, a)
    K.logits_adjust(ctx, dev, 7, 5001, K.logit_rules(), argmax=b)
    ctx.sync()
    assert np.array_equal(a.download(), b.download())


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_more_named_tokens_than_are_kept_at_a_time(env, f32, in_place):
    rng, c = case(31, 2, 90000, 60000, 4000)
    c["history"] = [rng.permutation(90000)[:70000], rng.integers(0, 9000, 50000)]  # ... in every slice, and in one
    c["n_prompt"] = [35000, 20000]
    check(env, f32=f32, in_place=in_place, allowed=rng.random((2, 90000)) < 0.5, **c)

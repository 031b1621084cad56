"""The 4-bit key/value cache against its statement in 64 bits: append (bit for bit), attention of single tokens and of runs of tokens.

Tolerance of the attention.  A score is a sum of at most 128 products in f32, times a constant: off by at most (128 + 4) 2^-24 S in all, S the
largest sum |q||k| scale.  A weight exp(score) is then off by that, relatively, twice (the reference point's score and its own), the exponential by
2^-22 and P, as a bf16 head and remainder, by 2^-17; weights and their sum enter the result.  The sums over n tokens in f32 add at most n 2^-24,
parts of a run and of blocks included.  So |error| <= (2 (264 2^-24 S + 2^-22 + 2^-17 + n 2^-24)) max|v|, and then the result is rounded to bf16:
2^-8 of it.
With many query tokens P may be one bf16 number: every weight is off by at most 2^-8 of itself (half a step) and their sum, taken before, is not, so
|error| grows by at most 2^-8 sum(w |v|) / sum(w) <= 2^-8 max|v|."""
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


def tolerance(ref, size, vmax, n, many=False):
    return (2.0 ** -8 * vmax if many else 0) + 2 * (264 * 2.0 ** -24 * size + 2.0 ** -22 + 2.0 ** -17 + n * 2.0 ** -24) * vmax + 2.0 ** -8 * np.abs(ref)


def as_bf16(x):
    return H.f32_to_bf16_np(np.asarray(x, np.float32))


# ---- append ------------------------------------------------------------------------------------------------------------
def rope_in_64(x, cos, sin):
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half], x[..., half:], cos[:, None], sin[:, None]
    return O.bf16(np.concatenate([O.bf16(a * c) + O.bf16(-b * s), O.bf16(b * c) + O.bf16(a * s)], -1))


def append_case(seed, T, hq, hkv, hd, page, pages):
    rng = np.random.default_rng(seed)
    qkv = O.bf16(rng.standard_normal((T, hq + 2 * hkv, hd)) * np.exp(0.4 * rng.standard_normal((1, hq + 2 * hkv, hd))))
    pos = rng.integers(0, 300, T).astype(np.int32)
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    angle = np.arange(300)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)
    return rng, qkv, pos, slots, O.bf16(np.cos(angle)), O.bf16(np.sin(angle))


def run_append(env, qkv, pos, slots, cos, sin, q_norm, k_norm, page, pages, hq, hkv, hd, values=True):
    ctx, K = env
    T = len(qkv)
    pool = np.full(K.kv_q4_pool_bytes(pages, hkv, hd, page), 0xA5, np.uint8)
    dev = ctx.buf(pool)
    q_out = ctx.empty((T, hq, hd), np.uint16)
    kv = [ctx.empty((T, hkv, hd), np.uint16) if values else None for _ in range(2)]
    K.rope_kv_append_q4(ctx, ctx.buf(as_bf16(qkv)), T, hq, hkv, hd, ctx.buf(pos), ctx.buf(slots), ctx.buf(as_bf16(cos)), ctx.buf(as_bf16(sin)),
                        None if q_norm is None else ctx.buf(as_bf16(q_norm)), None if k_norm is None else ctx.buf(as_bf16(k_norm)), 1e-6, page, dev, pages,
                        q_out, *kv)
    ctx.sync()
    return pool, dev.download(), q_out.download(), [b.download() if values else None for b in kv]


@pytest.mark.parametrize("T, hq, hkv, hd, page, seed", [(1, 4, 2, 128, 16, 0), (5, 8, 8, 64, 16, 1), (33, 6, 2, 128, 32, 2), (40, 7, 1, 64, 48, 3), (130, 3, 3, 128, 16, 4)])
def test_append_bit_for_bit(env, T, hq, hkv, hd, page, seed):
    pages = 2 * T // page + 2
    rng, qkv, pos, slots, cos, sin = append_case(seed, T, hq, hkv, hd, page, pages)
    if T > 4:
        slots[1], slots[3] = -1, pages * page + 5  # tokens that are not to be kept
        # groups that are special: equal values, zeros, ends that are as far from zero as one another, one sign only, one large value
        qkv[2, hq + hkv] = 0.75
        qkv[2, hq] = 0.0
        qkv[4, hq + hkv, :64] = np.linspace(-2, 2, 64)
        qkv[0, hq + hkv, :64] = 100 + np.arange(64) / 64
        qkv[0, hq, 7] = 5000.0
        qkv[1, hq, 0] = 5000.0
    qkv = O.bf16(qkv)  # what the call is given
    before, after, q, (k, v) = run_append(env, qkv, pos, slots, cos, sin, None, None, page, pages, hq, hkv, hd)
    turned = rope_in_64(qkv[:, :hq + hkv], cos[pos], sin[pos])
    assert np.array_equal(q, as_bf16(turned[:, :hq]))
    want = before.copy()
    for t in range(T):
        for h in range(hkv):
            for is_v, x, got in ((False, turned[t, hq + h], k), (True, qkv[t, hq + hkv + h], v)):
                codes, scale, bias = O.quantize(x)
                assert np.array_equal(got[t, h], as_bf16(O.values(codes, scale, bias)))
                if 0 <= slots[t] < pages * page:
                    O.put(want, page, hkv, hd, int(slots[t]), h, is_v, codes, scale, bias)
    assert np.array_equal(after, want)  # the neighbours' bytes too


@pytest.mark.parametrize("hd", [64, 128])
def test_append_with_norms(env, hd):
    """The norm is a sum in f32: values may round to the neighbouring bf16 number, and a code with them.  Everything within one step."""
    T, hq, hkv, page, pages = 50, 4, 2, 16, 8
    rng, qkv, pos, slots, cos, sin = append_case(9, T, hq, hkv, hd, page, pages)
    qn, kn = (O.bf16(1 + 0.2 * rng.standard_normal(hd)) for _ in range(2))
    _, _, q, (k, v) = run_append(env, qkv, pos, slots, cos, sin, qn, kn, page, pages, hq, hkv, hd)

    def normed(x, w):
        return O.bf16(x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w)

    # bf16 2^-8 of each of the three roundings' operands, which are at most sqrt 2 of the pair's size
    ref = rope_in_64(normed(qkv[:, :hq], qn), cos[pos], sin[pos])
    assert (np.abs(H.bf16_to_f32_np(q) - ref) <= 6 * 2.0 ** -8 * np.abs(normed(qkv[:, :hq], qn)).max()).all()
    ref = rope_in_64(normed(qkv[:, hq:hq + hkv], kn), cos[pos], sin[pos])
    codes, scale, bias = O.quantize(ref)
    step = np.repeat(np.abs(scale), 64, -1)
    diff = np.abs(H.bf16_to_f32_np(k) - O.values(codes, scale, bias))
    assert (diff <= 1.1 * step + 2.0 ** -6 * np.abs(ref).max()).all()
    assert (diff == 0).mean() > 0.99
    codes, scale, bias = O.quantize(qkv[:, hq + hkv:])
    assert np.array_equal(v, as_bf16(O.values(codes, scale, bias)))


def test_append_matches_the_16_bit_append(env):
    """Queries carry the same bits as those of the append into bf16 pages, norms included."""
    ctx, K = env
    T, hq, hkv, hd, page, pages = 37, 8, 2, 128, 16, 6
    rng, qkv, pos, slots, cos, sin = append_case(12, T, hq, hkv, hd, page, pages)
    qn, kn = (O.bf16(1 + 0.2 * rng.standard_normal(hd)) for _ in range(2))
    _, _, q, _ = run_append(env, qkv, pos, slots, cos, sin, qn, kn, page, pages, hq, hkv, hd, values=False)
    wide = [ctx.buf(np.zeros((pages, hkv, page, hd), np.uint16)) for _ in range(2)]
    q16 = ctx.empty((T, hq, hd), np.uint16)
    K.rope_kv_append(ctx, ctx.buf(as_bf16(qkv)), T, hq, hkv, hd, ctx.buf(pos), ctx.buf(slots), ctx.buf(as_bf16(cos)), ctx.buf(as_bf16(sin)),
                     ctx.buf(as_bf16(qn)), ctx.buf(as_bf16(kn)), 1e-6, page, wide[0], wide[1], q16)
    ctx.sync()
    assert np.array_equal(q, q16.download())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_poisons_the_group_of_a_bad_value_only(env, hd, bad):
    T, hq, hkv, page, pages = 3, 2, 1, 16, 1
    _, qkv, pos, slots, cos, sin = append_case(20, T, hq, hkv, hd, page, pages)
    qkv[1, hq + hkv, 5] = bad
    _, _, _, (k, v) = run_append(env, qkv, pos, slots, cos, sin, None, None, page, pages, hq, hkv, hd)
    v = H.bf16_to_f32_np(v)
    assert np.isnan(v[1, 0, :64]).all() and np.isfinite(v[1, 0, 64:]).all()
    assert np.isfinite(v[[0, 2]]).all() and np.isfinite(H.bf16_to_f32_np(k)).all()


def test_append_of_nothing(env):
    ctx, K = env
    K.rope_kv_append_q4(ctx, None, 0, 2, 1, 64, None, None, None, None, None, None, 1e-6, 16, ctx.buf(np.zeros(1152, np.uint8)), 1, None)
    ctx.sync()


# ---- attention ---------------------------------------------------------------------------------------------------------
class Cache:
    """Sequences of given lengths in a 4-bit pool, in pages of any order; bytes behind a sequence's end are NaN scales."""

    def __init__(self, env, seed, lengths, hkv, hd, page, spare=2, extra_blocks=0):
        ctx, K = env
        rng = np.random.default_rng(seed)
        blocks = [(n + page - 1) // page for n in lengths]
        self.pages, self.max_blocks = sum(blocks) + spare, max(max(blocks), 1) + extra_blocks
        order = rng.permutation(self.pages)
        self.tables = np.full((len(lengths), self.max_blocks), -7, np.int32)  # (entries behind a sequence's end are not looked at)
        pool = np.full((self.pages, hkv, page // 16, O.record_bytes(hd)), 0xFF, np.uint8)
        self.k, self.v = [], []
        at = 0
        for i, n in enumerate(lengths):
            self.tables[i, :blocks[i]] = order[at:at + blocks[i]]
            at += blocks[i]
            got = []
            for is_v in (False, True):
                rows = blocks[i] * page
                codes = np.clip(np.rint(7.5 + 3 * rng.standard_normal((hkv, rows, hd))), 0, 15)
                scale = O.bf16(0.3 * np.exp(0.3 * rng.standard_normal((hkv, rows, hd // 64))) * rng.choice([-1, 1], (hkv, rows, hd // 64)))
                bias = O.bf16(-scale * (7.5 + rng.standard_normal(scale.shape)))
                got.append(O.values(codes, scale, bias)[:, :n])
                scale[:, n:], bias[:, n:] = np.nan, np.nan
                self._write(pool, self.tables[i, :blocks[i]], page, hkv, hd, is_v, codes, scale, bias)
            self.k.append(got[0])
            self.v.append(got[1])
        self.pool = ctx.buf(pool)
        self.dev_tables = ctx.buf(self.tables)

    @staticmethod
    def _write(pool, pages, page, hkv, hd, is_v, codes, scale, bias):
        """O.put for whole pages (compared with it in test_cache_builder)."""
        n = len(pages)
        tiles = lambda x: x.reshape(hkv, n, page // 16, 16, x.shape[-1]).transpose(1, 0, 2, 3, 4)
        c = tiles(codes).astype(np.uint8)
        bytes_ = c[..., 0::2] | c[..., 1::2] << 4
        if is_v:  # token 8h + 2c + j, byte of block g, word d, byte b
            b = bytes_.reshape(n, hkv, page // 16, 2, 4, 2, 8, hd // 32, 2).transpose(0, 1, 2, 3, 6, 4, 7, 5, 8)
            pool[pages, ..., 8 * hd:16 * hd] = b.reshape(n, hkv, page // 16, 8 * hd)
        else:
            pool[pages, ..., :8 * hd] = bytes_.reshape(n, hkv, page // 16, 8 * hd)
        words = (O.bits(tiles(scale)) | O.bits(tiles(bias)) << 16).transpose(0, 1, 2, 4, 3)
        groups = hd // 64
        at = 16 * hd + (64 * groups if is_v else 0)
        pool[pages, ..., at:at + 64 * groups] = np.ascontiguousarray(words).view(np.uint8).reshape(n, hkv, page // 16, 64 * groups)


def test_cache_builder():
    for hd, page in ((64, 32), (128, 16)):
        rng = np.random.default_rng(1)
        codes, scale, bias = rng.integers(0, 16, (2, 2 * page, hd)), O.bf16(rng.standard_normal((2, 2 * page, hd // 64))), O.bf16(rng.standard_normal((2, 2 * page, hd // 64)))
        a, b = (np.zeros((3, 2, page // 16, O.record_bytes(hd)), np.uint8) for _ in range(2))
        for is_v in (False, True):
            Cache._write(a, np.array([2, 0]), page, 2, hd, is_v, codes, scale, bias)
            for t in range(2 * page):
                for h in range(2):
                    O.put(b.reshape(-1), page, 2, hd, [2, 0][t // page] * page + t % page, h, is_v, codes[h, t], scale[h, t], bias[h, t])
        assert np.array_equal(a, b)


def queries(seed, rows, hq, hd):
    return O.bf16(np.random.default_rng(seed + 1000).standard_normal((rows, hq, hd)))


def check_rows(got, q, cache, i, scale, many=False):
    ref, size = O.attention(q, cache.k[i], cache.v[i], scale)
    n = cache.k[i].shape[1]
    got = H.bf16_to_f32_np(got)
    tol = tolerance(ref, size, np.abs(cache.v[i]).max(), n, many)
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"sequence {i} ({n} tokens): {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - ref) - tol)}, nan {np.isnan(got).any()}"


def run_decode(env, cache, lengths, q, hq, hkv, hd, page, scale):
    ctx, K = env
    out = ctx.buf(np.full(q.shape, 0x7FC1, np.uint16))
    K.paged_attn_decode_q4(ctx, ctx.buf(as_bf16(q)), cache.pool, cache.pages, cache.dev_tables, ctx.buf(np.asarray(lengths, np.int32)), len(lengths), hq, hkv, hd,
                           page, scale, out, cache.max_blocks)
    ctx.sync()
    return out.download()


DECODE = [
    # lengths, hq, hkv, hd, page
    ([1], 1, 1, 128, 16),
    ([1], 8, 1, 64, 16),
    ([15, 16, 17, 31, 32, 33], 8, 2, 128, 16),
    ([0, 5, 0, 0, 300, 0], 4, 2, 64, 32),
    ([0, 0], 4, 1, 128, 16),
    ([777], 32, 8, 128, 16),
    ([5000, 3, 1200], 14, 2, 128, 48),
    ([600, 601], 3, 3, 64, 64),
    ([250, 90], 10, 2, 128, 16),
    ([130, 260, 2], 24, 4, 64, 16),
    ([511, 40], 36, 4, 128, 32),   # 9 heads a group: two blocks of columns
    ([70, 1000], 32, 2, 128, 16),  # 16
    ([64, 3], 40, 2, 64, 16),      # 20: three
    (list(range(1, 90)), 8, 2, 128, 16),
    ([(5 * i) % 23 for i in range(300)], 8, 2, 128, 16),       # each unit a warp's
    ([(37 * i) % 500 for i in range(300)], 4, 1, 64, 16),
    ([300 + i % 60 for i in range(60)], 16, 8, 128, 16),       # ... two warps'
    ([9000, 20000], 2, 1, 64, 16),
]


@pytest.mark.parametrize("lengths, hq, hkv, hd, page", DECODE)
def test_decode(env, lengths, hq, hkv, hd, page):
    cache = Cache(env, len(lengths) + hq, lengths, hkv, hd, page, extra_blocks=1)
    q = queries(hq, len(lengths), hq, hd)
    got = run_decode(env, cache, lengths, q, hq, hkv, hd, page, hd ** -0.5)
    for i, n in enumerate(lengths):
        if n == 0:
            assert (got[i] == 0).all()
        else:
            check_rows(got[i:i + 1], q[i:i + 1], cache, i, hd ** -0.5)
    assert np.array_equal(got, run_decode(env, cache, lengths, q, hq, hkv, hd, page, hd ** -0.5))


def test_decode_of_more_sequences_than_index_entries(env):
    lengths = [(7 * i) % 41 for i in range(2500)]
    cache = Cache(env, 5, lengths, 1, 64, 16)
    q = queries(5, len(lengths), 2, 64)
    got = run_decode(env, cache, lengths, q, 2, 1, 64, 16, 0.125)
    for i in range(0, len(lengths), 13):
        if lengths[i]:
            check_rows(got[i:i + 1], q[i:i + 1], cache, i, 0.125)
    assert (got[[i for i, n in enumerate(lengths) if n == 0]] == 0).all()


def test_decode_with_scores_far_apart(env):
    """Scores that rise by hundreds along the sequence, and that all lie far below zero: the running reference follows."""
    ctx, K = env
    hd, n = 128, 700
    for sign in (1.0, -1.0):
        pool = np.zeros((44, 1, 1, 2304), np.uint8)
        k, v = np.zeros((1, n, hd)), np.zeros((1, n, hd))
        for t in range(n):
            for is_v, x in ((False, np.full(hd, sign * t / 64)), (True, np.random.default_rng(t).standard_normal(hd))):
                codes, scale, bias = O.quantize(O.bf16(x))
                O.put(pool.reshape(-1), 16, 1, hd, t, 0, is_v, codes, scale, bias)
                (v if is_v else k)[0, t] = O.values(codes, scale, bias)
        cache = Cache.__new__(Cache)
        cache.pool, cache.pages, cache.max_blocks, cache.k, cache.v = ctx.buf(pool), 44, 44, [k], [v]
        cache.dev_tables = ctx.buf(np.arange(44, dtype=np.int32)[None])
        q = O.bf16(np.full((1, 1, hd), 3.0))
        check_rows(run_decode(env, cache, [n], q, 1, 1, hd, 16, 1.0), q, cache, 0, 1.0)


def test_decode_of_contexts_longer_than_their_tables(env):
    cache = Cache(env, 6, [64], 2, 128, 16)
    q = queries(6, 1, 4, 128)
    assert np.array_equal(run_decode(env, cache, [64], q, 4, 2, 128, 16, 0.1), run_decode(env, cache, [90], q, 4, 2, 128, 16, 0.1))
    assert (run_decode(env, cache, [-3], q, 4, 2, 128, 16, 0.1) == 0).all()


@pytest.mark.parametrize("bad", [-1, 1 << 30, "pages"])
def test_decode_leaves_pages_outside_of_the_pool_out(env, bad):
    ctx, _ = env
    cache = Cache(env, 7, [60, 40, 16], 2, 128, 16)
    tables = cache.tables.copy()
    tables[0, 1] = tables[2, 0] = cache.pages if bad == "pages" else bad
    cache.dev_tables = ctx.buf(tables)
    q = queries(7, 3, 4, 128)
    got = run_decode(env, cache, [60, 40, 16], q, 4, 2, 128, 16, 0.1)
    cache.k[0], cache.v[0] = (np.delete(x, np.s_[16:32], 1) for x in (cache.k[0], cache.v[0]))
    for i in range(2):
        check_rows(got[i:i + 1], q[i:i + 1], cache, i, 0.1)
    assert (got[2] == 0).all()


def test_decode_carries_a_nan_of_the_cache(env):
    ctx, _ = env
    cache = Cache(env, 8, [100, 100], 1, 128, 16)
    pool = cache.pool.download()
    page = cache.tables[1, 2]
    pool[page, 0, 0, 2048 + 128 + 4:2048 + 128 + 8] = 0xFF  # V's scale of token 33 of sequence 1, first group
    cache.pool = ctx.buf(pool)
    got = H.bf16_to_f32_np(run_decode(env, cache, [100, 100], queries(8, 2, 2, 128), 2, 1, 128, 16, 0.1))
    assert np.isfinite(got[0]).all() and np.isnan(got[1, :, :64]).all() and np.isfinite(got[1, :, 64:]).all()


PREFILL = [
    # (new, cached) of every sequence, hq, hkv, hd, page
    ([(1, 0)], 4, 2, 128, 16),
    ([(3, 0)], 4, 2, 64, 16),
    ([(2, 30), (5, 1), (8, 100), (1, 17)], 8, 2, 128, 16),
    ([(6, 1500)], 32, 8, 128, 16),
    ([(7, 90), (4, 0)], 6, 2, 128, 32),
    ([(1, 600), (40, 3)], 12, 1, 64, 48),
    ([(200, 0)], 8, 2, 128, 16),
    ([(150, 70), (0, 9), (3, 40), (129, 0)], 8, 2, 128, 16),
    ([(70, 5), (64, 64)], 10, 2, 64, 32),
    ([(33, 3000)], 16, 2, 128, 64),
    ([(300, 500)], 6, 6, 128, 48),
    ([(65, 0)], 5, 1, 64, 16),
]


@pytest.mark.parametrize("seqs, hq, hkv, hd, page", PREFILL)
def test_prefill(env, seqs, hq, hkv, hd, page):
    ctx, K = env
    lengths = [a + b for a, b in seqs]
    cache = Cache(env, hq + len(seqs), lengths, hkv, hd, page)
    cu = np.concatenate([[0], np.cumsum([a for a, _ in seqs])]).astype(np.int32)
    q = queries(hq, int(cu[-1]), hq, hd)
    out = ctx.buf(np.full((cu[-1] + 2, hq, hd), 0x7FC1, np.uint16))
    K.paged_attn_prefill_q4(ctx, ctx.buf(as_bf16(q)), cache.pool, cache.pages, cache.dev_tables, cache.max_blocks, cu, lengths, hq, hkv, hd, page, hd ** -0.5, out)
    ctx.sync()
    got = out.download()
    assert (got[cu[-1]:] == 0x7FC1).all()  # rows behind the last sequence
    for i, (n, _) in enumerate(seqs):
        if n:
            check_rows(got[cu[i]:cu[i + 1]], q[cu[i]:cu[i + 1]], cache, i, hd ** -0.5, many=n * hq // hkv > 32)


# Long enough that the tensor cores' kernel is the cheaper one for some sequence, or all: keys split over blocks or not, rows of a block that
# no query fills, groups that do not divide a block of rows, and single tokens next to prompts.
@pytest.mark.parametrize("seqs, hq, hkv, hd, page", [
    ([(200, 300), (129, 700), (1, 40), (0, 9), (64, 64)], 32, 8, 128, 16),
    ([(512, 1000), (1, 9000), (1, 9000), (2, 8999)], 32, 8, 128, 16),  # both kernels
    ([(100, 6000)], 8, 1, 128, 16),   # 12 splits
    ([(300, 5001)], 4, 2, 64, 64),    # splits, the last of them shorter
    ([(300, 2000)], 6, 2, 128, 48),
    ([(130, 900)], 40, 8, 64, 32),
    ([(9, 2000)], 128, 1, 128, 16),   # one query a block of rows
    ([(5, 50)], 130, 1, 128, 16),     # a group that no block of rows holds
    ([(700, 500)], 8, 8, 128, 16),
    ([(1000, 0)], 16, 4, 128, 16),
    ([(1025, 0), (63, 1), (257, 0)], 14, 2, 64, 16),
])
def test_prefill_of_many(env, seqs, hq, hkv, hd, page):
    ctx, K = env
    lengths = [a + b for a, b in seqs]
    cache = Cache(env, hq + len(seqs), lengths, hkv, hd, page)
    cu = np.concatenate([[0], np.cumsum([a for a, _ in seqs])]).astype(np.int32)
    q = queries(hq, int(cu[-1]), hq, hd)
    out = ctx.buf(np.full((cu[-1] + 2, hq, hd), 0x7FC1, np.uint16))
    K.paged_attn_prefill_q4(ctx, ctx.buf(as_bf16(q)), cache.pool, cache.pages, cache.dev_tables, cache.max_blocks, cu, lengths, hq, hkv, hd, page, hd ** -0.5, out)
    ctx.sync()
    got = out.download()
    assert (got[cu[-1]:] == 0x7FC1).all()
    for i, (n, _) in enumerate(seqs):
        if n:
            check_rows(got[cu[i]:cu[i + 1]], q[cu[i]:cu[i + 1]], cache, i, hd ** -0.5, many=True)


@pytest.mark.parametrize("new", [2, 300])
def test_prefill_reads_nothing_outside_the_pool(env, new):
    """Page numbers outside the pool in one sequence's row: the other sequences' rows are as they were, and finite."""
    ctx, K = env
    hq, hkv, hd, page, seqs = 32, 8, 128, 16, [(new, 500), (new, 400), (new, 300)]
    lengths = [a + b for a, b in seqs]
    cache = Cache(env, 3, lengths, hkv, hd, page)
    cu = np.arange(4) * new
    q = queries(3, 3 * new, hq, hd)
    got = []
    for bad in (False, True):
        tables = cache.tables.copy()
        if bad:
            tables[1, :6] = [-1, cache.pages, 2 ** 31 - 1, -2 ** 31, 10 ** 6, -5]
        out = ctx.empty(q.shape, np.uint16)
        K.paged_attn_prefill_q4(ctx, ctx.buf(as_bf16(q)), cache.pool, cache.pages, ctx.buf(tables), cache.max_blocks, cu, lengths, hq, hkv, hd, page, hd ** -0.5, out)
        ctx.sync()
        got.append(out.download())
    for i in (0, 2):
        assert np.array_equal(got[0][cu[i]:cu[i + 1]], got[1][cu[i]:cu[i + 1]])
        check_rows(got[1][cu[i]:cu[i + 1]], q[cu[i]:cu[i + 1]], cache, i, hd ** -0.5, many=True)
    assert np.isfinite(H.bf16_to_f32_np(got[1])).all()


def test_one_query_is_decode(env):
    ctx, K = env
    lengths = [40, 333, 16, 1]
    cache = Cache(env, 31, lengths, 2, 128, 16)
    q = queries(31, 4, 8, 128)
    out = ctx.empty(q.shape, np.uint16)
    K.paged_attn_prefill_q4(ctx, ctx.buf(as_bf16(q)), cache.pool, cache.pages, cache.dev_tables, cache.max_blocks, [0, 1, 2, 3, 4], lengths, 8, 2, 128, 16, 0.1, out)
    ctx.sync()
    assert np.array_equal(out.download(), run_decode(env, cache, lengths, q, 8, 2, 128, 16, 0.1))


# ---- a sequence's life, as a model's layer goes through it --------------------------------------------------------------
@pytest.mark.parametrize("hd, hq, hkv", [(128, 8, 2), (64, 6, 3)])
def test_prompt_then_tokens_then_choices(env, hd, hq, hkv):
    ctx, K = env
    rng = np.random.default_rng(77)
    page, pages, prompts, vocab = 16, 40, [75, 9], 997
    pool = ctx.buf(rng.integers(0, 256, K.kv_q4_pool_bytes(pages, hkv, hd, page)).astype(np.uint8))  # whatever was there before
    order = rng.permutation(pages)
    tables = order[:16].reshape(2, 8).astype(np.int32)
    dev_tables = ctx.buf(tables)
    angle = np.arange(200)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)
    cos, sin = O.bf16(np.cos(angle)), O.bf16(np.sin(angle))
    dcos, dsin = ctx.buf(as_bf16(cos)), ctx.buf(as_bf16(sin))
    have = [(np.zeros((hkv, 0, hd)), np.zeros((hkv, 0, hd))) for _ in prompts]
    lengths = [0, 0]
    head = rng.standard_normal((vocab, hq * hd)) / 8
    history = [list(rng.integers(0, vocab, n)) for n in prompts]
    for step in range(6):
        new = prompts if step == 0 else [1, 1]
        T = sum(new)
        qkv = O.bf16(rng.standard_normal((T, hq + 2 * hkv, hd)))
        seq = np.repeat([0, 1], new)
        pos = np.concatenate([np.arange(l, l + n) for l, n in zip(lengths, new)]).astype(np.int32)
        slots = (tables[seq, pos // page] * page + pos % page).astype(np.int32)
        q_dev = ctx.empty((T, hq, hd), np.uint16)
        K.rope_kv_append_q4(ctx, ctx.buf(as_bf16(qkv)), T, hq, hkv, hd, ctx.buf(pos), ctx.buf(slots), dcos, dsin, None, None, 1e-6, page, pool, pages, q_dev)
        lengths = [l + n for l, n in zip(lengths, new)]
        out = ctx.empty((T, hq, hd), np.uint16)
        cu = np.concatenate([[0], np.cumsum(new)])
        if step == 0:
            K.paged_attn_prefill_q4(ctx, q_dev, pool, pages, dev_tables, 8, cu, lengths, hq, hkv, hd, page, hd ** -0.5, out)
        else:
            K.paged_attn_decode_q4(ctx, q_dev, pool, pages, dev_tables, ctx.buf(np.array(lengths, np.int32)), 2, hq, hkv, hd, page, hd ** -0.5, out, 8)
        ctx.sync()
        turned = rope_in_64(qkv[:, :hq + hkv], cos[pos], sin[pos])
        rows = []
        for i in range(2):
            r = slice(cu[i], cu[i + 1])
            k, v = (O.values(*O.quantize(x[r])).transpose(1, 0, 2) for x in (turned[:, hq:], qkv[:, hq + hkv:]))
            have[i] = tuple(np.concatenate([a, b], 1) for a, b in zip(have[i], (k, v)))
            cache = Cache.__new__(Cache)
            cache.k, cache.v = [have[i][0]], [have[i][1]]
            check_rows(out.download()[r], turned[r, :hq], cache, 0, hd ** -0.5, many=new[i] * hq // hkv > 32)
            rows.append(H.bf16_to_f32_np(out.download()[cu[i + 1] - 1]).astype(np.float64))
        # the step's logits under rules, and the tokens that come of them
        logits = O.bf16(np.stack([head @ r.reshape(-1) for r in rows]))
        allowed = rng.random((2, vocab)) < 0.5
        packed = np.zeros((2, (vocab + 31) // 32 * 32), bool)
        packed[:, :vocab] = allowed
        mask = np.packbits(packed, axis=1, bitorder="little").view(np.uint32)
        offs = np.concatenate([[0], np.cumsum([len(h) for h in history])]).astype(np.int32)
        tokens = ctx.empty((2,), np.int32)
        rules = K.logit_rules(history=ctx.buf(np.concatenate(history).astype(np.int32)), history_off=ctx.buf(offs), n_prompt=ctx.buf(np.array(prompts, np.int32)),
                              repetition=ctx.buf(np.array([1.3, 1.1], np.float32)), frequency=ctx.buf(np.array([0.1, 0.2], np.float32)),
                              mask=ctx.buf(mask), mask_words=mask.shape[1])
        K.logits_adjust(ctx, ctx.buf(as_bf16(logits)), 2, vocab, rules, argmax=tokens)
        ctx.sync()
        for i, t in enumerate(tokens.download()):
            _, want = O.adjust(logits[i], history[i], prompts[i], [1.3, 1.1][i], 0.0, [0.1, 0.2][i], allowed=allowed[i])
            assert t == want
            history[i].append(int(t))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("new, cached", [(3, 37), (60, 37), (400, 700), (900, 700)])
def test_prefill_keeps_a_bad_token_from_earlier_queries(env, hd, what, new, cached):
    """A token whose key or value is NaN: queries before it are as if it were not there, those that see it are NaN."""
    ctx, K = env
    hq, hkv, page = 4, 2, 16
    n = cached + new
    cache = Cache(env, 91, [n], hkv, hd, page)
    q = queries(91, new, hq, hd)
    bad = cached + new // 2
    pool = cache.pool.download()
    at = 16 * hd + (64 * (hd // 64) if what == "value" else 0) + (bad % 16) * 4
    pool[cache.tables[0, bad // page], 0, 0, at:at + 4] = 0xFF  # of kv head 0, first group
    out = ctx.empty(q.shape, np.uint16)
    K.paged_attn_prefill_q4(ctx, ctx.buf(as_bf16(q)), ctx.buf(pool), cache.pages, cache.dev_tables, cache.max_blocks, [0, new], [n], hq, hkv, hd, page, 0.1, out)
    ctx.sync()
    got = out.download()
    before = new // 2
    cache.k[0], cache.v[0] = cache.k[0][:, :cached + before], cache.v[0][:, :cached + before]
    check_rows(got[:before], q[:before], cache, 0, 0.1, many=new * hq // hkv > 32)
    got = H.bf16_to_f32_np(got[before:])
    assert np.isnan(got[:, :2, :64]).all() and np.isfinite(got[:, 2:]).all()


# ---- calls next to one another, and caches past 32 bits -------------------------------------------------------------------
def test_pool_past_four_gigabytes(env):
    """Pages whose bytes lie beyond 2^32: what is appended there is what attention reads, by single tokens, few and many."""
    ctx, K = env
    hq, hkv, hd, page, n = 8, 1, 128, 16, 700
    pages = (1 << 21) + 64
    pool = ctx.empty((K.kv_q4_pool_bytes(pages, hkv, hd, page),), np.uint8)
    assert pool.nbytes > 1 << 32
    tables = (pages - 1 - np.arange(44, dtype=np.int32))[None]
    pos = np.arange(n, dtype=np.int32)
    slots = (tables[0, pos // page] * page + pos % page).astype(np.int32)
    rng = np.random.default_rng(8)
    qkv = O.bf16(rng.standard_normal((n, hq + 2 * hkv, hd)))
    cos, sin = O.bf16(np.ones((n, hd // 2))), O.bf16(np.zeros((n, hd // 2)))
    q, k, v = ctx.empty((n, hq, hd), np.uint16), ctx.empty((n, hkv, hd), np.uint16), ctx.empty((n, hkv, hd), np.uint16)
    K.rope_kv_append_q4(ctx, ctx.buf(as_bf16(qkv)), n, hq, hkv, hd, ctx.buf(pos), ctx.buf(slots), ctx.buf(as_bf16(cos)), ctx.buf(as_bf16(sin)), None, None, 1e-6,
                        page, pool, pages, q, k, v)
    ctx.sync()
    cache = Cache.__new__(Cache)
    cache.pool, cache.pages, cache.max_blocks, cache.dev_tables = pool, pages, 44, ctx.buf(tables)
    cache.k, cache.v = ([H.bf16_to_f32_np(x.download()).astype(np.float64).transpose(1, 0, 2)] for x in (k, v))
    rows = qkv[:, :hq]
    check_rows(run_decode(env, cache, [n], rows[-1:], hq, hkv, hd, page, 0.1), rows[-1:], cache, 0, 0.1)
    for new in (3, n):
        out = ctx.empty((new, hq, hd), np.uint16)
        K.paged_attn_prefill_q4(ctx, ctx.buf(as_bf16(rows[-new:])), pool, pages, cache.dev_tables, 44, [0, new], [n], hq, hkv, hd, page, 0.1, out)
        ctx.sync()
        check_rows(out.download(), rows[-new:], cache, 0, 0.1, many=True)
        out.free()
    pool.free()


def attention_calls(env, ctx):
    """Calls of every kind and size on `ctx`, and where their results are."""
    _, K = env
    calls = []
    for seed, lengths, new in ((1, [700], None), (2, [3000, 5, 900, 64], None), (3, [16] * 20, None), (4, [900, 33], [200, 33]), (5, [2500], [300]),
                               (6, [400, 40, 1500], [2, 1, 4])):
        cache = Cache((ctx, K), seed, lengths, 2, 128, 16)
        cu = None if new is None else np.concatenate([[0], np.cumsum(new)])
        q = ctx.buf(as_bf16(queries(seed, len(lengths) if new is None else int(cu[-1]), 8, 128)))
        out, n = ctx.empty(q.shape, np.uint16), ctx.buf(np.asarray(lengths, np.int32))
        if new is None:
            calls.append((out, lambda q=q, c=cache, n=n, l=lengths, o=out: K.paged_attn_decode_q4(ctx, q, c.pool, c.pages, c.dev_tables, n, len(l), 8, 2, 128, 16,
                                                                                                  0.1, o, c.max_blocks)))
        else:
            calls.append((out, lambda q=q, c=cache, u=cu, l=lengths, o=out: K.paged_attn_prefill_q4(ctx, q, c.pool, c.pages, c.dev_tables, c.max_blocks, u, l, 8, 2,
                                                                                                    128, 16, 0.1, o)))
    return calls


def test_calls_one_after_the_other_and_two_contexts_at_once(env):
    from mlx_llm_b200 import _lib

    ctx, _ = env
    other = _lib.Context(0)
    try:
        here, there = attention_calls(env, ctx), attention_calls(env, other)
        alone = []
        for out, call in here:
            call()
            ctx.sync()
            alone.append(out.download())
        for _ in range(5):
            for out, _ in here + there:
                out.upload(np.full(out.shape, 0x7FC1, np.uint16))
            for i in np.random.default_rng(3).permutation(len(here) * 4) % len(here):  # nothing waits in between
                here[i][1]()
                there[len(here) - 1 - i][1]()
            ctx.sync()
            other.sync()
            for i, want in enumerate(alone):
                assert np.array_equal(here[i][0].download(), want) and np.array_equal(there[i][0].download(), want)
    finally:
        other.close()

"""Plain numpy statement of the 4-bit key/value cache and of rules on logits, in 64 bits (test infrastructure)."""
import numpy as np


def bf16(x):
    """Nearest bf16 numbers, ties to even, as float64; x float64 or anything that float32 holds exactly."""
    x = np.asarray(x, np.float64)
    u = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32).astype(np.float64)
    return np.where(np.isfinite(x), r, x)


def bits(x):
    """The 16 bits of numbers that bf16 holds."""
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint32)


def away(x):
    return np.trunc(x + np.copysign(0.5, x))


def quantize(x):
    """x [..., 64 g] -> codes, scales [..., g], biases [..., g]."""
    x = np.asarray(x, np.float64)
    x = x.reshape(x.shape[:-1] + (x.shape[-1] // 64, 64))
    lo, hi = x.min(-1), x.max(-1)
    edge, span = np.where(np.abs(lo) > np.abs(hi), lo, hi), hi - lo
    with np.errstate(all="ignore"):
        n = away(15 * np.abs(edge) / span)
        scale = np.where(span == 0, 0.0, bf16(-edge / n))
        scale = np.where((span == 0) | (15 * np.abs(edge) < 2.0 ** 128) & (np.abs(scale) < 2.0 ** 59), scale, np.nan)
        codes = np.clip(away((x - edge[..., None]) / scale[..., None]), 0, 15)
    codes = np.where((scale[..., None] == 0) | np.isnan(scale[..., None]), 0, codes)
    return codes.reshape(codes.shape[:-2] + (codes.shape[-2] * 64,)), scale, edge


def values(codes, scale, bias):
    c = codes.reshape(codes.shape[:-1] + (codes.shape[-1] // 64, 64))
    return bf16(c * scale[..., None] + bias[..., None]).reshape(codes.shape)


def record_bytes(hd):
    return 16 * hd + 128 * (hd // 64)


def put(pool, page_size, hkv, hd, slot, kvh, is_v, codes, scale, bias):
    """Writes one token's head into a pool (uint8 array) the way the header of the C ABI describes the record."""
    page, off = divmod(slot, page_size)
    t = off % 16
    base = ((page * hkv + kvh) * (page_size // 16) + off // 16) * record_bytes(hd)
    codes = codes.astype(np.uint8)
    if not is_v:
        pool[base + t * hd // 2: base + (t + 1) * hd // 2] = codes[0::2] | codes[1::2] << 4
    else:
        for d in range(0, hd, 4):  # four dims are a half word
            g, r = divmod(d, hd // 8)
            word = ((t // 8 * 8 + g) * 4 + t % 8 // 2) * (hd // 32) + r // 4
            at = base + 8 * hd + word * 4 + (t % 2) * 2
            pool[at] = codes[d] | codes[d + 1] << 4
            pool[at + 1] = codes[d + 2] | codes[d + 3] << 4
    for g in range(hd // 64):
        at = base + 16 * hd + ((hd // 64 if is_v else 0) + g) * 64 + t * 4
        pool[at:at + 4] = np.array([bits(scale[g]) | bits(bias[g]) << 16], np.uint32).view(np.uint8)


def attention(q, k, v, scale):
    """q [n, hq, hd], k and v [hkv, ctx, hd]; query r of n sees keys 0 .. ctx - n + r.  Also the largest sum |q||k| scale."""
    n, hq, hd = q.shape
    hkv, ctx, _ = k.shape
    out = np.zeros((n, hq, hd))
    size = 0.0
    for h in range(hq):
        kk, vv = k[h // (hq // hkv)], v[h // (hq // hkv)]
        s = q[:, h] @ kk.T * scale
        size = max(size, float((np.abs(q[:, h]) @ np.abs(kk).T * abs(scale)).max()) if ctx else 0.0)
        s[np.arange(ctx)[None] > ctx - n + np.arange(n)[:, None]] = -np.inf
        w = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = w @ vv / w.sum(-1, keepdims=True)
    return out, size


def adjust(row, history=(), n_prompt=0, repetition=1.0, presence=0.0, frequency=0.0, bias=(), allowed=None):
    """One row of logits under the rules, in f32 steps, and the greedy choice (-1: none)."""
    f = np.float32
    x = np.asarray(row, np.float32).copy()
    vocab = len(x)
    history = np.asarray(history, np.int64)
    seen = np.unique(history[(history >= 0) & (history < vocab)])
    with np.errstate(all="ignore"):
        x[seen] = np.where(x[seen] > 0, x[seen] / f(repetition), x[seen] * f(repetition))
        answer = history[n_prompt:]
        ids, n = np.unique(answer[(answer >= 0) & (answer < vocab)], return_counts=True)
        x[ids] = (x[ids] - n.astype(np.float32) * f(frequency)) - f(presence)
        done = set()
        for i, b in bias:
            if 0 <= i < vocab and i not in done:
                x[i] += f(b)
            done.add(i)
    if allowed is not None:
        x[~allowed] = -np.inf
    best = np.where(np.isnan(x), -np.inf, x)
    return x, int(best.argmax()) if best.max() > -np.inf else -1

"""The operators of serving from a 4-bit key/value cache, and of choosing tokens under rules, as cases that can be timed and compared.

append   rotation of a step's queries and keys and quantization of its keys and values into the pages of a 4-bit cache
decode   attention of one query token per sequence over such a cache
prefill  attention of prompts, portions of prompts and drafts to be verified (several query tokens per sequence) over such a cache
logits   penalties for repeated tokens, biases and grammar masks on a step's logits, with the greedy choice

The cache.  Sixteen tokens of one kv head are a record of bytes; the pool is [pages][kv heads][page size / 16][record].
  keys     [16 tokens][dim / 2] bytes: a token's dims along the row, the lower of two in the low nibble
  values   u32 [2][8][4][dim / 32]: word (h, g, c, d) has tokens 8h + 2c and 8h + 2c + 1 in its halves, and in each half the dims
           g dim / 8 + 4 d ... + 3 from the lowest nibble on
  keys' scales and biases, then the values': u32 [dim / 64][16 tokens], the bf16 scale in the low half, the bf16 bias in the high one
A code stands for bf16(code scale + bias), with a scale and a bias for each 64 dims of a token."""
import functools
import math

import numpy as np
import torch

own = False
GROUP = 64


def listed():
    return [
        # one user: the latency of a token
        _append("append_token", hq=32, hkv=8, dim=128, tokens=1),
        # a loaded server's iteration: everybody's next token and a 512-token portion of a prompt; narrow heads
        _append("append_serve_64", hq=32, hkv=8, dim=64, tokens=608),
        # prompts taken whole, of a model that normalises queries and keys
        _append("append_prompts_norm", hq=64, hkv=8, dim=128, tokens=6151, norm=True),
        # one user, a short conversation
        _decode("decode_1", hq=32, hkv=8, dim=128, seqs=1, lo=700, hi=700),
        # the library's ordinary batch: contexts of very different lengths
        _decode("decode_64", hq=32, hkv=8, dim=128, seqs=64, lo=128, hi=4096),
        # what the 4 bits are for: many long conversations at once
        _decode("decode_32_long", hq=32, hkv=8, dim=128, seqs=32, lo=8000, hi=16000, page=32),
        # drafts that are verified: a few query tokens per sequence
        _prefill("verify_8", hq=32, hkv=8, dim=128, seqs=8, new=6, cached=1500),
        # prompts that arrive together, of a size that divides nothing
        _prefill("prompts_3", hq=32, hkv=8, dim=128, seqs=3, new=1049, cached=0),
        # a portion far inside a long document, for the large model
        _prefill("document", hq=64, hkv=8, dim=128, seqs=1, new=512, cached=11800),
        # one user whose answer has to follow a grammar; the logits go on to a sampler
        _logits("logits_1", rows=1, vocab=128256, history=600, bias=12, masked=1.0, out=True),
        # a server's greedy step: the tokens are all that is wanted
        _logits("logits_96_greedy", rows=96, vocab=128256, history=1500, bias=30, masked=0.3, out=False),
        # the largest batch and vocabulary, logits in 32 bits
        _logits("logits_256_f32", rows=256, vocab=151936, history=1000, bias=300, masked=0.5, out=True, f32=True),
    ]


def _append(name, hq, hkv, dim, tokens, norm=False, page=16):
    return dict(name=name, kind="append", hq=hq, hkv=hkv, dim=dim, page=page, tokens=tokens, norm=norm)


def _decode(name, hq, hkv, dim, seqs, lo, hi, page=16):
    return dict(name=name, kind="decode", hq=hq, hkv=hkv, dim=dim, page=page, seqs=seqs, lo=lo, hi=hi)


def _prefill(name, hq, hkv, dim, seqs, new, cached, page=16):
    return dict(name=name, kind="prefill", hq=hq, hkv=hkv, dim=dim, page=page, seqs=seqs, new=new, cached=cached)


def _logits(name, rows, vocab, history, bias, masked, out, f32=False):
    return dict(name=name, kind="logits", rows=rows, vocab=vocab, history=history, bias=bias, masked=masked, out=out, f32=f32)


def _between(rng, lo, hi):
    """A whole number whose logarithm is spread evenly."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "logits"])
    if kind == "logits":
        rows, vocab = _between(rng, 1, 256), _between(rng, 1000, 151936)
        case = _logits("", rows, vocab, rng.choice([0, _between(rng, 1, 3000)]), rng.choice([0, _between(rng, 1, 300)]),
                       rng.choice([0.0, round(rng.random(), 2), 1.0]), rng.random() < 0.6, rng.random() < 0.4)
        del case["name"]
        return case
    dim, page, hkv = rng.choice([64, 128, 128]), rng.choice([16, 16, 32, 64]), rng.choice([1, 2, 4, 5, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    if kind == "append":
        case = _append("", hq, hkv, dim, _between(rng, 1, min(6151, 6151 * 80 // (hq + 2 * hkv))), rng.random() < 0.5, page)
    elif kind == "decode":
        seqs = _between(rng, 1, 256)
        hi = _between(rng, 1, min(16000, 12000 * 32 * 8 * 4 // (seqs * max(hq, hkv * 4))))
        case = _decode("", hq, hkv, dim, seqs, rng.choice([hi, _between(rng, 1, hi)]), hi, page)
    else:
        seqs = _between(rng, 1, 8)
        new = _between(rng, 1, 1600 // seqs)
        most = 512 * 12000 * 64 // (seqs * new * hq) - new
        case = _prefill("", hq, hkv, dim, seqs, new, rng.choice([0, _between(rng, 1, max(1, min(12000, most, 24000 // seqs)))]), page)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    return {"append": _prepare_append, "decode": _prepare_decode, "prefill": _prepare_prefill, "logits": _prepare_logits}[case["kind"]](case, gen, rng)


def _record(dim):
    return 16 * dim + 128 * (dim // GROUP)


def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(values, np.int32)).cuda()


def _prepare_append(case, gen, rng):
    t, hq, hkv, dim, page = (case[n] for n in ("tokens", "hq", "hkv", "dim", "page"))
    # a portion of a prompt behind the single tokens of other sequences: positions that run on, and positions from anywhere
    single = min(t, 96)
    positions = np.concatenate([rng.integers(0, 8192, single), 1000 + np.arange(t - single) % 7000])
    pages = 2 * ((t + page - 1) // page) + 1
    slots = rng.permutation(pages * page)[:single]
    free = np.setdiff1d(np.arange(pages * page), slots, assume_unique=True)
    slots = np.concatenate([slots, free[:t - single]])
    # some channels of the keys are larger than others, as those of trained models are
    wide = torch.exp(0.3 * torch.randn((hq + 2 * hkv) * dim, generator=gen, device="cuda"))
    qkv = (torch.randn(t, (hq + 2 * hkv) * dim, generator=gen, device="cuda") * wide).bfloat16()
    angle = torch.arange(8192, device="cuda", dtype=torch.float32)[:, None] * (500000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim))
    norms = [(1 + 0.1 * torch.randn(dim, generator=gen, device="cuda")).bfloat16() if case["norm"] else None for _ in range(2)]
    pool = torch.zeros(pages * hkv * (page // 16) * _record(dim), dtype=torch.uint8, device="cuda")
    return dict(case=case, qkv=qkv, positions=_ints(positions), slots=_ints(slots), cos=angle.cos().bfloat16(), sin=angle.sin().bfloat16(),
                q_norm=norms[0], k_norm=norms[1], pool=pool, pages=pages, q_out=torch.empty(t, hq, dim, dtype=torch.bfloat16, device="cuda"),
                k_out=torch.empty(t, hkv, dim, dtype=torch.bfloat16, device="cuda"), v_out=torch.empty(t, hkv, dim, dtype=torch.bfloat16, device="cuda"))


def _pool(gen, pages, hkv, dim, page):
    """A pool whose records hold quantized normal numbers, all of them: what lies behind a sequence's end was somebody else's."""
    n = pages * hkv * (page // 16)
    pool = torch.empty(n, _record(dim), dtype=torch.uint8, device="cuda")
    for at in range(0, n, 1 << 16):  # (a part at a time: the numbers behind the codes take eight times the room)
        part = pool[at:at + (1 << 16)]
        codes = (7.5 + 2.9 * torch.randn(len(part), 2, 16 * dim, generator=gen, device="cuda", dtype=torch.float16)).round().clamp(0, 15).to(torch.uint8)
        part[:, :16 * dim] = (codes[:, 0] | codes[:, 1] << 4)
        scale = 0.33 * torch.exp(0.15 * torch.randn(len(part), 2, dim // GROUP, 16, generator=gen, device="cuda"))
        bias = -scale * (7.5 + 0.5 * torch.randn(scale.shape, generator=gen, device="cuda"))
        part[:, 16 * dim:] = torch.stack([scale, bias], -1).bfloat16().view(torch.uint8).reshape(len(part), -1)
    return pool.reshape(-1)


def _tables(rng, ctx, page):
    blocks = (ctx + page - 1) // page
    pages = int(blocks.sum()) + max(1, int(blocks.sum()) // 8)
    tables, order, at = np.zeros((len(ctx), max(1, int(blocks.max()))), np.int32), rng.permutation(pages), 0
    for i, b in enumerate(blocks):
        tables[i, :b] = order[at:at + b]
        at += b
    return tables, pages


def _contexts(case):
    """Lengths spread evenly from the shortest to the longest."""
    return np.rint(np.linspace(case["lo"], case["hi"], case["seqs"])).astype(np.int64) if case["seqs"] > 1 else np.array([case["hi"]])


def _prepare_decode(case, gen, rng):
    ctx = rng.permutation(_contexts(case))
    tables, pages = _tables(rng, ctx, case["page"])
    q = torch.randn(len(ctx), case["hq"], case["dim"], generator=gen, device="cuda").bfloat16()
    return dict(case=case, q=q, pool=_pool(gen, pages, case["hkv"], case["dim"], case["page"]), pages=pages, tables=_ints(tables), ctx=_ints(ctx),
                out=torch.empty_like(q))


def _news(case):
    """New tokens of every sequence, from about half to one and a half times the middling number."""
    n = case["seqs"]
    return np.array([max(1, case["new"] * (n + 2 * i + 1) // (2 * n)) for i in range(n)] if n > 1 else [case["new"]], np.int64)


def _prepare_prefill(case, gen, rng):
    new = rng.permutation(_news(case))
    ctx = new + case["cached"]
    tables, pages = _tables(rng, ctx, case["page"])
    q = torch.randn(int(new.sum()), case["hq"], case["dim"], generator=gen, device="cuda").bfloat16()
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return dict(case=case, q=q, pool=_pool(gen, pages, case["hkv"], case["dim"], case["page"]), pages=pages, tables=_ints(tables), cu=cu,
                ctx=ctx.astype(np.int32), out=torch.empty_like(q))


def _prepare_logits(case, gen, rng):
    rows, vocab = case["rows"], case["vocab"]
    # histories of different lengths, in which a few tokens come again and again; the first half of each is the prompt
    lengths = rng.permutation(np.linspace(case["history"] // 2, case["history"] * 3 // 2, rows).astype(np.int64)) if rows > 1 else np.array([case["history"]])
    history = np.minimum((vocab * rng.random(int(lengths.sum())) ** 6).astype(np.int64), vocab - 1)
    n_bias = rng.integers(0, 2 * case["bias"] + 1, rows) if case["bias"] else np.zeros(rows, np.int64)
    n_bias = np.minimum(n_bias, vocab)
    bias_id = [np.unique(rng.integers(0, vocab, n)) for n in n_bias]
    bias_off = np.concatenate([[0], np.cumsum([len(b) for b in bias_id])])
    flat = np.concatenate(bias_id) if bias_off[-1] else np.zeros(0, np.int64)
    # a state of a grammar allows a few tokens or most of them; rows without a grammar have none
    words = (vocab + 31) // 32
    with_mask = rng.random(rows) < case["masked"]
    masks = max(1, int(with_mask.sum()))
    rate = torch.from_numpy(rng.choice([0.001, 0.3, 0.95], masks).astype(np.float32)).cuda()
    bits = torch.rand(masks, words * 32, generator=gen, device="cuda") < rate[:, None]
    weights = (1 << torch.arange(32, device="cuda", dtype=torch.int64))
    mask = torch.cat([(bits[i:i + 16].view(-1, words, 32) * weights).sum(-1) for i in range(0, masks, 16)])
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    mask_row = np.where(with_mask, np.cumsum(with_mask) - 1, -1)
    kind = torch.float32 if case["f32"] else torch.bfloat16
    logits = torch.empty(rows, vocab, dtype=kind, device="cuda")
    logits.copy_(3 * torch.randn(rows, vocab, generator=gen, device="cuda"))
    number = lambda lo, hi: torch.from_numpy(rng.uniform(lo, hi, rows).astype(np.float32)).cuda()
    return dict(case=case, logits=logits, history=_ints(history), history_off=_ints(np.concatenate([[0], np.cumsum(lengths)])),
                n_prompt=_ints(lengths // 2), repetition=number(1.0, 1.4), presence=number(0.0, 0.5), frequency=number(0.0, 0.2),
                bias_id=_ints(flat), bias_value=torch.from_numpy(rng.normal(0, 4, len(flat)).astype(np.float32)).cuda(), bias_off=_ints(bias_off),
                mask=mask, mask_row=_ints(mask_row), out=torch.empty_like(logits) if case["out"] else None,
                tokens=torch.empty(rows, dtype=torch.int32, device="cuda"))


# ---- one pass ----------------------------------------------------------------------------------------------------------
@functools.lru_cache(None)
def _context():
    from mlx_llm_b200 import _lib

    return _lib.Context(0)  # one per GPU and thread, as the library asks


def _at(tensor):
    return None if tensor is None else tensor.data_ptr()


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "prefill": _own_prefill, "logits": _own_logits}[kind](state)
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill, "logits": _plain_logits}[kind](state)


def _own_append(s):
    from mlx_llm_b200 import kernels

    c = s["case"]
    kernels.rope_kv_append_q4(_context(), _at(s["qkv"]), c["tokens"], c["hq"], c["hkv"], c["dim"], _at(s["positions"]), _at(s["slots"]), _at(s["cos"]),
                              _at(s["sin"]), _at(s["q_norm"]), _at(s["k_norm"]), 1e-6, c["page"], _at(s["pool"]), s["pages"], _at(s["q_out"]),
                              _at(s["k_out"]), _at(s["v_out"]))
    return [s["q_out"], s["k_out"], s["v_out"]]


def _own_decode(s):
    from mlx_llm_b200 import kernels

    c = s["case"]
    kernels.paged_attn_decode_q4(_context(), _at(s["q"]), _at(s["pool"]), s["pages"], _at(s["tables"]), _at(s["ctx"]), c["seqs"], c["hq"], c["hkv"],
                                 c["dim"], c["page"], c["dim"] ** -0.5, _at(s["out"]), s["tables"].shape[1])
    return s["out"]


def _own_prefill(s):
    from mlx_llm_b200 import kernels

    c = s["case"]
    kernels.paged_attn_prefill_q4(_context(), _at(s["q"]), _at(s["pool"]), s["pages"], _at(s["tables"]), s["tables"].shape[1], s["cu"], s["ctx"], c["hq"],
                                  c["hkv"], c["dim"], c["page"], c["dim"] ** -0.5, _at(s["out"]))
    return s["out"]


def _own_logits(s):
    from mlx_llm_b200 import kernels

    c = s["case"]
    rules = kernels.logit_rules(history=_at(s["history"]), history_off=_at(s["history_off"]), n_prompt=_at(s["n_prompt"]), repetition=_at(s["repetition"]),
                                presence=_at(s["presence"]), frequency=_at(s["frequency"]), bias_id=_at(s["bias_id"]), bias_value=_at(s["bias_value"]),
                                bias_off=_at(s["bias_off"]), mask=_at(s["mask"]), mask_words=s["mask"].shape[1], mask_row=_at(s["mask_row"]))
    kernels.logits_adjust(_context(), _at(s["logits"]), c["rows"], c["vocab"], rules, f32=c["f32"], out=_at(s["out"]), argmax=_at(s["tokens"]))
    return [s["tokens"]] if s["out"] is None else [s["out"], s["tokens"]]


def _rounded(x):
    return x.bfloat16().float()


def _plain_append(s):
    c = s["case"]
    hq, hkv, dim = c["hq"], c["hkv"], c["dim"]
    x = s["qkv"].float().view(c["tokens"], hq + 2 * hkv, dim)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    cos, sin = (s[n][s["positions"].long()].float()[:, None] for n in ("cos", "sin"))

    def turned(x, norm):
        if norm is not None:
            x = _rounded(x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)) * norm.float())
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return _rounded(torch.cat([_rounded(a * cos) - _rounded(b * sin), _rounded(b * cos) + _rounded(a * sin)], -1))

    k, v = (_quantized(x.reshape(-1, dim // GROUP, GROUP)) for x in (turned(k, s["k_norm"]), v))
    slots = s["slots"].long()
    _store(s["pool"], k, v, slots, c)
    return [turned(q, s["q_norm"]).bfloat16()] + [_values(codes, scale, bias).view(-1, hkv, dim).bfloat16() for codes, scale, bias in (k, v)]


def _away(x):
    """Rounded to the nearest whole number, halves away from zero."""
    x = x.double()
    return (torch.sign(x) * torch.floor(x.abs() + 0.5)).float()


def _quantized(x):
    """A scale with which zero and the value farthest from it are codes; then the codes nearest for the scale and bias as they are stored."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    edge, span = torch.where(lo.abs() > hi.abs(), lo, hi), hi - lo
    flat = span == 0
    count = _away(15 * edge.abs() / torch.where(flat, torch.ones_like(span), span))
    scale = torch.where(flat, torch.zeros_like(edge), -edge / torch.where(flat, torch.ones_like(count), count)).bfloat16()
    codes = _away((x - edge) / torch.where(flat, torch.ones_like(edge), scale.float()))
    return codes.clamp(0, 15), scale, edge.bfloat16()


def _values(codes, scale, bias):
    return _rounded(codes * scale.float() + bias.float())


def _store(pool, k, v, slots, c):
    """Codes, scales and biases of tokens into the records that their slots lie in."""
    hkv, dim, page = c["hkv"], c["dim"], c["page"]
    tile = page // 16
    tokens = len(slots)
    record = ((slots // page)[:, None] * hkv + torch.arange(hkv, device=slots.device)) * tile + (slots % page // 16)[:, None]
    base, at = record * _record(dim), (slots % 16)[:, None]
    pairs = k[0].to(torch.uint8).view(tokens, hkv, dim // 2, 2)
    pool[(base + at * (dim // 2))[..., None] + torch.arange(dim // 2, device=slots.device)] = pairs[..., 0] | pairs[..., 1] << 4
    pairs = v[0].to(torch.uint8).view(tokens, hkv, dim // 2, 2)
    byte = torch.arange(dim // 2, device=slots.device)  # byte of a token's row of values: block, word of the block, byte of the half word
    word = ((at // 8 * 8)[..., None] + byte // (dim // 16)) * 4 + (at % 8 // 2)[..., None]
    where = (word * (dim // 32) + byte % (dim // 16) // 2) * 4 + (at % 2)[..., None] * 2 + byte % 2
    pool[(base + 8 * dim)[..., None] + where] = pairs[..., 0] | pairs[..., 1] << 4
    groups = dim // GROUP
    for n, x in enumerate((k, v)):
        both = torch.stack([x[1], x[2]], -1).view(torch.uint8).view(tokens, hkv, groups, 4)
        where = ((n * groups + torch.arange(groups, device=slots.device)) * 16 + at[..., None]) * 4
        pool[(base + 16 * dim)[..., None, None] + where[..., None] + torch.arange(4, device=slots.device)] = both


def _loaded(s):
    """Keys and values of all sequences in 32 bits, [sequences, kv heads, positions, dim], whatever is in their tables."""
    c = s["case"]
    hkv, dim, tile = c["hkv"], c["dim"], c["page"] // 16
    seqs, blocks = s["tables"].shape
    records = s["pool"].view(-1, hkv, tile, _record(dim))[s["tables"].long()].permute(0, 2, 1, 3, 4).reshape(seqs, hkv, blocks * tile, _record(dim))
    groups = dim // GROUP
    sb = records[..., 16 * dim:].contiguous().view(torch.bfloat16).view(seqs, hkv, -1, 2, groups, 16, 2).transpose(-3, -2).float()

    def whole(codes, sb):
        codes = codes.reshape(seqs, hkv, -1, 16, groups, GROUP)
        return _rounded(codes * sb[..., :1] + sb[..., 1:]).reshape(seqs, hkv, -1, dim)

    def nibbles(b):
        return torch.stack([b & 15, b >> 4], -1)

    k = nibbles(records[..., :8 * dim]).float()
    v = nibbles(records[..., 8 * dim:16 * dim]).view(seqs, hkv, -1, 2, 8, 4, dim // 32, 2, 4)
    v = v.permute(0, 1, 2, 3, 5, 7, 4, 6, 8).float()  # ... half, pair, token of the pair, block, word, dim
    return whole(k, sb[..., 0, :, :, :]), whole(v, sb[..., 1, :, :, :])


def _attended(q, k, v, seen, scale):
    """q [sequences, queries, heads, dim]; seen [sequences, queries, positions]; rows that see nothing become zeros."""
    seqs, n, hq, dim = q.shape
    hkv = k.shape[1]
    q = q.view(seqs, n, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, -1, dim)
    scores = (torch.matmul(q, k.transpose(-1, -2)) * scale).view(seqs, hkv, hq // hkv, n, -1)
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(seqs, hkv, -1, weights.shape[-1]), v).view(seqs, hkv, hq // hkv, n, dim)
    return torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4).reshape(seqs, n, hq, dim)


def _plain_decode(s):
    k, v = _loaded(s)
    seen = torch.arange(k.shape[2], device="cuda") < s["ctx"][:, None, None]
    return _attended(s["q"].float()[:, None], k, v, seen, s["case"]["dim"] ** -0.5)[:, 0].bfloat16()


def _plain_prefill(s):
    k, v = _loaded(s)
    new = np.diff(s["cu"])
    most = int(new.max())
    row = np.minimum(s["cu"][:-1, None] + np.arange(most), len(s["q"]) - 1)
    real = torch.from_numpy(np.arange(most) < new[:, None]).cuda()
    last = torch.from_numpy((s["ctx"] - new)[:, None] + np.arange(most)).cuda()  # the last position that a query sees
    seen = torch.arange(k.shape[2], device="cuda") <= last[..., None]
    return _attended(s["q"][torch.from_numpy(row).cuda()].float(), k, v, seen, s["case"]["dim"] ** -0.5)[real].bfloat16()


def _plain_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    x = s["logits"].float()
    device = x.device
    at = torch.arange(len(s["history"]), device=device)
    row = torch.searchsorted(s["history_off"].long(), at, right=True) - 1
    place = row * vocab + s["history"].long()
    answer = at >= (s["history_off"][:-1] + s["n_prompt"]).long()[row]
    seen = torch.zeros(rows * vocab, device=device).index_fill_(0, place, 1.0).view(rows, vocab) > 0
    count = torch.zeros(rows * vocab, device=device).index_add_(0, place, answer.float()).view(rows, vocab)
    rate = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rate, x * rate), x)
    x = torch.where(count > 0, (x - count * s["frequency"][:, None]) - s["presence"][:, None], x)
    at = torch.arange(len(s["bias_id"]), device=device)
    row = torch.searchsorted(s["bias_off"].long(), at, right=True) - 1
    bias = torch.zeros(rows * vocab, device=device).index_add_(0, row * vocab + s["bias_id"].long(), s["bias_value"]).view(rows, vocab)
    x = x + bias
    bits = (s["mask"][..., None] >> torch.arange(32, device=device, dtype=torch.int32)) & 1
    allowed = bits.view(len(s["mask"]), -1)[:, :vocab].bool()[s["mask_row"].clamp(min=0).long()] | (s["mask_row"] < 0)[:, None]
    x = torch.where(allowed, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    index = torch.arange(vocab, device=device, dtype=torch.int32)
    tokens = torch.where(x == top, index, torch.full_like(index, vocab)).amin(-1)
    tokens = torch.where(top[:, 0] > -math.inf, tokens, torch.full_like(tokens, -1))
    return [x.to(s["logits"].dtype), tokens] if c["out"] else [tokens]


# ---- work and exact answers --------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "logits":
        size = (4 if case["f32"] else 2) * case["rows"] * case["vocab"]
        masks = case["masked"] * case["rows"] * case["vocab"] / 8
        return {"bytes": size * (2 if case["out"] else 1) + masks + case["rows"] * (4.0 * case["history"] + 8 * case["bias"]), "flops": float(case["rows"] * case["vocab"])}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    token = 2 * hkv * (dim / 2 + 4 * dim / GROUP)  # bytes of a token in the cache
    if case["kind"] == "append":
        t = case["tokens"]
        return {"bytes": t * (2.0 * (2 * hq + 4 * hkv) * dim + token + 2 * dim + 8), "flops": t * (6.0 * (hq + hkv) + 8.0 * hkv) * dim}
    if case["kind"] == "decode":
        keys = float(_contexts(case).sum())
        return {"bytes": keys * token + 4.0 * case["seqs"] * hq * dim, "flops": 4.0 * keys * hq * dim}
    new = _news(case).astype(np.float64)
    pairs = float((new * case["cached"] + new * (new + 1) / 2).sum())
    return {"bytes": float((new + case["cached"]).sum()) * token + 4.0 * new.sum() * hq * dim, "flops": 4.0 * pairs * hq * dim}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_attention, "prefill": _exact_attention, "logits": _exact_logits}[case["kind"]](s)


def _nearest(x):
    return x.to(torch.bfloat16).double()


def _exact_append(s):
    c = s["case"]
    hq, hkv, half = c["hq"], c["hkv"], c["dim"] // 2
    heads = s["qkv"].double().unflatten(1, (-1, 2, half))
    where = s["positions"].long()
    turn = torch.complex(s["cos"][where].double(), s["sin"][where].double())[:, None]

    def rotate(x, weight):
        if weight is not None:
            x = _nearest(x / (x.square().mean((-2, -1), keepdim=True) + 1e-6).sqrt() * weight.double().view(2, half))
        first = _nearest(x[:, :, 0] * turn.real) + _nearest(-x[:, :, 1] * turn.imag)
        second = _nearest(x[:, :, 1] * turn.real) + _nearest(x[:, :, 0] * turn.imag)
        return _nearest(torch.cat([first, second], -1))

    def kept(x):
        x = x.unflatten(-1, (-1, GROUP))
        low, high = torch.aminmax(x, dim=-1)
        end = low.where(low.abs() > high.abs(), high)
        n = torch.trunc(15 * end.abs() / (high - low) + 0.5)
        step = _nearest((-end / n).where(high > low, 0 * end))[..., None]
        code = ((x - end[..., None]) / step.where(step != 0, step + 1)).add(0.5).floor().clamp(0, 15)
        return _nearest(code * step + end[..., None]).flatten(-2)

    return [rotate(heads[:, :hq], s["q_norm"]), kept(rotate(heads[:, hq:hq + hkv], s["k_norm"])), kept(heads[:, hq + hkv:].flatten(-2))]


def _exact_attention(s):
    c = s["case"]
    hq, hkv, dim, page = c["hq"], c["hkv"], c["dim"], c["page"]
    ctx = [int(n) for n in s["ctx"]]
    cu = s["cu"] if "cu" in s else np.arange(len(ctx) + 1)
    pool = s["pool"].view(-1, hkv, page // 16, _record(dim))
    # the place of every nibble of a token's dims, and of its scales, in a record: one byte number and one shift each
    token, d = torch.arange(16, device="cuda")[:, None], torch.arange(dim, device="cuda")
    block, rest = d // (dim // 8), d % (dim // 8)
    word = ((token // 8 * 8 + block) * 4 + token % 8 // 2) * (dim // 32) + rest // 4
    places = [(token * (dim // 2) + d // 2, (d % 2) * 4), (8 * dim + word * 4 + token % 2 * 2 + rest % 4 // 2, (d % 2) * 4)]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(ctx):
        rows = slice(int(cu[i]), int(cu[i + 1]))
        new = rows.stop - rows.start
        if n == 0 or new == 0:
            continue
        records = pool[s["tables"][i, :(n + page - 1) // page].long()].transpose(0, 1).flatten(1, 2)
        values = []
        for j, (byte, shift) in enumerate(places):
            code = (records[..., byte] >> shift.to(torch.uint8)) & 15
            sb = records[..., 16 * dim:].contiguous().view(torch.bfloat16).unflatten(-1, (2, dim // GROUP, 16, 2))[..., j, :, :, :].double()
            sb = sb.transpose(-3, -2).repeat_interleave(GROUP, -2)
            values.append(_nearest(code.double() * sb[..., 0] + sb[..., 1]).flatten(1, 2)[:, :n])
        q = s["q"][rows].double().view(new, hkv, -1, dim)
        hidden = torch.arange(n, device="cuda") > n - new + torch.arange(new, device="cuda")[:, None]
        for h in range(hkv):
            weights = torch.einsum("rgd,kd->rgk", q[:, h], values[0][h]) * dim ** -0.5
            weights = torch.softmax(weights.masked_fill_(hidden[:, None], -math.inf), -1)
            out[rows, h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.einsum("rgk,kd->rgd", weights, values[1][h])
    return out


def _exact_logits(s):
    if s["out"] is None:
        return None
    x = s["logits"].double()
    history, off = s["history"].cpu().numpy(), s["history_off"].cpu().numpy()
    prompt, bias_off, mask_row = s["n_prompt"].cpu().numpy(), s["bias_off"].cpu().numpy(), s["mask_row"].cpu().numpy()
    masks = s["mask"].cpu().numpy().view(np.uint8)
    for i in range(len(x)):
        ids = history[off[i]:off[i + 1]]
        if len(ids):
            seen = torch.from_numpy(np.unique(ids).astype(np.int64)).cuda()
            r = s["repetition"][i].double()
            x[i, seen] = torch.where(x[i, seen] > 0, x[i, seen] / r, x[i, seen] * r)
            told, times = np.unique(ids[prompt[i]:], return_counts=True)
            told, times = torch.from_numpy(told.astype(np.int64)).cuda(), torch.from_numpy(times).cuda().double()
            x[i, told] -= times * s["frequency"][i].double() + s["presence"][i].double()
        a, b = int(bias_off[i]), int(bias_off[i + 1])
        x[i, s["bias_id"][a:b].long()] += s["bias_value"][a:b].double()
        if mask_row[i] >= 0:
            bits = np.unpackbits(masks[mask_row[i]], bitorder="little")[:x.shape[1]]
            x[i, torch.from_numpy(bits == 0).cuda()] = -math.inf
    return [x, None]

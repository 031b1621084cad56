"""Kernel-level entry points of the C ABI as Python callables (device buffers in, device buffers
out).  Used by the parity tests and the microbenchmarks; the engine API lives in engine.py."""
import ctypes as C
import operator

import numpy as np

from ._lib import DevBuf, check, load, ptr


def paged_attn_decode(ctx, q, k_pool, v_pool, block_tables, ctx_lens, num_seqs, hq, hkv, head_dim, page_size, scale,
                      out, max_blocks, chunk_tokens=0):
    check(load().b2_paged_attn_decode(ctx.h, ptr(q), ptr(k_pool), ptr(v_pool), ptr(block_tables), int(max_blocks), ptr(ctx_lens),
                                      int(num_seqs), int(hq), int(hkv), int(head_dim), int(page_size), C.c_float(scale),
                                      int(chunk_tokens), ptr(out)))


def paged_attn_decode_host(ctx, q_host, k_pool, v_pool, block_tables, ctx_lens, num_seqs, hq, hkv, head_dim, page_size, scale,
                           out_host, max_blocks, chunk_tokens=0):
    check(load().b2_paged_attn_decode_host(ctx.h, ptr(q_host), ptr(k_pool), ptr(v_pool), ptr(block_tables), int(max_blocks),
                                           ptr(ctx_lens), int(num_seqs), int(hq), int(hkv), int(head_dim), int(page_size),
                                           C.c_float(scale), int(chunk_tokens), ptr(out_host)))


def paged_attn_prefill(ctx, q, k_pool, v_pool, block_tables, max_blocks, cu_seqlens, ctx_lens, hq, hkv, head_dim, page_size,
                       scale, out):
    cu = np.ascontiguousarray(cu_seqlens, np.int32)
    cl = np.ascontiguousarray(ctx_lens, np.int32)
    check(load().b2_paged_attn_prefill(ctx.h, ptr(q), ptr(k_pool), ptr(v_pool), ptr(block_tables), int(max_blocks), ptr(cu), ptr(cl),
                                       int(cl.size), int(hq), int(hkv), int(head_dim), int(page_size), C.c_float(scale), ptr(out)))


_TYPES = {"p": C.c_void_p, "i": C.c_int32, "l": C.c_int64, "f": C.c_float}


class _Entry:
    """An entry point with declared argument types: numbers and addresses go as they are, which saves a call of many arguments a few microseconds."""

    def __init__(self, name, types):
        self.name, self.types, self.fn = name, [_TYPES[t] for t in types], None

    def __call__(self, *args):
        if self.fn is None:
            self.fn = getattr(load(), self.name)
            self.fn.argtypes = self.types
        try:
            rc = self.fn(*args)
        except C.ArgumentError:  # numbers that are not Python's own, an array's length in numpy for one
            rc = self.fn(*[a if a is None or isinstance(a, C.c_void_p) else float(a) if t is C.c_float else operator.index(a) for t, a in zip(self.types, args)])
        if rc:
            check(rc)


def _at(a):
    """Address of a device buffer (DevBuf, or a number), or nothing."""
    if a is None or type(a) is int:
        return a
    if isinstance(a, DevBuf):
        return a.ptr
    if isinstance(a, np.ndarray):  # (a kernel that reads host memory faults)
        raise TypeError("a host array where a device buffer is needed: upload it with Context.buf")
    return int(a)


_append_q4 = _Entry("b2_rope_kv_append_q4", "ppiiiippppppfipippp")
_decode_q4 = _Entry("b2_paged_attn_decode_q4", "pppipipiiiiifp")
_prefill_q4 = _Entry("b2_paged_attn_prefill_q4", "pppipippiiiiifp")
_adjust = _Entry("b2_logits_adjust", "ppiiilppp")


def kv_q4_pool_bytes(n_pages, hkv, head_dim, page_size):
    lib = load()
    lib.b2_kv_q4_pool_bytes.restype = C.c_int64
    return lib.b2_kv_q4_pool_bytes(C.c_int64(n_pages), int(hkv), int(head_dim), int(page_size))


def rope_kv_append_q4(ctx, qkv, T, hq, hkv, head_dim, positions, slot_mapping, cos, sin, q_norm, k_norm, eps, page_size, kv_pool, n_pages, q_out,
                      k_out=None, v_out=None):
    _append_q4(ctx.h, _at(qkv), T, hq, hkv, head_dim, _at(positions), _at(slot_mapping), _at(cos), _at(sin), _at(q_norm), _at(k_norm), eps, page_size,
               _at(kv_pool), n_pages, _at(q_out), _at(k_out), _at(v_out))


def paged_attn_decode_q4(ctx, q, kv_pool, n_pages, block_tables, ctx_lens, num_seqs, hq, hkv, head_dim, page_size, scale, out, max_blocks):
    _decode_q4(ctx.h, _at(q), _at(kv_pool), n_pages, _at(block_tables), max_blocks, _at(ctx_lens), num_seqs, hq, hkv, head_dim, page_size, scale, _at(out))


def paged_attn_prefill_q4(ctx, q, kv_pool, n_pages, block_tables, max_blocks, cu_seqlens, ctx_lens, hq, hkv, head_dim, page_size, scale, out):
    cu = np.ascontiguousarray(cu_seqlens, np.int32)
    cl = np.ascontiguousarray(ctx_lens, np.int32)
    if cu.ndim != 1 or cl.ndim != 1 or cu.size != cl.size + 1:  # (the library reads one more of the first)
        raise ValueError(f"paged_attn_prefill_q4: {cl.size} contexts need {cl.size + 1} cu_seqlens, not {cu.size}")
    _prefill_q4(ctx.h, _at(q), _at(kv_pool), n_pages, _at(block_tables), max_blocks, cu.ctypes.data, cl.ctypes.data, cl.size, hq, hkv, head_dim, page_size,
                scale, _at(out))


def quantize(ctx, w, out_dim, in_dim, bits, packed, scales, biases, group=64):
    check(load().b2_quantize(ctx.h, ptr(w), C.c_int64(out_dim), C.c_int64(in_dim), int(group), int(bits), ptr(packed), ptr(scales),
                             ptr(biases)))


def dequantize(ctx, packed, scales, biases, out_dim, in_dim, bits, w, group=64):
    check(load().b2_dequantize(ctx.h, ptr(packed), ptr(scales), ptr(biases), C.c_int64(out_dim), C.c_int64(in_dim), int(group),
                               int(bits), ptr(w)))


def unpack_codes(ctx, packed, out_dim, in_dim, bits, codes):
    check(load().b2_unpack_codes(ctx.h, ptr(packed), C.c_int64(out_dim), C.c_int64(in_dim), int(bits), ptr(codes)))


def qmm(ctx, x, packed, scales, biases, m, out_dim, in_dim, bits, y_bf16=None, y_f32=None, group=64):
    check(load().b2_qmm(ctx.h, ptr(x), ptr(packed), ptr(scales), ptr(biases), int(m), int(out_dim), int(in_dim), int(group),
                        int(bits), ptr(y_bf16), ptr(y_f32)))


def qmm_residual(ctx, x, packed, scales, biases, m, out_dim, in_dim, bits, h, group=64):
    check(load().b2_qmm_residual(ctx.h, ptr(x), ptr(packed), ptr(scales), ptr(biases), int(m), int(out_dim), int(in_dim), int(group),
                                 int(bits), ptr(h)))


def qmm_host(ctx, x_host, packed, scales, biases, m, out_dim, in_dim, bits, y_host, group=64):
    check(load().b2_qmm_host(ctx.h, ptr(x_host), ptr(packed), ptr(scales), ptr(biases), int(m), int(out_dim), int(in_dim), int(group),
                             int(bits), ptr(y_host)))


def linear(ctx, x, w, m, out_dim, in_dim, y_bf16=None, y_f32=None):
    check(load().b2_linear(ctx.h, ptr(x), ptr(w), int(m), int(out_dim), int(in_dim), ptr(y_bf16), ptr(y_f32)))


def projection(ctx, x, w, scales, biases, m, out_dim, in_dim, bits, y_bf16=None, y_f32=None, h=None):
    """One projection as a model's layers run it; returns (kernel, table used, K ranges, blocks per cluster)."""
    route = (C.c_int32 * 4)()
    check(load().b2_projection(ctx.h, ptr(x), ptr(w), ptr(scales), ptr(biases), int(m), int(out_dim), int(in_dim), int(bits), ptr(y_bf16),
                               ptr(y_f32), ptr(h), route))
    return tuple(route)


def rms_norm(ctx, x, w, eps, rows, dim, out):
    check(load().b2_rms_norm(ctx.h, ptr(x), ptr(w), C.c_float(eps), int(rows), int(dim), ptr(out)))


def swiglu(ctx, gate, up, n, out):
    check(load().b2_swiglu(ctx.h, ptr(gate), ptr(up), C.c_int64(n), ptr(out)))


def add(ctx, a, b, n, out):
    check(load().b2_add(ctx.h, ptr(a), ptr(b), C.c_int64(n), ptr(out)))


def embed(ctx, table, ids, n, dim, vocab, out):
    check(load().b2_embed(ctx.h, ptr(table), ptr(ids), int(n), int(dim), int(vocab), ptr(out)))


def argmax(ctx, logits, rows, vocab, out):
    check(load().b2_argmax(ctx.h, ptr(logits), int(rows), int(vocab), ptr(out)))


class LogitRules(C.Structure):
    """b2_logit_rules: device pointers, null where a rule is not used."""

    __slots__ = ()  # no attributes but the fields: a misspelt rule must not vanish in one

    _fields_ = [(n, C.c_void_p) for n in ("history", "history_off", "n_prompt", "repetition", "presence", "frequency", "bias_id", "bias_value", "bias_off",
                                          "mask")] + [("mask_words", C.c_int64), ("mask_row", C.c_void_p)]


def logit_rules(mask_words=0, **arrays):
    """Rules for logits_adjust: history, history_off, n_prompt, repetition, presence, frequency, bias_id, bias_value, bias_off, mask, mask_row as device
    buffers (None: not used), and the words of a mask's row."""
    rules = LogitRules()
    rules.mask_words = mask_words if type(mask_words) is int else operator.index(mask_words)
    try:
        for name, a in arrays.items():
            setattr(rules, name, _at(a))
    except AttributeError:
        raise TypeError(f"logit_rules: no rule is called {name}; there are {', '.join(n for n, _ in LogitRules._fields_ if n != 'mask_words')}") from None
    return rules


def logits_adjust(ctx, logits, rows, vocab, rules, f32=False, ld=None, out=None, argmax=None):
    _adjust(ctx.h, _at(logits), f32, rows, vocab, vocab if ld is None else ld, C.addressof(rules), _at(out), _at(argmax))


def rope_inv_freq(head_dim, theta, kind=0, factor=1.0, low=1.0, high=4.0, orig=8192.0):
    out = np.empty(head_dim // 2, np.float32)
    check(load().b2_rope_inv_freq(int(head_dim), C.c_float(theta), int(kind), C.c_float(factor), C.c_float(low), C.c_float(high),
                                  C.c_float(orig), ptr(out)))
    return out


def rope_tables(inv_freq, n_pos):
    inv = np.ascontiguousarray(inv_freq, np.float32)
    cos = np.empty((n_pos, inv.size), np.uint16)
    sin = np.empty_like(cos)
    check(load().b2_rope_tables(ptr(inv), int(inv.size), int(n_pos), ptr(cos), ptr(sin)))
    return cos, sin


def rope_kv_append(ctx, qkv, T, hq, hkv, head_dim, positions, slot_mapping, cos, sin, q_norm, k_norm, eps, page_size, k_pool,
                   v_pool, q_out):
    check(load().b2_rope_kv_append(ctx.h, ptr(qkv), int(T), int(hq), int(hkv), int(head_dim), ptr(positions), ptr(slot_mapping),
                                   ptr(cos), ptr(sin), ptr(q_norm), ptr(k_norm), C.c_float(eps), int(page_size), ptr(k_pool),
                                   ptr(v_pool), ptr(q_out)))


META_FIELDS = ["cu_seqlens", "context_lens", "positions", "token_seq", "slot_mapping", "logit_rows", "logit_seq", "dec_ctx",
               "dec_qrow", "dec_slot", "dec_work_off", "dec_work_seq", "dec_work_chunk", "pf_seq", "pf_qstart", "counts"]


def meta_layout(B, T, W, P):
    sizes = [B + 1, B, T, T, T, B, B, B, B, B, B + 1, W, W, P, P, 8]
    off, out = 0, {}
    for name, n in zip(META_FIELDS, sizes):
        out[name] = (off, n)
        off += n
    return out, off


def build_batch_metadata(ctx, seq_slot, q_len, ctx_before, want_logits, upd, chunk_tokens, q_tile, page_size, max_blocks,
                         max_dec_work, max_pf_work, block_tables_dev):
    """Runs the packer; returns a dict of numpy arrays trimmed to their valid lengths."""
    seq_slot = np.ascontiguousarray(seq_slot, np.int32)
    q_len = np.ascontiguousarray(q_len, np.int32)
    ctx_before = np.ascontiguousarray(ctx_before, np.int32)
    want_logits = np.ascontiguousarray(want_logits, np.int32)
    us = np.ascontiguousarray([u[0] for u in upd], np.int32)
    ui = np.ascontiguousarray([u[1] for u in upd], np.int32)
    up = np.ascontiguousarray([u[2] for u in upd], np.int32)
    B, T = int(seq_slot.size), int(q_len.sum())
    lay, total = meta_layout(B, T, max_dec_work, max_pf_work)
    lib = load()
    lib.b2_batch_metadata_elems.restype = C.c_int64
    assert lib.b2_batch_metadata_elems(B, T, max_dec_work, max_pf_work) == total
    out = ctx.empty((total,), np.int32)
    check(lib.b2_memset(ctx.h, ptr(out), 0xFF, C.c_size_t(total * 4)))
    check(lib.b2_build_batch_metadata(ctx.h, ptr(seq_slot), ptr(q_len), ptr(ctx_before), ptr(want_logits), B, ptr(us), ptr(ui), ptr(up),
                                      int(us.size), int(chunk_tokens), int(q_tile), int(page_size), int(max_blocks),
                                      int(max_dec_work), int(max_pf_work), ptr(block_tables_dev), ptr(out)))
    ctx.sync()
    flat = out.download()
    out.free()
    res = {k: flat[o:o + n].copy() for k, (o, n) in lay.items()}
    n_logits, n_dec, n_dw, n_pw = (int(x) for x in res["counts"][:4])
    res["logit_rows"], res["logit_seq"] = res["logit_rows"][:n_logits], res["logit_seq"][:n_logits]
    for k in ("dec_ctx", "dec_qrow", "dec_slot"):
        res[k] = res[k][:n_dec]
    res["dec_work_off"] = res["dec_work_off"][: n_dec + 1]
    res["dec_work_seq"], res["dec_work_chunk"] = res["dec_work_seq"][:n_dw], res["dec_work_chunk"][:n_dw]
    res["pf_seq"], res["pf_qstart"] = res["pf_seq"][:n_pw], res["pf_qstart"][:n_pw]
    res["counts"] = res["counts"][:6]
    return res

// Fused (optional per-head q/k RMSNorm) -> NeoX RoPE -> quantization to 4 bits -> append into the records of a 4-bit cache.
//
// The rotation is rope_kv.cu's, rounding for rounding; what differs is where keys and values go.  Each 64 dims of a token's head get a
// scale and a bias such that the value farthest from zero, e, and zero itself are codes:
//   n = round(15 |e| / (max - min)),  scale = bf16(-e / n),  bias = e,  code = clamp(round((x - bias) / scale), 0, 15)
// (e the maximum in a tie; halves away from zero).  Codes are taken for the scale as it is stored, so that its rounding costs nothing
// again; all values equal: scale 0.  A NaN or an infinity makes the scale a NaN, and with it the group's values, as they would be in bf16;
// so do values that are too large for 15 |e| or for a scale that attention takes (q4::kScaleEnd), so that all readers have the same values.
//
// Bound by instructions and by the wait for its loads, not by HBM alone (6151 tokens of 64 + 16 heads with norms: 261 MB in 59 us, 4.4 TB/s, while
// 68 % of the issue slots are taken and a warp, one of 26 on an SM, waits for what it loads a third of its time).  So instructions are few: HD / 16
// lanes take a head, each 8 adjacent dims of either half, so that reads and writes are 16 bytes, the rotation's roundings come with bf16x2 instructions
// (a product or a sum of two bf16 numbers rounded once is what they give), and a lane's codes of a group are one word.  The lanes go through
// two heads of a token with one set of positions and norm weights (one head: 65.7 us, four: 60.5 us, and few tokens wait longer: 608 take
// 6.5, 6.8 and 12.9 us).  Queries, keys and values are warps of their own, keys first, since they take longest (queries first: 60.3 us).
#include "kernels.h"
#include "kv_q4.cuh"

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 4;
constexpr int kHeads = 2;  // heads of a token that a group of lanes goes through

__device__ __forceinline__ uint32_t add_bf2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.bf16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
struct Eight {
    uint32_t w[4];
    __device__ __forceinline__ float operator[](int i) const { return i & 1 ? bfhi(w[i >> 1]) : bflo(w[i >> 1]); }
};
__device__ __forceinline__ Eight load8(const uint16_t* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    return {{v.x, v.y, v.z, v.w}};
}
__device__ __forceinline__ void store8(uint16_t* p, const Eight& v) { *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]); }

// Per-head RMSNorm of queries: rope_kv.cu's sum, term for term (its lane l has HD / 64 dims of either half, from HD / 64 l on, and it adds lanes 16, 8, ... 1
// apart), so that a model's queries do not depend on what holds its cache.
template <int HD>
__device__ __forceinline__ void norm_query(Eight& a, Eight& b, const Eight& wa, const Eight& wb, float eps) {
    constexpr int L = HD / 16, V = HD / 64, P = 8 / V;  // lanes of a head, elements and lanes of the other kernel
    float ss[P];
#pragma unroll
    for (int i = 0; i < P; i++) {
        ss[i] = 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) ss[i] += a[i * V + j] * a[i * V + j] + b[i * V + j] * b[i * V + j];
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < P; i++) ss[i] += __shfl_xor_sync(kFull, ss[i], o);
#pragma unroll
    for (int o = P / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < o; i++) ss[i] += ss[i + o];
    const float inv = 1.0f / sqrtf(ss[0] / (float)HD + eps);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a.w[i] = pack_bf2(a[2 * i] * inv * wa[2 * i], a[2 * i + 1] * inv * wa[2 * i + 1]);
        b.w[i] = pack_bf2(b[2 * i] * inv * wb[2 * i], b[2 * i + 1] * inv * wb[2 * i + 1]);
    }
}
// ... of keys: in f64, since one bit of a group's farthest value moves its scale, and with it the whole group.
template <int HD>
__device__ __forceinline__ void norm_key(Eight& a, Eight& b, const Eight& wa, const Eight& wb, float eps) {
    double ss = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) ss += (double)a[i] * a[i] + (double)b[i] * b[i];
#pragma unroll
    for (int o = HD / 32; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
    const double inv = 1.0 / sqrt(ss / HD + (double)eps);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a.w[i] = pack_bf2((float)(a[2 * i] * wa[2 * i] * inv), (float)(a[2 * i + 1] * wa[2 * i + 1] * inv));
        b.w[i] = pack_bf2((float)(b[2 * i] * wb[2 * i] * inv), (float)(b[2 * i + 1] * wb[2 * i + 1] * inv));
    }
}

struct Group {
    float scale, edge;  // (the scale as stored)
};
__device__ __forceinline__ Group group_of(float lo, float hi) {
    const float edge = fabsf(lo) > fabsf(hi) ? lo : hi, span = hi - lo;
    if (span == 0.f) return {0.f, edge};
    const float most = 15.f * fabsf(edge), scale = rbf(__fdiv_rn(-edge, roundf(__fdiv_rn(most, span))));
    return {most < INFINITY && fabsf(scale) < q4::kScaleEnd ? scale : __int_as_float(0x7fc00000), edge};
}
// smallest and largest of a lane's eight; NaN where one is NaN or infinite (0 x is, then)
__device__ __forceinline__ void ends_of(const Eight& v, float& lo, float& hi) {
    lo = hi = v[0];
    float bad = 0.f * v[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        lo = fminf(lo, v[i]), hi = fmaxf(hi, v[i]);
        bad = fmaf(0.f, v[i], bad);
    }
    lo += bad, hi += bad;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The eight codes of a lane, lowest nibble first.  The quotient comes from a reciprocal; what it misses is put right by the sign of an fma:
// (x - edge) / scale is never negative, and halves go up.
__device__ __forceinline__ uint32_t codes_of(const Eight& v, const Group& q) {
    // (a scale below 2^-126 has no reciprocal: such a group, whose values are below 2^-87, is taken 2^64 times as large, exactly)
    const float up = fabsf(q.scale) < 0x1p-100f ? 0x1p64f : 1.f, edge = q.edge * up;
    const float s = fabsf(q.scale) * up, inv = s > 0.f ? __fdividef(1.f, s) : 0.f, half = 0.5f * s;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float d = fabsf(fmaf(v[i], up, -edge));
        const float magic = fminf(d * inv, 15.f) + 8388608.f;  // 2^23: the sum's low bits are the whole number
        const float r = fmaf(8388608.f - magic, s, d);         // d - code s
        int code = (__float_as_int(magic) & 31) + (r >= half) - (r < -half);
        code = s > 0.f ? min(max(code, 0), 15) : 0;
        word |= (uint32_t)code << (4 * i);
    }
    return word;
}
// the values that codes stand for
__device__ __forceinline__ Eight values_of(uint32_t word, const Group& q) {
    const uint32_t s2 = pack_bf2(q.scale, q.scale), e2 = pack_bf2(q.edge, q.edge);
    Eight v;
#pragma unroll
    for (int i = 0; i < 4; i++) v.w[i] = fma_bf2(pack_bf2((float)(word >> (8 * i) & 15), (float)(word >> (8 * i + 4) & 15)), s2, e2);
    return v;
}

template <int HD>
__global__ void __launch_bounds__(kWarps * 32) rope_kv_q4_kernel(const RopeKvQ4Params a, int kv_blocks) {
    using Rec = q4::Record<HD>;
    constexpr int L = HD / 16, R = kHeads;  // L lanes a head
    const RopeKvParams& p = a.rope;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    pdl_wait();
    // keys, values, queries: those that take longest come first
    const int kind = blockIdx.x < kv_blocks ? 1 : blockIdx.x < 2 * kv_blocks ? 2 : 0;
    const int block = blockIdx.x - (kind == 1 ? 0 : kind == 2 ? kv_blocks : 2 * kv_blocks);
    const int lane = threadIdx.x & 31, j = lane % L;
    const int heads = kind == 0 ? p.hq : p.hkv, chunks = (heads + R - 1) / R;  // of R heads of a token
    const int chunk = (block * kWarps + (threadIdx.x >> 5)) * (32 / L) + lane / L, last = p.T * chunks - 1;
    const int tok = min(chunk, last) / chunks, head0 = (min(chunk, last) - tok * chunks) * R;  // (lanes without heads go through the motions of the last)
    const int real_heads = chunk <= last ? min(heads - head0, R) : 0;
    const uint16_t* src = p.qkv + (size_t)tok * p.ld + (size_t)(head0 + (kind == 0 ? 0 : kind == 1 ? p.hq : p.hq + p.hkv)) * HD + 8 * j;
    Eight xs[R], ys[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        const uint16_t* at = src + min(r, heads - 1 - head0) * HD;
        xs[r] = load8(at), ys[r] = load8(at + HD / 2);
    }
    const uint16_t* nw = kind == 0 ? p.q_norm : p.k_norm;
    Eight c, s, wa, wb;
    if (kind < 2) {
        const size_t at = (size_t)p.positions[tok] * (HD / 2) + 8 * j;
        c = load8(p.cos_table + at), s = load8(p.sin_table + at);
        if (nw) wa = load8(nw + 8 * j), wb = load8(nw + HD / 2 + 8 * j);
    }
    auto rotate = [&](Eight& x, Eight& y) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t u = sub_bf2(mul_bf2(x.w[i], c.w[i]), mul_bf2(y.w[i], s.w[i])), v = add_bf2(mul_bf2(y.w[i], c.w[i]), mul_bf2(x.w[i], s.w[i]));
            x.w[i] = u, y.w[i] = v;
        }
    };
    if (kind == 0) {
        uint16_t* dst = p.q_out + ((size_t)tok * p.hq + head0) * HD + 8 * j;
#pragma unroll
        for (int r = 0; r < R; r++) {
            if (nw) norm_query<HD>(xs[r], ys[r], wa, wb, p.eps);
            rotate(xs[r], ys[r]);
            if (r < real_heads) {
                store8(dst + r * HD, xs[r]);
                store8(dst + r * HD + HD / 2, ys[r]);
            }
        }
        return;
    }
    const bool is_k = kind == 1;
    const int slot = p.slot_mapping[tok];
#pragma unroll
    for (int r = 0; r < R; r++) {
        Eight &x = xs[r], &y = ys[r];
        const int head = head0 + r;
        if (is_k) {
            if (nw) norm_key<HD>(x, y, wa, wb, p.eps);
            rotate(x, y);
        }
        float lo1, hi1, lo2, hi2;
        ends_of(x, lo1, hi1);
        ends_of(y, lo2, hi2);
        if (Rec::kGroups == 1) lo1 = lo2 = min_nan(lo1, lo2), hi1 = hi2 = max_nan(hi1, hi2);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) {
            lo1 = min_nan(lo1, __shfl_xor_sync(kFull, lo1, o)), hi1 = max_nan(hi1, __shfl_xor_sync(kFull, hi1, o));
            if (Rec::kGroups == 2) lo2 = min_nan(lo2, __shfl_xor_sync(kFull, lo2, o)), hi2 = max_nan(hi2, __shfl_xor_sync(kFull, hi2, o));
        }
        const Group q1 = group_of(lo1, hi1), q2 = Rec::kGroups == 2 ? group_of(lo2, hi2) : q1;
        const uint32_t c1 = codes_of(x, q1), c2 = codes_of(y, q2);
        if (r < real_heads && slot >= 0 && slot < a.n_slots) {
            const int page = slot / p.page_size, off = slot - page * p.page_size, t = off & 15;
            uint8_t* rec = a.pool + (((size_t)page * p.hkv + head) * (p.page_size >> 4) + (off >> 4)) * Rec::kBytes;
            if (is_k) {  // a word has eight dims
                uint32_t* row = reinterpret_cast<uint32_t*>(rec) + t * (HD / 8) + j;
                row[0] = c1;
                row[HD / 16] = c2;
            } else {  // a half word has four: word d of block g, for dims 8 j + 4 i and HD/2 + 8 j + 4 i
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int d = (i >> 1) * (HD / 2) + 8 * j + 4 * (i & 1);
                    const int word = (((t >> 3) * 8 + d / (HD / 8)) * 4 + ((t & 7) >> 1)) * (HD / 32) + d % (HD / 8) / 4;
                    reinterpret_cast<uint16_t*>(rec + Rec::kV)[2 * word + (t & 1)] = (uint16_t)((i >> 1 ? c2 : c1) >> (16 * (i & 1)));
                }
            }
            if (j < Rec::kGroups)
                reinterpret_cast<uint32_t*>(rec + (is_k ? Rec::kKsb : Rec::kVsb))[j * 16 + t] = pack_bf2(j ? q2.scale : q1.scale, j ? q2.edge : q1.edge);
        }
        uint16_t* dst = is_k ? a.k_out : a.v_out;
        if (dst && r < real_heads) {
            dst += ((size_t)tok * p.hkv + head) * HD + 8 * j;
            store8(dst, values_of(c1, q1));
            store8(dst + HD / 2, values_of(c2, q2));
        }
    }
}

}  // namespace

int32_t b2_rope_kv_q4_launch(b2_ctx* ctx, const RopeKvQ4Params& a) {
    const RopeKvParams& p = a.rope;
    if (p.T <= 0) return B2_OK;
    const int per = kWarps * 512 / p.hd;  // chunks of a block
    auto blocks = [&](int heads) { return (int)(((long)p.T * ((heads + kHeads - 1) / kHeads) + per - 1) / per); };
    const int q_blocks = blocks(p.hq), kv_blocks = blocks(p.hkv);
    auto kernel = p.hd == 128 ? rope_kv_q4_kernel<128> : rope_kv_q4_kernel<64>;
    B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kernel, dim3(q_blocks + 2 * kv_blocks), dim3(kWarps * 32), 0, ctx->stream, a, kv_blocks));
    B2_LAUNCHED(ctx);
    B2_CUDA(cudaGetLastError());
    return B2_OK;
}

extern "C" int32_t b2_rope_kv_append_q4(b2_ctx* ctx, const uint16_t* qkv_dev, int32_t T, int32_t hq, int32_t hkv, int32_t head_dim, const int32_t* positions_dev,
                                        const int32_t* slot_mapping_dev, const uint16_t* cos_dev, const uint16_t* sin_dev, const uint16_t* q_norm_dev,
                                        const uint16_t* k_norm_dev, float eps, int32_t page_size, uint8_t* kv_pool_dev, int32_t n_pages, uint16_t* q_out_dev,
                                        uint16_t* k_out_dev, uint16_t* v_out_dev) {
    B2_REQUIRE(ctx && T >= 0 && (T == 0 || (qkv_dev && positions_dev && slot_mapping_dev && cos_dev && sin_dev && q_out_dev)) && kv_pool_dev, B2_ERR_MSG,
               "b2_rope_kv_append_q4: null argument");
    B2_CHECK(b2_kv_q4_check("b2_rope_kv_append_q4", kv_pool_dev, n_pages, hq, hkv, head_dim, page_size));
    B2_REQUIRE((long)T * (hq + 2 * hkv) < (1l << 31), B2_ERR_UNSUPPORTED, "b2_rope_kv_append_q4: too many tokens for one call");
    B2_REQUIRE((((uintptr_t)qkv_dev | (uintptr_t)q_out_dev | (uintptr_t)k_out_dev | (uintptr_t)v_out_dev | (uintptr_t)cos_dev | (uintptr_t)sin_dev |
                 (uintptr_t)q_norm_dev | (uintptr_t)k_norm_dev) & 15) == 0,
               B2_ERR_UNSUPPORTED, "b2_rope_kv_append_q4: bf16 arrays must be 16-byte aligned");
    RopeKvQ4Params a{};
    RopeKvParams& p = a.rope;
    p.qkv = const_cast<uint16_t*>(qkv_dev);
    p.ld = (hq + 2 * hkv) * head_dim;
    p.positions = positions_dev;
    p.slot_mapping = slot_mapping_dev;
    p.cos_table = cos_dev;
    p.sin_table = sin_dev;
    p.q_norm = q_norm_dev;
    p.k_norm = k_norm_dev;
    p.eps = eps;
    p.T = T;
    p.hq = hq;
    p.hkv = hkv;
    p.hd = head_dim;
    p.page_size = page_size;
    p.q_out = q_out_dev;
    a.pool = kv_pool_dev;
    a.n_slots = n_pages * page_size;
    a.k_out = k_out_dev;
    a.v_out = v_out_dev;
    B2_CUDA(cudaSetDevice(ctx->device));
    return b2_rope_kv_q4_launch(ctx, a);
}

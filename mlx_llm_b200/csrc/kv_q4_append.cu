// Fused (optional per-head q/k RMSNorm) -> NeoX RoPE -> quantization to 4 bits -> append into the records of a 4-bit cache.
//
// The rotation is rope_kv.cu's, rounding for rounding; what differs is where keys and values go.  Each 64 dims of a token's head get a
// scale and a bias such that the value farthest from zero, e, and zero itself are codes:
//   n = round(15 |e| / (max - min)),  scale = bf16(-e / n),  bias = e,  code = clamp(round((x - bias) / scale), 0, 15)
// (e the maximum in a tie; halves away from zero).  Codes are taken for the scale as it is stored, so that its rounding costs nothing
// again; all values equal: scale 0.  A NaN or an infinity makes the scale a NaN, and with it the group's values, as they would be in bf16.
//
// One warp per (token, head); a lane owns HD/64 adjacent elements of each half.
#include "kernels.h"
#include "kv_q4.cuh"

namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float warp_min_nan(float v) {
    float r;
    asm("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;\n" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;\n" : "=f"(r) : "f"(v));
    return r;
}
struct Group {
    float scale, edge;  // (the scale as stored)
};
__device__ __forceinline__ Group group_of(float lo, float hi) {
    const float edge = fabsf(lo) > fabsf(hi) ? lo : hi, span = hi - lo;
    if (span == 0.f) return {0.f, edge};
    const float scale = rbf(__fdiv_rn(-edge, roundf(__fdiv_rn(15.f * fabsf(edge), span))));
    // a bias of infinity is a NaN too: 0 scale + bias would keep it
    return {isfinite(span) ? scale : __int_as_float(0x7fc00000), edge};
}
__device__ __forceinline__ uint32_t code_of(float x, const Group& q) {
    return q.scale == 0.f ? 0u : (uint32_t)fminf(fmaxf(roundf(__fdiv_rn(x - q.edge, q.scale)), 0.f), 15.f);
}

template <int HD>
__global__ void rope_kv_q4_kernel(const RopeKvQ4Params a) {
    constexpr int V = HD / 64;  // elements per lane per half (1 or 2)
    using Rec = q4::Record<HD>;
    const RopeKvParams& p = a.rope;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    pdl_wait();
    const int heads_total = p.hq + 2 * p.hkv;
    const int wid = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (wid >= p.T * heads_total) return;
    const int lane = threadIdx.x & 31;
    const int tok = wid / heads_total, head = wid % heads_total;
    const uint16_t* src = p.qkv + (size_t)tok * p.ld + (size_t)head * HD;
    const bool is_q = head < p.hq, is_k = !is_q && head < p.hq + p.hkv;
    float x1[V], x2[V];  // first-half and second-half elements of this lane
    if (V == 2) {
        const uint32_t lo = reinterpret_cast<const uint32_t*>(src)[lane], hi = reinterpret_cast<const uint32_t*>(src)[32 + lane];
        x1[0] = bflo(lo), x1[V - 1] = bfhi(lo);
        x2[0] = bflo(hi), x2[V - 1] = bfhi(hi);
    } else {
        x1[0] = bf2f(src[lane]);
        x2[0] = bf2f(src[32 + lane]);
    }
    if (is_q || is_k) {
        const uint16_t* nw = is_q ? p.q_norm : p.k_norm;
        if (nw) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < V; j++) ss += x1[j] * x1[j] + x2[j] * x2[j];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
            const float inv = 1.0f / sqrtf(ss / (float)HD + p.eps);
#pragma unroll
            for (int j = 0; j < V; j++) {
                x1[j] = rbf(x1[j] * inv * bf2f(nw[lane * V + j]));
                x2[j] = rbf(x2[j] * inv * bf2f(nw[HD / 2 + lane * V + j]));
            }
        }
        const int pos = p.positions[tok];
        const uint16_t* ct = p.cos_table + (size_t)pos * (HD / 2);
        const uint16_t* st = p.sin_table + (size_t)pos * (HD / 2);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float c = bf2f(ct[lane * V + j]), s = bf2f(st[lane * V + j]);
            const float y1 = rbf(rbf(x1[j] * c) + rbf(-x2[j] * s)), y2 = rbf(rbf(x2[j] * c) + rbf(x1[j] * s));
            x1[j] = y1, x2[j] = y2;
        }
    }
    if (is_q) {
        uint16_t* dst = p.q_out + ((size_t)tok * p.hq + head) * HD;
        if (V == 2) {
            reinterpret_cast<uint32_t*>(dst)[lane] = pack_bf2(x1[0], x1[V - 1]);
            reinterpret_cast<uint32_t*>(dst)[32 + lane] = pack_bf2(x2[0], x2[V - 1]);
        } else {
            dst[lane] = f2bf(x1[0]);
            dst[32 + lane] = f2bf(x2[0]);
        }
        return;
    }
    const int kvh = head - p.hq - (is_k ? 0 : p.hkv);
    Group q1, q2;  // of the first and the second half; one group for both at head size 64
    if (V == 2) {
        q1 = group_of(warp_min_nan(fminf(x1[0], x1[V - 1]) + 0.f * (x1[0] + x1[V - 1])), warp_max_nan(fmaxf(x1[0], x1[V - 1])));
        q2 = group_of(warp_min_nan(fminf(x2[0], x2[V - 1]) + 0.f * (x2[0] + x2[V - 1])), warp_max_nan(fmaxf(x2[0], x2[V - 1])));
    } else {
        q1 = q2 = group_of(warp_min_nan(fminf(x1[0], x2[0]) + 0.f * (x1[0] + x2[0])), warp_max_nan(fmaxf(x1[0], x2[0])));
    }
    uint32_t c1[V], c2[V];
#pragma unroll
    for (int j = 0; j < V; j++) c1[j] = code_of(x1[j], q1), c2[j] = code_of(x2[j], q2);
    const int slot = p.slot_mapping[tok];
    if (slot >= 0 && slot < a.n_slots) {
        const int page = slot / p.page_size, off = slot % p.page_size, t = off & 15;
        uint8_t* rec = a.pool + (((size_t)page * p.hkv + kvh) * (p.page_size >> 4) + (off >> 4)) * Rec::kBytes;
        // a byte of a token's row holds dims 2b, 2b + 1: this lane's of either half, or, at head size 64, a pair of lanes'
        uint32_t b1, b2;
        if (V == 2) {
            b1 = c1[0] | c1[V - 1] << 4, b2 = c2[0] | c2[V - 1] << 4;
        } else {
            b1 = c1[0] | __shfl_down_sync(kFull, c1[0], 1) << 4, b2 = c2[0] | __shfl_down_sync(kFull, c2[0], 1) << 4;
        }
        if (V == 2 || (lane & 1) == 0) {
            const int at = V == 2 ? lane : lane >> 1;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int b = at + half * (HD / 4);
                int where = t * (HD / 2) + b;
                if (!is_k) {
                    constexpr int per = HD / 16;  // bytes of a token in a block
                    where = Rec::kV + ((((t >> 3) * 8 + b / per) * 4 + ((t & 7) >> 1)) * (HD / 32) + (b % per >> 1)) * 4 + (t & 1) * 2 + (b & 1);
                }
                rec[where] = (uint8_t)(half ? b2 : b1);
            }
        }
        if (lane < Rec::kGroups)
            reinterpret_cast<uint32_t*>(rec + (is_k ? Rec::kKsb : Rec::kVsb))[lane * 16 + t] = pack_bf2(lane ? q2.scale : q1.scale, lane ? q2.edge : q1.edge);
    }
    uint16_t* dst = is_k ? a.k_out : a.v_out;
    if (dst) {
        dst += ((size_t)tok * p.hkv + kvh) * HD;
        const uint32_t s1 = pack_bf2(q1.scale, q1.scale), e1 = pack_bf2(q1.edge, q1.edge), s2 = pack_bf2(q2.scale, q2.scale), e2 = pack_bf2(q2.edge, q2.edge);
        const uint32_t v1 = fma_bf2(pack_bf2((float)c1[0], (float)c1[V - 1]), s1, e1), v2 = fma_bf2(pack_bf2((float)c2[0], (float)c2[V - 1]), s2, e2);
        if (V == 2) {
            reinterpret_cast<uint32_t*>(dst)[lane] = v1;
            reinterpret_cast<uint32_t*>(dst)[32 + lane] = v2;
        } else {
            dst[lane] = (uint16_t)v1;
            dst[32 + lane] = (uint16_t)v2;
        }
    }
}

}  // namespace

int32_t b2_rope_kv_q4_launch(b2_ctx* ctx, const RopeKvQ4Params& a) {
    const RopeKvParams& p = a.rope;
    if (p.T <= 0) return B2_OK;
    const long warps = (long)p.T * (p.hq + 2 * p.hkv);
    const int wpb = 8;
    const unsigned grid = (unsigned)((warps + wpb - 1) / wpb);
    auto kernel = p.hd == 128 ? rope_kv_q4_kernel<128> : rope_kv_q4_kernel<64>;
    B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kernel, dim3(grid), dim3(wpb * 32), 0, ctx->stream, a));
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
    B2_REQUIRE((((uintptr_t)qkv_dev | (uintptr_t)q_out_dev | (uintptr_t)k_out_dev | (uintptr_t)v_out_dev) & 3) == 0, B2_ERR_UNSUPPORTED,
               "b2_rope_kv_append_q4: qkv, q_out, k_out and v_out must be 4-byte aligned");
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

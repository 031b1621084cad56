// Rules on a step's logits, and the greedy choice under them, in one pass over the logits:
//   penalties for tokens that came before (repetition: prompt and answer; presence, frequency: the answer), biases, a grammar's mask.
//
// A token's value v, in f32, each step with one rounding:  seen before: v / r where v > 0, else v r;  n times in the answer: (v - n f) - p;
// with a bias: v + b;  not allowed: -inf.  The choice is made among these; written out they are rounded to the logits' type.
//
// Bound by the bytes of the logits for many rows and by the latency of its phases for few.  A cluster of eight blocks takes a row, each
// block one eighth of the vocabulary, whose counters lie in its shared memory.  The row's history is read once: block i reads its i-th
// eighth and counts in the shared memory of whichever block has the token (integers: the order of the atomics changes nothing).  A bit
// per token says whether any rule names it, so that the pass over the logits looks at counters and biases for those alone.
#include <algorithm>

#include "elt.cuh"
#include "kernels.h"

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kBlocks = 8, kThreads = 512;
constexpr int kMaxSlice = 24576;  // tokens of a block at a time: 96 KB of counters, two blocks on an SM
constexpr uint32_t kInPrompt = 0x80000000u;

__device__ __forceinline__ uint32_t at_block(uint32_t addr, uint32_t block) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(block));
    return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }

struct AdjustParams {
    b2_logit_rules r;
    const void* in;
    void* out;  // nullable; may be `in`
    int32_t* argmax;
    int64_t ld;
    int vocab, slice;  // tokens of a block in one round: a multiple of 32
};

template <typename T>
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads, 2) logits_adjust_kernel(const AdjustParams p) {
    constexpr int V = 16 / sizeof(T);
    extern __shared__ __align__(16) uint32_t smem[];
    uint32_t* const counts = smem;            // [slice]: kInPrompt if seen at all, and how often in the answer
    uint32_t* const named = smem + p.slice;   // [slice / 32] a bit per token that a rule names
    __shared__ float sv[kThreads / 32], cv[kBlocks];
    __shared__ int si[kThreads / 32], ci[kBlocks];
    pdl_wait();
    const int block = blockIdx.x % kBlocks, row = blockIdx.x / kBlocks, tid = threadIdx.x;
    const b2_logit_rules& r = p.r;
    const T* in = reinterpret_cast<const T*>(p.in) + (size_t)row * p.ld;
    T* out = p.out ? reinterpret_cast<T*>(p.out) + (size_t)row * p.ld : nullptr;
    const int h0 = r.history_dev ? r.history_off_dev[row] : 0, h1 = r.history_dev ? r.history_off_dev[row + 1] : 0;
    const int answer = h0 + (r.n_prompt_dev ? r.n_prompt_dev[row] : 0);
    const int b0 = r.bias_id_dev ? r.bias_off_dev[row] : 0, b1 = r.bias_id_dev ? r.bias_off_dev[row + 1] : 0;
    const bool any = h1 > h0 || b1 > b0;
    const float rep = r.repetition_dev ? r.repetition_dev[row] : 1.f, pres = r.presence_dev ? r.presence_dev[row] : 0.f,
                freq = r.frequency_dev ? r.frequency_dev[row] : 0.f;
    const int mask_row = !r.mask_dev ? -1 : r.mask_row_dev ? r.mask_row_dev[row] : row;
    const uint32_t* mask = mask_row < 0 ? nullptr : r.mask_dev + (size_t)mask_row * r.mask_words;
    const bool vec = ((uintptr_t)in & 15) == 0 && ((uintptr_t)out & 15) == 0;
    float best = -INFINITY;
    int bi = 0x7fffffff;
    const int round = kBlocks * p.slice;
    for (int base = 0; base < p.vocab; base += round) {
        const int first = base + block * p.slice, last = min(first + p.slice, p.vocab);  // this block's tokens
        if (any) {
            for (int i = tid; i < p.slice / 4; i += kThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
            for (int i = tid; i < p.slice / 32; i += kThreads) named[i] = 0;
            cluster_sync();
            const int n = min(p.vocab - base, round);
            for (int i = h0 + block * kThreads + tid; i < h1; i += kBlocks * kThreads) {
                const uint32_t t = (uint32_t)(r.history_dev[i] - base);
                if (t >= (uint32_t)n || r.history_dev[i] < 0) continue;
                const uint32_t owner = t / p.slice, at = t - owner * p.slice;
                const uint32_t c = at_block(smem_u32(counts + at), owner), b = at_block(smem_u32(named + (at >> 5)), owner);
                asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;\n" ::"r"(b), "r"(1u << (at & 31)) : "memory");
                if (i >= answer)
                    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], 1;\n" ::"r"(c) : "memory");
                asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;\n" ::"r"(c), "r"(kInPrompt) : "memory");
            }
            for (int i = b0 + block * kThreads + tid; i < b1; i += kBlocks * kThreads) {
                const int id = r.bias_id_dev[i];
                const uint32_t t = (uint32_t)(id - base);
                if (id < 0 || t >= (uint32_t)n) continue;
                const uint32_t owner = t / p.slice, at = t - owner * p.slice;
                asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;\n" ::"r"(at_block(smem_u32(named + (at >> 5)), owner)), "r"(1u << (at & 31)) : "memory");
            }
            cluster_sync();
        }
        auto value = [&](float v, int i, bool is_named, bool allowed) {
            if (is_named) {
                const uint32_t c = counts[i - first];
                if (c & kInPrompt) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                if (c & ~kInPrompt) v = __fsub_rn(__fsub_rn(v, __fmul_rn((float)(c & ~kInPrompt), freq)), pres);
                int lo = b0, hi = b1;  // the bias of this token, if it has one: ids ascend
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (r.bias_id_dev[mid] < i)
                        lo = mid + 1;
                    else
                        hi = mid;
                }
                if (lo < b1 && r.bias_id_dev[lo] == i) v = __fadd_rn(v, r.bias_value_dev[lo]);
            }
            if (!allowed) v = -INFINITY;
            if (v > best) best = v, bi = i;  // a thread's indices ascend, so its first maximum is kept
            return v;
        };
        const int whole = vec && last > first ? (last - first) / V * V : 0;
#pragma unroll 2
        for (int at = tid * V; at < whole; at += kThreads * V) {
            uint4 raw = *reinterpret_cast<const uint4*>(in + first + at);
            uint32_t flags = any ? named[at >> 5] >> (at & 31) : 0u, ok = ~0u;
            if (mask) ok = mask[(first + at) >> 5] >> (at & 31);
            float v[V];
            {
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (V == 8)
                        v[2 * j] = bflo(w[j]), v[2 * j + 1] = bfhi(w[j]);
                    else
                        v[j] = __uint_as_float(w[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < V; j++) v[j] = value(v[j], first + at + j, flags >> j & 1, ok >> j & 1);
            if (out) {
                if constexpr (V == 8)
                    Elt<T>::st8(out + first + at, v);
                else
                    Elt<T>::st4(out + first + at, v);
            }
        }
        for (int at = whole + tid; at < last - first; at += kThreads) {
            const int i = first + at;
            const float v = value(Elt<T>::ld(in + i), i, any && (named[at >> 5] >> (at & 31) & 1), !mask || (mask[i >> 5] >> (i & 31) & 1));
            if (out) Elt<T>::st(out + i, v);
        }
        if (any && base + round < p.vocab) cluster_sync();  // the counters are cleared for the next round
    }
    if (!p.argmax) {
        return;
    }
    auto take = [&](float ov, int oi) {
        if (ov > best || (ov == best && oi < bi)) best = ov, bi = oi;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) take(__shfl_xor_sync(kFull, best, o), __shfl_xor_sync(kFull, bi, o));
    if ((tid & 31) == 0) sv[tid >> 5] = best, si[tid >> 5] = bi;
    cluster_sync();  // (and all blocks of the cluster run)
    if (tid < 32) {
        best = tid < kThreads / 32 ? sv[tid] : -INFINITY;
        bi = tid < kThreads / 32 ? si[tid] : 0x7fffffff;
#pragma unroll
        for (int o = kThreads / 64; o > 0; o >>= 1) take(__shfl_xor_sync(kFull, best, o), __shfl_xor_sync(kFull, bi, o));
        if (tid == 0) {
            asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(at_block(smem_u32(cv + block), 0)), "f"(best) : "memory");
            asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(at_block(smem_u32(ci + block), 0)), "r"(bi) : "memory");
        }
    }
    cluster_sync();
    if (block == 0 && tid == 0) {
        best = -INFINITY, bi = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < kBlocks; j++) take(cv[j], ci[j]);
        p.argmax[row] = bi == 0x7fffffff ? -1 : bi;
    }
}

}  // namespace

int32_t b2_logits_adjust_launch(b2_ctx* ctx, const b2_logit_rules& rules, const void* logits, bool f32, int rows, int vocab, int64_t ld, void* out, int32_t* argmax) {
    if (rows <= 0) return B2_OK;
    AdjustParams p{};
    p.r = rules;
    p.in = logits;
    p.out = out;
    p.argmax = argmax;
    p.ld = ld;
    p.vocab = vocab;
    p.slice = std::min(kMaxSlice, ((vocab + kBlocks - 1) / kBlocks + 31) / 32 * 32);
    const bool counters = rules.history_dev || rules.bias_id_dev;
    const size_t smem = counters ? (size_t)p.slice * 4 + p.slice / 8 : 16;
    const int most = kMaxSlice * 4 + kMaxSlice / 8;
    if (f32) {
        B2_SMEM_ONCE(ctx, logits_adjust_kernel<float>, most);
        B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, logits_adjust_kernel<float>, dim3(rows * kBlocks), dim3(kThreads), smem, ctx->stream, p));
    } else {
        B2_SMEM_ONCE(ctx, logits_adjust_kernel<uint16_t>, most);
        B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, logits_adjust_kernel<uint16_t>, dim3(rows * kBlocks), dim3(kThreads), smem, ctx->stream, p));
    }
    B2_LAUNCHED(ctx);
    B2_CUDA(cudaGetLastError());
    return B2_OK;
}

extern "C" int32_t b2_logits_adjust(b2_ctx* ctx, const void* logits_dev, int32_t f32, int32_t rows, int32_t vocab, int64_t ld, const b2_logit_rules* rules,
                                    void* out_dev, int32_t* argmax_dev) {
    B2_REQUIRE(ctx && logits_dev && rules && (out_dev || argmax_dev), B2_ERR_MSG, "b2_logits_adjust: null argument");
    B2_REQUIRE(rows >= 0 && vocab > 0 && ld >= vocab && rows < (1 << 27), B2_ERR_MSG, "b2_logits_adjust: bad sizes");
    B2_REQUIRE(!rules->history_dev || rules->history_off_dev, B2_ERR_MSG, "b2_logits_adjust: a history needs its rows' offsets");
    B2_REQUIRE(!rules->bias_id_dev || (rules->bias_off_dev && rules->bias_value_dev), B2_ERR_MSG, "b2_logits_adjust: biases need their values and their rows' offsets");
    B2_REQUIRE(!rules->mask_dev || rules->mask_words >= ((int64_t)vocab + 31) / 32, B2_ERR_MSG, "b2_logits_adjust: a mask's row must hold a bit for every token");
    const uintptr_t size = f32 ? 4 : 2;
    B2_REQUIRE((uintptr_t)logits_dev % size == 0 && (uintptr_t)out_dev % size == 0, B2_ERR_UNSUPPORTED, "b2_logits_adjust: logits and out must be aligned to their elements");
    B2_CUDA(cudaSetDevice(ctx->device));
    return b2_logits_adjust_launch(ctx, *rules, logits_dev, f32 != 0, rows, vocab, ld, out_dev, argmax_dev);
}

// Rules on a step's logits, and the greedy choice under them, in one pass over the logits:
//   penalties for tokens that came before (repetition: prompt and answer; presence, frequency: the answer), biases, a grammar's mask.
//
// A token's value v, in f32, each step with one rounding:  seen before: v / r where v > 0, else v r;  n times in the answer: (v - n f) - p;
// with a bias: v + b;  not allowed: -inf.  The choice is made among these; written out they are rounded to the logits' type.
//
// Bound by the bytes of the logits for many rows and by the latency of its phases for few.  A cluster of eight blocks takes a row, each
// block one eighth of the vocabulary.  A block reads the row's whole history and biases (from L2, but for the first block) and keeps what
// falls into its eighth: a bit per token that a rule names, and, ranked by these bits, a counter and a bias for each named token.  Shared
// memory does not grow with the vocabulary that way, so that several blocks fit an SM and one's phases hide behind another's loads; the
// first logits and mask words are on their way before the first phase.  Counters are integers, so the order of the atomics changes nothing.
#include <algorithm>

#include "elt.cuh"
#include "kernels.h"

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kBlocks = 8, kThreads = 512;
constexpr int kMaxSlice = 24576;        // tokens of a block at a time
constexpr int kWords = kMaxSlice / 32;
constexpr int kNamed = 4096;            // named tokens that are kept at a time
constexpr int kAhead = 4;               // 16-byte pieces of logits that a thread asks for at the start
constexpr uint32_t kSeen = 0x80000000u;

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
    __shared__ uint32_t named[kWords];       // a bit per token of the slice
    __shared__ uint32_t rank_of[kWords];     // named tokens before a word's
    __shared__ uint32_t counts[kNamed];      // by rank: kSeen, and how often in the answer
    __shared__ float biases[kNamed];
    __shared__ uint32_t s_scan[kThreads / 32];
    __shared__ float sv[kThreads / 32], cv[kBlocks];
    __shared__ int si[kThreads / 32], ci[kBlocks];
    pdl_wait();
    const int block = blockIdx.x % kBlocks, row = blockIdx.x / kBlocks, tid = threadIdx.x, lane = tid & 31;
    const b2_logit_rules& r = p.r;
    const T* in = reinterpret_cast<const T*>(p.in) + (size_t)row * p.ld;
    T* out = p.out ? reinterpret_cast<T*>(p.out) + (size_t)row * p.ld : nullptr;
    const bool vec = ((uintptr_t)in & 15) == 0 && ((uintptr_t)out & 15) == 0;
    const int mask_row = !r.mask_dev ? -1 : r.mask_row_dev ? r.mask_row_dev[row] : row;
    const uint32_t* mask = mask_row < 0 ? nullptr : r.mask_dev + (size_t)mask_row * r.mask_words;
    const int h0 = r.history_dev ? r.history_off_dev[row] : 0, h1 = r.history_dev ? r.history_off_dev[row + 1] : 0;
    const int answer = h0 + (r.n_prompt_dev ? r.n_prompt_dev[row] : 0);
    const int b0 = r.bias_id_dev ? r.bias_off_dev[row] : 0, b1 = r.bias_id_dev ? r.bias_off_dev[row + 1] : 0;
    const float rep = r.repetition_dev ? r.repetition_dev[row] : 1.f, pres = r.presence_dev ? r.presence_dev[row] : 0.f,
                freq = r.frequency_dev ? r.frequency_dev[row] : 0.f;
    float best = -INFINITY;
    int bi = 0x7fffffff;
    auto take = [&](float ov, int oi) {
        if (ov > best || (ov == best && oi < bi)) best = ov, bi = oi;
    };
    for (int base = 0; base < p.vocab; base += kBlocks * p.slice) {
        const int first = base + block * p.slice, n = max(0, min(p.slice, p.vocab - first));  // this block's tokens
        const int whole = vec ? n / V * V : 0;
        uint4 ahead[kAhead];
        uint32_t allow[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int at = (tid + k * kThreads) * V;
            allow[k] = ~0u;
            if (at < whole) {
                ahead[k] = *reinterpret_cast<const uint4*>(in + first + at);
                if (mask) allow[k] = mask[(first + at) >> 5];  // (first is a multiple of 32)
            }
        }
        uint32_t total = 0;  // named tokens
        if (h1 > h0 || b1 > b0) {
            for (int i = tid; i < p.slice / 32; i += kThreads) named[i] = 0;
            __syncthreads();
            auto mark = [&](int id) {
                const uint32_t t = (uint32_t)(id - first);
                if (id >= first && t < (uint32_t)n) atomicOr(&named[t >> 5], 1u << (t & 31));
            };
            for (int i = h0 + tid; i < h1; i += kThreads) mark(r.history_dev[i]);
            for (int i = b0 + tid; i < b1; i += kThreads) mark(r.bias_id_dev[i]);
            __syncthreads();
            static_assert(kWords <= 2 * kThreads, "two words a thread");
            const int w = 2 * tid;
            const uint32_t n0 = w < p.slice / 32 ? __popc(named[w]) : 0, n1 = w + 1 < p.slice / 32 ? __popc(named[w + 1]) : 0;
            uint32_t incl = n0 + n1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(kFull, incl, o);
                if (lane >= o) incl += v;
            }
            if (lane == 31) s_scan[tid >> 5] = incl;
            __syncthreads();
            uint32_t before = incl - n0 - n1;
#pragma unroll
            for (int i = 0; i < kThreads / 32; i++) {
                if (i < tid >> 5) before += s_scan[i];
                total += s_scan[i];
            }
            if (w < p.slice / 32) rank_of[w] = before;
            if (w + 1 < p.slice / 32) rank_of[w + 1] = before + n0;
        }
        auto rank = [&](uint32_t t) { return rank_of[t >> 5] + __popc(named[t >> 5] & ((1u << (t & 31)) - 1)); };
        for (uint32_t from = 0; from == 0 || from < total; from += kNamed) {  // (one round, unless rules name more than kNamed of the slice)
            const uint32_t kept = min((uint32_t)kNamed, total - from);
            if (from > 0) __syncthreads();  // the counters of the round before have been read, and this round's tokens written as they are
            if (kept) {
                for (uint32_t i = tid; i < kept; i += kThreads) counts[i] = 0, biases[i] = 0.f;
                __syncthreads();
                for (int i = h0 + tid; i < h1; i += kThreads) {
                    const int id = r.history_dev[i];
                    const uint32_t t = (uint32_t)(id - first);
                    if (id < first || t >= (uint32_t)n) continue;
                    const uint32_t at = rank(t) - from;
                    if (at >= kept) continue;
                    if (i >= answer)
                        atomicAdd(&counts[at], 1u);
                    else
                        atomicOr(&counts[at], kSeen);
                }
                for (int i = b0 + tid; i < b1; i += kThreads) {
                    const int id = r.bias_id_dev[i];
                    const uint32_t t = (uint32_t)(id - first);
                    if (id < first || t >= (uint32_t)n || (i > b0 && r.bias_id_dev[i - 1] == id)) continue;
                    const uint32_t at = rank(t) - from;
                    if (at < kept) biases[at] = r.bias_value_dev[i];
                }
                __syncthreads();
            }
            auto ruled = [&](float v, uint32_t at) {
                const uint32_t c = counts[at];
                if (c) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                if (c & ~kSeen) v = __fsub_rn(__fsub_rn(v, __fmul_rn((float)(c & ~kSeen), freq)), pres);
                return __fadd_rn(v, biases[at]);
            };
            auto allowed = [&](int i) { return !mask || (mask[i >> 5] >> (i & 31) & 1); };
            if (from > 0) {  // only the tokens of these ranks
                for (int w = tid; w < (n + 31) / 32; w += kThreads)
                    for (uint32_t bits = named[w]; bits; bits &= bits - 1) {
                        const uint32_t t = w * 32 + __ffs(bits) - 1, at = rank(t) - from;
                        if (at >= kept) continue;
                        const float v = allowed(first + t) ? ruled(Elt<T>::ld(in + first + t), at) : -INFINITY;
                        take(v > -INFINITY ? v : -INFINITY, v > -INFINITY ? first + t : 0x7fffffff);
                        if (out) Elt<T>::st(out + first + t, v);
                    }
                continue;
            }
            // value of token first + t; a named one of a later round stays as it is
            auto value = [&](float v, uint32_t t, bool is_named, bool ok) {
                bool later = false;
                if (is_named) {
                    const uint32_t at = rank(t);
                    later = at >= kept;
                    if (!later) v = ruled(v, at);
                }
                if (later) return v;
                if (!ok) v = -INFINITY;
                if (v > best) best = v, bi = first + t;  // a thread's indices ascend here, so its first maximum is kept
                return v;
            };
            auto piece = [&](const uint4& raw, int at, uint32_t ok) {
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
                float v[V];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (V == 8)
                        v[2 * j] = bflo(w[j]), v[2 * j + 1] = bfhi(w[j]);
                    else
                        v[j] = __uint_as_float(w[j]);
                }
                constexpr uint32_t kAll = (1u << V) - 1;
                const uint32_t flags = total ? named[at >> 5] >> (at & 31) & kAll : 0u;
                ok = ok >> (at & 31) & kAll;
                if (flags == 0 && ok == kAll) {
#pragma unroll
                    for (int j = 0; j < V; j++)
                        if (v[j] > best) best = v[j], bi = first + at + j;
                    if (out && (const void*)out != (const void*)in) *reinterpret_cast<uint4*>(out + first + at) = raw;
                    return;
                }
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = value(v[j], at + j, flags >> j & 1, ok >> j & 1);
                if (out) {
                    if constexpr (V == 8)
                        Elt<T>::st8(out + first + at, v);
                    else
                        Elt<T>::st4(out + first + at, v);
                }
            };
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int at = (tid + k * kThreads) * V;
                if (at < whole) piece(ahead[k], at, allow[k]);
            }
            for (int at = (tid + kAhead * kThreads) * V; at < whole; at += kThreads * V)
                piece(*reinterpret_cast<const uint4*>(in + first + at), at, mask ? mask[(first + at) >> 5] : ~0u);
            for (int t = whole + tid; t < n; t += kThreads) {
                const float v = value(Elt<T>::ld(in + first + t), t, total && (named[t >> 5] >> (t & 31) & 1), allowed(first + t));
                if (out) Elt<T>::st(out + first + t, v);
            }
        }
        if (total) __syncthreads();  // what names tokens has been read
    }
    if (!p.argmax) return;
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
    auto kernel = f32 ? logits_adjust_kernel<float> : logits_adjust_kernel<uint16_t>;
    B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kernel, dim3(rows * kBlocks), dim3(kThreads), 0, ctx->stream, p));
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

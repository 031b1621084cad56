// Rules on a step's logits, and the greedy choice under them, in one pass over the logits:
//   penalties for tokens that came before (repetition: prompt and answer; presence, frequency: the answer), biases, a grammar's mask.
//
// A token's value v, in f32, each step with one rounding:  seen before: v / r where v > 0, else v r;  n times in the answer: (v - n f) - p;
// with a bias: v + b;  not allowed: -inf.  The choice is made among these; written out they are rounded to the logits' type.
//
// Bound by the bytes of the logits for many rows and by the latency of its phases for few.  A cluster of blocks takes a row, each
// block its share of the vocabulary.  A block reads the row's whole history and biases (from L2, but for the first block) and marks what
// falls into its share: a bit per token that a rule names.  The pass over the logits leaves these out; they are listed, counted by their
// rank among the bits, and dealt out to the threads one by one, so that a history's favourites, which lie close together in a vocabulary,
// hold no warp up.  Shared memory does not grow with the vocabulary that way, and several blocks fit an SM, one's phases behind another's
// loads.  The first logits, mask words and tokens of the history are on their way before the first phase.  Counters are integers, so the
// order of the atomics changes nothing.
#include <algorithm>

#include "elt.cuh"
#include "kernels.h"

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxSlice = 40960;        // tokens of a block at a time
constexpr int kWords = kMaxSlice / 32;
constexpr int kNamed = 2048;            // named tokens that are listed at a time
constexpr uint32_t kSeen = 0x80000000u;

__device__ __forceinline__ uint32_t at_block(uint32_t addr, uint32_t block) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(block));
    return r;
}
// Word j of a 16-byte piece of V logits with -inf in the place of those whose bit in `which` is set.
template <int V>
__device__ __forceinline__ uint32_t hide(uint32_t u, uint32_t which, int j) {
    if constexpr (V == 4) {
        return which >> j & 1 ? 0xff800000u : u;
    } else {
        const uint32_t m = which >> (2 * j) & 3, mask = ((m | m << 15) & 0x00010001u) * 0xffffu;
        return (u & ~mask) | (0xff80ff80u & mask);
    }
}
template <int V>
__device__ __forceinline__ float largest(const uint32_t (&u)[4]) {  // NaNs do not count
    if constexpr (V == 4) {
        return fmaxf(fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1])), fmaxf(__uint_as_float(u[2]), __uint_as_float(u[3])));
    } else {
        auto max2 = [](uint32_t a, uint32_t b) {
            uint32_t d;
            asm("max.bf16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
            return d;
        };
        const uint32_t m = max2(max2(u[0], u[1]), max2(u[2], u[3]));
        return fmaxf(bflo(m), bfhi(m));
    }
}

struct AdjustParams {
    b2_logit_rules r;
    const void* in;
    void* out;  // nullable; may be `in`
    int32_t* argmax;
    int64_t ld;
    int vocab, slice;  // tokens of a block in one round: a multiple of 32
};

// kAhead: 16-byte pieces of logits that a thread asks for together, and tokens of the history
template <typename T, int kBlocks, int kThreads, int kAhead, int kPerSm>
__global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads, kPerSm) logits_adjust_kernel(const AdjustParams p) {
    constexpr int V = 16 / sizeof(T);
    __shared__ uint32_t named[kWords];       // a bit per token of the slice
    __shared__ uint32_t rank_of[kWords];     // named tokens before a word's
    __shared__ uint16_t ids[kNamed];         // by rank: the token,
    __shared__ uint32_t counts[kNamed];      // kSeen and how often it is in the answer,
    __shared__ float biases[kNamed];         // its bias
    __shared__ uint32_t s_scan[kThreads / 32];
    __shared__ float sv[kThreads / 32], cv[kBlocks];
    __shared__ int si[kThreads / 32], ci[kBlocks];
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");  // (waited for before another block's shared memory is written)
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
#pragma unroll 1
    for (int base = 0; base < p.vocab; base += kBlocks * p.slice) {
        const int first = base + block * p.slice, n = max(0, min(p.slice, p.vocab - first));  // this block's tokens
        const int whole = vec ? n / V * V : 0;
        uint4 ahead[kAhead];
        uint32_t allow[kAhead];
        auto ask = [&](int from) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int at = (from + tid + k * kThreads) * V;
                if (at < whole) ahead[k] = *reinterpret_cast<const uint4*>(in + first + at);
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int at = (from + tid + k * kThreads) * V;
                allow[k] = mask && at < whole ? mask[(first + at) >> 5] : ~0u;  // (first is a multiple of 32)
            }
        };
        ask(0);
        // calls f(place of the token in the slice, index) for what this thread has of a list of ids
        int head[kAhead];  // the first of the history
#pragma unroll
        for (int k = 0; k < kAhead; k++) head[k] = h0 + tid + k * kThreads < h1 ? r.history_dev[h0 + tid + k * kThreads] : -1;
        auto in_slice = [&](int id, int i, auto f) {
            const uint32_t t = (uint32_t)(id - first);
            if (id >= first && t < (uint32_t)n) f(t, i);
        };
        auto each_seen = [&](auto f) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) in_slice(head[k], h0 + tid + k * kThreads, f);
#pragma unroll 1
            for (int i = h0 + tid + kAhead * kThreads; i < h1; i += 4 * kThreads) {
                int id[4];
#pragma unroll
                for (int k = 0; k < 4; k++) id[k] = i + k * kThreads < h1 ? r.history_dev[i + k * kThreads] : -1;
#pragma unroll
                for (int k = 0; k < 4; k++) in_slice(id[k], i + k * kThreads, f);
            }
        };
        auto each_bias = [&](auto f) {
#pragma unroll 1
            for (int i = b0 + tid; i < b1; i += kThreads) in_slice(r.bias_id_dev[i], i, f);
        };
        uint32_t total = 0;  // named tokens
        if (h1 > h0 || b1 > b0) {
#pragma unroll 1
            for (int i = tid; i < p.slice / 32; i += kThreads) named[i] = 0;
            __syncthreads();
            auto mark = [&](uint32_t t, int) {  // (a look first: atomics on one word wait for one another, and favourites come in crowds)
                if (!(named[t >> 5] >> (t & 31) & 1)) atomicOr(&named[t >> 5], 1u << (t & 31));
            };
            each_seen(mark);
            each_bias(mark);
            __syncthreads();
            // rank of every word's first bit: a thread has kMine words
            constexpr int kMine = (kWords + kThreads - 1) / kThreads;
            const int w = kMine * tid;
            uint32_t bits[kMine], mine = 0;
#pragma unroll
            for (int j = 0; j < kMine; j++) {
                bits[j] = w + j < p.slice / 32 ? __popc(named[w + j]) : 0;
                mine += bits[j];
            }
            uint32_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(kFull, incl, o);
                if (lane >= o) incl += v;
            }
            if (lane == 31) s_scan[tid >> 5] = incl;
            __syncthreads();
            uint32_t at = incl - mine;
#pragma unroll
            for (int i = 0; i < kThreads / 32; i++) {
                if (i < tid >> 5) at += s_scan[i];
                total += s_scan[i];
            }
#pragma unroll
            for (int j = 0; j < kMine; j++) {
                if (w + j < p.slice / 32) rank_of[w + j] = at;
                at += bits[j];
            }
        }
        // The others, as they are or -inf: and of a piece only its largest value, a few instructions for eight logits;
        // which of its tokens that is is looked up at the end.
        auto allowed = [&](int i) { return !mask || (mask[i >> 5] >> (i & 31) & 1); };
        float top = -INFINITY;
        int place = 0;  // its piece, which `keep` holds, or its token behind the pieces
        uint32_t keep[4] = {};
        auto piece = [&](const uint4& raw, int at, uint32_t ok) {
            uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
            constexpr uint32_t kAll = (1u << V) - 1;
            const uint32_t flags = total ? named[at >> 5] >> (at & 31) & kAll : 0u;
            ok = ok >> (at & 31) & kAll;
            if (out) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = hide<V>(u[j], ~(ok | flags), j);
                if ((const void*)out != (const void*)in || ok != kAll) *reinterpret_cast<uint4*>(out + first + at) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            const uint32_t bad = flags | (ok ^ kAll);
            if (bad) {
#pragma unroll
                for (int j = 0; j < 4; j++) u[j] = hide<V>(u[j], bad, j);
            }
            const float x = largest<V>(u);
            if (x > top) {  // a thread's places ascend, so its first maximum is kept
                top = x, place = at;
#pragma unroll
                for (int j = 0; j < 4; j++) keep[j] = u[j];
            }
        };
#pragma unroll 1
        for (int from = 0; from * V < whole; from += kAhead * kThreads) {
            if (from > 0) ask(from);
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int at = (from + tid + k * kThreads) * V;
                if (at < whole) piece(ahead[k], at, allow[k]);
            }
        }
#pragma unroll 1
        for (int t = whole + tid; t < n; t += kThreads) {
            if (total && (named[t >> 5] >> (t & 31) & 1)) continue;
            const float v = allowed(first + t) ? Elt<T>::ld(in + first + t) : -INFINITY;
            if (v > top) top = v, place = t;
            if (out) Elt<T>::st(out + first + t, v);
        }
        if (top > -INFINITY) {
            int found = first + place;
            if (place < whole) {
#pragma unroll
                for (int j = V - 1; j >= 0; j--) {
                    const uint32_t u = keep[j * 4 / V];
                    const float v = V == 4 ? __uint_as_float(u) : j & 1 ? bfhi(u) : bflo(u);
                    if (v == top) found = first + place + j;
                }
            }
            take(top, found);
        }
        // the named ones, kNamed at a time
#pragma unroll 1
        for (uint32_t from = 0; from < total; from += kNamed) {
            const uint32_t kept = min((uint32_t)kNamed, total - from);
#pragma unroll 1
            for (uint32_t i = tid; i < kept; i += kThreads) counts[i] = 0, biases[i] = 0.f;
            __syncthreads();
            auto rank = [&](uint32_t t) { return rank_of[t >> 5] + __popc(named[t >> 5] & ((1u << (t & 31)) - 1)) - from; };
            each_seen([&](uint32_t t, int i) {
                const uint32_t at = rank(t);
                if (at >= kept) return;
                ids[at] = (uint16_t)t;  // (whoever writes it writes the same)
                if (i >= answer)
                    atomicAdd(&counts[at], 1u);
                else
                    atomicOr(&counts[at], kSeen);
            });
            each_bias([&](uint32_t t, int i) {
                const uint32_t at = rank(t);
                if (at >= kept) return;
                ids[at] = (uint16_t)t;
                if (i == b0 || r.bias_id_dev[i - 1] != r.bias_id_dev[i]) biases[at] = r.bias_value_dev[i];
            });
            __syncthreads();
#pragma unroll 1
            for (uint32_t at = tid; at < kept; at += kThreads) {
                const int i = first + ids[at];
                float v = Elt<T>::ld(in + i);
                const uint32_t c = counts[at];
                if (c) v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                if (c & ~kSeen) v = __fsub_rn(__fsub_rn(v, __fmul_rn((float)(c & ~kSeen), freq)), pres);
                v = __fadd_rn(v, biases[at]);
                if (!allowed(i)) v = -INFINITY;
                if (v > -INFINITY) take(v, i);
                if (out) Elt<T>::st(out + i, v);
            }
            __syncthreads();  // lists and marks have been read
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) take(__shfl_xor_sync(kFull, best, o), __shfl_xor_sync(kFull, bi, o));
    if (lane == 0) sv[tid >> 5] = best, si[tid >> 5] = bi;
    asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    __syncthreads();
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
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    if (block != 0) return;  // (the first block's shared memory is the one that is written)
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    if (tid == 0 && p.argmax) {
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
    // Few rows: as many blocks, threads and loads as a row can use.  More: fewer blocks, each of which reads the history, so that all rows'
    // phases overlap.  More blocks than SMs hold at once: smaller ones, of which a last wave leaves less idle.  128256 tokens, bf16, 18 / 48 /
    // 256 rows: eight blocks 10.1 / 16.4 / 56 us, four of 512 threads 10.4 / 13.0 / 37.9, four of 256 12.3 / 14.8 / 34.1.
    const bool few = (int64_t)rows * 8 <= ctx->sm_count, many = (int64_t)rows * 4 > 3 * ctx->sm_count;
    const int blocks = few ? 8 : 4;
    p.slice = std::min(kMaxSlice, ((vocab + blocks - 1) / blocks + 31) / 32 * 32);
    auto kernel = f32 ? few ? logits_adjust_kernel<float, 8, 512, 4, 2> : many ? logits_adjust_kernel<float, 4, 256, 4, 4> : logits_adjust_kernel<float, 4, 512, 2, 3>
                  : few ? logits_adjust_kernel<uint16_t, 8, 512, 4, 2> : many ? logits_adjust_kernel<uint16_t, 4, 256, 4, 4> : logits_adjust_kernel<uint16_t, 4, 512, 2, 3>;
    B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kernel, dim3(rows * blocks), dim3(many ? 256 : 512), 0, ctx->stream, p));
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
    B2_REQUIRE(vocab <= 1 << 30, B2_ERR_UNSUPPORTED, "b2_logits_adjust: a vocabulary of more than 2^30 tokens");
    const uintptr_t size = f32 ? 4 : 2;
    B2_REQUIRE((uintptr_t)logits_dev % size == 0 && (uintptr_t)out_dev % size == 0, B2_ERR_UNSUPPORTED, "b2_logits_adjust: logits and out must be aligned to their elements");
    B2_CUDA(cudaSetDevice(ctx->device));
    return b2_logits_adjust_launch(ctx, *rules, logits_dev, f32 != 0, rows, vocab, ld, out_dev, argmax_dev);
}

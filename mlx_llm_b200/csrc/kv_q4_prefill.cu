// Attention over a 4-bit paged cache for any number of query tokens per sequence: prompts, portions of prompts, drafts.
//
// Few columns (query tokens x q heads of a group) go through kv_q4_attn.cu, which reads and converts the 4 bits once per 8 columns.  With
// many, the products decide, not the bytes: kv_q4_prefill_kernel (tcgen05) converts the codes of a tile of 128 keys into the bf16 operands
// that the tensor cores read from shared memory, once for 256 rows of queries.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "kv_q4.cuh"
#include "tc5.cuh"

namespace {

using namespace tc5;

// Which of the two, for all sequences of a call, by what they cost in records x blocks of 8 columns.  Both kernels at work on 64 sequences
// behind 2000 tokens, 4 q heads a kv head: 8 new tokens (~36 columns) 160 and 186 us, 16 new 300 and 189 us; so a tile of 128 keys counts
// like 41.  The second kernel has ~6 us more of start and end (64 tokens behind 100: 14 and 21 us), and two kernels, one after the other,
// cost the shorter one's latency (8 sequences of 4 to 12 new tokens behind 1500: 31 us with either kernel, 49 with both).
constexpr double kTileCost = 41, kStartCost = 8e3, kBothCost = 2e4;
constexpr int KT = 128;  // keys of a tile

// A tile of K or V: [HD / 64 halves][128 keys][64 dims] bf16, rows of 128 bytes whose 16-byte pieces are swapped as the 128-byte swizzle
// wants (piece ^ row % 8).  K is read from it as a K-major operand, V as an MN-major one.
template <int HD>
constexpr int tile_bytes() {
    return KT * HD * 2;
}
__device__ __forceinline__ uint32_t tile_at(int row, int dim) {  // of 8 dims
    return (uint32_t)(dim >> 6) * (KT * 128) + (uint32_t)row * 128u + ((((uint32_t)dim >> 3) & 7u) ^ ((uint32_t)row & 7u)) * 16u;
}

// CTA = (two blocks of query rows, kv head[, split of the keys]).  A row is a (query token, q head of the group) pair, the heads of a token
// next to one another, so that a group shares every tile of K and V, and the two blocks of 128 rows share them again.
//   warps 0-3, 4-7  softmax of block A, B: thread = row = TMEM lane.  exp2 against a running reference that is raised only when a tile exceeds
//                   it by more than 2^8 (O is touched only then); P goes as bf16 over the scores' columns.
//   warps 8-11      codes to operands: a warp has two of the eight records of a tile, reads the next tile's while it converts this one's, and
//                   fills a ring of five tiles K0 V0 K1 V1 ...  K keeps the order that nibbles come out in, 0 4 1 5 2 6 3 7 of eight dims, and Q is
//                   put in the same; both carry the conversion's 2^-64 (kv_q4.cuh), which the softmax scale and the division take back.
//   warp 12         one thread issues S = Q K^T and O += P V with P from tensor memory, for A and B in turn: while one block's softmax runs,
//                   the tensor cores have the other's products.  S(j + 1) of a block goes over P(j), which the in-order pipe has read by then;
//                   and when S(j) is there, P V of j - 1 has completed, so O may be rescaled.
// Bound by a block's chain of product, softmax, product (two thirds of it are the tensor cores').  Converting in here costs each CTA what an
// own kernel would do once per 128 keys, in warps that the chain leaves idle: 512 tokens behind 11800 that read bf16 tiles, made by such a
// kernel, from L2 took 210 us instead of 236, but 64 tokens behind 12000 took 60 instead of 45, and eight sequences of 16 behind 1500 took 47 instead of 33.
// A value that is NaN must reach the rows that see it and no others, but a row that does not still multiplies it, with zero: it goes into the
// token's keys, whose scores are masked by choice and not by multiplication, and the value becomes zero.
// P carries 8 bits (one rounding of each weight, relative 2^-9; their sum is taken before the rounding, whose errors have no sign of their
// own): a second product for the rest of P would cost half as much again.
constexpr int kRows = 128, kSlots = 5, kConvert = 8, kIssuer = 12, kThreads = 416;
constexpr float kRaise = 8.f, kFloor = -1e30f;
template <int HD>
struct Smem {
    static constexpr int kQ = 0, kRing = 2 * tile_bytes<HD>(), kBar = kRing + kSlots * tile_bytes<HD>(), kBytes = kBar + 256;
};
constexpr uint32_t kIdesc128 = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
template <int HD>
constexpr uint32_t idesc_pv() {  // N = HD, B MN-major
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

struct ProductParams {
    const uint16_t* q;
    const uint8_t* pool;
    int64_t n_pages;
    const int32_t* block_tables;
    int max_blocks, page_tiles;
    const int32_t *bt_row, *q_row, *q_len, *ctx;  // [seqs]
    const int32_t *work_seq, *work_q;             // [items] sequence, first query token
    int hq, hkv, group, per_block;                // query tokens of a block of rows
    float scale_log2;                             // times 2^64
    uint16_t* out;
    int splits;
    float* part_o;   // [item][kv head][split][256 rows][HD], unnormalised, times 2^-64
    float* part_ml;  // [item][kv head][split][256 rows][2]: reference (log2 domain), sum
    int* err;
};
struct Item {
    int seq, q0, queries, ctx, before, tiles, first_tile, n_tiles;
};
__device__ __forceinline__ Item item_of(const ProductParams& p, int item, int split) {
    Item w;
    w.seq = p.work_seq[item];
    w.q0 = p.work_q[item];
    w.queries = min(2 * p.per_block, p.q_len[w.seq] - w.q0);
    w.ctx = p.ctx[w.seq];
    w.before = w.ctx - p.q_len[w.seq];
    w.tiles = (w.before + w.q0 + w.queries - 1) / KT + 1;  // up to the last key that its last query sees
    const int per = (w.tiles + p.splits - 1) / p.splits;
    w.first_tile = split * per;
    w.n_tiles = min(per, w.tiles - w.first_tile);
    return w;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t two(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ uint64_t twice(float x) { return two(__float_as_uint(x), __float_as_uint(x)); }
__device__ __forceinline__ float low(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float high(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }

// What a lane has of two records' keys, or values: the words of tokens g and g + 8 (or of the pairs c and c + 4), their scales, and for keys
// the scales of the same tokens' values.  Nothing is decided by them before they are used, so that they may still be on their way.
template <int HD>
struct Words {
    static constexpr int kGroups = HD / 64;
    uint32_t w[2][2][HD / 32], sb[2][2][2], other[2][2][kGroups];
    int left[2];  // tokens of the records that belong to the context
};
template <int HD>
struct Source {  // the two records of a converting warp in a tile
    const uint8_t* rec[2];
    int left[2];
    __device__ __forceinline__ void find(const ProductParams& p, const Item& w, int kvh, int t, int warp) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = t * 8 + warp * 2 + i;
            left[i] = w.ctx - r * 16;
            rec[i] = p.pool;
            if (left[i] <= 0) continue;
            const int index = r / p.page_tiles, page = p.block_tables[(size_t)p.bt_row[w.seq] * p.max_blocks + index];
            if (page < 0 || page >= p.n_pages)
                left[i] = 0;  // nothing there: zeros
            else
                rec[i] += (((size_t)page * p.hkv + kvh) * p.page_tiles + r - index * p.page_tiles) * q4::Record<HD>::kBytes;
        }
    }
    __device__ __forceinline__ void read(Words<HD>& x, bool values, int lane) const {
        using Rec = q4::Record<HD>;
        const int g = lane >> 2, c = lane & 3;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            x.left[i] = left[i];
            if (left[i] <= 0) continue;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t* at = rec[i] + (values ? Rec::kV : 0) + h * 4 * HD;
                if constexpr (HD == 128) {
                    const uint4 v = reinterpret_cast<const uint4*>(at)[lane];
                    x.w[i][h][0] = v.x, x.w[i][h][1] = v.y, x.w[i][h][2] = v.z, x.w[i][h][3] = v.w;
                } else {
                    const uint2 v = reinterpret_cast<const uint2*>(at)[lane];
                    x.w[i][h][0] = v.x, x.w[i][h][1] = v.y;
                }
                if (values) {  // tokens 8 h + 2 c and the next
                    const uint2 sb = *reinterpret_cast<const uint2*>(rec[i] + Rec::kVsb + ((g * (HD / 8) / 64) * 16 + 8 * h + 2 * c) * 4);
                    x.sb[i][h][0] = sb.x, x.sb[i][h][1] = sb.y;
                } else {  // token 8 h + g
                    x.sb[i][h][0] = reinterpret_cast<const uint32_t*>(rec[i] + Rec::kKsb)[(c * (HD / 4) / 64) * 16 + 8 * h + g];
#pragma unroll
                    for (int k = 0; k < Rec::kGroups; k++) x.other[i][h][k] = reinterpret_cast<const uint32_t*>(rec[i] + Rec::kVsb)[k * 16 + 8 * h + g];
                }
            }
        }
    }
};
template <int HD>
__device__ __forceinline__ void put_keys(uint8_t* tile, int row0, const Words<HD>& x, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint32_t sb = x.sb[i][h][0];
#pragma unroll
            for (int k = 0; k < Words<HD>::kGroups; k++)
                if (q4::poisoned(x.other[i][h][k])) sb = 0x7fc07fc0u;
            const bool real = 8 * h + g < x.left[i];
            const q4::Scales q = q4::scales_twice(real ? sb : 0u);
#pragma unroll
            for (int k = 0; k < HD / 32; k++) {
                // (at head size 128 lanes c and c + 2 have pieces that the swizzle puts into the same banks: the latter take another one first)
                const int w = HD == 128 ? k ^ (c & 2) : k;
                const uint32_t word = HD == 128 && (c & 2) ? x.w[i][h][k ^ (HD / 64)] : x.w[i][h][k];
                uint32_t v[4];
                q4::values(real ? word : 0u, q, v);
                *reinterpret_cast<uint4*>(tile + tile_at(row0 + 16 * i + 8 * h + g, c * (HD / 4) + 8 * w)) = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
}
template <int HD>
__device__ __forceinline__ void put_values(uint8_t* tile, int row0, const Words<HD>& x, int lane) {
    const int g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int t = 8 * h + 2 * c;
            const uint32_t sb0 = t >= x.left[i] || q4::poisoned(x.sb[i][h][0]) ? 0u : x.sb[i][h][0];
            const uint32_t sb1 = t + 1 >= x.left[i] || q4::poisoned(x.sb[i][h][1]) ? 0u : x.sb[i][h][1];
            const q4::Scales q = q4::scales_pair(sb0, sb1);
            const int row = row0 + 16 * i + t;
#pragma unroll
            for (int k = 0; k < HD / 32; k += 2) {
                const bool other = HD == 128 && (g & 1);  // (as above, lanes g and g + 1)
                const int w = other ? k ^ 2 : k;
                uint32_t a[4], b[4];
                q4::values(other ? x.w[i][h][(k ^ 2) % (HD / 32)] : x.w[i][h][k], q, a);  // dim i of both tokens
                q4::values(other ? x.w[i][h][(k ^ 2) % (HD / 32) + 1] : x.w[i][h][k + 1], q, b);
                const int d = g * (HD / 8) + 4 * w;
                *reinterpret_cast<uint4*>(tile + tile_at(row, d)) =
                    make_uint4(prmt(a[0], a[1], 0x5410u), prmt(a[2], a[3], 0x5410u), prmt(b[0], b[1], 0x5410u), prmt(b[2], b[3], 0x5410u));
                *reinterpret_cast<uint4*>(tile + tile_at(row + 1, d)) =
                    make_uint4(prmt(a[0], a[1], 0x7632u), prmt(a[2], a[3], 0x7632u), prmt(b[0], b[1], 0x7632u), prmt(b[2], b[3], 0x7632u));
            }
        }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) kv_q4_prefill_kernel(const ProductParams p) {
    using S = Smem<HD>;
    constexpr int TILE = tile_bytes<HD>(), HALF = KT * 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    pdl_wait();
    const uint32_t base = smem_u32(smem);
    if (base & 1023u) {  // the swizzled tiles need this alignment; every thread sees the same value
        if (threadIdx.x == 0) atomicExch(p.err, 7);
        return;
    }
    const int kvh = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Item w = item_of(p, blockIdx.y, blockIdx.z);
    if (w.n_tiles <= 0) return;  // (the merge leaves such splits out)
    const uint32_t bar = base + S::kBar;
    const uint32_t q_full = bar;
    auto full = [&](int s) { return bar + 8u * (1 + s); };
    auto empty = [&](int s) { return bar + 8u * (6 + s); };
    auto s_ready = [&](int x) { return bar + 8u * (11 + x); };
    auto p_ready = [&](int x) { return bar + 8u * (13 + x); };
    const uint32_t o_ready = bar + 8u * 15, slot_addr = bar + 8u * 16;
    if (tid == 0) {
        mbar_init(q_full, 8);
        for (int s = 0; s < kSlots; s++) mbar_init(full(s), 4), mbar_init(empty(s), 1);
        for (int x = 0; x < 2; x++) mbar_init(s_ready(x), 1), mbar_init(p_ready(x), 4);
        mbar_init(o_ready, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(slot_addr), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + (slot_addr - base));
    const int n = w.n_tiles;
    bool alive = true;

    if (warp >= kConvert && warp < kIssuer) {
        const int row0 = (warp - kConvert) * 32;
        Source<HD> from;
        Words<HD> keys, vals;
        from.find(p, w, kvh, w.first_tile, warp - kConvert);
        from.read(keys, false, lane);
        from.read(vals, true, lane);
        int slot = 0;
        uint32_t parity = 0;  // of the slot's present use
        auto fill = [&](auto put) {
            alive = __all_sync(0xffffffffu, mbar_wait(empty(slot), parity ^ 1u));
            if (!alive) return;
            put(smem + S::kRing + slot * TILE);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full(slot));
            if (++slot == kSlots) slot = 0, parity ^= 1u;
        };
        for (int j = 0; j < n && alive; j++) {
            if (j + 1 < n) from.find(p, w, kvh, w.first_tile + j + 1, warp - kConvert);
            fill([&](uint8_t* tile) { put_keys<HD>(tile, row0, keys, lane); });
            if (!alive) break;
            if (j + 1 < n) from.read(keys, false, lane);
            fill([&](uint8_t* tile) { put_values<HD>(tile, row0, vals, lane); });
            if (j + 1 < n) from.read(vals, true, lane);
        }
        if (!alive && lane == 0) atomicExch(p.err, 2);
    } else if (warp == kIssuer) {
        if (lane == 0) {
            // This thread's instructions per step set how soon the next products are queued, so descriptors are made once: the address is
            // the low word's (no carry leaves it), and all offsets but the ring's slot are constants.
            const uint64_t dq = desc_kmajor(base + S::kQ), dk = desc_kmajor(base + S::kRing), dv = desc_mnmajor(base + S::kRing, HALF);
            const uint32_t q_lo = (uint32_t)dq, k_lo = (uint32_t)dk, v_lo = (uint32_t)dv, k_hi = (uint32_t)(dk >> 32), v_hi = (uint32_t)(dv >> 32);
            auto issue_s = [&](int x, int slot) {  // S of block x
                const uint32_t at = k_lo + slot * (TILE >> 4);
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t off = ((k >> 2) * HALF + (k & 3) * 32) >> 4;
                    tc_mma(tmem + x * 128u, two(q_lo + x * (TILE >> 4) + off, k_hi), two(at + off, k_hi), kIdesc128, k > 0 ? 1u : 0u);
                }
                tc_commit(s_ready(x));
            };
            auto issue_o = [&](int x, int slot, uint32_t add) {  // O of block x
                const uint32_t at = v_lo + slot * (TILE >> 4);
#pragma unroll
                for (int k = 0; k < KT / 16; k++)
                    tc_mma_ts(tmem + 256u + x * 128u, tmem + x * 128u + k * 8u, two(at + k * (2048 >> 4), v_hi), idesc_pv<HD>(), k > 0 ? 1u : add);
            };
            int slot = 0;
            uint32_t parity = 0;
            auto advance = [&] {  // along the ring: K0 V0 K1 V1 ...
                if (++slot == kSlots) slot = 0, parity ^= 1u;
            };
            alive = mbar_wait(q_full, 0) && mbar_wait(full(0), 0);
            if (alive) {
                tc_fence_after();
                issue_s(0, 0);
                issue_s(1, 0);
                tc_commit(empty(0));
                advance();
            }
            for (int j = 0; j < n && alive; j++) {
                const int v = slot;
                alive = mbar_wait(full(v), parity) && mbar_wait(p_ready(0), (uint32_t)j & 1u);
                if (!alive) break;
                tc_fence_after();
                issue_o(0, v, j > 0);
                advance();
                const int k = slot;
                if (j + 1 < n) {
                    alive = mbar_wait(full(k), parity);
                    if (!alive) break;
                    tc_fence_after();
                    issue_s(0, k);
                }
                alive = mbar_wait(p_ready(1), (uint32_t)j & 1u);
                if (!alive) break;
                tc_fence_after();
                issue_o(1, v, j > 0);
                tc_commit(empty(v));
                if (j + 1 < n) {
                    issue_s(1, k);
                    tc_commit(empty(k));
                    advance();
                }
            }
            tc_commit(o_ready);  // (also after a wait that ran out: what is under way ends before the block does)
            if (!alive) {
                atomicExch(p.err, 3);
                mbar_wait(o_ready, 0);
            }
        }
        __syncwarp();
    } else {
        const int x = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int query = x * p.per_block + r / p.group, head = kvh * p.group + r % p.group;  // query: of the item
        const bool row_ok = r < p.per_block * p.group && query < w.queries;
        const size_t row = (size_t)(p.q_row[w.seq] + w.q0 + (row_ok ? query : 0)) * p.hq + head % p.hq;
        {  // this thread's row of Q
            const uint4* src = reinterpret_cast<const uint4*>(p.q + row * HD);
            uint8_t* dst = smem + S::kQ + x * TILE;
            uint4 v[HD / 8];
#pragma unroll
            for (int i = 0; i < HD / 8; i++) v[i] = row_ok ? src[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < HD / 8; i++)
                *reinterpret_cast<uint4*>(dst + tile_at(r, 8 * i)) =
                    make_uint4(prmt(v[i].x, v[i].z, 0x5410u), prmt(v[i].x, v[i].z, 0x7632u), prmt(v[i].y, v[i].w, 0x5410u), prmt(v[i].y, v[i].w, 0x7632u));
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        // last key that the row sees; rows without a query see all (nothing comes of them)
        const int sees = row_ok ? w.before + w.q0 + query : 0x3fffffff;
        const uint32_t ts = tmem + lanes + x * 128u, to = tmem + lanes + 256u + x * 128u;
        float m = kFloor, l = 0.f;
        for (int j = 0; j < n; j++) {
            if (!__all_sync(0xffffffffu, mbar_wait(s_ready(x), (uint32_t)j & 1u))) {
                alive = false;
                break;
            }
            tc_fence_after();
            // The upper 64 scores are read for the maximum and, once the lower ones have become P, again: a thread has 128 registers.
            const int key0 = (w.first_tile + j) * KT;
            const bool masked = key0 + KT - 1 > sees;
            uint32_t s[2][32];
            auto read = [&](int half) {
#pragma unroll
                for (int c = 0; c < 2; c++) tc_ld32_nowait(ts + half * 64u + c * 32u, s[c]);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 64; i++)
                        if (key0 + half * 64 + i > sees) s[i >> 5][i & 31] = 0xff800000u;
                }
            };
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int half = 1; half >= 0; half--) {
                read(half);
#pragma unroll
                for (int i = 0; i < 32; i += 4)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        mx[c] = max3(mx[c], __uint_as_float(s[c >> 1][i + 2 * (c & 1)]), __uint_as_float(s[c >> 1][i + 2 * (c & 1) + 1]));
            }
            const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.scale_log2;  // (the scale is positive)
            float alpha = 1.f;
            if (j == 0) {
                m = top < kFloor ? kFloor : top;
            } else if (!(top <= m + kRaise)) {  // (a NaN too, which makes all of the row NaN)
                alpha = fast_exp2(m - top);
                m = top;
            }
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                l *= alpha;
#pragma unroll 1
                for (int c = 0; c < HD / 32; c++) {
                    uint32_t v[32];
                    tc_ld32(to + c * 32u, v);
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                    tc_st32(to + c * 32u, v);
                }
            }
            const uint64_t sc = twice(p.scale_log2), neg = twice(-m);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (half == 1) read(1);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t h[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const uint64_t e = fma2(two(s[c][2 * i], s[c][2 * i + 1]), sc, neg);
                        const float a = fast_exp2(low(e)), b = fast_exp2(high(e));
                        sum[i & 1] = add2(sum[i & 1], two(__float_as_uint(a), __float_as_uint(b)));
                        h[i] = pack_bf2(a, b);
                    }
                    tc_st16_nowait(ts + (half * 2 + c) * 16u, h);
                }
            }
            const uint64_t both = add2(sum[0], sum[1]);
            l += low(both) + high(both);
            asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_ready(x));
        }
        if (alive && !__all_sync(0xffffffffu, mbar_wait(o_ready, 0))) alive = false;
        if (alive) {
            tc_fence_after();
            const bool part = p.splits > 1;
            const float inv = l == 0.f ? 0.f : q4::kUnscale / l;
            const size_t at = (((size_t)blockIdx.y * p.hkv + kvh) * p.splits + blockIdx.z) * (2 * kRows) + x * kRows + r;
#pragma unroll 1
            for (int c = 0; c < HD / 32; c++) {
                uint32_t v[32];
                tc_ld32(to + c * 32u, v);
                if (!row_ok) continue;
                if (part) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        reinterpret_cast<uint4*>(p.part_o + at * HD + c * 32)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                } else {
                    uint32_t h[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) h[i] = pack_bf2(__uint_as_float(v[2 * i]) * inv, __uint_as_float(v[2 * i + 1]) * inv);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        reinterpret_cast<uint4*>(p.out + row * HD + c * 32)[i] = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
                }
            }
            if (part && row_ok) p.part_ml[2 * at] = m, p.part_ml[2 * at + 1] = l;
        } else if (lane == 0) {
            atomicExch(p.err, 4);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

// Sum of the splits of an item, in their order: a warp per row, HD / 32 dims a lane.
template <int HD>
__global__ void __launch_bounds__(256) kv_q4_prefill_merge_kernel(const ProductParams p) {
    constexpr int D = HD / 32;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    pdl_wait();
    const int kvh = blockIdx.x, item = blockIdx.y, lane = threadIdx.x & 31;
    const int r = blockIdx.z * 8 + (threadIdx.x >> 5);  // row of the item
    const Item w = item_of(p, item, 0);
    const int in_block = r & (kRows - 1), query = (r / kRows) * p.per_block + in_block / p.group;
    if (in_block >= p.per_block * p.group || query >= w.queries) return;
    const int per = (w.tiles + p.splits - 1) / p.splits, used = (w.tiles + per - 1) / per;  // splits that had tiles
    const size_t at = (((size_t)item * p.hkv + kvh) * p.splits) * (2 * kRows) + r;
    float m = kFloor;
    for (int z = 0; z < used; z++) m = fmaxf(m, p.part_ml[2 * (at + (size_t)z * 2 * kRows)]);
    float l = 0.f, o[D] = {};
    for (int z = 0; z < used; z++) {
        const size_t s = at + (size_t)z * 2 * kRows;
        const float f = fast_exp2(p.part_ml[2 * s] - m);
        l += f * p.part_ml[2 * s + 1];
#pragma unroll
        for (int i = 0; i < D; i += 2) {
            const float2 v = *reinterpret_cast<const float2*>(p.part_o + s * HD + lane * D + i);
            o[i] += f * v.x, o[i + 1] += f * v.y;
        }
    }
    const float inv = l == 0.f ? 0.f : q4::kUnscale / l;
    uint16_t* dst = p.out + ((size_t)(p.q_row[w.seq] + w.q0 + query) * p.hq + (size_t)kvh * p.group + in_block % p.group) * HD + lane * D;
#pragma unroll
    for (int i = 0; i < D; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf2(o[i] * inv, o[i + 1] * inv);
}

}  // namespace

int32_t b2_kv_q4_plan(b2_ctx* ctx, const std::vector<Q4Seq>& seqs, int hq, int hkv, int head_dim, Q4Plan& plan) {
    (void)head_dim;
    plan = Q4Plan{};
    const int group = hq / hkv, step = 2 * (kRows / group);  // query tokens of an item
    auto few_cost = [&](const Q4Seq& s) { return (double)((s.ctx + 15) / 16) * hkv * (((int64_t)s.q_len * group + 7) / 8); };
    auto many_cost = [&](const Q4Seq& s) {
        return group > kRows ? INFINITY : kTileCost * ((s.ctx + KT - 1) / KT) * hkv * ((s.q_len + step - 1) / step);
    };
    double all_few = 0, all_many = kStartCost, each = kStartCost + kBothCost;
    for (const Q4Seq& s : seqs)
        if (s.q_len > 0) all_few += few_cost(s), all_many += many_cost(s), each += std::min(few_cost(s), many_cost(s));
    const bool by_few = all_few <= std::min(all_many, each), by_many = all_many <= each;
    std::vector<Q4Seq> few, many;
    for (const Q4Seq& s : seqs)
        if (s.q_len > 0) (by_few || (!by_many && few_cost(s) <= many_cost(s)) ? few : many).push_back(s);
    double line = 0;
    for (const Q4Seq& s : few) line += few_cost(s);
    B2_REQUIRE(line < 1073741824.0, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: more than 2^30 records in one call; make fewer sequences a call");
    plan.few = (int)few.size();
    for (const Q4Seq& s : few) plan.host.push_back(s.bt_row);
    for (const Q4Seq& s : few) plan.host.push_back(s.q_row);
    for (const Q4Seq& s : few) plan.host.push_back(s.q_len);
    for (const Q4Seq& s : few) plan.host.push_back(s.ctx);
    plan.many = (int)many.size();
    if (many.empty()) return B2_OK;
    plan.list = plan.host.size();
    for (const Q4Seq& s : many) plan.host.push_back(s.bt_row);
    for (const Q4Seq& s : many) plan.host.push_back(s.q_row);
    for (const Q4Seq& s : many) plan.host.push_back(s.q_len);
    for (const Q4Seq& s : many) plan.host.push_back(s.ctx);
    // the longest items first, so that the last ones to start are short
    struct Work {
        int32_t seq, q, tiles;
    };
    std::vector<Work> work;
    for (int i = 0; i < plan.many; i++)
        for (int q = 0; q < many[i].q_len; q += step)
            work.push_back({i, q, (many[i].ctx - many[i].q_len + std::min(q + step, many[i].q_len) - 1) / KT + 1});
    std::stable_sort(work.begin(), work.end(), [](const Work& a, const Work& b) { return a.tiles > b.tiles; });
    plan.work = (int)work.size();
    plan.longest = work[0].tiles;
    for (const Work& x : work) plan.host.push_back(x.seq);
    for (const Work& x : work) plan.host.push_back(x.q);
    return B2_OK;
}

template <int HD>
static int32_t launch_many(b2_ctx* ctx, const Q4PrefillParams& p, const Q4Plan& plan, const int32_t* plan_dev) {
    ProductParams a{};
    a.q = p.q;
    a.pool = p.pool;
    a.n_pages = p.n_pages;
    a.block_tables = p.block_tables;
    a.max_blocks = p.max_blocks;
    a.page_tiles = p.page_tiles;
    a.bt_row = plan_dev + plan.list;
    a.q_row = a.bt_row + plan.many;
    a.q_len = a.q_row + plan.many;
    a.ctx = a.q_len + plan.many;
    a.work_seq = a.ctx + plan.many;
    a.work_q = a.work_seq + plan.work;
    a.hq = p.hq;
    a.hkv = p.hkv;
    a.group = p.hq / p.hkv;
    a.per_block = kRows / a.group;
    a.scale_log2 = p.scale_log2 * q4::kUnscale;
    a.out = p.out;
    a.err = ctx->dev_err;
    // A CTA fills an SM.  Where the items leave half of the SMs idle, the keys are split as well, four tiles a split at least.
    const int ctas = plan.work * p.hkv;
    a.splits = ctas * 2 <= ctx->sm_count ? std::max(1, std::min({ctx->sm_count / ctas, plan.longest / 4, 16})) : 1;
    if (a.splits > 1) {
        const size_t slots = (size_t)ctas * a.splits * 2 * kRows, bytes = slots * (HD + 2) * sizeof(float);
        if (bytes > ctx->pf_part_bytes) {
            B2_CUDA(cudaStreamSynchronize(ctx->stream));
            if (ctx->pf_part) B2_CUDA(cudaFree(ctx->pf_part));
            ctx->pf_part = nullptr;
            ctx->pf_part_bytes = 0;
            B2_CUDA(cudaMalloc((void**)&ctx->pf_part, bytes + (bytes >> 2)));
            ctx->pf_part_bytes = bytes + (bytes >> 2);
        }
        a.part_o = ctx->pf_part;
        a.part_ml = ctx->pf_part + slots * HD;
    }
    B2_SMEM_ONCE(ctx, kv_q4_prefill_kernel<HD>, Smem<HD>::kBytes);
    B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kv_q4_prefill_kernel<HD>, dim3(p.hkv, plan.work, a.splits), dim3(kThreads), (size_t)Smem<HD>::kBytes, ctx->stream, a));
    B2_LAUNCHED(ctx);
    if (a.splits > 1) {
        B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kv_q4_prefill_merge_kernel<HD>, dim3(p.hkv, plan.work, 2 * kRows / 8), dim3(256), 0, ctx->stream, a));
        B2_LAUNCHED(ctx);
    }
    B2_CUDA(cudaGetLastError());
    return B2_OK;
}

int32_t b2_kv_q4_prefill_launch(b2_ctx* ctx, const Q4PrefillParams& p, int head_dim, const Q4Plan& plan, const int32_t* plan_dev) {
    if (plan.few > 0) {
        Q4AttnParams a{};
        a.q = p.q;
        a.pool = p.pool;
        a.n_pages = p.n_pages;
        a.block_tables = p.block_tables;
        a.max_blocks = p.max_blocks;
        a.bt_rows = plan_dev;
        a.q_rows = plan_dev + plan.few;
        a.q_lens = plan_dev + 2 * plan.few;
        a.ctx_lens = plan_dev + 3 * plan.few;
        a.num_seqs = plan.few;
        a.hq = p.hq;
        a.hkv = p.hkv;
        a.page_tiles = p.page_tiles;
        a.scale_log2 = p.scale_log2;
        a.out = p.out;
        B2_CHECK(b2_kv_q4_attn_launch(ctx, a, head_dim));
    }
    if (plan.many == 0) return B2_OK;
    B2_REQUIRE(plan.work <= 65535, B2_ERR_UNSUPPORTED, "attention over a 4-bit cache: too many query tokens for one call");
    return head_dim == 128 ? launch_many<128>(ctx, p, plan, plan_dev) : launch_many<64>(ctx, p, plan, plan_dev);
}

extern "C" int32_t b2_paged_attn_prefill_q4(b2_ctx* ctx, const uint16_t* q_dev, const uint8_t* kv_pool_dev, int32_t n_pages, const int32_t* block_tables_dev,
                                            int32_t max_blocks, const int32_t* cu_seqlens_host, const int32_t* ctx_lens_host, int32_t num_seqs, int32_t hq,
                                            int32_t hkv, int32_t head_dim, int32_t page_size, float scale, uint16_t* out_dev) {
    B2_REQUIRE(ctx && q_dev && kv_pool_dev && block_tables_dev && cu_seqlens_host && ctx_lens_host && out_dev, B2_ERR_MSG, "b2_paged_attn_prefill_q4: null argument");
    B2_CHECK(b2_kv_q4_check("b2_paged_attn_prefill_q4", kv_pool_dev, n_pages, hq, hkv, head_dim, page_size));
    B2_REQUIRE(num_seqs >= 0 && max_blocks > 0, B2_ERR_MSG, "b2_paged_attn_prefill_q4: bad sizes");
    B2_REQUIRE(scale > 0.f && scale < INFINITY, B2_ERR_MSG, "b2_paged_attn_prefill_q4: the scale must be positive");
    B2_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) == 0, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: q and out must be 16-byte aligned");
    if (num_seqs == 0) return B2_OK;
    std::vector<Q4Seq> seqs;
    for (int i = 0; i < num_seqs; i++) {
        const int n = cu_seqlens_host[i + 1] - cu_seqlens_host[i], ctx_len = ctx_lens_host[i];
        B2_REQUIRE(cu_seqlens_host[i] >= 0 && n >= 0 && ctx_len >= n, B2_ERR_MSG, "b2_paged_attn_prefill_q4: ctx_lens must include the new tokens, and cu_seqlens ascend");
        B2_REQUIRE(((int64_t)ctx_len + page_size - 1) / page_size <= max_blocks, B2_ERR_MSG,
                   "b2_paged_attn_prefill_q4: a context needs more blocks than a block-table row holds");
        seqs.push_back(Q4Seq{i, cu_seqlens_host[i], n, ctx_len});
    }
    B2_CUDA(cudaSetDevice(ctx->device));
    Q4Plan plan;
    B2_CHECK(b2_kv_q4_plan(ctx, seqs, hq, hkv, head_dim, plan));
    if (plan.host.empty()) return B2_OK;
    void* dev = nullptr;
    B2_CHECK(b2_ctx_stage(ctx, plan.host.size() * 4, &dev));
    // (pageable memory: the call returns when it has been read)
    B2_CUDA(cudaMemcpyAsync(dev, plan.host.data(), plan.host.size() * 4, cudaMemcpyHostToDevice, ctx->stream));
    Q4PrefillParams p{};
    p.q = q_dev;
    p.pool = kv_pool_dev;
    p.n_pages = n_pages;
    p.block_tables = block_tables_dev;
    p.max_blocks = max_blocks;
    p.hq = hq;
    p.hkv = hkv;
    p.page_tiles = page_size / 16;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.out = out_dev;
    return b2_kv_q4_prefill_launch(ctx, p, head_dim, plan, reinterpret_cast<const int32_t*>(dev));
}

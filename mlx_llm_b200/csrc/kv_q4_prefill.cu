// Attention over a 4-bit paged cache for any number of query tokens per sequence: prompts, portions of prompts, drafts.
//
// Few columns (query tokens x q heads of a group) go through kv_q4_attn.cu, which reads and converts the 4 bits once per 8 columns.  With
// many, the products decide, not the bytes: kv_q4_prefill_kernel (tcgen05) converts the codes of a tile of 128 keys into the bf16 operands
// that the tensor cores read from shared memory, once for 256 rows of queries.
#include <algorithm>
#include <cmath>
#include <functional>
#include <type_traits>

#include "kernels.h"
#include "kv_q4.cuh"
#include "tc5.cuh"

namespace {

using namespace tc5;

// Which of the two, for all sequences of a call, by what they cost in records x blocks of 8 columns.  Both kernels at work on 64 sequences
// behind 2000 tokens, 4 q heads a kv head: 8 new tokens (32 columns) 156 and 173 us, 16 new 292 and 175 us; so a tile of 128 keys counts
// like 41.  The second kernel has 5 to 8 us more of start and end (32 tokens behind 1500: 20.8 and 28.2 us; but 16 behind 12000 42.9 and
// 37.3), and two kernels, one after the other, cost the shorter one's latency (8 sequences of 4 to 12 new tokens behind 1500: 25 and 31 us,
// 48 with both; 31 of 4 and one of 512 behind 2000: 226, 122 and 101 with both).  The same rule serves head size 64, where both kernels save
// alike (64 of 8 behind 2000: 112 and 136 us, of 16 206 and 136, 32 behind 1500 17.6 and 23.1, 16 behind 12000 33.2 and 30.4).  Where it is
// off: short prompts with nothing before them, of which the second kernel takes only what the mask leaves (200 tokens: 22 us for 19).
constexpr double kTileCost = 41, kStartCost = 1.4e4, kBothCost = 2e4;
// In tiles (2.4 us): what a segment costs besides its tiles, what joining parts does, and the shortest run worth a CTA.
constexpr double kSegmentCost = 2, kJoinCost = 4, kShortRun = 4;
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

// A CTA fills an SM and goes through segments: two blocks of 128 query rows, a kv head, and tiles of their keys.  A row is a (query token,
// q head of the group) pair, the heads of a token next to one another, so that a group shares every tile of K and V, and the two blocks share
// them again.  The host, which knows all lengths, deals the segments out (b2_kv_q4_plan).  The warps that convert are at the next segment's
// keys, and the other block at its products, while a block writes its rows out: three prompts of ~1049 took 65 us (now 60), with a CTA for
// each segment 72.
//   warps 0-3, 4-7  softmax of block A, B: thread = row = TMEM lane.  exp2 against a running reference that is raised only when a tile exceeds
//                   it by more than 2^8 (O is touched only then); P goes as bf16 over the scores' columns.
//   warps 8-11      codes to operands: a warp has two of the eight records of a tile, reads the next tile's while it converts this one's, and
//                   fills a ring of five tiles K0 V0 K1 V1 ...  K keeps the order that nibbles come out in, 0 4 1 5 2 6 3 7 of eight dims, and Q is
//                   put in the same; both carry the conversion's 2^-64 (kv_q4.cuh), which the softmax scale and the division take back.
//   warp 12         one thread issues S = Q K^T and O += P V with P from tensor memory, for A and B in turn: while one block's softmax runs,
//                   the tensor cores have the other's products.  P comes by halves of the keys, and the first half's product runs beside the
//                   second half's exponentials.  S(j + 1) of a block goes over P(j), which the in-order pipe has read by then; and when S(j) is
//                   there, P V of j - 1 has completed, so O may be rescaled.
// Bound by a block's chain of product, softmax, product (two thirds of it are the tensor cores').  Converting in here costs each CTA what an
// own kernel would do once per 128 keys, in warps that the chain leaves idle: 512 tokens behind 11800 that read bf16 tiles, made by such a
// kernel, from L2 took 210 us where this took 236, but 64 tokens behind 12000 took 60 instead of 45, and eight sequences of 16 behind 1500 took 47
// instead of 33.  The three roles' code competes for the SM's instruction cache: loops that could be unrolled are not (512 behind 11800, each step
// timed on the same inputs again and again: masks in place 234 -> 228 us, exponentials 222, the maximum and P by halves 218; on new inputs each
// time 235 in the end), but for the issuing thread's, whose latency counts.
// A value that is NaN must reach the rows that see it and no others, but a row that does not still multiplies it, with zero: it goes into the
// token's keys, whose scores are masked by choice and not by multiplication, and the value becomes zero.
// P carries 8 bits (one rounding of each weight, 2^-8 of it at most; their sum is taken before the rounding, whose errors have no sign of their
// own).  A second product for the rest of P brings the error to that of the other kernels (512 behind 11800: 0.0023 to 0.0017 of the values'
// size, most of it the result's rounding) and takes a third more time (239 -> 315 us, three prompts 63 -> 77).
constexpr int kRows = 128, kSlots = 5, kConvert = 8, kIssuer = 12, kThreads = 416;
constexpr float kRaise = 8.f, kFloor = -3e38f;
template <int HD>
struct Smem {
    static constexpr int kQ = 0, kRing = 2 * tile_bytes<HD>(), kBar = kRing + kSlots * tile_bytes<HD>(), kBytes = kBar + 256;
    // Records of a tile that are not there, a bit each: a byte per converting warp, a word per tile, of the last four tiles.  (The ring has
    // room for K of tile t when P V of t - 3 is done, and with it all that the softmax reads of that tile.)
    static constexpr int kAbsent = kBar + 192;
};
constexpr uint32_t kIdesc128 = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
template <int HD>
constexpr uint32_t idesc_pv() {  // N = HD, B MN-major
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// What a CTA does at a time: 256 rows of queries of a kv head over some tiles of their keys.
struct alignas(16) Segment {
    int32_t bt_row, q_row, queries, ctx;        // q_row: of the first query token
    int32_t sees, kvh, first_tile, n_tiles;     // sees: the last key that the first query token sees
    int32_t part, unused[3];                    // where the sum goes that other segments complete, or -1: these are all tiles
};
struct alignas(16) Join {
    int32_t q_row, queries, kvh, first_part, parts, unused[3];
};
struct ProductParams {
    const uint16_t* q;
    const uint8_t* pool;
    int64_t n_pages;
    const int32_t* block_tables;
    int max_blocks, page_tiles;
    const Segment* segments;
    const int32_t* first_segment;  // [CTAs + 1]
    const Join* joins;
    int hq, hkv, group, per_block;  // query tokens of a block of rows
    float scale_log2;               // times 2^64
    uint16_t* out;
    float* part_o;   // [part][256 rows][HD], unnormalised, times 2^-64
    float* part_ml;  // [part][256 rows][2]: reference (log2 domain), sum
    int* err;
};
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
    __device__ __forceinline__ void find(const ProductParams& p, const Segment& w, int t, int warp) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = t * 8 + warp * 2 + i;
            left[i] = w.ctx - r * 16;
            rec[i] = p.pool;
            if (left[i] <= 0) continue;
            const int index = r / p.page_tiles, page = p.block_tables[(size_t)w.bt_row * p.max_blocks + index];
            if (page < 0 || page >= p.n_pages)
                left[i] = 0;  // nothing there: zeros, which the softmax leaves out
            else
                rec[i] += (((size_t)page * p.hkv + w.kvh) * p.page_tiles + r - index * p.page_tiles) * q4::Record<HD>::kBytes;
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
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int begin = p.first_segment[blockIdx.x], end = p.first_segment[blockIdx.x + 1];
    const uint32_t bar = base + S::kBar;
    auto full = [&](int s) { return bar + 8u * s; };
    auto empty = [&](int s) { return bar + 8u * (5 + s); };
    auto s_ready = [&](int x) { return bar + 8u * (10 + x); };
    auto p_ready = [&](int x, int half) { return bar + 8u * (12 + 2 * x + half); };
    auto q_full = [&](int x) { return bar + 8u * (16 + x); };   // once a segment: Q is there, and O of the last one has been read
    auto o_ready = [&](int x) { return bar + 8u * (18 + x); };  // once a segment
    const uint32_t gone = bar + 8u * 20, slot_addr = bar + 8u * 21;
    if (tid == 0) {
        for (int s = 0; s < kSlots; s++) mbar_init(full(s), 4), mbar_init(empty(s), 1);
        for (int x = 0; x < 2; x++) mbar_init(s_ready(x), 1), mbar_init(p_ready(x, 0), 4), mbar_init(p_ready(x, 1), 4), mbar_init(q_full(x), 4), mbar_init(o_ready(x), 1);
        mbar_init(gone, 1);
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
    bool alive = true;

    if (warp >= kConvert && warp < kIssuer) {
        const int row0 = (warp - kConvert) * 32;
        Source<HD> from;
        Words<HD> keys, vals;
        Segment w = p.segments[begin];
        int segment = begin, j = 0;
        auto next = [&] {  // the tile after this one; false if there is none
            if (++j == w.n_tiles) {
                if (++segment == end) return false;
                w = p.segments[segment], j = 0;
            }
            from.find(p, w, w.first_tile + j, warp - kConvert);
            return true;
        };
        from.find(p, w, w.first_tile, warp - kConvert);
        from.read(keys, false, lane);
        from.read(vals, true, lane);
        int slot = 0, tile = 0;
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
        for (bool more = true; more;) {
            more = next();
            fill([&](uint8_t* at) {
                put_keys<HD>(at, row0, keys, lane);
                if (lane == 0) smem[S::kAbsent + (tile & 3) * 4 + warp - kConvert] = (uint8_t)((keys.left[0] <= 0) | (keys.left[1] <= 0) << 1);
            });
            if (!alive) break;
            tile++;
            if (more) from.read(keys, false, lane);
            fill([&](uint8_t* at) { put_values<HD>(at, row0, vals, lane); });
            if (!alive) break;
            if (more) from.read(vals, true, lane);
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
            auto issue_o = [&](int x, int half, int slot, uint32_t add) {  // O of block x, by half of the keys
                const uint32_t at = v_lo + slot * (TILE >> 4);
#pragma unroll
                for (int i = 0; i < KT / 32; i++) {
                    const int k = half * (KT / 32) + i;
                    tc_mma_ts(tmem + 256u + x * 128u, tmem + x * 128u + k * 8u, two(at + k * (2048 >> 4), v_hi), idesc_pv<HD>(), k > 0 ? 1u : add);
                }
            };
            int slot = 0;
            uint32_t parity = 0;
            auto advance = [&] {  // along the ring: K0 V0 K1 V1 ...
                if (++slot == kSlots) slot = 0, parity ^= 1u;
            };
            uint32_t phase = 0, seg_phase = 0;  // of a tile's barriers, of a segment's
            for (int segment = begin; segment < end && alive; segment++, seg_phase ^= 1u) {
                const int n = p.segments[segment].n_tiles, first = slot;
                alive = mbar_wait(full(first), parity) && mbar_wait(q_full(0), seg_phase);
                if (!alive) break;
                tc_fence_after();
                issue_s(0, first);
                alive = mbar_wait(q_full(1), seg_phase);
                if (!alive) break;
                tc_fence_after();
                issue_s(1, first);
                tc_commit(empty(first));
                advance();
                for (int j = 0; j < n; j++, phase ^= 1u) {
                    const int v = slot;
                    alive = mbar_wait(full(v), parity) && mbar_wait(p_ready(0, 0), phase);
                    if (!alive) break;
                    tc_fence_after();
                    issue_o(0, 0, v, j > 0);
                    alive = mbar_wait(p_ready(0, 1), phase);
                    if (!alive) break;
                    tc_fence_after();
                    issue_o(0, 1, v, 1);
                    advance();
                    const int k = slot;
                    if (j + 1 < n) {
                        alive = mbar_wait(full(k), parity);
                        if (!alive) break;
                        tc_fence_after();
                        issue_s(0, k);
                    } else {
                        tc_commit(o_ready(0));
                    }
                    alive = mbar_wait(p_ready(1, 0), phase);
                    if (!alive) break;
                    tc_fence_after();
                    issue_o(1, 0, v, j > 0);
                    alive = mbar_wait(p_ready(1, 1), phase);
                    if (!alive) break;
                    tc_fence_after();
                    issue_o(1, 1, v, 1);
                    tc_commit(empty(v));
                    if (j + 1 < n) {
                        issue_s(1, k);
                        tc_commit(empty(k));
                        advance();
                    } else {
                        tc_commit(o_ready(1));
                    }
                }
            }
            if (!alive) {  // what is under way ends before the block does
                atomicExch(p.err, 3);
                tc_commit(gone);
                mbar_wait(gone, 0);
            }
        }
        __syncwarp();
    } else {
        const int x = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + x * 128u, to = tmem + lanes + 256u + x * 128u;
        const int query = x * p.per_block + r / p.group;  // of the segment's
        const bool in_block = r < p.per_block * p.group;
        auto row_of = [&](const Segment& w) { return ((size_t)(w.q_row + query) * p.hq + w.kvh * p.group + r % p.group) * HD; };
        auto copy_q = [&](const Segment& w) {  // this thread's row
            const bool ok = in_block && query < w.queries;
            const uint4* src = reinterpret_cast<const uint4*>(p.q + (ok ? row_of(w) : 0));
            uint8_t* dst = smem + S::kQ + x * TILE;
            uint4 v[HD / 8];
#pragma unroll
            for (int i = 0; i < HD / 8; i++) v[i] = ok ? src[i] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < HD / 8; i++)
                *reinterpret_cast<uint4*>(dst + tile_at(r, 8 * i)) =
                    make_uint4(prmt(v[i].x, v[i].z, 0x5410u), prmt(v[i].x, v[i].z, 0x7632u), prmt(v[i].y, v[i].w, 0x5410u), prmt(v[i].y, v[i].w, 0x7632u));
            fence_proxy_async();
        };
        auto q_there = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(x));
        };
        copy_q(p.segments[begin]);
        q_there();
        uint32_t phase = 0, seg_phase = 0, tile = 0;
        for (int segment = begin; segment < end; segment++, seg_phase ^= 1u) {
            // last key that the row sees; rows without a query see all (nothing comes of them)
            const Segment* const work = p.segments + segment;
            const int n = work->n_tiles, first_key = work->first_tile * KT, sees = in_block && query < work->queries ? work->sees + query : 0x3fffffff;
            float m = kFloor, l = 0.f;
            for (int j = 0; j < n; j++, tile++, phase ^= 1u) {
                if (!__all_sync(0xffffffffu, mbar_wait(s_ready(x), phase))) {
                    alive = false;
                    break;
                }
                tc_fence_after();
                // The upper 64 scores are read for the maximum and, once the lower ones have become P, again: a thread has 128 registers.
                const int key0 = first_key + j * KT;
                const uint32_t absent = *reinterpret_cast<volatile uint32_t*>(smem + S::kAbsent + (tile & 3) * 4);
                if (__any_sync(0xffffffffu, key0 + KT - 1 > sees || absent != 0)) {  // in place, so that the code for other tiles is without it
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t v[32];
                        tc_ld32(ts + c * 32u, v);
                        const int sees0 = absent >> (8 * c) & 1 ? -1 : sees, sees1 = absent >> (8 * c) & 2 ? -1 : sees;  // of two records
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (key0 + c * 32 + i > (i < 16 ? sees0 : sees1)) v[i] = 0xff800000u;
                        tc_st32(ts + c * 32u, v);
                    }
                }
                uint32_t s[2][32];
                auto read = [&](int half) {
#pragma unroll
                    for (int c = 0; c < 2; c++) tc_ld32_nowait(ts + half * 64u + c * 32u, s[c]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                };
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
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
#pragma unroll 1
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
                    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready(x, half));
                }
                const uint64_t both = add2(sum[0], sum[1]);
                l += low(both) + high(both);
            }
            if (!alive) break;
            if (segment + 1 < end) copy_q(work[1]);  // (all of this segment's scores are there, so its Q is not read any more)
            alive = __all_sync(0xffffffffu, mbar_wait(o_ready(x), seg_phase));
            if (!alive) break;
            tc_fence_after();
            const bool row_ok = in_block && query < work->queries;
            const size_t row = row_of(*work);
            const int part = work->part;
            const float inv = l == 0.f ? 0.f : q4::kUnscale / l;
            const size_t at = (size_t)part * (2 * kRows) + x * kRows + r;
#pragma unroll 1
            for (int c = 0; c < HD / 32; c++) {
                uint32_t o[32];
                tc_ld32(to + c * 32u, o);
                if (!row_ok) continue;
                if (part >= 0) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        reinterpret_cast<uint4*>(p.part_o + at * HD + c * 32)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                } else {
                    uint32_t h[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) h[i] = pack_bf2(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
                    for (int i = 0; i < 4; i++) reinterpret_cast<uint4*>(p.out + row + c * 32)[i] = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
                }
            }
            if (part >= 0 && row_ok) p.part_ml[2 * at] = m, p.part_ml[2 * at + 1] = l;
            if (segment + 1 < end) q_there();
        }
        if (!alive && lane == 0) atomicExch(p.err, 4);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

// Sum of the segments of a query's rows, in their order: a warp has four rows, HD / 32 dims a lane, and reads two segments of all four at
// once (most rows have two; 36 MB behind 512 tokens: one row and one segment at a time took 16 us).
constexpr int kJoinRows = 4;
template <int HD>
__global__ void __launch_bounds__(256) kv_q4_prefill_merge_kernel(const ProductParams p) {
    constexpr int D = HD / 32, N = kJoinRows;
    using Vec = std::conditional_t<HD == 128, float4, float2>;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    pdl_wait();
    const int lane = threadIdx.x & 31, row0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * N;
    const Join w = p.joins[blockIdx.x];
    const int last = p.per_block * p.group, end = (w.queries - (row0 >= kRows ? p.per_block : 0)) * p.group;  // rows of the block that there are
    const int in_block = row0 & (kRows - 1), rows = min(min(last, end) - in_block, N);
    if (rows <= 0) return;
    float m[N], l[N], o[N][D];
#pragma unroll
    for (int i = 0; i < N; i++) {
        m[i] = kFloor, l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < D; d++) o[i][d] = 0.f;
    }
    for (int z = 0; z < w.parts; z += 2) {
        float2 ml[2][N];
        union {
            Vec v;
            float f[D];
        } x[2][N];
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const size_t at = (size_t)(w.first_part + min(z + k, w.parts - 1)) * (2 * kRows) + row0 + min(i, rows - 1);
                ml[k][i] = reinterpret_cast<const float2*>(p.part_ml)[at];
                x[k][i].v = reinterpret_cast<const Vec*>(p.part_o + at * HD)[lane];
            }
        if (z + 1 == w.parts) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                ml[1][i] = make_float2(kFloor, 0.f);
#pragma unroll
                for (int d = 0; d < D; d++) x[1][i].f[d] = 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float top = fmaxf(m[i], ml[k][i].x), f = fast_exp2(m[i] - top), g = fast_exp2(ml[k][i].x - top);
                m[i] = top, l[i] = l[i] * f + ml[k][i].y * g;  // (a row that is NaN has a NaN sum)
#pragma unroll
                for (int d = 0; d < D; d++) o[i][d] = o[i][d] * f + x[k][i].f[d] * g;
            }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i >= rows) break;
        const float inv = l[i] == 0.f ? 0.f : q4::kUnscale / l[i];
        const int query = (row0 / kRows) * p.per_block + (in_block + i) / p.group;
        uint16_t* dst = p.out + ((size_t)(w.q_row + query) * p.hq + (size_t)w.kvh * p.group + (in_block + i) % p.group) * HD + lane * D;
#pragma unroll
        for (int d = 0; d < D; d += 2) *reinterpret_cast<uint32_t*>(dst + d) = pack_bf2(o[i][d] * inv, o[i][d + 1] * inv);
    }
}

}  // namespace

int32_t b2_kv_q4_plan(b2_ctx* ctx, const std::vector<Q4Seq>& seqs, int hq, int hkv, Q4Plan& plan) {
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
    for (const Q4Seq& s : few) line += few_cost(s), plan.few_columns = std::max(plan.few_columns, (int64_t)s.q_len * group);
    B2_REQUIRE(line < 1073741824.0, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: more than 2^30 records in one call; make fewer sequences a call");
    plan.few = (int)few.size();
    for (const Q4Seq& s : few) plan.host.push_back(s.bt_row);
    for (const Q4Seq& s : few) plan.host.push_back(s.q_row);
    for (const Q4Seq& s : few) plan.host.push_back(s.q_len);
    for (const Q4Seq& s : few) plan.host.push_back(s.ctx);
    if (many.empty()) return B2_OK;
    struct Work {
        int32_t seq, q, tiles;
    };
    std::vector<Work> work;
    for (int i = 0; i < (int)many.size(); i++)
        for (int q = 0; q < many[i].q_len; q += step)
            work.push_back({i, q, (many[i].ctx - many[i].q_len + std::min(q + step, many[i].q_len) - 1) / KT + 1});
    std::stable_sort(work.begin(), work.end(), [](const Work& a, const Work& b) { return a.tiles > b.tiles; });
    // Two ways to give a GPU's CTAs (one fills an SM) their segments.  Whole: every (item, kv head) in one segment, the longest first, each to
    // the CTA that has least.  Cut: all their tiles in one line, cut into runs that cost the same; what is cut is joined by another kernel.
    const double units = (double)work.size() * hkv;
    double tiles = 0;
    for (const Work& x : work) tiles += (double)x.tiles * hkv;
    std::vector<std::pair<double, int>> load;  // a heap with the least loaded CTA first
    const int whole_ctas = (int)std::min((double)ctx->sm_count, units);
    for (int i = 0; i < whole_ctas; i++) load.push_back({0, i});
    std::vector<int32_t> owner;
    double whole = 0;
    for (const Work& x : work)
        for (int h = 0; h < hkv; h++) {
            std::pop_heap(load.begin(), load.end(), std::greater<>());
            owner.push_back(load.back().second);
            whole = std::max(whole, load.back().first += x.tiles + kSegmentCost);
            std::push_heap(load.begin(), load.end(), std::greater<>());
        }
    const int cut_ctas = (int)std::max(1.0, std::min((double)ctx->sm_count, tiles / kShortRun));
    const double run = std::ceil((tiles + kSegmentCost * (units + cut_ctas)) / cut_ctas);
    std::vector<Segment> segments;
    std::vector<Join> joins;
    std::vector<int32_t> first;
    auto segment = [&](const Work& x, int h, int from, int n, int part) {
        const Q4Seq& s = many[x.seq];
        return Segment{s.bt_row, s.q_row + x.q, std::min(step, s.q_len - x.q), s.ctx, s.ctx - s.q_len + x.q, h, from, n, part, {}};
    };
    if (whole <= run + kJoinCost) {
        std::vector<int32_t> count(whole_ctas + 1, 0);
        for (int o : owner) count[o + 1]++;
        for (int i = 0; i < whole_ctas; i++) count[i + 1] += count[i];
        first = count;
        segments.resize(owner.size());
        size_t i = 0;
        for (const Work& x : work)
            for (int h = 0; h < hkv; h++) segments[count[owner[i++]]++] = segment(x, h, 0, x.tiles, -1);
    } else {
        double left = run;
        first.push_back(0);
        for (const Work& x : work)
            for (int h = 0; h < hkv; h++) {
                const int start = plan.parts;
                for (int t = 0; t < x.tiles;) {
                    const bool last = (int)first.size() >= cut_ctas;
                    if (!last && left < kSegmentCost + 1) first.push_back((int)segments.size()), left = run;
                    const int n = (int)first.size() >= cut_ctas ? x.tiles - t : std::min(x.tiles - t, (int)(left - kSegmentCost));
                    const bool all = n == x.tiles;
                    segments.push_back(segment(x, h, t, n, all ? -1 : plan.parts));
                    if (!all) plan.parts++;
                    t += n, left -= n + kSegmentCost;
                }
                if (plan.parts > start)
                    joins.push_back(Join{segments.back().q_row, segments.back().queries, h, start, plan.parts - start, {}});
            }
        first.push_back((int)segments.size());
    }
    plan.ctas = (int)first.size() - 1;
    plan.joins = (int)joins.size();
    while (plan.host.size() % 4) plan.host.push_back(0);
    auto add = [&](const void* x, size_t n) { plan.host.insert(plan.host.end(), (const int32_t*)x, (const int32_t*)x + n); };
    plan.segments = plan.host.size();
    add(segments.data(), segments.size() * (sizeof(Segment) / 4));
    plan.join_list = plan.host.size();
    add(joins.data(), joins.size() * (sizeof(Join) / 4));
    plan.first = plan.host.size();
    add(first.data(), first.size());
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
    a.segments = reinterpret_cast<const Segment*>(plan_dev + plan.segments);
    a.joins = reinterpret_cast<const Join*>(plan_dev + plan.join_list);
    a.first_segment = plan_dev + plan.first;
    a.hq = p.hq;
    a.hkv = p.hkv;
    a.group = p.hq / p.hkv;
    a.per_block = kRows / a.group;
    a.scale_log2 = p.scale_log2 * q4::kUnscale;
    a.out = p.out;
    a.err = ctx->dev_err;
    if (plan.parts > 0) {
        const size_t rows = (size_t)plan.parts * 2 * kRows, bytes = rows * (HD + 2) * sizeof(float);
        B2_CHECK(b2_ctx_grow(ctx, &ctx->pf_part, &ctx->pf_part_bytes, bytes));
        a.part_o = ctx->pf_part;
        a.part_ml = ctx->pf_part + rows * HD;
    }
    B2_SMEM_ONCE(ctx, kv_q4_prefill_kernel<HD>, Smem<HD>::kBytes);
    B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kv_q4_prefill_kernel<HD>, dim3(plan.ctas), dim3(kThreads), (size_t)Smem<HD>::kBytes, ctx->stream, a));
    B2_LAUNCHED(ctx);
    if (plan.joins > 0) {
        B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kv_q4_prefill_merge_kernel<HD>, dim3(plan.joins, 2 * kRows / (8 * kJoinRows)), dim3(256), 0, ctx->stream, a));
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
        a.columns = plan.few_columns;
        a.hq = p.hq;
        a.hkv = p.hkv;
        a.page_tiles = p.page_tiles;
        a.scale_log2 = p.scale_log2;
        a.out = p.out;
        B2_CHECK(b2_kv_q4_attn_launch(ctx, a, head_dim));
    }
    if (plan.ctas == 0) return B2_OK;
    return head_dim == 128 ? launch_many<128>(ctx, p, plan, plan_dev) : launch_many<64>(ctx, p, plan, plan_dev);
}

extern "C" int32_t b2_paged_attn_prefill_q4(b2_ctx* ctx, const uint16_t* q_dev, const uint8_t* kv_pool_dev, int32_t n_pages, const int32_t* block_tables_dev,
                                            int32_t max_blocks, const int32_t* cu_seqlens_host, const int32_t* ctx_lens_host, int32_t num_seqs, int32_t hq,
                                            int32_t hkv, int32_t head_dim, int32_t page_size, float scale, uint16_t* out_dev) {
    B2_REQUIRE(ctx && q_dev && kv_pool_dev && block_tables_dev && cu_seqlens_host && ctx_lens_host && out_dev, B2_ERR_MSG, "b2_paged_attn_prefill_q4: null argument");
    B2_CHECK(b2_kv_q4_check("b2_paged_attn_prefill_q4", kv_pool_dev, n_pages, hq, hkv, head_dim, page_size));
    B2_REQUIRE(num_seqs >= 0 && max_blocks > 0, B2_ERR_MSG, "b2_paged_attn_prefill_q4: bad sizes");
    B2_REQUIRE(scale > 0.f && scale < kQ4SoftmaxScaleEnd, B2_ERR_MSG, "b2_paged_attn_prefill_q4: the scale must be positive and below 2^62");
    B2_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) == 0, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: q and out must be 16-byte aligned");
    if (num_seqs == 0) return B2_OK;
    std::vector<Q4Seq> seqs;
    double segments = 0;  // of 256 rows, about: the plan's lists would outgrow the host's memory long before a GPU holds such queries
    for (int i = 0; i < num_seqs; i++) {
        const int64_t n = (int64_t)cu_seqlens_host[i + 1] - cu_seqlens_host[i];
        const int ctx_len = ctx_lens_host[i];
        B2_REQUIRE(cu_seqlens_host[i] >= 0 && n >= 0 && ctx_len >= n, B2_ERR_MSG, "b2_paged_attn_prefill_q4: ctx_lens must include the new tokens, and cu_seqlens ascend");
        B2_REQUIRE(((int64_t)ctx_len + page_size - 1) / page_size <= max_blocks, B2_ERR_MSG,
                   "b2_paged_attn_prefill_q4: a context needs more blocks than a block-table row holds");
        B2_REQUIRE(ctx_len <= 0x7fffff00, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: a context of more than 2^31 - 256 tokens");
        segments += std::ceil((double)n * (hq / hkv) / (2 * kRows)) * hkv;
        B2_REQUIRE(segments < 16777216.0, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: more than 2^24 x 256 queries of q heads; make fewer sequences a call");
        seqs.push_back(Q4Seq{i, cu_seqlens_host[i], (int32_t)n, ctx_len});
    }
    B2_CUDA(cudaSetDevice(ctx->device));
    Q4Plan plan;
    B2_CHECK(b2_kv_q4_plan(ctx, seqs, hq, hkv, plan));
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

// Attention over a 4-bit paged cache for few query tokens per sequence: single-token decode, and the short runs of tokens that a
// verification step checks.
//
// Byte streaming, 144 bytes per token and kv head (head size 128), that is bound by its instructions: 377 a record, with 64 % of the issue
// slots taken; 32 sequences of 8000 to 16000 tokens stream at 4.1 of the 6.5 TB/s that a copy reaches (109 us in a row of calls; 116
// with nothing in the caches, 3.8).
//
//   unit    = (sequence, kv head, block of 8 columns); a column is one (query token, q head of the group).  Its work is the sequence's
//             16-token records.
//   split   = all units' records form one line, which is cut into equal runs, one per warp: every warp streams the same number of
//             records whatever the lengths of the sequences, and no warp of a block waits for another before its run is done.  Short
//             units of much the same length have 1, 2, 4 or 8 warps of a block to themselves instead, and no blocks share one.
//             A unit inside one run is written out at once.  Runs that share a unit leave (maximum, sum, unnormalised output): first
//             in shared memory, where the block adds up its warps', then in global memory, where the block that arrives last adds up
//             the blocks', both in the order of the line, so that results do not depend on timing.
//   tensor  = mma.sync m16n8k16 with the record's 16 tokens on M and the columns on N: S^T = K Q^T, then O^T += V^T P^T.  Codes become
//             A operands in place (9 instructions for 8 codes, kv_q4.cuh); the order of dims inside a product is free, so Q is read in
//             the order that the nibbles come out.  P^T reaches the B layout with one movmatrix per 8 tokens; it is split into a bf16
//             head and remainder, so that P V keeps ~16 bits.  Where no unit has more than 4 columns (single tokens of groups of 4) the other
//             four carry the remainder: Q is there twice, P's lanes take one or the other, and one product does for two (HD / 16 fewer
//             a record; 64 sequences of 8192 150 -> 143 us).
//   softmax = in the log2 domain against a running reference that is raised only when a score exceeds it by more than 2^8.
#include <algorithm>

#include "kernels.h"
#include "kv_q4.cuh"

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 8;
constexpr int kStages = 4;             // records of a warp in shared memory: the two that it works on, the two that are on their way
constexpr float kFloor = -3e38f;     // reference of a column that has seen nothing: exp2(-inf - floor) is 0; scores down to it count
constexpr float kSlack = 8.f;
constexpr int kMinRun = 4;           // records of a run at least (one sequence of 4000: 18.0 us, 2 records 18.1, 8 records 20.3)
// Where units have warps to themselves: the records that the longest may have beyond an equal run, and the longest such run.  64 sequences
// of 16-128 tokens 10.9 us (equal runs: 19.0), of 128 11.1 (13.6), of 512 18.1 (21.1), of 1024 27.4 (29.0), of 2048 47.7 (47.0).
// Less of it where a unit would have a whole block, which is where warps are not short of units: 8 sequences of 1500 17.1 us (21.0 with 8),
// 32 of 50-1000 17.0 (18.1 with 3).
constexpr int kUnitSlack = 8, kBlockSlack = 4, kUnitRun = 20;
constexpr int kBlocksPerSm = 2;

template <int HD>
constexpr int part_floats() {
    return 8 * HD + 16;  // [8 columns][HD] outputs, 8 maxima, 8 sums
}
template <int HD>
constexpr int ring_bytes() {
    return kWarps * kStages * q4::Record<HD>::kBytes;
}
template <int HD>
constexpr int smem_bytes() {
    return ring_bytes<HD>() + kWarps * part_floats<HD>() * 4;
}

struct Lengths {  // of one sequence
    int ctx, tiles, columns, blocks;
};
__device__ __forceinline__ Lengths lengths_of(const Q4AttnParams& p, int seq) {
    Lengths l;
    l.ctx = min(max(p.ctx_lens[seq], 0), p.max_ctx);
    l.columns = p.q_lens ? p.q_lens[seq] * p.group : p.group;
    l.tiles = (l.ctx + 15) >> 4;
    l.blocks = l.tiles ? (l.columns + 7) >> 3 : 0;
    return l;
}
// A place on the line.
struct Cursor {
    int seq, kvh, block, tile;
    Lengths len;
    __device__ __forceinline__ void at_seq(const Q4AttnParams& p, int s) {  // the first sequence from s on that has work
        kvh = block = tile = 0;
        for (seq = s; seq < p.num_seqs; seq++) {
            len = lengths_of(p, seq);
            if (len.blocks > 0) return;
        }
    }
    __device__ __forceinline__ void at_unit(int unit) {
        kvh = unit / len.blocks;
        block = unit - kvh * len.blocks;
    }
    __device__ __forceinline__ void next_unit(const Q4AttnParams& p) {
        tile = 0;
        if (++block < len.blocks) return;
        block = 0;
        if (++kvh < p.hkv) return;
        at_seq(p, seq + 1);
    }
};
struct Part {  // what a run leaves of a unit that it shares with others
    int seq, kvh, block, start, tiles, first, last, cols;  // start: the unit's place on the line; records first .. last - 1 of its `tiles`
};

// W words of this lane
template <int W>
__device__ __forceinline__ void lane_words(const uint8_t* at, int lane, uint32_t (&w)[W]) {
    if constexpr (W == 4) {
        const uint4 v = reinterpret_cast<const uint4*>(at)[lane];
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
        const uint2 v = reinterpret_cast<const uint2*>(at)[lane];
        w[0] = v.x, w[1] = v.y;
    }
}
// S^T[token, column] of a record: tokens g and g + 8, columns 2c and 2c + 1
template <int HD>
__device__ __forceinline__ void scores(const uint8_t* rec, int lane, const uint32_t (&qf)[HD / 16][2], float to_log2, float (&s)[4]) {
    using Rec = q4::Record<HD>;
    constexpr int W = HD / 32;
    const int g = lane >> 2, c = lane & 3;
    const uint32_t* sb = reinterpret_cast<const uint32_t*>(rec + Rec::kKsb) + (c * (HD / 4) / 64) * 16 + g;
    const q4::Scales qa = q4::scales_twice(sb[0]), qb = q4::scales_twice(sb[8]);
    uint32_t ka[W], kb[W];
    lane_words<W>(rec, lane, ka);
    lane_words<W>(rec + 4 * HD, lane, kb);
    float s2[4] = {0.f, 0.f, 0.f, 0.f};
    s[0] = s[1] = s[2] = s[3] = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) {
        uint32_t va[4], vb[4];
        q4::values(ka[w], qa, va);
        q4::values(kb[w], qb, vb);
        const uint32_t a0[4] = {va[0], vb[0], va[1], vb[1]}, a1[4] = {va[2], vb[2], va[3], vb[3]};
        mma_bf16_16816(s, a0, qf[2 * w]);
        mma_bf16_16816(s2, a1, qf[2 * w + 1]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) s[j] = (s[j] + s2[j]) * to_log2;
}
// Where columns see different tokens: a value that is NaN must reach those that see it and no others, but the others multiply it too, with
// zero.  So it makes the token's scores NaN instead, which are masked by choice.
template <int HD>
__device__ __forceinline__ void hidden_values(const uint8_t* rec, int lane, float (&s)[4]) {
    using Rec = q4::Record<HD>;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < Rec::kGroups; i++)
            if (q4::poisoned(reinterpret_cast<const uint32_t*>(rec + Rec::kVsb)[i * 16 + (lane >> 2) + 8 * h])) s[2 * h] = s[2 * h + 1] = __int_as_float(0x7fc00000);
}
// O^T[dim, column] += V^T P^T of a record; rows g and g + 8 of tile mt are dims 2 mt and 2 mt + 1 of this lane's block.  `left`: tokens of
// the record that belong to the context; what lies behind them may be anything, and 0 * NaN is NaN.  `some`: not every column sees every
// token, so that values that are NaN have gone into the scores (hidden_values)
template <int HD, bool kNarrow>
__device__ __forceinline__ void add_values(const uint8_t* rec, int lane, const float (&p)[4], int left, bool some, float (&o)[HD / 16][4]) {
    using Rec = q4::Record<HD>;
    constexpr int W = HD / 32;
    const int g = lane >> 2, c = lane & 3;
    const uint32_t* vsb = reinterpret_cast<const uint32_t*>(rec + Rec::kVsb) + (g * (HD / 8) / 64) * 16 + 2 * c;
    uint2 sb0 = *reinterpret_cast<const uint2*>(vsb), sb1 = *reinterpret_cast<const uint2*>(vsb + 8);
    if (left < 16) {
        if (2 * c >= left) sb0.x = 0;
        if (2 * c + 1 >= left) sb0.y = 0;
        if (2 * c + 8 >= left) sb1.x = 0;
        if (2 * c + 9 >= left) sb1.y = 0;
    }
    if (some) {
        if (q4::poisoned(sb0.x)) sb0.x = 0;
        if (q4::poisoned(sb0.y)) sb0.y = 0;
        if (q4::poisoned(sb1.x)) sb1.x = 0;
        if (q4::poisoned(sb1.y)) sb1.y = 0;
    }
    uint32_t pb[2], pl[2];
    const uint32_t h01 = pack_bf2(p[0], p[1]), h23 = pack_bf2(p[2], p[3]);
    const uint32_t r01 = pack_bf2(p[0] - bflo(h01), p[1] - bfhi(h01)), r23 = pack_bf2(p[2] - bflo(h23), p[3] - bfhi(h23));
    if constexpr (kNarrow) {
        pb[0] = movmatrix_trans(c < 2 ? h01 : r01), pb[1] = movmatrix_trans(c < 2 ? h23 : r23);
    } else {
        pb[0] = movmatrix_trans(h01), pb[1] = movmatrix_trans(h23);
        pl[0] = movmatrix_trans(r01), pl[1] = movmatrix_trans(r23);
    }
    const q4::Scales qa = q4::scales_pair(sb0.x, sb0.y), qb = q4::scales_pair(sb1.x, sb1.y);
    uint32_t wa[W], wb[W];
    lane_words<W>(rec + Rec::kV, lane, wa);
    lane_words<W>(rec + Rec::kV + 4 * HD, lane, wb);
#pragma unroll
    for (int w = 0; w < W; w++) {
        uint32_t va[4], vb[4];
        q4::values(wa[w], qa, va);
        q4::values(wb[w], qb, vb);
        const uint32_t a0[4] = {va[0], va[1], vb[0], vb[1]}, a1[4] = {va[2], va[3], vb[2], vb[3]};
        mma_bf16_16816(o[2 * w], a0, pb);
        mma_bf16_16816(o[2 * w + 1], a1, pb);
        if constexpr (!kNarrow) {
            mma_bf16_16816(o[2 * w], a0, pl);
            mma_bf16_16816(o[2 * w + 1], a1, pl);
        }
    }
}

template <int HD, bool kNarrow>
__global__ void __launch_bounds__(kWarps * 32, kBlocksPerSm) kv_q4_attn_kernel(const Q4AttnParams p) {
    using Rec = q4::Record<HD>;
    constexpr int W = HD / 32;  // words of a lane per token (K) or token pair (V)
    constexpr int KS = HD / 16, MT = HD / 16;
    constexpr int kChunks = Rec::kBytes / 16;
    constexpr int kThreads = kWarps * 32, kParts = 2 * kWarps;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Part s_part[kParts];
    __shared__ int4 s_scan[kWarps];
    __shared__ int s_first[2][kThreads];  // records, units of the sequences before a thread's
    __shared__ float s_m[kParts][8], s_l[kParts][8], s_weight[kParts][8], s_sum[kParts][8], s_max[kParts][8];
    __shared__ int s_last[2];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int group = p.group;

    if (lane < 2) s_part[2 * warp + lane].tiles = 0;
    int run = 0, team_log2 = 0, team = 1, block_units = kWarps, block_start = 0, longest = 0, total = 0, units = 0;
    bool by_unit = false;
    int lo = 0, span = p.num_seqs, left = 0;  // sequences that hold the place where this warp's run begins, and the place among theirs
    auto add_up = [&](int from, int to, int& n, int& u, int& most, int& none) {  // records, units, the longest unit, an empty context
#pragma unroll 1
        for (int s = from; s < to; s++) {
            const Lengths l = lengths_of(p, s);
            u += l.blocks * p.hkv;
            n += l.tiles * l.blocks * p.hkv;
            most = max(most, l.tiles);
            none |= l.tiles == 0;
        }
    };
    auto scan = [&](int& n, int& u) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(kFull, n, o), b = __shfl_up_sync(kFull, u, o);
            if (lane >= o) n += a, u += b;
        }
    };
    auto deal = [&](bool none) {  // false: nothing for this block
        if (__builtin_expect(none, 0))  // an empty context attends to nothing: rows of zeros
#pragma unroll 1
            for (int s = blockIdx.x; s < p.num_seqs; s += gridDim.x) {
                if (lengths_of(p, s).tiles > 0) continue;
                const size_t row = p.q_rows ? p.q_rows[s] : s;
                const int count = (p.q_lens ? p.q_lens[s] : 1) * p.hq * HD;
#pragma unroll 1
                for (int e = threadIdx.x; e < count; e += kThreads) p.out[row * p.hq * HD + e] = 0;
            }
        // Units of much the same length, as many as there are warps or fewer: each has a team of warps of a block to itself, and no block
        // shares one with another.  Else equal runs.
        const int warps = (int)gridDim.x * kWarps;
        run = max(min(kMinRun, longest), (total + warps - 1) / warps);
        team_log2 = 3;
        static_assert(kWarps == 8, "a team is 1, 2, 4 or 8 of a block's warps");
#pragma unroll 1
        while (team_log2 > 0 && units > warps >> team_log2) team_log2--;
        team = 1 << team_log2, block_units = kWarps >> team_log2;
        by_unit = units <= warps >> team_log2 && run <= kUnitRun &&
                  (longest + team - 1) >> team_log2 <= run + (team == kWarps ? kBlockSlack : kUnitSlack);
        block_start = blockIdx.x * kWarps * run;
        left = by_unit ? min((int)blockIdx.x * block_units + (warp >> team_log2), units - 1) : min(block_start + warp * run, total - 1);
        return by_unit ? (int)blockIdx.x * block_units < units : block_start < total;
    };
    // With many sequences a block looks at all of them together, a thread at 1/256 (4096 sequences of 100: 160 us; each warp by itself 191) ...
    const bool many = p.num_seqs > kThreads;
    if (__builtin_expect(many, 0)) {
        const int per = (span + kThreads - 1) / kThreads;
        int n = 0, u = 0, most = 0, none = 0;
        add_up(threadIdx.x * per, min((int)(threadIdx.x + 1) * per, span), n, u, most, none);
        int ni = n, ui = u;
        scan(ni, ui);
        most = __reduce_max_sync(kFull, most);
        none = __any_sync(kFull, none);
        if (lane == 31) s_scan[warp] = make_int4(ni, ui, most, none);
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < kWarps; w++) {
            const int4 v = s_scan[w];
            if (w < warp) ni += v.x, ui += v.y;
            total += v.x, units += v.y, longest = max(longest, v.z), none |= v.w;
        }
        s_first[0][threadIdx.x] = ni - n, s_first[1][threadIdx.x] = ui - u;
        __syncthreads();
        if (!deal(none)) return;
        const int* first = s_first[by_unit];
        int at = 0;  // the last thread whose sequences begin at or before the place; of equal ones all but the last have nothing
#pragma unroll 1
        for (int step = kThreads / 2; step > 0; step >>= 1)
            if (first[at + step] <= left) at += step;
        left -= first[at];
        lo = at * per, span = min(per, span - lo);
    }
    // ... and else every warp finds its place by itself, without waiting for others: its lanes add up what 1/32 of the sequences have each, and
    // then the same of the lane that holds the place, until that is one sequence.
    for (bool all = !many;; all = false) {
        const int per = (span + 31) >> 5, from = lo + lane * per;
        int n = 0, u = 0, most = 0, none = 0;
        add_up(from, min(from + per, lo + span), n, u, most, none);
        int ni = n, ui = u;
        scan(ni, ui);
        if (all) {
            total = __shfl_sync(kFull, ni, 31), units = __shfl_sync(kFull, ui, 31), longest = __reduce_max_sync(kFull, most);
            if (!deal(__any_sync(kFull, none))) return;
        }
        const int size = by_unit ? u : n, before = (by_unit ? ui : ni) - size;
        const int owner = __ffs(__ballot_sync(kFull, left >= before && left - before < size)) - 1;
        left -= __shfl_sync(kFull, before, owner);
        lo += owner * per, span = min(per, span - owner * per);
        if (per == 1) break;
    }
    const uint32_t ring = smem_u32(smem) + warp * kStages * Rec::kBytes;
    float4* const parts = reinterpret_cast<float4*>(smem + ring_bytes<HD>());
    const float to_log2 = p.scale_log2 * q4::kUnscale;

    // row of the output that a unit's column belongs to
    auto out_row = [&](int seq, int kvh, int col) {
        const int query = col / group;
        const int row = (p.q_rows ? p.q_rows[seq] : seq) + query;
        return p.out + ((size_t)row * p.hq + (size_t)kvh * group + (col - query * group)) * HD;
    };

    Cursor use;
    int pos, end;
    {
        use.at_seq(p, lo);
        if (by_unit) {
            use.at_unit(left);
            const int each = (use.len.tiles + team - 1) >> team_log2, line = (warp >> team_log2) * longest;  // (a line for every unit of the block)
            use.tile = min((warp & (team - 1)) * each, use.len.tiles);
            pos = line + use.tile;
            end = (int)blockIdx.x * block_units + (warp >> team_log2) < units ? line + min(use.tile + each, use.len.tiles) : pos;
        } else {
            const int unit = left / use.len.tiles;
            use.tile = left - unit * use.len.tiles;
            use.at_unit(unit);
            pos = min(block_start + warp * run, total);
            end = min(pos + run, total);
        }
    }
    if (pos < end) {
        // The records of a run are looked up 32 at a time, a lane each, whatever units they belong to, and a window ahead: a look into the
        // block table is not waited for.
        const int begin = pos;
        int asked = pos, look_from = pos, look_seq = use.seq, look_at = (use.kvh * use.len.blocks + use.block) * use.len.tiles + use.tile;
        uint32_t absent = 0;  // bit s: the record of stage s lies on a page outside of the pool
        auto look = [&] {  // record number of place look_from + lane, -1 for none
            int seq = look_seq, at = look_at + lane, record = -1;  // `at`: in the line of the sequence
            if (look_from + lane < end) {
                Lengths l = lengths_of(p, seq);
                for (int all = l.tiles * l.blocks * p.hkv; at >= all; all = l.tiles * l.blocks * p.hkv) {
                    at -= all;
                    l = lengths_of(p, ++seq);
                }
                const int unit = at / l.tiles, tile = at - unit * l.tiles, index = tile / p.page_tiles;
                const int page = p.block_tables[(size_t)(p.bt_rows ? p.bt_rows[seq] : seq) * p.max_blocks + index];
                if (page >= 0 && page < p.n_pages) record = (page * p.hkv + unit / l.blocks) * p.page_tiles + tile - index * p.page_tiles;
            }
            look_seq = __shfl_sync(kFull, seq, 31), look_at = __shfl_sync(kFull, at, 31) + 1, look_from += 32;
            return record;
        };
        int record = look(), later = -1;
        auto ask_until = [&](int upto) {
            for (; asked < upto; asked++) {
                const int i = asked - begin, stage = i % kStages;
                if (i > 0 && i % 32 == 0) record = later;
                if (i % 32 == kStages && look_from < end) later = look();
                const int rec = __shfl_sync(kFull, record, i % 32);
                absent = (absent & ~(1u << stage)) | (rec < 0 ? 1u << stage : 0u);
                if (rec >= 0) {
                    const uint8_t* src = p.pool + (size_t)rec * Rec::kBytes + lane * 16;
                    const uint32_t dst = ring + stage * Rec::kBytes + lane * 16;
#pragma unroll
                    for (int k = 0; k < kChunks; k += 32)
                        if (k + 32 <= kChunks || k + lane < kChunks) cp_async16(dst + k * 16, src + k * 16);
                }
            }
            cp_async_commit();
        };
        uint32_t qf[KS][2];
        auto load_q = [&] {  // Q as the B operand, in the order of the nibbles; columns past the last are zeros
            const int cols = min(8, use.len.columns - use.block * 8), col = use.block * 8 + min(kNarrow ? g & 3 : g, cols - 1), query = col / group;
            const size_t row = (p.q_rows ? p.q_rows[use.seq] : use.seq) + query;
            const uint16_t* q = p.q + (row * p.hq + (size_t)use.kvh * group + (col - query * group)) * HD + c * (HD / 4);
#pragma unroll
            for (int w = 0; w < W; w++) {
                uint4 u = *reinterpret_cast<const uint4*>(q + 8 * w);
                if (!kNarrow && g >= cols) u = make_uint4(0, 0, 0, 0);
                qf[2 * w][0] = prmt(u.x, u.z, 0x5410u);
                qf[2 * w][1] = prmt(u.x, u.z, 0x7632u);
                qf[2 * w + 1][0] = prmt(u.y, u.w, 0x5410u);
                qf[2 * w + 1][1] = prmt(u.y, u.w, 0x7632u);
            }
        };
        load_q();  // before the records: they would queue up ahead of it
        ask_until(min(end, pos + kStages));
        bool first_of_run = true;
        while (pos < end) {
            const int t0 = use.tile, t1 = min(use.len.tiles, t0 + end - pos);
            const int start = pos - t0;
            const int cols = min(8, use.len.columns - use.block * 8);
            if (!first_of_run) load_q();
            if (pos + use.len.tiles - use.tile < end) {  // the next unit's queries, into L1, where its columns begin in this sequence or the next one
                int seq = use.seq, kvh = use.kvh, block = use.block + 1;
                if (block == use.len.blocks) block = 0, kvh++;
                if (kvh == p.hkv) kvh = 0, seq++;
                if (seq == use.seq || (!p.q_rows && seq < p.num_seqs)) {
                    constexpr int kLines = HD / 64;
                    const int col = block * 8 + lane / kLines, query = col / group;
                    if (lane < (kNarrow ? 4 : 8) * kLines && col < use.len.columns) {
                        const size_t row = (p.q_rows ? p.q_rows[seq] : seq) + query;
                        const uint16_t* q = p.q + (row * p.hq + (size_t)kvh * group + (col - query * group)) * HD + lane % kLines * 64;
                        uint32_t x;
                        asm volatile("ld.global.ca.u32 %0, [%1];\n" : "=r"(x) : "l"(q));
                    }
                }
            }
            // keys that columns 2c and 2c + 1 see; all columns see those before `sure`
            int lim0 = use.len.ctx, lim1 = lim0, sure = lim0;
            if (p.q_lens) {
                const int hidden = use.len.ctx - p.q_lens[use.seq] + 1;
                const int col = use.block * 8 + 2 * (kNarrow ? c & 1 : c);
                lim0 = hidden + col / group, lim1 = hidden + (col + 1) / group;
                sure = hidden + use.block * 8 / group;
            }
            float m0 = kFloor, m1 = kFloor, l0 = 0.f, l1 = 0.f;
            float o[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;

            for (int t = t0; t < t1; t += 2) {
                // two records at a time, so that their chains of instructions overlap; at an odd end the second is left out
                const int at = pos + t - t0;
                cp_async_wait<0>();
                __syncwarp();  // everyone's copies have landed, and everyone is done with the records that are overwritten now
                ask_until(min(end, at + kStages));
                const int st0 = (at - begin) % kStages, st1 = (st0 + 1) % kStages;
                const bool one = !(absent >> st0 & 1), two = t + 1 < t1 && !(absent >> st1 & 1);
                const uint8_t *rec0 = smem + (warp * kStages + st0) * Rec::kBytes, *rec1 = smem + (warp * kStages + st1) * Rec::kBytes;
                float s0[4], s1[4];
                if (one)
                    scores<HD>(rec0, lane, qf, to_log2, s0);
                else
                    s0[0] = s0[1] = s0[2] = s0[3] = -INFINITY;
                if (two)
                    scores<HD>(rec1, lane, qf, to_log2, s1);
                else
                    s1[0] = s1[1] = s1[2] = s1[3] = -INFINITY;
                const int tok0 = t * 16;
                const bool edge = tok0 > sure - 32, some = edge && p.q_lens;  // (tok0 + 32 may be 2^31)
                if (some) {
                    if (one) hidden_values<HD>(rec0, lane, s0);
                    if (two) hidden_values<HD>(rec1, lane, s1);
                }
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int lim = j & 1 ? lim1 : lim0, tok = tok0 + g + (j >> 1) * 8;
                        if (tok >= lim) s0[j] = -INFINITY;
                        if (tok + 16 >= lim) s1[j] = -INFINITY;
                    }
                }
                float mx0 = fmaxf(fmaxf(s0[0], s0[2]), fmaxf(s1[0], s1[2])), mx1 = fmaxf(fmaxf(s0[1], s0[3]), fmaxf(s1[1], s1[3]));
                if (__any_sync(kFull, mx0 > m0 + kSlack || mx1 > m1 + kSlack)) {
#pragma unroll
                    for (int sh = 4; sh <= 16; sh <<= 1) {
                        mx0 = fmaxf(mx0, __shfl_xor_sync(kFull, mx0, sh));
                        mx1 = fmaxf(mx1, __shfl_xor_sync(kFull, mx1, sh));
                    }
                    mx0 = fmaxf(m0, mx0), mx1 = fmaxf(m1, mx1);
                    const float a0 = fast_exp2(m0 - mx0), a1 = fast_exp2(m1 - mx1);
                    m0 = mx0, m1 = mx1;
                    l0 *= a0, l1 *= a1;
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) o[mt][0] *= a0, o[mt][1] *= a1, o[mt][2] *= a0, o[mt][3] *= a1;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) s0[j] = fast_exp2(s0[j] - (j & 1 ? m1 : m0)), s1[j] = fast_exp2(s1[j] - (j & 1 ? m1 : m0));
                l0 += (s0[0] + s0[2]) + (s1[0] + s1[2]);
                l1 += (s0[1] + s0[3]) + (s1[1] + s1[3]);
                if (one) add_values<HD, kNarrow>(rec0, lane, s0, use.len.ctx - tok0, some, o);
                if (two) add_values<HD, kNarrow>(rec1, lane, s1, use.len.ctx - tok0 - 16, some, o);
            }
            pos += t1 - t0;
#pragma unroll
            for (int sh = 4; sh <= 16; sh <<= 1) {
                l0 += __shfl_xor_sync(kFull, l0, sh);
                l1 += __shfl_xor_sync(kFull, l1, sh);
            }
            if constexpr (kNarrow) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[mt][j] += __shfl_xor_sync(kFull, o[mt][j], 2);
            }
            if (t0 == 0 && t1 == use.len.tiles) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int col = 2 * c + h;
                    if (col >= cols) continue;
                    const float l = h ? l1 : l0, f = l == 0.f ? 0.f : q4::kUnscale / l;
                    uint32_t v[MT];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) v[mt] = pack_bf2(o[mt][h] * f, o[mt][h + 2] * f);
                    uint4* dst = reinterpret_cast<uint4*>(out_row(use.seq, use.kvh, use.block * 8 + col) + g * (HD / 8));
#pragma unroll
                    for (int i = 0; i < MT / 4; i++) dst[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                }
            } else {
                // as it lies in the lanes.  The first part of a run has a place of its own; the last one lies where the run's records were
                __syncwarp();
                const int i = 2 * warp + !first_of_run;
                float4* dst = first_of_run ? parts + warp * MT * 32 : reinterpret_cast<float4*>(smem + warp * kStages * Rec::kBytes);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) dst[mt * 32 + lane] = make_float4(o[mt][0], o[mt][1], o[mt][2], o[mt][3]);
                if (g == 0) s_m[i][2 * c] = m0, s_m[i][2 * c + 1] = m1, s_l[i][2 * c] = l0, s_l[i][2 * c + 1] = l1;
                if (lane == 0) s_part[i] = Part{use.seq, use.kvh, use.block, start, use.len.tiles, t0, t1, cols};
            }
            first_of_run = false;
            use.tile = t1;
            if (t1 == use.len.tiles) use.next_unit(p);
        }
    }
    __syncthreads();

    // ---- the block's parts, unit by unit in the order of the line.  A thread has what a lane had of one tile: 2 dims of 2 columns.
    const Part mine = s_part[lane % kParts];
    const unsigned there = __ballot_sync(kFull, lane < kParts && mine.tiles > 0);
    unsigned heads, unit;  // the first part of every unit; the parts of this lane's
    {
        const unsigned before = there & ((1u << lane) - 1);
        const int prev_start = __shfl_sync(kFull, mine.start, before ? 31 - __clz(before) : 0);
        heads = __ballot_sync(kFull, (there >> lane & 1) && (!before || prev_start != mine.start));
        const unsigned up_to = (2u << lane) - 1, head = heads & up_to, later = heads & ~up_to;
        unit = there & (later ? (later & -later) - 1 : ~0u) & ~(head ? (1u << (31 - __clz(head))) - 1 : ~0u);
    }
    {  // a warp per column, a lane per part: weight of the part, and its unit's maximum and sum
        static_assert(kWarps == 8 && kParts <= 32, "a warp has a column, a lane a part");
        const bool is = there >> lane & 1;
        const unsigned so_far = heads & ((2u << lane) - 1);
        const int head = so_far ? 31 - __clz(so_far) : 0, last = unit ? 31 - __clz(unit) : 0;
        const float own = is ? s_m[lane][warp] : kFloor;
        float m = own;
#pragma unroll
        for (int o = 1; o < kParts; o <<= 1) {
            const float other = __shfl_up_sync(kFull, m, o);
            if (lane - o >= head) m = fmaxf(m, other);
        }
        m = __shfl_sync(kFull, m, last);
        const float f = fast_exp2(own - m);
        float l = is ? s_l[lane][warp] * f : 0.f;
#pragma unroll
        for (int o = 1; o < kParts; o <<= 1) {
            const float other = __shfl_up_sync(kFull, l, o);
            if (lane - o >= head) l += other;
        }
        l = __shfl_sync(kFull, l, last);
        if (is) s_weight[lane][warp] = f, s_max[lane][warp] = m, s_sum[lane][warp] = l;
    }
    __syncthreads();
    const int mt = warp;
    auto store = [&](const Part& u, const float4& v, float l0, float l1) {
        const float f0 = l0 == 0.f ? 0.f : q4::kUnscale / l0, f1 = l1 == 0.f ? 0.f : q4::kUnscale / l1;
        const int d = g * (HD / 8) + 2 * mt;
        if (2 * c < u.cols) *reinterpret_cast<uint32_t*>(out_row(u.seq, u.kvh, u.block * 8 + 2 * c) + d) = pack_bf2(v.x * f0, v.z * f0);
        if (2 * c + 1 < u.cols) *reinterpret_cast<uint32_t*>(out_row(u.seq, u.kvh, u.block * 8 + 2 * c + 1) + d) = pack_bf2(v.y * f1, v.w * f1);
    };
    auto add = [](float4& sum, const float4& v, float f0, float f1) { sum.x += v.x * f0, sum.y += v.y * f1, sum.z += v.z * f0, sum.w += v.w * f1; };
    static_assert(MT <= kWarps, "a warp has a tile of the output");
    int crossing[2] = {-1, -1};  // parts of the units that other blocks share: this block's first and its last one
    // (kept short: the tail of a kernel is fetched when all blocks come to it)
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    int head = 0;
#pragma unroll 1
    for (unsigned rest = there; rest; rest &= rest - 1) {
        const int i = __ffs(rest) - 1;
        if (heads >> i & 1) head = i, sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mt < MT) {
            const float4* part = (i & 1) ? reinterpret_cast<const float4*>(smem + (i >> 1) * kStages * Rec::kBytes) : parts + (i >> 1) * MT * 32;
            add(sum, part[mt * 32 + lane], s_weight[i][2 * c], s_weight[i][2 * c + 1]);
        }
        const unsigned later = rest & (rest - 1);
        if (later && !(heads >> (__ffs(later) - 1) & 1)) continue;  // the unit has more parts here
        const Part u = s_part[head];
        const bool whole = u.first == 0 && s_part[i].last == u.tiles;
        const int side = u.start <= block_start ? 0 : 1;
        if (!whole) crossing[side] = head;
        if (mt >= MT) continue;
        if (whole) {
            store(u, sum, s_sum[head][2 * c], s_sum[head][2 * c + 1]);
        } else {
            float* dst = p.parts + (size_t)(blockIdx.x * 2 + side) * part_floats<HD>();
            reinterpret_cast<float4*>(dst)[mt * 32 + lane] = sum;
            if (warp == 0 && lane < 8) dst[8 * HD + 2 * lane] = s_max[head][lane], dst[8 * HD + 2 * lane + 1] = s_sum[head][lane];
        }
    }
    if (crossing[0] < 0 && crossing[1] < 0) return;
    // ---- units of several blocks: whoever arrives last adds up their parts.  All blocks come here at the same time, so what counts is the
    // number of trips to L2, one after the other: fence, arrival, parts.
    const int block_run = kWarps * run;
    __syncthreads();
    if (lane == 0 && warp < 2) {
        int last = 0;
        const int mine = crossing[warp];
        if (mine >= 0) {
            const Part u = s_part[mine];
            const int from = u.start / block_run, to = (u.start + u.tiles - 1) / block_run;
            __threadfence();  // the block's parts are visible before its arrival is counted
            if (atomicAdd(p.counters + from, 1) == to - from) {
                last = 1;
                p.counters[from] = 0;
                __threadfence();
            }
        }
        s_last[warp] = last;
    }
    __syncthreads();
    if (mt >= MT) return;
#pragma unroll 1
    for (int side = 0; side < 2; side++) {
        if (!s_last[side]) continue;
        const Part u = s_part[side ? crossing[1] : crossing[0]];
        const int from = u.start / block_run, to = (u.start + u.tiles - 1) / block_run;
        constexpr int N = 4;
        sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float m0 = kFloor, m1 = kFloor, l0 = 0.f, l1 = 0.f;
        for (int b0 = from; b0 <= to; b0 += N) {
            float4 v[N], ml[N];  // ml: maximum and sum of columns 2c and 2c + 1
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int b = min(b0 + i, to);
                const float* part = p.parts + (size_t)(b * 2 + (u.start <= b * block_run ? 0 : 1)) * part_floats<HD>();
                ml[i] = __ldcg(reinterpret_cast<const float4*>(part + 8 * HD) + c);
                v[i] = __ldcg(reinterpret_cast<const float4*>(part) + mt * 32 + lane);
            }
            float top0 = m0, top1 = m1;
#pragma unroll
            for (int i = 0; i < N; i++) top0 = fmaxf(top0, ml[i].x), top1 = fmaxf(top1, ml[i].z);
            const float a0 = fast_exp2(m0 - top0), a1 = fast_exp2(m1 - top1);
            m0 = top0, m1 = top1;
            l0 *= a0, l1 *= a1;
            sum.x *= a0, sum.y *= a1, sum.z *= a0, sum.w *= a1;
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (b0 + i > to) break;
                const float f0 = fast_exp2(ml[i].x - m0), f1 = fast_exp2(ml[i].z - m1);
                l0 += ml[i].y * f0, l1 += ml[i].w * f1;
                add(sum, v[i], f0, f1);
            }
        }
        store(u, sum, l0, l1);
    }
}

template <int HD, bool kNarrow>
int32_t launch(b2_ctx* ctx, Q4AttnParams p) {
    const int grid = kBlocksPerSm * ctx->sm_count;
    if (!ctx->q4_parts) {  // two parts per block, and an arrival counter each (zero between launches)
        const size_t bytes = (size_t)grid * (2 * part_floats<128>() + 1) * 4;
        B2_CUDA(cudaMalloc((void**)&ctx->q4_parts, bytes));
        B2_CUDA(cudaMemsetAsync(ctx->q4_parts, 0, bytes, ctx->stream));
    }
    p.group = p.hq / p.hkv;
    p.max_ctx = (int)std::min<int64_t>((int64_t)p.max_blocks * p.page_tiles * 16, 0x7ffffff0);
    p.parts = ctx->q4_parts;
    p.counters = reinterpret_cast<int*>(ctx->q4_parts + (size_t)grid * 2 * part_floats<128>());
    const auto kernel = kv_q4_attn_kernel<HD, kNarrow>;
    B2_SMEM_ONCE(ctx, kernel, smem_bytes<HD>());
    B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, kernel, dim3(grid), dim3(kWarps * 32), (size_t)smem_bytes<HD>(), ctx->stream, p));
    B2_LAUNCHED(ctx);
    B2_CUDA(cudaGetLastError());
    return B2_OK;
}

}  // namespace

int32_t b2_kv_q4_check(const char* who, const void* pool, int64_t n_pages, int32_t hq, int32_t hkv, int32_t head_dim, int32_t page_size) {
    const std::string name = who;
    B2_REQUIRE(hkv > 0 && hq > 0 && hq % hkv == 0, B2_ERR_MSG, name + ": hq must be a multiple of hkv");
    B2_REQUIRE(head_dim == 64 || head_dim == 128, B2_ERR_UNSUPPORTED, name + ": head_dim must be 64 or 128");
    B2_REQUIRE(page_size > 0 && page_size % 16 == 0, B2_ERR_UNSUPPORTED, name + ": page_size must be a multiple of 16");
    B2_REQUIRE(n_pages > 0 && n_pages * page_size < (1ll << 31) && n_pages * hkv * (page_size / 16) < (1ll << 31), B2_ERR_MSG,
               name + ": the pool must have pages, and fewer than 2^31 tokens and records");
    B2_REQUIRE(((uintptr_t)pool & 15) == 0, B2_ERR_UNSUPPORTED, name + ": the pool must be 16-byte aligned");
    return B2_OK;
}

int32_t b2_kv_q4_attn_launch(b2_ctx* ctx, const Q4AttnParams& p, int head_dim) {
    if (p.num_seqs <= 0) return B2_OK;
    if (p.columns <= 4) return head_dim == 128 ? launch<128, true>(ctx, p) : launch<64, true>(ctx, p);
    return head_dim == 128 ? launch<128, false>(ctx, p) : launch<64, false>(ctx, p);
}

extern "C" int64_t b2_kv_q4_pool_bytes(int64_t n_pages, int32_t hkv, int32_t head_dim, int32_t page_size) {
    if (b2_kv_q4_check("b2_kv_q4_pool_bytes", nullptr, n_pages, hkv, hkv, head_dim, page_size) != B2_OK) return 0;
    return n_pages * hkv * (page_size / 16) * q4::record_bytes(head_dim);
}

extern "C" int32_t b2_paged_attn_decode_q4(b2_ctx* ctx, const uint16_t* q_dev, const uint8_t* kv_pool_dev, int32_t n_pages, const int32_t* block_tables_dev,
                                           int32_t max_blocks, const int32_t* ctx_lens_dev, int32_t num_seqs, int32_t hq, int32_t hkv, int32_t head_dim,
                                           int32_t page_size, float scale, uint16_t* out_dev) {
    B2_REQUIRE(ctx && q_dev && kv_pool_dev && block_tables_dev && ctx_lens_dev && out_dev, B2_ERR_MSG, "b2_paged_attn_decode_q4: null argument");
    B2_CHECK(b2_kv_q4_check("b2_paged_attn_decode_q4", kv_pool_dev, n_pages, hq, hkv, head_dim, page_size));
    B2_REQUIRE(num_seqs >= 0 && max_blocks > 0, B2_ERR_MSG, "b2_paged_attn_decode_q4: bad sizes");
    B2_REQUIRE((double)num_seqs * max_blocks * (page_size / 16) * hkv * ((hq / hkv + 7) / 8) < 1073741824.0, B2_ERR_UNSUPPORTED,
               "b2_paged_attn_decode_q4: the block tables reach more than 2^30 records; make fewer sequences a call");
    B2_REQUIRE(scale > 0.f && scale < kQ4SoftmaxScaleEnd, B2_ERR_MSG, "b2_paged_attn_decode_q4: the scale must be positive and below 2^62");
    B2_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) == 0, B2_ERR_UNSUPPORTED, "b2_paged_attn_decode_q4: q and out must be 16-byte aligned");
    B2_CUDA(cudaSetDevice(ctx->device));
    Q4AttnParams p{};
    p.q = q_dev;
    p.pool = kv_pool_dev;
    p.n_pages = n_pages;
    p.block_tables = block_tables_dev;
    p.max_blocks = max_blocks;
    p.ctx_lens = ctx_lens_dev;
    p.num_seqs = num_seqs;
    p.columns = hq / hkv;
    p.hq = hq;
    p.hkv = hkv;
    p.page_tiles = page_size / 16;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.out = out_dev;
    return b2_kv_q4_attn_launch(ctx, p, head_dim);
}

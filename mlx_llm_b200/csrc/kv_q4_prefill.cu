// Attention over a 4-bit paged cache for any number of query tokens per sequence: prompts, portions of prompts, drafts.
//
// Few columns (query tokens x q heads of a group) go through kv_q4_attn.cu, which reads the 4 bits once per 8 columns.  With many, the
// products decide, not the bytes: the keys and values of a sequence are widened once to bf16 in a workspace, [16-token tile][kv head]
// [16][head size], and the prefill kernels of the 16-bit cache multiply from there, so that a code is converted once and not once per
// query tile and head.  The workspace takes whole sequences, up to kPassBytes at a time (a longer sequence alone).
#include <algorithm>

#include "kernels.h"
#include "kv_q4.cuh"

namespace {

constexpr size_t kPassBytes = 1ull << 30;
constexpr int kFewColumns = 32;

struct WidenParams {
    const uint8_t* pool;
    int64_t n_pages;
    const int32_t* block_tables;
    int max_blocks, hkv, page_tiles;
    const int32_t *rows, *ctx, *first;  // [seqs] block-table row, context, first tile
    int seqs;
    int64_t tiles;
    int max_tiles;
    uint16_t *k, *v;       // [tiles][hkv][16][HD]
    int32_t* table;        // [seqs][max_tiles] tile numbers: the workspace's block table
};

// One warp per record.  Bound by its writes, four times what it reads; they stay in L2 for the attention behind it where they fit.
// Tokens behind the context, and pages outside of the pool, become zeros.
template <int HD>
__global__ void __launch_bounds__(256) kv_q4_widen_kernel(const WidenParams p) {
    using Rec = q4::Record<HD>;
    constexpr int W = HD / 32;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    pdl_wait();
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= p.tiles * p.hkv) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int tile = (int)(item / p.hkv), kvh = (int)(item - (int64_t)tile * p.hkv);
    int lo = 0, hi = p.seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.first[mid] <= tile)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int t = tile - p.first[lo], left = p.ctx[lo] - t * 16;  // tokens of this tile that belong to the context
    const int index = t / p.page_tiles;
    const int page = p.block_tables[(size_t)p.rows[lo] * p.max_blocks + index];
    const bool there = page >= 0 && page < p.n_pages;
    if (kvh == 0 && lane == 0) p.table[(size_t)lo * p.max_tiles + t] = tile;
    const uint8_t* rec = p.pool + (((size_t)(there ? page : 0) * p.hkv + kvh) * p.page_tiles + t - index * p.page_tiles) * Rec::kBytes;
    auto wide = [](uint32_t v) { return mul_bf2(v, 0x5f805f80u); };  // times 2^64
    auto store = [](uint16_t* dst, const uint32_t (&v)[W * 2]) {     // W * 4 values
#pragma unroll
        for (int i = 0; i < W / 2; i++) reinterpret_cast<uint4*>(dst)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    };
    const size_t base = (size_t)item * 16 * HD;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        {  // K: token g + 8 half, dims c HD/4 ...
            const int tok = g + 8 * half;
            const q4::Scales q = q4::scales_twice(reinterpret_cast<const uint32_t*>(rec + Rec::kKsb)[(c * (HD / 4) / 64) * 16 + tok]);
            const uint32_t* src = reinterpret_cast<const uint32_t*>(rec) + (half * 32 + lane) * W;
            uint16_t* dst = p.k + base + (size_t)tok * HD + c * (HD / 4);
#pragma unroll
            for (int w = 0; w < W; w++) {
                uint32_t v[4];
                q4::values(src[w], q, v);  // (0,4) (1,5) (2,6) (3,7)
                const bool ok = there && tok < left;
                const uint4 r = make_uint4(wide(prmt(v[0], v[1], 0x5410u)), wide(prmt(v[2], v[3], 0x5410u)), wide(prmt(v[0], v[1], 0x7632u)), wide(prmt(v[2], v[3], 0x7632u)));
                reinterpret_cast<uint4*>(dst)[w] = ok ? r : make_uint4(0, 0, 0, 0);
            }
        }
        {  // V: tokens 8 half + 2c and the next, dims g HD/8 ...
            const int tok = 8 * half + 2 * c;
            const uint2 sb = *reinterpret_cast<const uint2*>(rec + Rec::kVsb + ((g * (HD / 8) / 64) * 16 + tok) * 4);
            const q4::Scales q = q4::scales_pair(sb.x, sb.y);
            const uint32_t* src = reinterpret_cast<const uint32_t*>(rec + Rec::kV) + (half * 32 + lane) * W;
            uint32_t a[2 * W], b[2 * W];
            const bool ok0 = there && tok < left, ok1 = there && tok + 1 < left;
#pragma unroll
            for (int w = 0; w < W; w++) {
                uint32_t v[4];
                q4::values(src[w], q, v);  // dim i of both tokens
                a[2 * w] = ok0 ? wide(prmt(v[0], v[1], 0x5410u)) : 0u, a[2 * w + 1] = ok0 ? wide(prmt(v[2], v[3], 0x5410u)) : 0u;
                b[2 * w] = ok1 ? wide(prmt(v[0], v[1], 0x7632u)) : 0u, b[2 * w + 1] = ok1 ? wide(prmt(v[2], v[3], 0x7632u)) : 0u;
            }
            uint16_t* dst = p.v + base + (size_t)tok * HD + g * (HD / 8);
            store(dst, a);
            store(dst + HD, b);
        }
    }
}

}  // namespace

int32_t b2_kv_q4_plan(b2_ctx* ctx, const std::vector<Q4Seq>& seqs, int hq, int hkv, int head_dim, Q4Plan& plan) {
    plan = Q4Plan{};
    const int group = hq / hkv, q_tile = b2_prefill_q_tile(ctx, head_dim);
    std::vector<Q4Seq> few, many;
    for (const Q4Seq& s : seqs)
        if (s.q_len > 0) ((long)s.q_len * group <= kFewColumns ? few : many).push_back(s);
    plan.few = (int)few.size();
    for (const Q4Seq& s : few) plan.host.push_back(s.bt_row);
    for (const Q4Seq& s : few) plan.host.push_back(s.q_row);
    for (const Q4Seq& s : few) plan.host.push_back(s.q_len);
    for (const Q4Seq& s : few) plan.host.push_back(s.ctx);
    const size_t tile_bytes = (size_t)hkv * 16 * head_dim * 4;
    for (size_t from = 0; from < many.size();) {
        Q4Pass pass{};
        size_t to = from;
        for (; to < many.size(); to++) {
            const int64_t tiles = (many[to].ctx + 15) / 16;
            if (to > from && (pass.tiles + tiles) * tile_bytes > kPassBytes) break;
            pass.tiles += tiles;
            pass.max_tiles = std::max(pass.max_tiles, (int)tiles);
            pass.max_ctx = std::max(pass.max_ctx, many[to].ctx);
        }
        const int n = pass.seqs = (int)(to - from);
        pass.list = plan.host.size();
        int32_t tile = 0;
        for (size_t i = from; i < to; i++) plan.host.push_back(many[i].bt_row);
        for (size_t i = from; i < to; i++) plan.host.push_back(many[i].ctx);
        for (size_t i = from; i < to; i++) {
            plan.host.push_back(tile);
            tile += (many[i].ctx + 15) / 16;
        }
        // The prefill kernels take the rows of sequence b from cu[b] and cu[b + 1].  Theirs need not lie behind one another here, so
        // sequence i is number 2i, and the odd numbers have no work: rows [2n], then contexts [2n], workspace table rows [2n].
        pass.cu = plan.host.size();
        for (size_t i = from; i < to; i++) plan.host.insert(plan.host.end(), {many[i].q_row, many[i].q_row + many[i].q_len});
        for (size_t i = from; i < to; i++) plan.host.insert(plan.host.end(), {many[i].ctx, 0});
        for (int i = 0; i < n; i++) plan.host.insert(plan.host.end(), {i, 0});
        for (int i = 0; i < n; i++)
            for (int r = 0; r < many[from + i].q_len; r += q_tile) pass.work++;
        for (int i = 0; i < n; i++)
            for (int r = 0; r < many[from + i].q_len; r += q_tile) plan.host.push_back(2 * i);
        for (int i = 0; i < n; i++)
            for (int r = 0; r < many[from + i].q_len; r += q_tile) plan.host.push_back(r);
        plan.host.push_back(pass.work);
        plan.passes.push_back(pass);
        from = to;
    }
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
    size_t need = 0;
    for (const Q4Pass& pass : plan.passes)
        need = std::max(need, (size_t)pass.tiles * p.hkv * 16 * head_dim * 4 + (size_t)pass.seqs * pass.max_tiles * 4);
    if (need > ctx->q4_wide_bytes) {
        B2_CUDA(cudaStreamSynchronize(ctx->stream));
        if (ctx->q4_wide) B2_CUDA(cudaFree(ctx->q4_wide));
        ctx->q4_wide = nullptr;
        ctx->q4_wide_bytes = 0;
        B2_CUDA(cudaMalloc((void**)&ctx->q4_wide, need + (need >> 2)));
        ctx->q4_wide_bytes = need + (need >> 2);
    }
    for (const Q4Pass& pass : plan.passes) {
        const size_t elems = (size_t)pass.tiles * p.hkv * 16 * head_dim;
        WidenParams w{};
        w.pool = p.pool;
        w.n_pages = p.n_pages;
        w.block_tables = p.block_tables;
        w.max_blocks = p.max_blocks;
        w.hkv = p.hkv;
        w.page_tiles = p.page_tiles;
        w.rows = plan_dev + pass.list;
        w.ctx = w.rows + pass.seqs;
        w.first = w.ctx + pass.seqs;
        w.seqs = pass.seqs;
        w.tiles = pass.tiles;
        w.max_tiles = pass.max_tiles;
        w.k = reinterpret_cast<uint16_t*>(ctx->q4_wide);
        w.v = w.k + elems;
        w.table = reinterpret_cast<int32_t*>(w.v + elems);
        const dim3 grid((unsigned)((pass.tiles * p.hkv + 7) / 8));
        B2_CUDA(b2_launch_pdl(ctx->pdl_consumers, head_dim == 128 ? kv_q4_widen_kernel<128> : kv_q4_widen_kernel<64>, grid, dim3(256), 0, ctx->stream, w));
        B2_LAUNCHED(ctx);
        PrefillAttnParams a{};
        a.q = p.q;
        a.k_pool = w.k;
        a.v_pool = w.v;
        a.block_tables = w.table;
        a.max_blocks = pass.max_tiles;
        a.cu_seqlens = plan_dev + pass.cu;
        a.context_lens = a.cu_seqlens + 2 * pass.seqs;
        a.seq_slot = a.context_lens + 2 * pass.seqs;
        a.pf_seq = a.seq_slot + 2 * pass.seqs;
        a.pf_qstart = a.pf_seq + pass.work;
        a.n_work = a.pf_qstart + pass.work;
        a.hq = p.hq;
        a.hkv = p.hkv;
        a.page_tiles = 1;
        a.scale_log2 = p.scale_log2;
        a.out = p.out;
        a.q_tile = b2_prefill_q_tile(ctx, head_dim);
        a.q_rows = p.q_rows;
        a.pool_rows = pass.tiles * p.hkv * 16;
        a.max_ctx = pass.max_ctx;
        B2_CHECK(b2_prefill_attn_launch(ctx, a, head_dim, pass.work));
    }
    return B2_OK;
}

extern "C" int32_t b2_paged_attn_prefill_q4(b2_ctx* ctx, const uint16_t* q_dev, const uint8_t* kv_pool_dev, int32_t n_pages, const int32_t* block_tables_dev,
                                            int32_t max_blocks, const int32_t* cu_seqlens_host, const int32_t* ctx_lens_host, int32_t num_seqs, int32_t hq,
                                            int32_t hkv, int32_t head_dim, int32_t page_size, float scale, uint16_t* out_dev) {
    B2_REQUIRE(ctx && q_dev && kv_pool_dev && block_tables_dev && cu_seqlens_host && ctx_lens_host && out_dev, B2_ERR_MSG, "b2_paged_attn_prefill_q4: null argument");
    B2_CHECK(b2_kv_q4_check("b2_paged_attn_prefill_q4", kv_pool_dev, n_pages, hq, hkv, head_dim, page_size));
    B2_REQUIRE(num_seqs >= 0 && max_blocks > 0, B2_ERR_MSG, "b2_paged_attn_prefill_q4: bad sizes");
    B2_REQUIRE((((uintptr_t)q_dev | (uintptr_t)out_dev) & 15) == 0, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: q and out must be 16-byte aligned");
    if (num_seqs == 0) return B2_OK;
    std::vector<Q4Seq> seqs;
    double records = 0;
    for (int i = 0; i < num_seqs; i++) {
        const int n = cu_seqlens_host[i + 1] - cu_seqlens_host[i], ctx_len = ctx_lens_host[i];
        B2_REQUIRE(cu_seqlens_host[i] >= 0 && n >= 0 && ctx_len >= n, B2_ERR_MSG, "b2_paged_attn_prefill_q4: ctx_lens must include the new tokens, and cu_seqlens ascend");
        B2_REQUIRE(((int64_t)ctx_len + page_size - 1) / page_size <= max_blocks, B2_ERR_MSG,
                   "b2_paged_attn_prefill_q4: a context needs more blocks than a block-table row holds");
        seqs.push_back(Q4Seq{i, cu_seqlens_host[i], n, ctx_len});
        records += (ctx_len + 15) / 16 * (double)hkv * (kFewColumns / 8 + 1);
    }
    B2_REQUIRE(records < 1073741824.0, B2_ERR_UNSUPPORTED, "b2_paged_attn_prefill_q4: more than 2^30 records in one call; make fewer sequences a call");
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
    p.q_rows = cu_seqlens_host[num_seqs];
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

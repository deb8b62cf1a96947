// Attention of new tokens over a cache in pages: the choice of kernel, the split of long contexts and the joining of their parts.
// (paged_attention_rows.cuh: few rows; paged_attention_tc.cu: many.)
#include <algorithm>

#include "paged_attention.cuh"

namespace lv {

// A warp per (token, head): the splits of its row in their order.
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttn p, uint32_t block_rows) {
    pdl_launch_dependents();
    pdl_wait();
    const lv_paged_attention_args& a = p.a;
    const PagedCache& c = p.c;
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t job = uint64_t(blockIdx.x) * 4 + threadIdx.x / 32;
    const uint32_t t = uint32_t(job / a.heads), h = uint32_t(job - uint64_t(t) * a.heads);
    if (t >= a.tokens) return;
    // the first parts are asked for before it is known how many there are (all places lie in the scratch)
    const size_t part = (size_t(t) * a.heads + h) * p.splits;
    const float2 first = lane < p.splits ? p.part_rl[part + lane] : make_float2(-INFINITY, 0.f);
    float4 x[4][2];
    auto ask = [&](uint32_t i0, uint32_t end) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t d = 4 * (lane + 32 * k);
                x[e][k] = i0 + e < end && d < c.dim ? *reinterpret_cast<const float4*>(p.part_o + (part + i0 + e) * c.dim + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
    };
    ask(0, p.splits);
    const uint32_t s = paged_owner(c, t);
    PagedSeq q;
    if (s == c.seqs || !paged_seq(c, s, a.tokens, &q) || !paged_holds(q, t) || q.n > a.max_new || q.len > a.max_len) return;       // (reported)
    const uint32_t r = (t - q.row0) * p.group + h % p.group, r0 = r / block_rows * block_rows;
    const PagedRange all = paged_range(p, q, r0, min(r0 + block_rows, q.n * p.group) - 1);
    const uint32_t n = min((all.hi - (all.lo & ~p.align) + p.chunk - 1) / p.chunk, p.splits);
    const float sink = paged_sink(p, h);
    float top = sink - kPaLift;
    float2 mine = lane < n ? first : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, mine.x);
    for (uint32_t i = lane + 32; i < n; i += 32) top = fmaxf(top, p.part_rl[part + i].x);
    top = warp_max(top);
    float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    float total = 0.f;
    for (uint32_t b = 0; b < n; b += 32) {
        if (b != 0) mine = b + lane < n ? p.part_rl[part + b + lane] : make_float2(-INFINITY, 0.f);
        // weight of this lane's split; one that saw nothing has none
        const float mine_f = mine.x == -INFINITY ? mine.y : exp2_fast(mine.x - top);          // (0, or NaN)
        if (!(mine.x == -INFINITY && mine.y == 0.f)) total = fmaf(mine.y, mine_f, total);
        const uint32_t end = min(32u, n - b);
        for (uint32_t i = 0; i < end; i += 4) {
            if (b + i != 0) ask(b + i, n);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float f = __shfl_sync(0xffffffffu, mine_f, int(min(i + e, 31u)));
                if (i + e >= end || f == 0.f) continue;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    v[k] = make_float4(fmaf(x[e][k].x, f, v[k].x), fmaf(x[e][k].y, f, v[k].y), fmaf(x[e][k].z, f, v[k].z), fmaf(x[e][k].w, f, v[k].w));
            }
        }
    }
    total = warp_sum(total) + paged_sink_weight(sink, top);
    const float f = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t d = 4 * (lane + 32 * k);
        if (d < c.dim) store_values4(a.out, size_t(t) * a.out_ld + size_t(h) * c.dim + d, a.out_type, make_float4(v[k].x * f, v[k].y * f, v[k].z * f, v[k].w * f));
    }
}

// ---- choice of kernel and split ------------------------------------------------------------------

struct PagedPlan {
    uint32_t rows, blocks;       // rows of a block, blocks of the longest chunk of new tokens
    uint32_t chunk, splits, box;
    size_t bytes;
    bool many;
};

static PagedPlan paged_plan(const lv_ctx* ctx, const lv_paged_attention_args& a) {
    PagedPlan plan{};
    if (!a.tokens || !a.max_new) {                                       // nobody has new tokens: nothing is launched
        plan.bytes = 16;
        return plan;
    }
    const uint32_t group = a.heads / a.cache.kv_heads, rows = a.max_new * group;
    // 16-bit outputs of more than 32 rows that share their keys (8-bit caches: of more than 96): tiles of the tensor cores, whose copies take eight rows of a page at least.  Both sides,
    // us in blocks of 32 rows against tiles, 8 key/value heads, rows of the longest sequence:
    //   16 sequences of 200 to 6000 keys, bf16   40 rows  99, 114    48  110, 114    64  121, 116     96  156, 120
    //   64 of 500 to 8192, bf16                  40      373, 369                    64  523, 379    128  835, 405        one of 4096   48  31.7, 17.0
    //   16, e4m3                                 40       83, 213    64  102, 216    96  131, 228    128  165, 240       192  232, 277       320  338, 309
    //   64, int8                                 40      303, 720    64  430, 739                    128  685, 784       320  1506, 1261
    //   one of 12000, int8                       40       43, 42     64   47, 44                     128   64, 47         one of 2000, e4m3   96  26.5, 23.4
    // (a tile's codes are taken apart by four warps, whatever its rows)
    plan.box = std::min(a.cache.page_rows & (0u - a.cache.page_rows), uint32_t(kPtKeys));
    plan.many = a.out_type != LV_TYPE_F32 && a.cache.dim <= 128 && rows > (paged_is8(a.cache.type) ? 96 : 32) && plan.box >= 8 && uint64_t(a.cache.pages) * a.cache.kv_heads * a.cache.page_rows < (uint64_t(1) << 31);
    plan.rows = plan.many ? kPtRows : std::min((rows + 7) / 8 * 8, a.cache.dim > 128 ? 16u : 32u);
    plan.blocks = (rows + plan.rows - 1) / plan.rows;
    const uint64_t seen = a.window ? std::min<uint64_t>(a.max_len, uint64_t(a.window) + std::min(a.max_new, plan.rows)) : a.max_len;
    const uint32_t unit = plan.many ? kPtKeys : kPrWarps * (paged_is8(a.cache.type) ? kPrKeys8 : kPrKeys16);
    const uint64_t ctas = uint64_t(a.cache.seqs) * a.cache.kv_heads * plan.blocks;
    const uint64_t most = std::max<uint64_t>(1, (seen + unit - 1) / unit);
    uint64_t splits = 1;
    if (plan.many) {
        // the split with the fewest steps of 128 keys one after the other: rounds of CTAs, each with about kPtSetUp steps' time beside its own, and the joining, which
        // moves 8 bytes a value and split at the memory's rate (a step takes about 2 us: 13 MB)
        uint64_t best = ~uint64_t(0);
        for (uint64_t n = 1; n <= std::min<uint64_t>(most, 32); ++n) {
            // (in halves: a last round that is not full costs half a round on average, lengths differ)
            const uint64_t rounds = ctas * n <= uint64_t(ctx->sm_count) ? 2 : 2 * ctas * n / ctx->sm_count + 1, join = n == 1 ? 0 : 2 + uint64_t(a.tokens) * a.heads * a.cache.dim * 8 * n / (13u << 20);
            const uint64_t cost = rounds * ((most + n - 1) / n + kPtSetUp) / 2 + join;
            if (cost < best) { best = cost; splits = n; }
        }
    } else {
        // Three CTAs per SM hold blocks of up to 16 rows, two the larger ones.  Where there are fewer blocks than SMs (larger ones: than half of the SMs), splits fill the GPU once: more would be short
        // ones, each with its start and a part to join.  Where there are more blocks, sequences of different lengths share the GPU evenly when there are several rounds of CTAs.  us with 3, 6 and 12
        // CTAs per SM, 8 key/value heads, one token (blocks of 8 rows):
        //   int8  2 sequences of 4096 keys  12.8, 14.6, 14.5    8  21.2, 22.8, 22.3    16 of 500 to 2000  18.8, 21.4, 20.7    24 of 500 to 8192  60, 60, 56    64  145, 134, 125
        //   bf16  2                         13.6, 15.9, 21.6    8  24.8, 27.9, 29.1    16                 22.0, 25.9, 25.7    24                 80, 91, 84    64  208, 208, 188
        // six drafts of sequences of 200 to 6000 keys (blocks of 24), e4m3:  2  25.5, 32.5, 32.5    8  30.8, 38.6, 50.7    16  53.5, 52.2, 57.8    32  92, 86, 92    64  163, 148, 145    (bf16  4  40.3, 35.6, 50.6)
        const bool free_sms = a.cache.seqs == 1 || ctas * (plan.rows <= 16 ? 1 : 2) <= uint64_t(ctx->sm_count);
        const uint64_t want = uint64_t(ctx->sm_count) * (free_sms ? 3 : plan.rows <= 16 ? 12 : 6);
        splits = std::max<uint64_t>(1, std::min<uint64_t>((want + ctas - 1) / ctas, most));
    }
    uint64_t chunk = ((seen + splits - 1) / splits + unit - 1) / unit * unit;
    plan.chunk = uint32_t(std::max<uint64_t>(chunk, unit));
    plan.splits = uint32_t((seen + (plan.many ? kPtKeys - 1 : 0) + plan.chunk - 1) / plan.chunk);
    if (plan.splits == 0) plan.splits = 1;
    plan.bytes = plan.splits == 1 ? 16 : (size_t(a.tokens) * a.heads * plan.splits * (a.cache.dim + 2)) * 4 + 32;
    return plan;
}

static int paged_attention_check(const lv_paged_attention_args* a) {
    LV_REQUIRE(a && a->q && a->out, "paged attention: null argument");
    if (const int rc = paged_check(&a->cache)) return rc;
    LV_REQUIRE(a->heads && a->heads % a->cache.kv_heads == 0 && a->heads <= 65535, "paged attention: heads are a multiple of the key/value heads");
    LV_REQUIRE(paged_value_type(a->q_type) && paged_value_type(a->out_type), "paged attention: unsupported type");
    const uint64_t width = uint64_t(a->heads) * a->cache.dim;
    LV_REQUIRE(a->q_ld >= width && a->out_ld >= width, "paged attention: bad strides");
    LV_REQUIRE(uint64_t(a->q_ld) * paged_bytes(a->q_type) % 16 == 0 && uint64_t(a->out_ld) * paged_bytes(a->out_type) % 16 == 0 && aligned16(a->q) && aligned16(a->out),
               "paged attention: rows of q and out are 16-byte aligned");
    LV_REQUIRE(a->max_new <= a->tokens && a->max_new <= a->max_len && a->max_len <= uint64_t(a->cache.table_ld) * a->cache.page_rows, "paged attention: bad upper bounds");
    LV_REQUIRE(uint64_t(a->tokens) * a->heads < (uint64_t(1) << 31), "paged attention: too many tokens");
    LV_REQUIRE(a->scale > 0.f && isfinite(a->scale), "paged attention: scale");
    LV_REQUIRE(words_aligned(a->sink), "paged attention: 32-bit values are 4-byte aligned");
    return paged_check_rotation(a->angles, a->angle_ld, a->angle_pairs, a->cache.dim);
}

}  // namespace lv

using namespace lv;

extern "C" size_t lv_paged_attention_scratch_bytes(lv_ctx* ctx, const lv_paged_attention_args* a) {
    if (paged_attention_check(a) != LV_OK || !ctx) return 0;
    return paged_plan(ctx, *a).bytes;
}

extern "C" int lv_paged_attention(lv_ctx* ctx, const lv_paged_attention_args* a, void* scratch, size_t scratch_bytes) {
    if (const int rc = paged_attention_check(a)) return rc;
    LV_REQUIRE(scratch && aligned16(scratch), "paged attention: scratch is 16-byte aligned");
    LV_ENTER(ctx);
    const PagedPlan plan = paged_plan(ctx, *a);
    LV_REQUIRE(scratch_bytes >= plan.bytes, "paged attention: scratch too small");
    if (!a->tokens || !a->max_new) return LV_OK;
    PagedAttn p{};
    p.a = *a;
    p.c = paged_cache(a->cache);
    p.group = a->heads / a->cache.kv_heads;
    p.factor = paged_factor(a->scale * kPaLog2e, 1.f);
    p.chunk = plan.chunk;
    p.splits = plan.splits;
    p.align = plan.many ? kPtKeys - 1 : 0;
    p.box = plan.box;
    p.part_rl = static_cast<float2*>(scratch);
    p.part_o = static_cast<float*>(scratch) + (size_t(a->tokens) * a->heads * plan.splits * 2 + 3) / 4 * 4;
    p.err = ctx->d_err;
    p.data_err = ctx->data_err();
    int rc = LV_OK;
    if (plan.many) rc = paged_tc_launch(ctx, p, plan.blocks);
    else switch (a->cache.type) {
        case LV_TYPE_BF16: rc = paged_rows_launch_bf16(ctx, p, plan.rows, plan.blocks); break;
        case LV_TYPE_F16: rc = paged_rows_launch_f16(ctx, p, plan.rows, plan.blocks); break;
        case LV_TYPE_I8: rc = paged_rows_launch_i8(ctx, p, plan.rows, plan.blocks); break;
        default: rc = paged_rows_launch_e4m3(ctx, p, plan.rows, plan.blocks); break;
    }
    if (rc != LV_OK || plan.splits == 1) return rc;
    const uint64_t warps = uint64_t(a->tokens) * a->heads;
    LV_CUDA(launch_pdl(ctx, paged_join_kernel, dim3(uint32_t((warps + 3) / 4)), dim3(128), 0, p, plan.rows));
    return LV_OK;
}

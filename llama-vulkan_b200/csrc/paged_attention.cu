// Attention of new tokens over a cache in pages.
//
//   s_j = scale (q . k_j),  m = max s_j,  out = sum_j e^(s_j - m) v_j / (e^(sink - m) + sum_j e^(s_j - m))
#include <algorithm>

#include "paged.cuh"

namespace lv {

constexpr int kPaWarps = 4;

struct PagedAttn {
    lv_paged_attention_args a;
    uint32_t* err;
};

// A CTA per query head and token; every warp takes each fourth key, with a running maximum and sum of its own.
__global__ void __launch_bounds__(32 * kPaWarps) paged_plain_kernel(const PagedAttn p) {
    pdl_launch_dependents();
    pdl_wait();
    const lv_paged_attention_args& a = p.a;
    const lv_paged_cache& c = a.cache;
    __shared__ float s_m[kPaWarps], s_l[kPaWarps], s_o[kPaWarps][256];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x / 32, h = blockIdx.x, t = blockIdx.y + blockIdx.z * 65535u, kv = h / (a.heads / c.kv_heads);
    if (t >= a.tokens) return;
    const uint32_t s = paged_owner(c, t);
    if (s == c.seqs) return;
    PagedSeq q;
    if (!paged_seq(c, s, a.tokens, &q) || q.n > a.max_new || q.len > a.max_len) {
        if (threadIdx.x == 0) atomicOr(p.err, ERR_BAD_INDEX);
        return;
    }
    const uint32_t at = q.len - q.n + (t - q.row0), first = a.window != 0 && at + 1 > a.window ? at + 1 - a.window : 0;
    float4 x[2], o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t d = 4 * (lane + 32 * i);
        x[i] = o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d >= c.dim) continue;
        x[i] = load_values4(a.q, size_t(t) * a.q_ld + size_t(h) * c.dim + d, a.q_type);
        if (a.angles != nullptr) x[i] = rotate4(x[i], a.angles + size_t(t) * a.angle_ld, d, a.angle_pairs);
    }
    float m = -INFINITY, l = 0.f;
    for (uint32_t j = first + warp; j <= at; j += kPaWarps) {
        uint64_t row;
        if (!paged_row(c, c.table + size_t(s) * c.table_ld, j, kv, &row)) {
            if (lane == 0) atomicOr(p.err, ERR_BAD_INDEX);
            continue;
        }
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t d = 4 * (lane + 32 * i);
            if (d >= c.dim) continue;
            const float4 k = load_cached4(c.k, row * c.dim + d, c.type);
            dot = fmaf(x[i].x, k.x, fmaf(x[i].y, k.y, fmaf(x[i].z, k.z, fmaf(x[i].w, k.w, dot))));
        }
        dot = warp_sum(dot) * a.scale * (paged_is8(c.type) ? c.k_scale[row] : 1.f);
        const float top = fmaxf(m, dot), keep = top == -INFINITY ? 1.f : expf(m - top), w = top == -INFINITY ? 0.f : expf(dot - top);
        const float vw = w * (paged_is8(c.type) ? c.v_scale[row] : 1.f);
        l = l * keep + w;
        m = top;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t d = 4 * (lane + 32 * i);
            if (d >= c.dim) continue;
            const float4 v = load_cached4(c.v, row * c.dim + d, c.type);
            o[i] = make_float4(fmaf(vw, v.x, o[i].x * keep), fmaf(vw, v.y, o[i].y * keep), fmaf(vw, v.z, o[i].z * keep), fmaf(vw, v.w, o[i].w * keep));
        }
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (4 * (lane + 32 * i) < c.dim) *reinterpret_cast<float4*>(&s_o[warp][4 * (lane + 32 * i)]) = o[i];
    __syncthreads();
    const float sink = a.sink ? a.sink[h] : -INFINITY;
    float top = sink;
    for (int w = 0; w < kPaWarps; ++w) top = fmaxf(top, s_m[w]);
    float total = sink == -INFINITY ? 0.f : expf(sink - top);
    for (int w = 0; w < kPaWarps; ++w) total += s_m[w] == -INFINITY ? 0.f : s_l[w] * expf(s_m[w] - top);
    for (uint32_t d = 4 * threadIdx.x; d < c.dim; d += 4 * blockDim.x) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < kPaWarps; ++w) {
            const float f = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - top);
            if (f == 0.f) continue;
            v = make_float4(fmaf(f, s_o[w][d], v.x), fmaf(f, s_o[w][d + 1], v.y), fmaf(f, s_o[w][d + 2], v.z), fmaf(f, s_o[w][d + 3], v.w));
        }
        const float f = total == 0.f ? 0.f : 1.f / total;
        store_values4(a.out, size_t(t) * a.out_ld + size_t(h) * c.dim + d, a.out_type, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    }
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
    LV_REQUIRE(uint64_t(a->tokens) * (a->heads / a->cache.kv_heads) < (uint64_t(1) << 31), "paged attention: too many tokens");
    LV_REQUIRE(isfinite(a->scale), "paged attention: scale");
    return paged_check_rotation(a->angles, a->angle_ld, a->angle_pairs, a->cache.dim);
}

}  // namespace lv

using namespace lv;

extern "C" size_t lv_paged_attention_scratch_bytes(lv_ctx* ctx, const lv_paged_attention_args* a) {
    if (paged_attention_check(a) != LV_OK || !ctx) return 0;
    return 16;
}

extern "C" int lv_paged_attention(lv_ctx* ctx, const lv_paged_attention_args* a, void* scratch, size_t scratch_bytes) {
    if (const int rc = paged_attention_check(a)) return rc;
    LV_REQUIRE(scratch && aligned16(scratch), "paged attention: scratch is 16-byte aligned");
    LV_ENTER(ctx);
    LV_REQUIRE(scratch_bytes >= lv_paged_attention_scratch_bytes(ctx, a), "paged attention: scratch too small");
    if (!a->tokens || !a->max_new) return LV_OK;
    PagedAttn p{};
    p.a = *a;
    p.err = ctx->d_err;
    LV_CUDA(launch_pdl(ctx, paged_plain_kernel, dim3(a->heads, std::min(a->tokens, 65535u), (a->tokens + 65534u) / 65535u), dim3(32 * kPaWarps), 0, p));
    return LV_OK;
}

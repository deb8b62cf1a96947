// A cache in pages: new keys and values on their way in, rows on their way out.
//
// lv_paged_append    x' = rotated x (keys);  16 bits: x' rounded;  8 bits: a = max |x'|, scale = a / top, code = round(x' * (top / a))
// lv_paged_read      value = code * scale
//
// Both move bytes: a value is read once and written once, with a handful of operations in between.
#include "paged.cuh"

namespace lv {

struct PagedAppend {
    lv_paged_cache c;
    const void* in[2];
    const float* angles;
    uint32_t ld, angle_ld, angle_pairs, tokens;
    int in_type;
    uint32_t* err;
};

// A warp per row (token, head, key or value).  The values are asked for before the places are looked up, which is a chain of four dependent loads.
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppend p) {
    pdl_launch_dependents();
    pdl_wait();
    const lv_paged_cache& c = p.c;
    const uint32_t lane = threadIdx.x & 31u, H = c.kv_heads;
    const uint64_t job = uint64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
    if (job >= uint64_t(p.tokens) * H * 2) return;
    const uint32_t t = uint32_t(job / (2 * H)), which = uint32_t(job - uint64_t(t) * 2 * H) / H, h = uint32_t(job - uint64_t(t) * 2 * H) - which * H;
    constexpr int kParts = 2;                    // of 128 values
    float4 v[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        const uint32_t at = 4 * (lane + 32 * i);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (at < c.dim) v[i] = load_values4(p.in[which], size_t(t) * p.ld + h * c.dim + at, p.in_type);
    }
    if (which == 0 && p.angles != nullptr) {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const uint32_t at = 4 * (lane + 32 * i);
            if (at < c.dim) v[i] = rotate4(v[i], p.angles + size_t(t) * p.angle_ld, at, p.angle_pairs);
        }
    }
    const uint32_t s = paged_owner(c, t);
    PagedSeq q;
    if (s == c.seqs) return;
    uint64_t row;
    if (!paged_seq(c, s, p.tokens, &q) || !paged_row(c, c.table + size_t(s) * c.table_ld, q.len - q.n + (t - q.row0), h, &row)) {
        if (lane == 0) atomicOr(p.err, ERR_BAD_INDEX);
        return;
    }
    void* out = which ? c.v : c.k;
    if (!paged_is8(c.type)) {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            const uint32_t at = 4 * (lane + 32 * i);
            if (at < c.dim) store_values4(out, row * c.dim + at, c.type, v[i]);
        }
        return;
    }
    float a = 0.f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        a = fmaxf(fmaxf(a, fmaxf(fabsf(v[i].x), fabsf(v[i].y))), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
        fine = fine && fabsf(v[i].x) < INFINITY && fabsf(v[i].y) < INFINITY && fabsf(v[i].z) < INFINITY && fabsf(v[i].w) < INFINITY;
    }
    a = warp_max(a);
    fine = __all_sync(0xffffffffu, fine);
    const float top = c.type == LV_TYPE_I8 ? 127.f : 448.f;
    const bool live = fine && a >= kPagedTiny;
    const float f = live ? top / a : 0.f;
    if (lane == 0) (which ? c.v_scale : c.k_scale)[row] = live ? a / top : fine ? 0.f : NAN;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        const uint32_t at = 4 * (lane + 32 * i);
        if (at >= c.dim) continue;
        const float x = live ? v[i].x * f : 0.f, y = live ? v[i].y * f : 0.f, z = live ? v[i].z * f : 0.f, w = live ? v[i].w * f : 0.f;
        uint32_t u;
        if (c.type == LV_TYPE_I8) {
            u = (uint32_t(__float2int_rn(x)) & 0xffu) | ((uint32_t(__float2int_rn(y)) & 0xffu) << 8) | ((uint32_t(__float2int_rn(z)) & 0xffu) << 16) |
                (uint32_t(__float2int_rn(w)) << 24);
        } else {
            u = uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3)) |
                (uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(z, w), __NV_SATFINITE, __NV_E4M3)) << 16);
        }
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out) + row * c.dim + at) = u;
    }
}

struct PagedRead {
    lv_paged_cache c;
    void* out[2];
    int out_type;
    size_t seq_stride, head_stride, row_stride;
    uint32_t first, rows;
    uint32_t* err;
};

// A thread per 16 values of a row: a 16-byte load of codes, 32 or 64 bytes out.  Grid: (units of the rows of one head, heads x {k, v}, sequences).
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedRead p) {
    pdl_launch_dependents();
    pdl_wait();
    const lv_paged_cache& c = p.c;
    const uint32_t units = c.dim / 16, H = c.kv_heads, s = blockIdx.z, which = blockIdx.y / H, h = blockIdx.y - which * H;
    const uint32_t len = c.lens[s];
    const uint64_t job = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    const uint32_t i = uint32_t(job / units), u = uint32_t(job - uint64_t(i) * units);
    if (len > uint64_t(c.table_ld) * c.page_rows) {
        if (threadIdx.x == 0) atomicOr(p.err, ERR_BAD_INDEX);
        return;
    }
    if (i >= p.rows || p.first >= len || i >= len - p.first) return;
    uint64_t row;
    if (!paged_row(c, c.table + size_t(s) * c.table_ld, p.first + i, h, &row)) {
        atomicOr(p.err, ERR_BAD_INDEX);
        return;
    }
    const void* in = which ? c.v : c.k;
    const float f = paged_is8(c.type) ? (which ? c.v_scale : c.k_scale)[row] : 1.f;
    const size_t to = s * p.seq_stride + h * p.head_stride + i * p.row_stride + 16 * u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float4 v = load_cached4(in, row * c.dim + 16 * u + 4 * k, c.type);
        if (paged_is8(c.type)) v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
        store_values4(p.out[which], to + 4 * k, p.out_type, v);
    }
}

}  // namespace lv

using namespace lv;

extern "C" int lv_paged_locate(const lv_paged_cache* cache, const uint32_t* table_row, uint32_t position, uint32_t head, uint64_t* value_index) {
    if (const int rc = paged_check(cache)) return rc;
    LV_REQUIRE(table_row && value_index, "null argument");
    LV_REQUIRE(head < cache->kv_heads && position < uint64_t(cache->table_ld) * cache->page_rows, "paged cache: no such head or position");
    uint64_t row;
    LV_REQUIRE(paged_row(*cache, table_row, position, head, &row), "paged cache: the table names no page of the cache there");
    *value_index = row * cache->dim;
    return LV_OK;
}

extern "C" int lv_paged_append(lv_ctx* ctx, const lv_paged_cache* cache, const void* k, const void* v, int in_type, uint32_t ld, const float* angles, uint32_t angle_ld,
                               uint32_t angle_pairs, uint32_t tokens) {
    if (const int rc = paged_check(cache)) return rc;
    LV_REQUIRE(k && v && paged_value_type(in_type), "paged append: bad input");
    LV_REQUIRE(ld >= uint64_t(cache->kv_heads) * cache->dim && uint64_t(ld) * paged_bytes(in_type) % 16 == 0 && aligned16(k) && aligned16(v), "paged append: rows of k and v are 16-byte aligned");
    if (const int rc = paged_check_rotation(angles, angle_ld, angle_pairs, cache->dim)) return rc;
    const uint64_t warps = uint64_t(tokens) * cache->kv_heads * 2;
    LV_REQUIRE(warps < (uint64_t(1) << 31), "paged append: too many tokens");
    LV_ENTER(ctx);
    if (!tokens) return LV_OK;
    PagedAppend p{};
    p.c = *cache;
    p.in[0] = k;
    p.in[1] = v;
    p.angles = angles;
    p.ld = ld;
    p.angle_ld = angle_ld;
    p.angle_pairs = angle_pairs;
    p.tokens = tokens;
    p.in_type = in_type;
    p.err = ctx->d_err;
    LV_CUDA(launch_pdl(ctx, paged_append_kernel, dim3(uint32_t((warps + 7) / 8)), dim3(256), 0, p));
    return LV_OK;
}

extern "C" int lv_paged_read(lv_ctx* ctx, const lv_paged_cache* cache, void* k_out, void* v_out, int out_type, size_t seq_stride, size_t head_stride, size_t row_stride,
                             uint32_t first, uint32_t rows) {
    if (const int rc = paged_check(cache)) return rc;
    LV_REQUIRE(k_out && v_out && paged_value_type(out_type), "paged read: bad output");
    const size_t unit = 16 / paged_bytes(out_type);
    LV_REQUIRE(seq_stride % unit == 0 && head_stride % unit == 0 && row_stride % unit == 0 && aligned16(k_out) && aligned16(v_out), "paged read: rows are 16-byte aligned");
    const uint64_t blocks = (uint64_t(rows) * (cache->dim / 16) + 255) / 256;
    LV_REQUIRE(cache->kv_heads <= 32767 && blocks < (uint64_t(1) << 31), "paged read: too many heads or rows");
    LV_ENTER(ctx);
    if (!rows) return LV_OK;
    PagedRead p{};
    p.c = *cache;
    p.out[0] = k_out;
    p.out[1] = v_out;
    p.out_type = out_type;
    p.seq_stride = seq_stride;
    p.head_stride = head_stride;
    p.row_stride = row_stride;
    p.first = first;
    p.rows = rows;
    p.err = ctx->d_err;
    LV_CUDA(launch_pdl(ctx, paged_read_kernel, dim3(uint32_t(blocks), 2 * cache->kv_heads, cache->seqs), dim3(256), 0, p));
    return LV_OK;
}

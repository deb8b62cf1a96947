// A cache in pages: new keys and values on their way in, rows on their way out.
//
// lv_paged_append    x' = rotated x (keys);  16 bits: x' rounded;  8 bits: a = max |x'|, scale = a / top, code = round(x' * (top / a))
// lv_paged_read      value = code * scale
//
// Both move bytes: a value is read once and written once, with a handful of operations in between.
#include "paged.cuh"

namespace lv {

struct PagedAppend {
    PagedCache c;
    const void* in[2];
    const float* angles;
    uint32_t ld, angle_ld, angle_pairs, tokens;
    int in_type;
    uint32_t* err;
};

// A warp takes the keys or the values of four (L = 16: eight) heads of a token: L lanes a head, four values a lane and part.  All values are asked for before the
// places are looked up, which is a chain of four dependent loads, once for the heads of a warp.
// FIGURES_APPEND
constexpr int kAppendRows = 4;
template <int L, int PARTS>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppend p) {
    pdl_launch_dependents();
    pdl_wait();
    const PagedCache& c = p.c;
    constexpr uint32_t kHeads = kAppendRows * (32 / L);
    const uint32_t lane = threadIdx.x & 31u, H = c.kv_heads, groups = (H + kHeads - 1) / kHeads;
    const uint64_t job = uint64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
    const uint32_t t = uint32_t(job / (2 * groups)), in_t = uint32_t(job - uint64_t(t) * 2 * groups), which = in_t / groups, h0 = (in_t - which * groups) * kHeads + lane / L;
    if (t >= p.tokens) return;
    const uint32_t at0 = 4 * (lane % L);
    float4 v[kAppendRows][PARTS];
#pragma unroll
    for (int k = 0; k < kAppendRows; ++k)
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const uint32_t at = at0 + 4 * L * i, h = h0 + k * (32 / L);
            v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at < c.dim && h < H) v[k][i] = load_values4(p.in[which], size_t(t) * p.ld + size_t(h) * c.dim + at, p.in_type);
        }
    const uint32_t s = paged_owner(c, t);
    PagedSeq q;
    if (s == c.seqs) return;
    uint64_t row0;                                                       // of head 0
    if (!paged_seq(c, s, p.tokens, &q) || !paged_row(c, c.table + size_t(s) * c.table_ld, q.len - q.n + (t - q.row0), 0, &row0)) {
        if (lane == 0) atomicOr(p.err, ERR_BAD_INDEX);
        return;
    }
    if (which == 0 && p.angles != nullptr) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const uint32_t at = at0 + 4 * L * i;
            if (at >= c.dim) continue;
#pragma unroll
            for (int k = 0; k < kAppendRows; ++k) v[k][i] = rotate4(v[k][i], p.angles + size_t(t) * p.angle_ld, at, p.angle_pairs);
        }
    }
    void* out = which ? c.v : c.k;
    const float top = c.type == LV_TYPE_I8 ? 127.f : 448.f;
#pragma unroll
    for (int k = 0; k < kAppendRows; ++k) {
        const uint32_t h = h0 + k * (32 / L);
        const uint64_t row = row0 + uint64_t(h) * c.page_rows;
        if (!paged_is8(c.type)) {
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                const uint32_t at = at0 + 4 * L * i;
                if (at < c.dim && h < H) store_values4(out, row * c.dim + at, c.type, v[k][i]);
            }
            continue;
        }
        // the largest magnitude by its bits, which are in the order of the numbers; infinities and NaN are above all numbers
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const float4 x = v[k][i];
            most = max(most, max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu), max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu)));
        }
        if constexpr (L == 32) {
            most = __reduce_max_sync(0xffffffffu, most);
        } else {
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        const float a = __uint_as_float(most);
        const bool fine = most < 0x7f800000u, live = fine && a >= kPagedTiny;
        const float f = live ? top / a : 0.f;
        if (h >= H) continue;
        if (lane % L == 0) (which ? c.v_scale : c.k_scale)[row] = live ? a / top : fine ? 0.f : NAN;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const uint32_t at = at0 + 4 * L * i;
            if (at >= c.dim) continue;
            const float4 x = v[k][i];
            const float4 y = live ? make_float4(x.x * f, x.y * f, x.z * f, x.w * f) : make_float4(0.f, 0.f, 0.f, 0.f);
            uint32_t u;
            if (c.type == LV_TYPE_I8) {
                u = (uint32_t(__float2int_rn(y.x)) & 0xffu) | ((uint32_t(__float2int_rn(y.y)) & 0xffu) << 8) | ((uint32_t(__float2int_rn(y.z)) & 0xffu) << 16) |
                    (uint32_t(__float2int_rn(y.w)) << 24);
            } else {
                u = uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(y.x, y.y), __NV_SATFINITE, __NV_E4M3)) |
                    (uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(y.z, y.w), __NV_SATFINITE, __NV_E4M3)) << 16);
            }
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out) + row * c.dim + at) = u;
        }
    }
}

struct PagedRead {
    PagedCache c;
    void* out[2];
    int out_type;
    size_t seq_stride, head_stride, row_stride;
    uint32_t first, rows;
    uint32_t* err;
};

// A thread takes eight neighbouring values of four rows: 8 or 16 bytes in, 16 (f32: 32) out, in step with its neighbours.  Grid: (rows of one head, heads x {keys, values},
// sequences).
// FIGURES_READ
constexpr int kReadRows = 4;
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedRead p) {
    pdl_launch_dependents();
    pdl_wait();
    const PagedCache& c = p.c;
    const uint32_t units = c.dim / 8, each = blockDim.x / units, H = c.kv_heads, s = blockIdx.z, which = blockIdx.y / H, h = blockIdx.y - which * H;
    const uint32_t len = c.lens[s], i0 = threadIdx.x / units, u = threadIdx.x - i0 * units;
    if (len > uint64_t(c.table_ld) * c.page_rows) {
        if (threadIdx.x == 0) atomicOr(p.err, ERR_BAD_INDEX);
        return;
    }
    if (p.first >= len || uint64_t(blockIdx.x) * each * kReadRows >= len - p.first) return;
    const uint32_t rows = min(p.rows, len - p.first);
    const void* in = which ? c.v : c.k;
    const float* scales = which ? c.v_scale : c.k_scale;
    // the rows of a warp, looked up by a lane each: 32 / units (rounded up) of every pass
    const uint32_t lane = threadIdx.x & 31u, first_i0 = (threadIdx.x & ~31u) / units, span = (threadIdx.x | 31u) / units - first_i0 + 1;
    uint64_t row[kReadRows];
    bool here[kReadRows];
    auto look_up = [&](uint32_t k, uint32_t at, uint64_t* found) {
        const uint64_t i = uint64_t(blockIdx.x) * each * kReadRows + k * each + at;
        if (k >= kReadRows || at >= each || i >= rows) return false;
        if (paged_row(c, c.table + size_t(s) * c.table_ld, p.first + uint32_t(i), h, found)) return true;
        atomicOr(p.err, ERR_BAD_INDEX);
        return false;
    };
    if (kReadRows * span <= 32) {
        uint64_t mine = 0;
        const bool there = look_up(lane / span, first_i0 + lane % span, &mine);
        const uint32_t all_there = __ballot_sync(0xffffffffu, there);
#pragma unroll
        for (int k = 0; k < kReadRows; ++k) {
            const uint32_t from = k * span + i0 - first_i0;
            row[k] = __shfl_sync(0xffffffffu, mine, int(from));
            here[k] = ((all_there >> from) & 1u) != 0;
        }
    } else {                                                             // (heads of 16 values)
#pragma unroll
        for (int k = 0; k < kReadRows; ++k) here[k] = look_up(k, i0, &row[k]);
    }
    uint4 v[kReadRows];                                                  // eight values, or (the first two words) codes
    float f[kReadRows];
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
        if (!here[k]) continue;
        const size_t at = row[k] * c.dim + 8 * u;
        if (paged_is8(c.type)) {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(in) + at);
            v[k] = make_uint4(w.x, w.y, 0u, 0u);
            f[k] = scales[row[k]];
        } else {
            v[k] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(in) + at);
        }
    }
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
        if (!here[k]) continue;
        float4 x, y;
        if (paged_is8(c.type)) {
            x = code_values4(v[k].x, c.type);
            y = code_values4(v[k].y, c.type);
            x = make_float4(x.x * f[k], x.y * f[k], x.z * f[k], x.w * f[k]);
            y = make_float4(y.x * f[k], y.y * f[k], y.z * f[k], y.w * f[k]);
        } else {
            x = unpack_values4(make_uint2(v[k].x, v[k].y), c.type);
            y = unpack_values4(make_uint2(v[k].z, v[k].w), c.type);
        }
        const size_t to = s * p.seq_stride + h * p.head_stride + (uint64_t(blockIdx.x) * each * kReadRows + k * each + i0) * p.row_stride + 8 * u;
        if (p.out_type == LV_TYPE_F32) {
            store_values4(p.out[which], to, LV_TYPE_F32, x);
            store_values4(p.out[which], to + 4, LV_TYPE_F32, y);
        } else {
            const uint2 a = pack_values4(x, p.out_type), b = pack_values4(y, p.out_type);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out[which]) + to) = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
}

}  // namespace lv

using namespace lv;

extern "C" int lv_paged_locate(const lv_paged_cache* cache, const uint32_t* table_row, uint32_t position, uint32_t head, uint64_t* value_index) {
    if (const int rc = paged_check(cache)) return rc;
    LV_REQUIRE(table_row && value_index, "null argument");
    LV_REQUIRE(head < cache->kv_heads && position < uint64_t(cache->table_ld) * cache->page_rows, "paged cache: no such head or position");
    uint64_t row;
    LV_REQUIRE(paged_row(paged_cache(*cache), table_row, position, head, &row), "paged cache: the table names no page of the cache there");
    *value_index = row * cache->dim;
    return LV_OK;
}

extern "C" int lv_paged_append(lv_ctx* ctx, const lv_paged_cache* cache, const void* k, const void* v, int in_type, uint32_t ld, const float* angles, uint32_t angle_ld,
                               uint32_t angle_pairs, uint32_t tokens) {
    if (const int rc = paged_check(cache)) return rc;
    LV_REQUIRE(k && v && paged_value_type(in_type), "paged append: bad input");
    LV_REQUIRE(ld >= uint64_t(cache->kv_heads) * cache->dim && uint64_t(ld) * paged_bytes(in_type) % 16 == 0 && aligned16(k) && aligned16(v), "paged append: rows of k and v are 16-byte aligned");
    if (const int rc = paged_check_rotation(angles, angle_ld, angle_pairs, cache->dim)) return rc;
    const uint32_t heads = kAppendRows * (cache->dim <= 64 ? 2 : 1);
    const uint64_t warps = uint64_t(tokens) * 2 * ((cache->kv_heads + heads - 1) / heads);
    LV_REQUIRE(warps < (uint64_t(1) << 31), "paged append: too many tokens");
    LV_ENTER(ctx);
    if (!tokens) return LV_OK;
    PagedAppend p{};
    p.c = paged_cache(*cache);
    p.in[0] = k;
    p.in[1] = v;
    p.angles = angles;
    p.ld = ld;
    p.angle_ld = angle_ld;
    p.angle_pairs = angle_pairs;
    p.tokens = tokens;
    p.in_type = in_type;
    p.err = ctx->d_err;
    const dim3 grid(uint32_t((warps + 7) / 8));
    if (cache->dim <= 64) LV_CUDA(launch_pdl(ctx, paged_append_kernel<16, 1>, grid, dim3(256), 0, p));
    else if (cache->dim <= 128) LV_CUDA(launch_pdl(ctx, paged_append_kernel<32, 1>, grid, dim3(256), 0, p));
    else LV_CUDA(launch_pdl(ctx, paged_append_kernel<32, 2>, grid, dim3(256), 0, p));
    return LV_OK;
}

extern "C" int lv_paged_read(lv_ctx* ctx, const lv_paged_cache* cache, void* k_out, void* v_out, int out_type, size_t seq_stride, size_t head_stride, size_t row_stride,
                             uint32_t first, uint32_t rows) {
    if (const int rc = paged_check(cache)) return rc;
    LV_REQUIRE(k_out && v_out && paged_value_type(out_type), "paged read: bad output");
    const size_t unit = 16 / paged_bytes(out_type);
    LV_REQUIRE(seq_stride % unit == 0 && head_stride % unit == 0 && row_stride % unit == 0 && aligned16(k_out) && aligned16(v_out), "paged read: rows are 16-byte aligned");
    const uint32_t block_rows = 256 / (cache->dim / 8) * kReadRows;
    const uint64_t blocks = (uint64_t(rows) + block_rows - 1) / block_rows;
    LV_REQUIRE(cache->kv_heads <= 32767 && blocks < (uint64_t(1) << 31), "paged read: too many heads or rows");
    LV_ENTER(ctx);
    if (!rows) return LV_OK;
    PagedRead p{};
    p.c = paged_cache(*cache);
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

// A cache in pages: new keys and values on their way in, rows on their way out.
//
// lv_paged_append    x' = rotated x (keys);  16 bits: x' rounded;  8 bits: a = max |x'|, scale = a / top, code = round(x' * (top / a))
// lv_paged_read      value = code * scale
//
// Both move bytes: a value is read once and written once, with a handful of operations in between.
#include <algorithm>

#include "paged.cuh"

namespace lv {

struct PagedAppend {
    PagedCache c;
    const void* in[2];
    const float* angles;
    uint32_t ld, angle_ld, angle_pairs, tokens;
    uint32_t* err;
};

// A warp takes the keys or the values of four (L = 16: eight) heads of a token: L lanes a head, four values a lane and part.  All values are asked for before the
// places are looked up, which is a chain of four dependent loads, once for the heads of a warp.
// 8 sequences of 2048 tokens, f32 to int8, 8 heads of 128: 30.7 us, 4.4 TB/s of 135 MB (a warp per head: 72 us; four heads: 43; types known when compiled: 30); f32 to bf16 28.8, 5.6 TB/s.
// Counters of the former: issue 73 % of the busy cycles, integer pipe 46 %, memory 47 %: instructions, then loads.  One token: 4.7 us, a launch and its chain of loads.
constexpr int kAppendRows = 4;
// IN, KIND: types of the values given and stored
template <int IN, int KIND, int L, int PARTS>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppend p) {
    pdl_launch_dependents();
    pdl_wait();
    const PagedCache& c = p.c;
    constexpr uint32_t kHeads = kAppendRows * (32 / L);
    const uint32_t lane = threadIdx.x & 31u, H = c.kv_heads, groups = (H + kHeads - 1) / kHeads;
    const uint64_t job = uint64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
    const uint32_t t = uint32_t(job / (2 * groups)), in_t = uint32_t(job - uint64_t(t) * 2 * groups), which = in_t / groups, h0 = (in_t - which * groups) * kHeads + lane / L;
    // every sequence is looked at by one thread: one whose rows all lie behind the step's has no warp that would find out
    for (uint64_t s = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; s < c.seqs; s += uint64_t(gridDim.x) * blockDim.x) {
        PagedSeq q;
        if (!paged_seq(c, uint32_t(s), p.tokens, &q)) atomicOr(p.err, ERR_BAD_INDEX);
    }
    if (t >= p.tokens) return;
    const uint32_t at0 = 4 * (lane % L);
    float4 v[kAppendRows][PARTS];
#pragma unroll
    for (int k = 0; k < kAppendRows; ++k)
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const uint32_t at = at0 + 4 * L * i, h = h0 + k * (32 / L);
            v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at < c.dim && h < H) v[k][i] = load_values4(p.in[which], size_t(t) * p.ld + size_t(h) * c.dim + at, IN);
        }
    const uint32_t s = paged_owner(c, t);
    PagedSeq q;
    if (s == c.seqs) return;
    uint32_t row0;                                                       // of head 0
    if (!paged_seq(c, s, p.tokens, &q) || !paged_holds(q, t) || !paged_row(c, c.table + size_t(s) * c.table_ld, q.len - q.n + (t - q.row0), 0, &row0)) {
        if (lane == 0) atomicOr(p.err, ERR_BAD_INDEX);
        return;
    }
    if (which == 0 && p.angles != nullptr) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const uint32_t at = at0 + 4 * L * i;
            if (at >= c.dim) continue;
            if (at + 2 < 2 * p.angle_pairs) {                            // (both pairs)
                const float2 t0 = *reinterpret_cast<const float2*>(p.angles + size_t(t) * p.angle_ld + at), t1 = *reinterpret_cast<const float2*>(p.angles + size_t(t) * p.angle_ld + at + 2);
#pragma unroll
                for (int k = 0; k < kAppendRows; ++k) v[k][i] = rotate4(v[k][i], t0, t1);
            } else {
#pragma unroll
                for (int k = 0; k < kAppendRows; ++k) v[k][i] = rotate4(v[k][i], p.angles + size_t(t) * p.angle_ld, at, p.angle_pairs);
            }
        }
    }
    constexpr bool kEight = KIND == LV_TYPE_I8 || KIND == LV_TYPE_E4M3;
    uint8_t* out = static_cast<uint8_t*>(which ? c.v : c.k) + (uint64_t(row0 + h0 * c.page_rows) * c.dim + at0) * (kEight ? 1 : 2);
    const size_t step = size_t(32 / L) * c.page_rows * c.dim * (kEight ? 1 : 2);
    if constexpr (!kEight) {
#pragma unroll
        for (int k = 0; k < kAppendRows; ++k)
#pragma unroll
            for (int i = 0; i < PARTS; ++i)
                if (at0 + 4 * L * i < c.dim && h0 + k * (32 / L) < H) store_values4(out + k * step, 4 * L * i, KIND, v[k][i]);
    } else {
        constexpr float top = KIND == LV_TYPE_I8 ? 127.f : 448.f;
        // the largest magnitudes, of each row in all its lanes: bits of non-negative numbers are in their order, NaN above all
        float most[kAppendRows];
#pragma unroll
        for (int k = 0; k < kAppendRows; ++k) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) m = max_nan(max_nan(m, max_nan(fabsf(v[k][i].x), fabsf(v[k][i].y))), max_nan(fabsf(v[k][i].z), fabsf(v[k][i].w)));
            uint32_t u = __float_as_uint(m);
            if constexpr (L == 32) {
                u = __reduce_max_sync(0xffffffffu, u);
            } else {
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) u = max(u, __shfl_xor_sync(0xffffffffu, u, o));
            }
            most[k] = __uint_as_float(u);
        }
        // a lane divides for a row: the k-th of a head's lanes for its row of step k
        static_assert(kAppendRows == 4, "");
        const uint32_t mine = lane % L;
        const float a = mine & 2u ? (mine & 1u ? most[3] : most[2]) : mine & 1u ? most[1] : most[0];
        const bool fine = a < INFINITY, live = fine && a >= kPagedTiny;
        const float f = live ? top / a : 0.f;
        const uint32_t h_mine = h0 + mine * (32 / L);
        if (mine < kAppendRows && h_mine < H) (which ? c.v_scale : c.k_scale)[row0 + h_mine * c.page_rows] = live ? a / top : fine ? 0.f : NAN;
#pragma unroll
        for (int k = 0; k < kAppendRows; ++k) {
            const float g = __shfl_sync(0xffffffffu, f, int((lane & ~uint32_t(L - 1)) + k));
            if (h0 + k * (32 / L) >= H) continue;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                if (at0 + 4 * L * i >= c.dim) continue;
                // (rounded by themselves: a product that is fused with the sum below would round values between two codes otherwise)
                float4 y = make_float4(__fmul_rn(v[k][i].x, g), __fmul_rn(v[k][i].y, g), __fmul_rn(v[k][i].z, g), __fmul_rn(v[k][i].w, g));
                if (g == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);       // (times infinity or NaN)
                uint32_t u;
                if constexpr (KIND == LV_TYPE_I8) {
                    // 1.5 2^23 + y: the sum's rounding to whole numbers (ties to even) is the code's, its low byte the code
                    constexpr float kWhole = 12582912.f;
                    u = __byte_perm(__byte_perm(__float_as_uint(y.x + kWhole), __float_as_uint(y.y + kWhole), 0x0040), __byte_perm(__float_as_uint(y.z + kWhole), __float_as_uint(y.w + kWhole), 0x0040), 0x5410);
                } else {
                    u = uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(y.x, y.y), __NV_SATFINITE, __NV_E4M3)) |
                        (uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(y.z, y.w), __NV_SATFINITE, __NV_E4M3)) << 16);
                }
                *reinterpret_cast<uint32_t*>(out + k * step + 4 * L * i) = u;
            }
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
// e4m3 to bf16, 8 sequences of 3000 to 20000 positions: 115 us, 5.9 TB/s of 675 MB (one row a thread: 229 us; four: 166; the row's place by multiplication instead of division: 139; types
// known when compiled: 117).  int8 to f16, 1531 positions of 32 heads: 8.7 us of which 5.8 are the memory's.
constexpr int kReadRows = 4;
template <int KIND, int OUT>
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
    constexpr bool kEight = KIND == LV_TYPE_I8 || KIND == LV_TYPE_E4M3;
    uint32_t row[kReadRows];
    bool here[kReadRows];
    auto look_up = [&](uint32_t k, uint32_t at, uint32_t* found) {
        const uint64_t i = uint64_t(blockIdx.x) * each * kReadRows + k * each + at;
        if (k >= kReadRows || at >= each || i >= rows) return false;
        if (paged_row(c, c.table + size_t(s) * c.table_ld, p.first + uint32_t(i), h, found)) return true;
        atomicOr(p.err, ERR_BAD_INDEX);
        return false;
    };
    if (kReadRows * span <= 32) {
        uint32_t mine = 0;
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
        const size_t at = uint64_t(row[k]) * c.dim + 8 * u;
        if constexpr (kEight) {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(in) + at);
            v[k] = make_uint4(w.x, w.y, 0u, 0u);
            f[k] = scales[row[k]];
        } else {
            v[k] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(in) + at);
        }
    }
    const size_t step = each * p.row_stride, base = s * p.seq_stride + h * p.head_stride + (uint64_t(blockIdx.x) * each * kReadRows + i0) * p.row_stride + 8 * u;
#pragma unroll
    for (int k = 0; k < kReadRows; ++k) {
        if (!here[k]) continue;
        float4 x, y;
        if constexpr (kEight) {
            x = code_values4(v[k].x, KIND);
            y = code_values4(v[k].y, KIND);
            x = make_float4(x.x * f[k], x.y * f[k], x.z * f[k], x.w * f[k]);
            y = make_float4(y.x * f[k], y.y * f[k], y.z * f[k], y.w * f[k]);
        } else {
            x = unpack_values4(make_uint2(v[k].x, v[k].y), KIND);
            y = unpack_values4(make_uint2(v[k].z, v[k].w), KIND);
        }
        const size_t to = base + k * step;
        if constexpr (OUT == LV_TYPE_F32) {
            store_values4(p.out[which], to, LV_TYPE_F32, x);
            store_values4(p.out[which], to + 4, LV_TYPE_F32, y);
        } else {
            const uint2 a = pack_values4(x, OUT), b = pack_values4(y, OUT);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out[which]) + to) = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
}

template <int IN, int KIND>
static int append_launch(lv_ctx* ctx, const PagedAppend& p, dim3 grid) {
    if (p.c.dim <= 64) LV_CUDA(launch_pdl(ctx, paged_append_kernel<IN, KIND, 16, 1>, grid, dim3(256), 0, p));
    else if (p.c.dim <= 128) LV_CUDA(launch_pdl(ctx, paged_append_kernel<IN, KIND, 32, 1>, grid, dim3(256), 0, p));
    else LV_CUDA(launch_pdl(ctx, paged_append_kernel<IN, KIND, 32, 2>, grid, dim3(256), 0, p));
    return LV_OK;
}
template <int IN>
static int append_launch_from(lv_ctx* ctx, const PagedAppend& p, dim3 grid) {
    switch (p.c.type) {
        case LV_TYPE_F16: return append_launch<IN, LV_TYPE_F16>(ctx, p, grid);
        case LV_TYPE_BF16: return append_launch<IN, LV_TYPE_BF16>(ctx, p, grid);
        case LV_TYPE_I8: return append_launch<IN, LV_TYPE_I8>(ctx, p, grid);
        default: return append_launch<IN, LV_TYPE_E4M3>(ctx, p, grid);
    }
}
template <int KIND>
static int read_launch_from(lv_ctx* ctx, const PagedRead& p, dim3 grid) {
    switch (p.out_type) {
        case LV_TYPE_F32: LV_CUDA(launch_pdl(ctx, paged_read_kernel<KIND, LV_TYPE_F32>, grid, dim3(256), 0, p)); break;
        case LV_TYPE_F16: LV_CUDA(launch_pdl(ctx, paged_read_kernel<KIND, LV_TYPE_F16>, grid, dim3(256), 0, p)); break;
        default: LV_CUDA(launch_pdl(ctx, paged_read_kernel<KIND, LV_TYPE_BF16>, grid, dim3(256), 0, p)); break;
    }
    return LV_OK;
}

}  // namespace lv

using namespace lv;

extern "C" int lv_paged_locate(const lv_paged_cache* cache, const uint32_t* table_row, uint32_t position, uint32_t head, uint64_t* value_index) {
    if (const int rc = paged_check(cache)) return rc;
    LV_REQUIRE(table_row && value_index, "null argument");
    LV_REQUIRE(head < cache->kv_heads && position < uint64_t(cache->table_ld) * cache->page_rows, "paged cache: no such head or position");
    uint32_t row;
    LV_REQUIRE(paged_row(paged_cache(*cache), table_row, position, head, &row), "paged cache: the table names no page of the cache there");
    *value_index = uint64_t(row) * cache->dim;
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
    PagedAppend p{};
    p.c = paged_cache(*cache);
    p.in[0] = k;
    p.in[1] = v;
    p.angles = angles;
    p.ld = ld;
    p.angle_ld = angle_ld;
    p.angle_pairs = angle_pairs;
    p.tokens = tokens;
    p.err = ctx->data_err();
    const dim3 grid(std::max(1u, uint32_t((warps + 7) / 8)));            // (without rows the sequences are looked at all the same)
    switch (in_type) {
        case LV_TYPE_F32: return append_launch_from<LV_TYPE_F32>(ctx, p, grid);
        case LV_TYPE_F16: return append_launch_from<LV_TYPE_F16>(ctx, p, grid);
        default: return append_launch_from<LV_TYPE_BF16>(ctx, p, grid);
    }
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
    p.err = ctx->data_err();
    const dim3 grid(uint32_t(blocks), 2 * cache->kv_heads, cache->seqs);
    switch (cache->type) {
        case LV_TYPE_F16: return read_launch_from<LV_TYPE_F16>(ctx, p, grid);
        case LV_TYPE_BF16: return read_launch_from<LV_TYPE_BF16>(ctx, p, grid);
        case LV_TYPE_I8: return read_launch_from<LV_TYPE_I8>(ctx, p, grid);
        default: return read_launch_from<LV_TYPE_E4M3>(ctx, p, grid);
    }
}

// What the kernels of a paged cache share: where a row lies, which sequence a token belongs to, and the types that values come in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>

#include "../../include/lv_b200.h"
#include "common.cuh"
#include "ctx.h"

namespace lv {

constexpr float kPagedTiny = 0x1p-100f;          // rows whose largest magnitude is below are stored as zeros

// n / d for n < 2^31: (n * mul) >> (31 + shift) with shift = ceil(log2 d) and mul = ceil(2^(31 + shift) / d), which has 32 bits.  Exact: mul * d exceeds
// 2^(31 + shift) by less than d, so that n * mul / 2^(31 + shift) exceeds n / d by less than n / 2^(31 + shift) < 2^-shift <= 1 / d.
struct PagedDiv {
    uint32_t mul, shift;
};
inline PagedDiv paged_div(uint32_t d) {
    uint32_t shift = 0;
    while ((uint64_t(1) << shift) < d) ++shift;
    return {uint32_t(((uint64_t(1) << (31 + shift)) + d - 1) / d), shift};
}

// A cache as the kernels get it
struct PagedCache : lv_paged_cache {
    PagedDiv by_rows;                            // a position's page
};
inline PagedCache paged_cache(const lv_paged_cache& c) {
    PagedCache p{};
    static_cast<lv_paged_cache&>(p) = c;
    p.by_rows = paged_div(c.page_rows);
    return p;
}

// Entry of a sequence's table row that a position lies in
__host__ __device__ __forceinline__ uint32_t paged_slot(const PagedCache& c, uint32_t position) { return uint32_t((uint64_t(position) * c.by_rows.mul) >> (31 + c.by_rows.shift)); }

// Row (of k or v, and of the scales) of a head's position; false: the table names no page of the cache.  A cache has fewer than 2^32 rows, whose bytes need 64 bits.
__host__ __device__ __forceinline__ bool paged_row(const PagedCache& c, const uint32_t* table_row, uint32_t position, uint32_t head, uint32_t* row) {
    const uint32_t slot = paged_slot(c, position), page = slot < c.table_ld ? table_row[slot] : c.pages;
    *row = (page * c.kv_heads + head) * c.page_rows + (position - slot * c.page_rows);
    return page < c.pages;
}

// New rows and length of a sequence; false: they contradict each other, the step's rows or the table.
struct PagedSeq {
    uint32_t row0, n, len;
};
__device__ __forceinline__ bool paged_seq(const lv_paged_cache& c, uint32_t s, uint32_t tokens, PagedSeq* out) {
    const uint32_t a = c.starts[s], b = c.starts[s + 1], len = c.lens[s];
    out->row0 = a;
    out->n = b - a;
    out->len = len;
    return a <= b && b <= tokens && b - a <= len && len <= uint64_t(c.table_ld) * c.page_rows;
}

// The sequence of row t: the last s with starts[s] <= t (seqs: t belongs to nobody); for a whole warp, 32 places at a time.  Ends for any contents of starts, but where
// they decrease its answer need not hold t: paged_holds tells.
__device__ __forceinline__ uint32_t paged_owner(const lv_paged_cache& c, uint32_t t) {
    const uint32_t lane = threadIdx.x & 31u, end = c.starts[c.seqs];
    uint32_t lo = 0, n = c.seqs;                 // of the places lo .. lo + n - 1
    while (true) {
        const uint32_t step = (n + 31) / 32;
        const uint32_t below = __ballot_sync(0xffffffffu, lane * step < n && c.starts[lo + lane * step] <= t);
        if (below == 0) return c.seqs;           // (in front of the first)
        const uint32_t last = uint32_t(__popc(below)) - 1;
        lo += last * step;
        n = min(step, n - last * step);
        if (step == 1) break;
    }
    return t < end ? lo : c.seqs;
}

__device__ __forceinline__ bool paged_holds(const PagedSeq& q, uint32_t t) { return t - q.row0 < q.n; }

__host__ __device__ __forceinline__ bool paged_is8(int type) { return type == LV_TYPE_I8 || type == LV_TYPE_E4M3; }
__host__ __device__ __forceinline__ uint32_t paged_bytes(int type) { return type == LV_TYPE_F32 ? 4u : paged_is8(type) ? 1u : 2u; }
inline bool paged_value_type(int type) { return type == LV_TYPE_F32 || type == LV_TYPE_F16 || type == LV_TYPE_BF16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
template <typename... P>
inline bool words_aligned(const P*... p) { return ((... | reinterpret_cast<uintptr_t>(p)) & 3u) == 0; }

// Four consecutive values of type f32, f16 or bf16 (the type is the same for a whole launch)
__device__ __forceinline__ float4 unpack_values4(uint2 u, int type) {
    float2 a, b;
    if (type == LV_TYPE_BF16) {
        a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
        b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    } else {
        a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
        b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    }
    return make_float4(a.x, a.y, b.x, b.y);
}
// as they lie in memory, to be unpacked behind the loads of several: a conversion in the branch of a load would make each wait for the one before
__device__ __forceinline__ uint4 load_raw4(const void* p, size_t at, int type) {
    if (type == LV_TYPE_F32) return *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + at);
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at);
    return make_uint4(u.x, u.y, 0u, 0u);
}
__device__ __forceinline__ float4 unpack_raw4(uint4 u, int type) {
    if (type == LV_TYPE_F32) return make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
    return unpack_values4(make_uint2(u.x, u.y), type);
}
__device__ __forceinline__ float4 load_values4(const void* p, size_t at, int type) {
    if (type == LV_TYPE_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    return unpack_values4(*reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at), type);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint2 pack_values4(const float4& v, int type) {
    return type == LV_TYPE_BF16 ? make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w)) : make_uint2(pack_f16(v.x, v.y), pack_f16(v.z, v.w));
}
__device__ __forceinline__ void store_values4(void* p, size_t at, int type, const float4& v) {
    if (type == LV_TYPE_F32) *reinterpret_cast<float4*>(static_cast<float*>(p) + at) = v;
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + at) = pack_values4(v, type);
}

// Values of a cache row; 8-bit codes come as whole numbers or e4m3 values, without their scale
__device__ __forceinline__ float4 code_values4(uint32_t u, int type) {
    if (type == LV_TYPE_I8)
        return make_float4(float(int8_t(u & 0xffu)), float(int8_t((u >> 8) & 0xffu)), float(int8_t((u >> 16) & 0xffu)), float(int8_t(u >> 24)));
    const float2 a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(u & 0xffffu), __NV_E4M3)));
    const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(u >> 16), __NV_E4M3)));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Two pairs of a head's vector turned by {cos, sin}: every product and sum rounded by itself, so that the codes that a rotated key is stored as are the same
// wherever it is rotated
__device__ __forceinline__ float4 rotate4(float4 v, float2 t0, float2 t1) {
    return make_float4(__fsub_rn(__fmul_rn(v.x, t0.x), __fmul_rn(v.y, t0.y)), __fadd_rn(__fmul_rn(v.y, t0.x), __fmul_rn(v.x, t0.y)),
                       __fsub_rn(__fmul_rn(v.z, t1.x), __fmul_rn(v.w, t1.y)), __fadd_rn(__fmul_rn(v.w, t1.x), __fmul_rn(v.z, t1.y)));
}
// values c .. c + 3 by a token's angles
__device__ __forceinline__ float4 rotate4(float4 v, const float* angles, uint32_t c, uint32_t pairs) {
    const float2 still = make_float2(1.f, 0.f);
    const float2 t0 = c < 2 * pairs ? *reinterpret_cast<const float2*>(angles + c) : still, t1 = c + 2 < 2 * pairs ? *reinterpret_cast<const float2*>(angles + c + 2) : still;
    const float4 u = rotate4(v, t0, t1);
    // (a value that is not turned is not multiplied either)
    return make_float4(c < 2 * pairs ? u.x : v.x, c < 2 * pairs ? u.y : v.y, c + 2 < 2 * pairs ? u.z : v.z, c + 2 < 2 * pairs ? u.w : v.w);
}

// What is wrong with a cache's description (LV_OK: nothing)
inline int paged_check(const lv_paged_cache* c) {
    LV_REQUIRE(c && c->k && c->v && c->table && c->lens && c->starts, "paged cache: null argument");
    LV_REQUIRE(c->type == LV_TYPE_F16 || c->type == LV_TYPE_BF16 || paged_is8(c->type), "paged cache: unsupported type");
    LV_REQUIRE(!paged_is8(c->type) || (c->k_scale && c->v_scale), "paged cache: 8-bit values need scales");
    LV_REQUIRE(c->dim && c->dim % 16 == 0 && c->dim <= 256, "paged cache: head size");
    LV_REQUIRE(c->pages && c->page_rows && c->kv_heads && c->kv_heads <= 65535 && c->table_ld && c->seqs && c->seqs <= 65535, "paged cache: bad sizes");
    LV_REQUIRE(uint64_t(c->table_ld) * c->page_rows <= 0x7fffffffull, "paged cache: positions of a sequence are below 2^31");
    LV_REQUIRE(uint64_t(c->pages) * c->page_rows <= 0xffffffffull && uint64_t(c->pages) * c->page_rows * c->kv_heads <= 0xffffffffull, "paged cache: rows are below 2^32");
    LV_REQUIRE(aligned16(c->k) && aligned16(c->v), "paged cache: k and v are 16-byte aligned");
    LV_REQUIRE(words_aligned(c->table, c->lens, c->starts) && (!paged_is8(c->type) || words_aligned(c->k_scale, c->v_scale)), "paged cache: 32-bit values are 4-byte aligned");
    return LV_OK;
}
inline int paged_check_rotation(const float* angles, uint32_t angle_ld, uint32_t angle_pairs, uint32_t dim) {
    LV_REQUIRE(!angles || (angle_pairs <= dim / 2 && angle_ld >= 2 * angle_pairs && angle_ld % 2 == 0 && (reinterpret_cast<uintptr_t>(angles) & 7u) == 0), "paged cache: bad angles");
    return LV_OK;
}

}  // namespace lv

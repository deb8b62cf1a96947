// Pieces of the two kernels of the attention over pages: what they are given, the rows that a sequence's new tokens are, and partial results.
#pragma once

#include <float.h>

#include "paged.cuh"

namespace lv {

constexpr float kPaLog2e = 1.4426950408889634f;
// Weights are e^(s - r) with a reference r that is 2^kPaLift below a row's maximum: the largest are near 2^kPaLift, so that f16 weights have their full
// precision down to 2^-24 of the largest (rounding to f16 starts to lose bits below 2^-14)
constexpr float kPaLift = 10.f;
// A new maximum becomes the reference when it is above the old one by more than this (log2): then weights stay below 2^(kPaLift + kPaStep + 1) < 65504
constexpr float kPaStep = 4.f;

// Rows of a block, keys of a step, and time of a CTA beside its steps (in steps), of the kernel for many rows.  (3 for the last chooses the same splits on twelve points, 12 worse ones on
// two: prompts of 300 tokens behind 4000 positions 97 us against 69.)
constexpr int kPtRows = 256, kPtKeys = 128, kPtSetUp = 6;

struct PagedAttn {
    lv_paged_attention_args a;
    PagedCache c;                // a.cache
    uint32_t group;              // query heads of a key/value head
    uint32_t chunk, splits;      // keys of a split (from the first key that a block of rows sees on), upper bound of the splits
    uint32_t align;              // splits begin at the block's first key with these bits cleared
    uint32_t box;                // rows of a TMA box (the kernel for many rows)
    float factor;                // the scale in log2 units
    float* part_o;               // [token][head][split][dim]: sums of the splits
    float2* part_rl;             // [token][head][split]: reference and sum of weights
    uint32_t *err, *data_err;    // of waits; of what sequences contain
};

// The keys that rows r0 .. r1 (of a sequence's n * group; row r is query head r mod group of new token r / group) see: lo .. hi - 1
struct PagedRange {
    uint32_t lo, hi;
};
__device__ __forceinline__ uint32_t paged_first_key(uint32_t position, uint32_t window) { return window != 0 && position + 1 > window ? position + 1 - window : 0; }
__device__ __forceinline__ PagedRange paged_range(const PagedAttn& p, const PagedSeq& q, uint32_t r0, uint32_t r1) {
    const uint32_t before = q.len - q.n;
    return {paged_first_key(before + r0 / p.group, p.a.window), before + r1 / p.group + 1};
}

// A sequence of the launch; false (reported): it contradicts itself or the stated bounds
__device__ __forceinline__ bool paged_attention_seq(const PagedAttn& p, uint32_t s, PagedSeq* q) {
    if (paged_seq(p.c, s, p.a.tokens, q) && q->n <= p.a.max_new && q->len <= p.a.max_len) return true;
    if (threadIdx.x == 0) atomicOr(p.data_err, ERR_BAD_INDEX);
    return false;
}

// What a row's products are multiplied by: the scale in log2 units, over the power of two of the row's queries.  Above zero and finite, so that it times zero is zero and times
// -infinity is that
__host__ __device__ __forceinline__ float paged_factor(float scale, float unit) { return fminf(fmaxf(scale / unit, 0x1p-149f), FLT_MAX); }

// the weight of a head's sink, and the least reference that it fits under
__device__ __forceinline__ float paged_sink(const PagedAttn& p, uint32_t head) { return p.a.sink ? p.a.sink[head] * kPaLog2e : -INFINITY; }
__device__ __forceinline__ float paged_sink_weight(float sink, float ref) { return sink == -INFINITY ? 0.f : exp2_fast(sink - ref); }

// paged_attention_rows.cuh: blocks of 8, 16, 24 or 32 rows (heads of more than 128 values: 8 or 16)
constexpr int kPrWarps = 4, kPrKeys16 = 16, kPrKeys8 = 32;          // warps; keys of a slice
int paged_rows_launch_bf16(lv_ctx* ctx, const PagedAttn& p, uint32_t rows, uint32_t blocks);
int paged_rows_launch_f16(lv_ctx* ctx, const PagedAttn& p, uint32_t rows, uint32_t blocks);
int paged_rows_launch_i8(lv_ctx* ctx, const PagedAttn& p, uint32_t rows, uint32_t blocks);
int paged_rows_launch_e4m3(lv_ctx* ctx, const PagedAttn& p, uint32_t rows, uint32_t blocks);

// paged_attention_tc.cu: blocks of kPtRows rows, 16-bit outputs, heads of up to 128 values
int paged_tc_launch(lv_ctx* ctx, const PagedAttn& p, uint32_t blocks);

// Value pairs as 16-bit operands, and two codes (the low or the high half of a word) as f16
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    return BF16 ? pack_bf16(lo, hi) : pack_f16(lo, hi);
}
template <int KIND>
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, bool high) {
    if constexpr (KIND == LV_TYPE_I8) {
        // 0x64xx is 1024 + xx in f16; the codes' sign bits are flipped before (128 + code)
        const uint32_t u = __byte_perm(w, 0x64646464u, high ? 0x4342u : 0x4140u);
        const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1152.f, 1152.f));
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        uint32_t v;
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(v) : "r"(high ? w >> 16 : w));
        return v;
    }
}

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async4_zfill(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 2^-e of a row's largest magnitude (f16 queries are divided by 2^e; rows below 2^-63 have no scores to speak of), and the exponent field of a value's scale (0 for one that is not finite)
__device__ __forceinline__ float paged_row_unit(float top) { return __uint_as_float((254u - min(max(__float_as_uint(top) >> 23, 64u), 253u)) << 23); }
__device__ __forceinline__ uint32_t paged_scale_exponent(float scale) {
    const uint32_t e = (__float_as_uint(scale) >> 23) & 255u;
    return e == 255u ? 0u : e;
}
// what outputs in units of 2^(from - 127) are multiplied by when the unit becomes 2^(to - 127); from 0: there are none yet
__device__ __forceinline__ float paged_unit_step(uint32_t from, uint32_t to) { return from == 0 ? 1.f : __uint_as_float((127u - min(to - from, 126u)) << 23); }

}  // namespace lv

// Pieces of the two kernels of the attention over pages: what they are given, the rows that a sequence's new tokens are, and partial results.
#pragma once

#include "paged.cuh"

namespace lv {

constexpr float kPaLog2e = 1.4426950408889634f;
// Weights are e^(s - r) with a reference r that is 2^kPaLift below a row's maximum: the largest are near 2^kPaLift, so that f16 weights have their full
// precision down to 2^-24 of the largest (rounding to f16 starts to lose bits below 2^-14)
constexpr float kPaLift = 10.f;
// A new maximum becomes the reference when it is above the old one by more than this (log2): then weights stay below 2^(kPaLift + kPaStep + 1) < 65504
constexpr float kPaStep = 4.f;

struct PagedAttn {
    lv_paged_attention_args a;
    uint32_t group;              // query heads of a key/value head
    uint32_t chunk, splits;      // keys of a split (from the first key that a block of rows sees), upper bound of the splits
    float* part_o;               // [token][head][split][dim]: sums of the splits
    float2* part_rl;             // [token][head][split]: reference and sum of weights
    uint32_t* err;
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
    if (paged_seq(p.a.cache, s, p.a.tokens, q) && q->n <= p.a.max_new && q->len <= p.a.max_len) return true;
    if (threadIdx.x == 0) atomicOr(p.err, ERR_BAD_INDEX);
    return false;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the weight of a head's sink, and the least reference that it fits under
__device__ __forceinline__ float paged_sink(const PagedAttn& p, uint32_t head) { return p.a.sink ? p.a.sink[head] * kPaLog2e : -INFINITY; }
__device__ __forceinline__ float paged_sink_weight(float sink, float ref) { return sink == -INFINITY ? 0.f : exp2_fast(sink - ref); }

}  // namespace lv

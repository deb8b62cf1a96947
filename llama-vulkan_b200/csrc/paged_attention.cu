// Attention of new tokens over a cache in pages: the kernel for few rows, and the joining of split contexts.
//
//   s_j = scale (q . k_j),  r = max_j s_j - lift,  w_j = 2^(s_j - r),  out = sum_j w_j v_j / (2^(sink - r) + sum_j w_j)      (s in log2 units)
//
// A key/value row is read for all query heads and new tokens that share it: the rows of a block are (token, head) pairs.  One token of 4 grouped
// heads does 8 operations per byte of a 16-bit cache, so the kernel is bound by memory, and what counts is that enough bytes are on
// their way: every warp has a ring of its own, filled by 16-byte cp.async (the page of a row is looked up by one lane a slice ahead), and takes slices of 16 or 32
// keys by itself -- running maximum, sum and output are the warp's, nothing in the loop waits for another warp.  The four warps meet at the end.
//
// The products are mma.sync m16n8k16: 16 rows are a whole instruction, a tcgen05 tile would be seven eighths empty.  Operands: bf16 for bf16 caches, else f16;
// 8-bit codes are exact in f16, their scales multiply the finished scores and the weights.  For f32 outputs queries and weights enter as two 16-bit numbers each (high and low
// part, 16 or 22 bits together), for 16-bit outputs as one: their rounding is half a step of the output's type at most.
// f16 operands: a query row is divided by a power of two (its largest value is near 1), and the scales of the values by the power of two of the largest so
// far, so that neither overflows nor loses bits.
#include <algorithm>

#include "paged_attention.cuh"

namespace lv {

constexpr int kPrWarps = 4, kPrStages = 2, kPrKeys8 = 32, kPrCtas = 3, kPrRounds = 8;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// what the rounding to 16 bits has left of two values, rounded in its turn
template <bool BF16>
__device__ __forceinline__ uint32_t pack16_rest(float lo, float hi, uint32_t rounded) {
    float2 r;
    if constexpr (BF16) r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&rounded));
    else r = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
    return pack16<BF16>(lo - r.x, hi - r.y);
}

// KIND: type of the cache; D: head size rounded up to 64, 128 or 256; EXACT: two 16-bit numbers per query value and weight; MT: blocks of 16 rows
template <int KIND, int D, bool EXACT, int MT>
struct RowsShape {
    static constexpr bool kEight = KIND == LV_TYPE_I8 || KIND == LV_TYPE_E4M3, kBf16 = KIND == LV_TYPE_BF16;
    static constexpr int kKeys = kEight ? kPrKeys8 : 16;                      // of a slice
    static constexpr int kRowBytes = kEight ? D : 2 * D, kUnits = kRowBytes / 16;
    static constexpr int kHalf = kKeys * kRowBytes;                      // bytes of the keys (or values) of a slice
    static constexpr int kStage = 2 * kHalf + (kEight ? 2 * kKeys * 4 : 0);
    static constexpr int kPlanes = EXACT ? 2 : 1, kRows = 16 * MT;
    static constexpr int kQ = kPlanes * kRows * D * 2;
    static constexpr int kRing = kPrWarps * kPrStages * kStage, kMerge = kPrWarps * kRows * D * 4;
    static constexpr int kSmem = kQ + (kRing > kMerge ? kRing : kMerge);
    // where 16-byte unit u of row r lies: the eight rows that one phase of an ldmatrix takes (16 bits), or the two keys, or the four values of one
    // phase of a 16-byte load (8 bits), fall into different banks
    __device__ static uint32_t at(uint32_t r, uint32_t u) {
        if constexpr (!kEight) return r * kRowBytes + ((u ^ (r & 7u)) << 4);
        else if constexpr (D == 64) return (r >> 1) * 128u + (((((r & 1u) << 2) | u) ^ (((r >> 1) & 3u) << 1)) << 4);
        else return r * kRowBytes + ((u ^ (r & 6u) ^ ((r & 1u) << 2)) << 4);
    }
    // column of a query value among the operand's, so that a thread's 16 bytes of an 8-bit key are its part of four instructions
    __device__ static uint32_t column(uint32_t d) {
        if constexpr (!kEight) return d;
        else return (d & ~63u) + 16 * ((d >> 2) & 3u) + ((d & 2u) << 2) + 2 * ((d >> 4) & 3u) + (d & 1u);
    }
};

// place of value d of row r where the warps' outputs meet: 16-byte units moved so that a store by eight rows and four columns falls into different banks
__device__ __forceinline__ uint32_t merged_at(uint32_t r, uint32_t d) {
    const uint32_t unit = d >> 2;
    return ((unit ^ (((unit >> 3) * 2 + r) & 7u)) << 2) + (d & 3u);
}

template <int KIND, int D, bool EXACT, int MT>
__global__ void __launch_bounds__(32 * kPrWarps, D <= 128 ? (MT == 1 ? kPrCtas : 2) : 1) paged_rows_kernel(const PagedAttn p) {
    using S = RowsShape<KIND, D, EXACT, MT>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_factor[S::kRows], s_ref[kPrWarps][S::kRows], s_l[kPrWarps][S::kRows];
    __shared__ uint32_t s_valid[kPrWarps][kPrStages];
    pdl_launch_dependents();
    pdl_wait();
    const lv_paged_attention_args& a = p.a;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, tq = lane & 3;
    const uint32_t split = blockIdx.x % p.splits, kv = blockIdx.y, r0 = blockIdx.x / p.splits * S::kRows;
    PagedSeq q;
    if (!paged_attention_seq(p, blockIdx.z, &q) || r0 >= q.n * p.group) return;
    const uint32_t rows = min(uint32_t(S::kRows), q.n * p.group - r0);
    const PagedRange all = paged_range(p, q, r0, r0 + rows - 1);
    const uint64_t begin = uint64_t(all.lo) + uint64_t(split) * p.chunk;
    if (begin >= all.hi) return;
    const uint32_t lo = uint32_t(begin), hi = uint32_t(min(uint64_t(all.hi), begin + p.chunk));
    const uint32_t* table = c.table + size_t(blockIdx.z) * c.table_ld;
    const uint32_t row_bytes = c.dim * (S::kEight ? 1u : 2u);

    // ---- the ring: slices warp, warp + 4, .. of the split ----
    uint8_t* ring = smem + S::kQ + warp * kPrStages * S::kStage;
    const uint32_t ring_at = smem_u32(ring);
    uint32_t next_row = 0;
    bool next_there = false;
    auto look_up = [&](uint32_t slice) {                                 // a lane per key
        const uint64_t j = uint64_t(lo) + uint64_t(slice) * S::kKeys + lane;
        next_there = lane < S::kKeys && j < hi;
        if (next_there && !paged_row(c, table, uint32_t(j), kv, &next_row)) {
            atomicOr(p.err, ERR_BAD_INDEX);
            next_there = false;
        }
        if (!next_there) next_row = 0;
    };
    // a lane copies the same unit of every row that is its
    constexpr int kPer = S::kKeys * S::kUnits / 32;                      // units of keys, and of values, per lane
    const uint32_t my_unit = lane % S::kUnits;
    const uint8_t *my_k = static_cast<const uint8_t*>(c.k) + my_unit * 16, *my_v = static_cast<const uint8_t*>(c.v) + my_unit * 16;
    const bool my_part = my_unit * 16 < row_bytes;
    auto issue = [&](uint32_t stage) {
        const uint32_t to = ring_at + stage * S::kStage;
        const uint32_t there = __ballot_sync(0xffffffffu, next_there);
        if (lane == 0) s_valid[warp][stage] = there;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t r = (lane + 32 * i) / S::kUnits;
            const uint64_t from = uint64_t(__shfl_sync(0xffffffffu, next_row, int(r))) * row_bytes;
            const bool here = ((there >> r) & 1u) != 0 && my_part;
            cp_async16_zfill(to + S::at(r, my_unit), here ? my_k + from : static_cast<const uint8_t*>(c.k), here);
            cp_async16_zfill(to + S::kHalf + S::at(r, my_unit), here ? my_v + from : static_cast<const uint8_t*>(c.v), here);
        }
        if constexpr (S::kEight) {
            if (S::kKeys == 32 || lane < S::kKeys) {
                cp_async4_zfill(to + 2 * S::kHalf + 4 * lane, c.k_scale + next_row, next_there);
                cp_async4_zfill(to + 2 * S::kHalf + 4 * (S::kKeys + lane), c.v_scale + next_row, next_there);
            }
        }
    };
    const uint32_t slices = (hi - lo + S::kKeys - 1) / S::kKeys;
    look_up(warp);
#pragma unroll
    for (int i = 0; i < kPrStages - 1; ++i) {
        if (warp + kPrWarps * i < slices) issue(i);
        look_up(warp + kPrWarps * (i + 1));
        cp_async_commit();
    }

    // ---- queries: rotated, divided by a power of two, in one or two 16-bit planes; all of a warp's rows are asked for at once ----
    {
        constexpr int kParts = D == 256 ? 2 : 1, kOwn = S::kRows / kPrWarps;
        float4 x[kOwn][kParts];
        float2 turn[kOwn][kParts][2];
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const uint32_t r = warp + kPrWarps * k, t = q.row0 + (r0 + r) / p.group, h = kv * p.group + (r0 + r) % p.group;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const uint32_t d = 4 * (lane + 32 * i);
                const bool here = r < rows && d < c.dim;
                x[k][i] = here ? load_values4(a.q, size_t(t) * a.q_ld + size_t(h) * c.dim + d, a.q_type) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    turn[k][i][e] = here && a.angles != nullptr && d + 2 * e < 2 * a.angle_pairs ? *reinterpret_cast<const float2*>(a.angles + size_t(t) * a.angle_ld + d + 2 * e) : make_float2(1.f, 0.f);
            }
        }
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const uint32_t r = warp + kPrWarps * k;
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                if (a.angles != nullptr) x[k][i] = rotate4(x[k][i], turn[k][i][0], turn[k][i][1]);
                top = fmaxf(fmaxf(top, fmaxf(fabsf(x[k][i].x), fabsf(x[k][i].y))), fmaxf(fabsf(x[k][i].z), fabsf(x[k][i].w)));
            }
            float f = 1.f;                                               // 2^-e of the largest value (f16 operands)
            if constexpr (!S::kBf16) f = paged_row_unit(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))));
            if (lane == 0) s_factor[r] = a.scale * kPaLog2e / f;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const uint32_t d = 4 * (lane + 32 * i);
                if (d >= D) continue;
                const float v[4] = {x[k][i].x * f, x[k][i].y * f, x[k][i].z * f, x[k][i].w * f};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t col = S::column(d + 2 * e), at = r * (2 * D) + (((col >> 3) ^ (r & 7u)) << 4) + (col & 7u) * 2;
                    const uint32_t u = pack16<S::kBf16>(v[2 * e], v[2 * e + 1]);
                    *reinterpret_cast<uint32_t*>(smem + at) = u;
                    if constexpr (EXACT) *reinterpret_cast<uint32_t*>(smem + S::kRows * D * 2 + at) = pack16_rest<S::kBf16>(v[2 * e], v[2 * e + 1], u);
                }
            }
        }
    }
    __syncthreads();

    // ---- this thread's rows: quad and quad + 8 of every block of 16 ----
    float factor[MT][2], ref[MT][2], l[MT][2];
    int key_hi[MT][2], key_lo[MT][2];                                    // visible keys, relative to lo: key_lo <= j <= key_hi
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t r = 16 * mt + quad + 8 * i, at = q.len - q.n + (r0 + min(r, rows - 1)) / p.group;
            factor[mt][i] = s_factor[r];
            ref[mt][i] = -INFINITY;
            l[mt][i] = 0.f;
            key_hi[mt][i] = r < rows ? int(at) - int(lo) : -1;
            key_lo[mt][i] = int(paged_first_key(at, a.window)) - int(lo);
        }
    const int all_hi = int(q.len - q.n + r0 / p.group) - int(lo), all_lo = int(paged_first_key(q.len - q.n + (r0 + rows - 1) / p.group, a.window)) - int(lo);
    constexpr int kNt = S::kKeys / 8, kOt = D / 8;
    float o[MT][kOt][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < kOt; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[mt][j][i] = 0.f;
    uint32_t unit = 0;                                                   // 8 bits: exponent field of the power of two that values' scales are divided by
    const uint32_t q_at = smem_u32(smem);

    uint32_t stage = 0;
    for (uint32_t slice = warp; slice < slices; slice += kPrWarps) {
        cp_async_wait<kPrStages - 2>();
        __syncwarp();
        {
            const uint32_t ahead = slice + kPrWarps * (kPrStages - 1), free_stage = stage == 0 ? kPrStages - 1 : stage - 1;
            if (ahead < slices) issue(free_stage);
            look_up(ahead + kPrWarps);
            cp_async_commit();
        }
        const uint8_t* here = ring + stage * S::kStage;
        const uint32_t here_at = ring_at + stage * S::kStage;
        const uint32_t there = s_valid[warp][stage];
        stage = stage + 1 == kPrStages ? 0 : stage + 1;

        // S = Q K^T
        float s[MT][kNt][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < kNt; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[mt][j][i] = 0.f;
        auto load_q = [&](uint32_t (&x)[4], int plane, int mt, int step) {
            const uint32_t r = 16 * mt + (lane & 15), u = 2 * step + (lane >> 4);
            ldsm4(x, q_at + plane * S::kRows * D * 2 + r * (2 * D) + ((u ^ (r & 7u)) << 4));
        };
        if constexpr (!S::kEight) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t b[4];
                ldsm4(b, here_at + S::at((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
#pragma unroll
                for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        uint32_t x[4];
                        load_q(x, plane, mt, k);
                        mma16<S::kBf16>(s[mt][0], x, b[0], b[1]);
                        mma16<S::kBf16>(s[mt][1], x, b[2], b[3]);
                    }
            }
        } else {
#pragma unroll
            for (int blk = 0; blk < D / 64; ++blk) {
                uint32_t x[S::kPlanes][MT][4][4];
#pragma unroll
                for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int k = 0; k < 4; ++k) load_q(x[plane][mt][k], plane, mt, 4 * blk + k);
                uint32_t w[kNt][4];
#pragma unroll
                for (int j = 0; j < kNt; ++j) {
                    const uint4 u = *reinterpret_cast<const uint4*>(here + S::at(8 * j + quad, 4 * blk + tq));
                    w[j][0] = u.x;
                    w[j][1] = u.y;
                    w[j][2] = u.z;
                    w[j][3] = u.w;
                }
                // (neighbouring products belong to different sums: none waits for the one before)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < kNt; ++j) {
                        const uint32_t v = KIND == LV_TYPE_I8 ? w[j][k] ^ 0x80808080u : w[j][k];
                        const uint32_t b0 = codes_f16<KIND>(v, false), b1 = codes_f16<KIND>(v, true);
#pragma unroll
                        for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) mma16<false>(s[mt][j], x[plane][mt][k], b0, b1);
                    }
            }
        }

        // scores in log2 units, hidden ones -inf
        const int j0 = int(slice * S::kKeys);
        const bool open = there == (S::kKeys == 32 ? 0xffffffffu : 0xffffu) && j0 + S::kKeys - 1 <= all_hi && j0 >= all_lo;
        float vs[kNt][2];
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
            float2 ks = make_float2(1.f, 1.f);
            if constexpr (S::kEight) {
                const float* scales = reinterpret_cast<const float*>(here + 2 * S::kHalf);
                ks = *reinterpret_cast<const float2*>(scales + 8 * j + 2 * tq);
                const float2 v2 = *reinterpret_cast<const float2*>(scales + S::kKeys + 8 * j + 2 * tq);
                vs[j][0] = v2.x;
                vs[j][1] = v2.y;
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = s[mt][j][i] * factor[mt][i >> 1];
                    if constexpr (S::kEight) v *= i & 1 ? ks.y : ks.x;
                    if (!open) {
                        const int at = 8 * j + 2 * tq + (i & 1), key = j0 + at;
                        v = ((there >> at) & 1u) != 0 && key <= key_hi[mt][i >> 1] && key >= key_lo[mt][i >> 1] ? v : -INFINITY;
                    }
                    s[mt][j][i] = v;
                }
        }
        // references, and the power of two of the values' scales
        float keep[MT][2];
        bool moved = false;
        if constexpr (S::kEight) {
            const uint32_t mine = paged_scale_exponent(reinterpret_cast<const float*>(here + 2 * S::kHalf)[S::kKeys + lane % S::kKeys]);
            const uint32_t top = min(max(__reduce_max_sync(0xffffffffu, mine), 1u), 253u);
            if (top > unit) {                                            // (unit 0: nothing yet, all outputs are zero)
                const float f = paged_unit_step(unit, top);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) keep[mt][0] = keep[mt][1] = f;
                unit = top;
                moved = true;
            } else {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) keep[mt][0] = keep[mt][1] = 1.f;
            }
        } else {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) keep[mt][0] = keep[mt][1] = 1.f;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < kNt; ++j) top = fmaxf(top, fmaxf(s[mt][j][2 * i], s[mt][j][2 * i + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                if (top > ref[mt][i] + (kPaLift + kPaStep)) {            // (-inf before the first visible key)
                    const float next = top - kPaLift, f = exp2_fast(ref[mt][i] - next);
                    l[mt][i] *= f;
                    keep[mt][i] *= f;
                    ref[mt][i] = next;
                    moved = true;
                }
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int j = 0; j < kOt; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[mt][j][i] *= keep[mt][i >> 1];
        }
        // weights; what they are as operands replaces the scores
        const float down = S::kEight ? __uint_as_float((254u - unit) << 23) : 1.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float at[2] = {ref[mt][0] == -INFINITY ? 0.f : ref[mt][0], ref[mt][1] == -INFINITY ? 0.f : ref[mt][1]};
#pragma unroll
            for (int j = 0; j < kNt; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = exp2_fast(s[mt][j][i] - at[i >> 1]);
                    l[mt][i >> 1] += w;
                    // (a hidden key's scale may be anything)
                    s[mt][j][i] = S::kEight ? (open || s[mt][j][i] != -INFINITY ? w * (vs[j][i & 1] * down) : 0.f) : w;
                }
        }

        // O += P V
        if constexpr (!S::kEight) {
            uint32_t x[S::kPlanes][MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = s[mt][i >> 1][2 * (i & 1)], v = s[mt][i >> 1][2 * (i & 1) + 1];
                    x[0][mt][i] = pack16<S::kBf16>(u, v);
                    if constexpr (EXACT) x[S::kPlanes - 1][mt][i] = pack16_rest<S::kBf16>(u, v, x[0][mt][i]);
                }
#pragma unroll
            for (int j = 0; j < kOt / 2; ++j) {
                uint32_t b[4];
                ldsm4_trans(b, here_at + S::kHalf + S::at((lane & 7) + (((lane >> 3) & 1) << 3), 2 * j + (lane >> 4)));
#pragma unroll
                for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        mma16<S::kBf16>(o[mt][2 * j], x[plane][mt], b[0], b[1]);
                        mma16<S::kBf16>(o[mt][2 * j + 1], x[plane][mt], b[2], b[3]);
                    }
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < S::kKeys / 16; ++kk) {
                uint32_t x[S::kPlanes][MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float u = s[mt][2 * kk + (i >> 1)][2 * (i & 1)], v = s[mt][2 * kk + (i >> 1)][2 * (i & 1) + 1];
                        x[0][mt][i] = pack16<false>(u, v);
                        if constexpr (EXACT) x[S::kPlanes - 1][mt][i] = pack16_rest<false>(u, v, x[0][mt][i]);
                    }
                // a thread takes 16 (8 for D = 64) neighbouring values of its four keys: its column of that many instructions
                constexpr int kWords = D == 64 ? 2 : 4;
#pragma unroll
                for (int part = 0; part < (D == 256 ? 2 : 1); ++part) {
                    uint32_t w[4][kWords];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t key = 16 * kk + 2 * tq + (k & 1) + 8 * (k >> 1);
                        if constexpr (D == 64) {
                            const uint2 u = *reinterpret_cast<const uint2*>(here + S::kHalf + S::at(key, quad >> 1) + 8 * (quad & 1));
                            w[k][0] = u.x;
                            w[k][1] = u.y;
                        } else {
                            const uint4 u = *reinterpret_cast<const uint4*>(here + S::kHalf + S::at(key, quad + 8 * part));
                            w[k][0] = u.x;
                            w[k][1] = u.y;
                            w[k][2] = u.z;
                            w[k][3] = u.w;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < kWords; ++n) {
#pragma unroll
                        for (int pair = 0; pair < 2; ++pair) {           // values 4 n + 2 pair, + 1 of the four keys
                            uint32_t lo2 = __byte_perm(w[0][n], w[1][n], pair ? 0x7362 : 0x5140), hi2 = __byte_perm(w[2][n], w[3][n], pair ? 0x7362 : 0x5140);
                            if constexpr (KIND == LV_TYPE_I8) {
                                lo2 ^= 0x80808080u;
                                hi2 ^= 0x80808080u;
                            }
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t b0 = codes_f16<KIND>(lo2, e != 0), b1 = codes_f16<KIND>(hi2, e != 0);
#pragma unroll
                                for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                                    for (int mt = 0; mt < MT; ++mt) mma16<false>(o[mt][16 * part + 4 * n + 2 * pair + e], x[plane][mt], b0, b1);
                            }
                        }
                    }
                }
            }
        }
    }
    cp_async_wait<0>();

    // ---- the four warps meet ----
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 1);
            l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 2);
            if (tq == 0) {
                s_ref[warp][16 * mt + quad + 8 * i] = ref[mt][i];
                s_l[warp][16 * mt + quad + 8 * i] = l[mt][i];
            }
        }
    __syncthreads();                                                     // the rings are empty: their place is the outputs' now
    float* merged = reinterpret_cast<float*>(smem + S::kQ);              // [warp][row][D]
    const float up = S::kEight ? __uint_as_float(max(unit, 1u) << 23) : 1.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t r = 16 * mt + quad + 8 * i;
            float* to = merged + (warp * S::kRows + r) * D;
            if constexpr (!S::kEight) {
#pragma unroll
                for (int j = 0; j < kOt; ++j) *reinterpret_cast<float2*>(to + merged_at(r, 8 * j + 2 * tq)) = make_float2(o[mt][j][2 * i], o[mt][j][2 * i + 1]);
            } else {
                constexpr int kRun = D == 64 ? 8 : 16;                   // neighbouring values of a column
#pragma unroll
                for (int j = 0; j < kOt; j += 4)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float4*>(to + merged_at(r, j / kRun * 128 + kRun * (2 * tq + e) + j % kRun)) =
                            make_float4(o[mt][j][2 * i + e] * up, o[mt][j + 1][2 * i + e] * up, o[mt][j + 2][2 * i + e] * up, o[mt][j + 3][2 * i + e] * up);
            }
        }
    __syncthreads();
    const bool whole = p.splits == 1;
    for (uint32_t at = threadIdx.x; at < rows * (D / 4); at += 32 * kPrWarps) {
        const uint32_t r = at / (D / 4), d = 4 * (at - r * (D / 4));
        if (d >= c.dim) continue;
        const uint32_t t = q.row0 + (r0 + r) / p.group, h = kv * p.group + (r0 + r) % p.group;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kPrWarps; ++w) top = fmaxf(top, s_ref[w][r]);
        const float sink = whole ? paged_sink(p, h) : -INFINITY;
        top = fmaxf(top, sink - kPaLift);                                // (the sink may be far above)
        float total = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kPrWarps; ++w) {
            const float f = s_ref[w][r] == -INFINITY ? 0.f : exp2_fast(s_ref[w][r] - top);
            const float4 x = *reinterpret_cast<const float4*>(merged + (w * S::kRows + r) * D + merged_at(r, d));
            if (s_ref[w][r] == -INFINITY && s_l[w][r] == 0.f) continue;
            total = fmaf(s_l[w][r], f, total);
            v = make_float4(fmaf(x.x, f, v.x), fmaf(x.y, f, v.y), fmaf(x.z, f, v.z), fmaf(x.w, f, v.w));
        }
        if (whole) {
            total += paged_sink_weight(sink, top);
            const float f = total == 0.f ? 0.f : 1.f / total;
            store_values4(a.out, size_t(t) * a.out_ld + size_t(h) * c.dim + d, a.out_type, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
        } else {
            const size_t part = (size_t(t) * a.heads + h) * p.splits + split;
            *reinterpret_cast<float4*>(p.part_o + part * c.dim + d) = v;
            if (d == 0) p.part_rl[part] = make_float2(top, total);
        }
    }
}

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
    const uint32_t s = paged_owner(c, t);
    PagedSeq q;
    if (s == c.seqs || !paged_seq(c, s, a.tokens, &q) || q.n > a.max_new || q.len > a.max_len) return;       // (reported)
    const uint32_t r = (t - q.row0) * p.group + h % p.group, r0 = r / block_rows * block_rows;
    const PagedRange all = paged_range(p, q, r0, min(r0 + block_rows, q.n * p.group) - 1);
    const uint32_t n = (all.hi - all.lo + p.chunk - 1) / p.chunk;
    const size_t part = (size_t(t) * a.heads + h) * p.splits;
    const float sink = paged_sink(p, h);
    float top = sink - kPaLift;
    float2 mine = lane < n ? p.part_rl[part + lane] : make_float2(-INFINITY, 0.f);
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
            float4 x[4][2];
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t d = 4 * (lane + 32 * k);
                    x[e][k] = i + e < end && d < c.dim ? *reinterpret_cast<const float4*>(p.part_o + (part + b + i + e) * c.dim + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
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
    uint32_t chunk, splits;
    size_t bytes;
    bool many;
};

static PagedPlan paged_plan(const lv_ctx* ctx, const lv_paged_attention_args& a) {
    PagedPlan plan{};
    const uint32_t group = a.heads / a.cache.kv_heads, rows = a.max_new * group;
    // 16-bit outputs of more than 32 rows that share their keys: a tile of the tensor cores
    plan.many = a.out_type != LV_TYPE_F32 && a.cache.dim <= 128 && rows > 32;
    plan.rows = plan.many ? kPtRows : rows <= 16 || a.cache.dim > 128 ? 16 : 32;
    plan.blocks = (rows + plan.rows - 1) / plan.rows;
    const uint64_t seen = a.window ? std::min<uint64_t>(a.max_len, uint64_t(a.window) + std::min(a.max_new, plan.rows)) : a.max_len;
    const uint32_t unit = plan.many ? kPtKeys : kPrWarps * (paged_is8(a.cache.type) ? kPrKeys8 : 16);
    const uint64_t ctas = uint64_t(a.cache.seqs) * a.cache.kv_heads * plan.blocks;
    const uint64_t want = plan.many ? uint64_t(ctx->sm_count) * (ctas > uint64_t(ctx->sm_count) ? 6 : 1) : uint64_t(kPrCtas) * ctx->sm_count * (a.cache.seqs > 1 ? kPrRounds : 1);
    uint64_t splits = std::max<uint64_t>(1, std::min<uint64_t>((want + ctas - 1) / ctas, (seen + unit - 1) / unit));
    uint64_t chunk = ((seen + splits - 1) / splits + unit - 1) / unit * unit;
    plan.chunk = uint32_t(std::max<uint64_t>(chunk, unit));
    plan.splits = uint32_t((seen + plan.chunk - 1) / plan.chunk);
    if (plan.splits == 0) plan.splits = 1;
    plan.bytes = plan.splits == 1 ? 16 : (size_t(a.tokens) * a.heads * plan.splits * (a.cache.dim + 2)) * 4 + 32;
    return plan;
}

template <int KIND, int D, bool EXACT, int MT>
static int rows_launch(lv_ctx* ctx, const PagedAttn& p, uint32_t blocks) {
    using S = RowsShape<KIND, D, EXACT, MT>;
    auto* kernel = paged_rows_kernel<KIND, D, EXACT, MT>;
    LV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    LV_CUDA(launch_pdl(ctx, kernel, dim3(p.splits * blocks, p.a.cache.kv_heads, p.a.cache.seqs), dim3(32 * kPrWarps), S::kSmem, p));
    return LV_OK;
}

template <int KIND, bool EXACT>
static int rows_launch_size(lv_ctx* ctx, const PagedAttn& p, const PagedPlan& plan) {
    if (p.a.cache.dim > 128) return rows_launch<KIND, 256, EXACT, 1>(ctx, p, plan.blocks);
    if (p.a.cache.dim > 64) return plan.rows == 16 ? rows_launch<KIND, 128, EXACT, 1>(ctx, p, plan.blocks) : rows_launch<KIND, 128, EXACT, 2>(ctx, p, plan.blocks);
    return plan.rows == 16 ? rows_launch<KIND, 64, EXACT, 1>(ctx, p, plan.blocks) : rows_launch<KIND, 64, EXACT, 2>(ctx, p, plan.blocks);
}

template <int KIND>
static int rows_launch_kind(lv_ctx* ctx, const PagedAttn& p, const PagedPlan& plan) {
    return p.a.out_type == LV_TYPE_F32 ? rows_launch_size<KIND, true>(ctx, p, plan) : rows_launch_size<KIND, false>(ctx, p, plan);
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
    p.chunk = plan.chunk;
    p.splits = plan.splits;
    p.part_rl = static_cast<float2*>(scratch);
    p.part_o = static_cast<float*>(scratch) + (size_t(a->tokens) * a->heads * plan.splits * 2 + 3) / 4 * 4;
    p.err = ctx->d_err;
    int rc = LV_OK;
    if (plan.many) rc = paged_tc_launch(ctx, p, plan.blocks);
    else switch (a->cache.type) {
        case LV_TYPE_BF16: rc = rows_launch_kind<LV_TYPE_BF16>(ctx, p, plan); break;
        case LV_TYPE_F16: rc = rows_launch_kind<LV_TYPE_F16>(ctx, p, plan); break;
        case LV_TYPE_I8: rc = rows_launch_kind<LV_TYPE_I8>(ctx, p, plan); break;
        default: rc = rows_launch_kind<LV_TYPE_E4M3>(ctx, p, plan); break;
    }
    if (rc != LV_OK || plan.splits == 1) return rc;
    const uint64_t warps = uint64_t(a->tokens) * a->heads;
    LV_CUDA(launch_pdl(ctx, paged_join_kernel, dim3(uint32_t((warps + 3) / 4)), dim3(128), 0, p, plan.rows));
    return LV_OK;
}

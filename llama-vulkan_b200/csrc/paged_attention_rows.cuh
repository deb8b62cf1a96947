// Attention of few new tokens over a cache in pages.
//
//   s_j = scale (q . k_j),  r = max_j s_j - lift,  w_j = 2^(s_j - r),  out = sum_j w_j v_j / (2^(sink - r) + sum_j w_j)      (s in log2 units)
//
// A key/value row is read for all query heads and new tokens that share it: the rows of a block are (token, head) pairs.  One token of 4 grouped
// heads does 8 operations per byte of a 16-bit cache, so the kernel is bound by memory, and what counts is that enough bytes are on
// their way: every warp has a ring of its own, filled by 16-byte cp.async (the page of a row is looked up by one lane a slice ahead), and takes slices of 16 or 32
// keys by itself -- running maximum, sum and output are the warp's, nothing in the loop waits for another warp.  The four warps meet at the end.
//
// The products are mma.sync m16n8k16, transposed: S^T = K Q^T and O^T = V^T P^T, keys and values the operand of 16 rows, queries and weights the one of 8 columns, so that
// 8 rows of queries (24, ..) are whole instructions; a tcgen05 tile of 128 would be mostly empty.  Weights change sides by movmatrix.  Operands: bf16 for bf16
// caches, else f16; 8-bit codes are exact in f16, their scales multiply the finished scores and the weights.  Queries and weights enter as one or more 16-bit numbers
// (each the rounding of what the ones before left): for f32 outputs with 22 or 24 bits together (f16 outputs over f16 caches: 22), for other 16-bit outputs with 11 (f16 operands) or 16 (bf16).
// f16 operands: a query row is divided by a power of two (its largest value is near 1), and the scales of the values by the power of two of the largest so
// far, so that neither overflows nor loses bits.
// 64 sequences of one token, 500 to 8192 keys, int8, 32/8 heads of 128: 126 us, 4.7 TB/s of 593 MB.  Counters: integer pipe 63 %, issue 64 %, memory 62 % of its peak, few waits for loads:
// the instructions that take codes apart share the time with memory (rows as the operand of 16 instead: 150 us; slices of 16 keys, so that a fourth CTA fits: 134).  One token of one sequence,
// 521 keys, 32 heads, f16: 8.8 us, two launches and a chain of loads.  16 sequences with 6 drafts over e4m3, blocks of 24 rows: 54 us where memory takes 15: 250 registers leave eight warps per SM, which issue
// in 44 % of the clocks and wait for their own results (three CTAs per SM, with spilled registers: 61); the tcgen05 kernel, with tiles four fifths empty: 160.
#pragma once

#include "paged_attention.cuh"

namespace lv {

constexpr int kPrStages = 2;

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
__device__ __forceinline__ uint32_t transposed8x8(uint32_t u) {
    uint32_t v;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(v) : "r"(u));
    return v;
}
// Two values rounded to 16 bits; what the rounding has left stays in them.
template <bool BF16>
__device__ __forceinline__ uint32_t take16(float& lo, float& hi) {
    const uint32_t u = pack16<BF16>(lo, hi);
    float2 r;
    if constexpr (BF16) r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
    else r = __half22float2(*reinterpret_cast<const __half2*>(&u));
    lo -= r.x;
    hi -= r.y;
    return u;
}

// KIND: type of the cache; D: head size rounded up to 64, 128 or 256; EXACT: f32 outputs (f16 caches: f16 ones too); NT: blocks of 8 rows
template <int KIND, int D, bool EXACT, int NT>
struct RowsShape {
    static constexpr bool kEight = KIND == LV_TYPE_I8 || KIND == LV_TYPE_E4M3, kBf16 = KIND == LV_TYPE_BF16;
    static constexpr int kKeys = kEight ? kPrKeys8 : kPrKeys16;          // of a slice
    static constexpr int kRowBytes = kEight ? D : 2 * D, kUnits = kRowBytes / 16;
    static constexpr int kHalf = kKeys * kRowBytes;                      // bytes of the keys (or values) of a slice
    static constexpr int kStage = 2 * kHalf + (kEight ? 2 * kKeys * 4 : 0);
    static constexpr int kPlanes = kBf16 ? (EXACT ? 3 : 2) : EXACT ? 2 : 1, kRows = 8 * NT;
    static constexpr bool kHoldQ = NT * kPlanes * D <= 256;              // queries stay in registers
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

// place of value d of row r where the warps' outputs meet: 16-byte units moved by the row, so that stores of several rows fall into different banks
__device__ __forceinline__ uint32_t merged_at(uint32_t r, uint32_t d) { return (((d >> 2) ^ (r & 7u)) << 2) + (d & 3u); }

template <int KIND, int D, bool EXACT, int NT>
__global__ void __launch_bounds__(32 * kPrWarps, D == 256 ? 1 : NT == 1 ? 4 : NT == 2 ? 3 : 2) paged_rows_kernel(const PagedAttn p) {
    using S = RowsShape<KIND, D, EXACT, NT>;
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
            atomicOr(p.data_err, ERR_BAD_INDEX);
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

    // ---- queries: rotated, divided by a power of two, in one to three 16-bit planes; all of a warp's rows are asked for at once ----
    {
        constexpr int kParts = D == 256 ? 2 : 1, kOwn = S::kRows / kPrWarps;
        uint4 raw[kOwn][kParts];
        float2 turn[kOwn][kParts][2];
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const uint32_t r = warp + kPrWarps * k, t = q.row0 + (r0 + r) / p.group, h = kv * p.group + (r0 + r) % p.group;
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const uint32_t d = 4 * (lane + 32 * i);
                const bool here = r < rows && d < c.dim;
                raw[k][i] = here ? load_raw4(a.q, size_t(t) * a.q_ld + size_t(h) * c.dim + d, a.q_type) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    turn[k][i][e] = here && a.angles != nullptr && d + 2 * e < 2 * a.angle_pairs ? *reinterpret_cast<const float2*>(a.angles + size_t(t) * a.angle_ld + d + 2 * e) : make_float2(1.f, 0.f);
            }
        }
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const uint32_t r = warp + kPrWarps * k;
            float top = 0.f;
            float4 x[kParts];
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                x[i] = unpack_raw4(raw[k][i], a.q_type);
                if (a.angles != nullptr) x[i] = rotate4(x[i], turn[k][i][0], turn[k][i][1]);
                top = fmaxf(fmaxf(top, fmaxf(fabsf(x[i].x), fabsf(x[i].y))), fmaxf(fabsf(x[i].z), fabsf(x[i].w)));
            }
            float f = 1.f;                                               // 2^-e of the largest value (f16 operands)
            if constexpr (!S::kBf16) f = paged_row_unit(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))));
            if (lane == 0) s_factor[r] = paged_factor(p.factor, f);
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const uint32_t d = 4 * (lane + 32 * i);
                if (d >= D) continue;
                float v[4] = {x[i].x * f, x[i].y * f, x[i].z * f, x[i].w * f};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t col = S::column(d + 2 * e), at = r * (2 * D) + (((col >> 3) ^ (r & 7u)) << 4) + (col & 7u) * 2;
#pragma unroll
                    for (int plane = 0; plane < S::kPlanes; ++plane) *reinterpret_cast<uint32_t*>(smem + plane * S::kRows * D * 2 + at) = take16<S::kBf16>(v[2 * e], v[2 * e + 1]);
                }
            }
        }
    }
    __syncthreads();

    // ---- this thread's rows: 2 tq and 2 tq + 1 of every block of 8 ----
    float factor[NT][2], ref[NT][2], l[NT][2];
    int key_hi[NT][2], key_lo[NT][2];                                    // visible keys, relative to lo: key_lo <= j <= key_hi
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t r = 8 * nt + 2 * tq + e, at = q.len - q.n + (r0 + min(r, rows - 1)) / p.group;
            factor[nt][e] = s_factor[r];
            ref[nt][e] = -INFINITY;
            l[nt][e] = 0.f;
            key_hi[nt][e] = r < rows ? int(at) - int(lo) : -1;
            key_lo[nt][e] = int(paged_first_key(at, a.window)) - int(lo);
        }
    const int all_hi = int(q.len - q.n + r0 / p.group) - int(lo), all_lo = int(paged_first_key(q.len - q.n + (r0 + rows - 1) / p.group, a.window)) - int(lo);
    constexpr int kMk = S::kKeys / 16, kMo = D / 16, kSteps = D / 16;
    const uint32_t q_at = smem_u32(smem);
    // operand of two steps (32 columns) of a block of queries
    auto load_q = [&](uint32_t (&x)[4], int plane, int nt, int pair) {
        const uint32_t r = 8 * nt + (lane & 7), u = 4 * pair + (lane >> 3);
        ldsm4(x, q_at + plane * S::kRows * D * 2 + r * (2 * D) + ((u ^ (r & 7u)) << 4));
    };
    [[maybe_unused]] uint32_t held[S::kHoldQ ? S::kPlanes : 1][S::kHoldQ ? NT : 1][S::kHoldQ ? kSteps / 2 : 1][4];
    if constexpr (S::kHoldQ) {
#pragma unroll
        for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < kSteps / 2; ++k) load_q(held[plane][nt][k], plane, nt, k);
    }
    float o[kMo][NT][4];
#pragma unroll
    for (int j = 0; j < kMo; ++j)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][nt][i] = 0.f;
    uint32_t unit = 0;                                                   // exponent field of the power of two that values' scales are divided by

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

        // S^T = K Q^T
        float s[kMk][NT][4];
#pragma unroll
        for (int m = 0; m < kMk; ++m)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[m][nt][i] = 0.f;
        [[maybe_unused]] uint4 word[S::kEight ? kMk : 1][2];
#pragma unroll
        for (int pair = 0; pair < kSteps / 2; ++pair) {
            // two steps of the keys, as operands
            uint32_t key[2][kMk][4];
            if constexpr (!S::kEight) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int m = 0; m < kMk; ++m) ldsm4(key[k][m], here_at + S::at(16 * m + (lane & 15), 2 * (2 * pair + k) + (lane >> 4)));
            } else {
                // a thread's 16 bytes of a key are its part of four steps: two pairs
#pragma unroll
                for (int m = 0; m < kMk; ++m)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (pair % 2 == 0) word[m][i] = *reinterpret_cast<const uint4*>(here + S::at(16 * m + 8 * i + quad, 4 * (pair >> 1) + tq));
                        const uint2 u = pair % 2 == 0 ? make_uint2(word[m][i].x, word[m][i].y) : make_uint2(word[m][i].z, word[m][i].w);
                        const uint32_t w0 = KIND == LV_TYPE_I8 ? u.x ^ 0x80808080u : u.x, w1 = KIND == LV_TYPE_I8 ? u.y ^ 0x80808080u : u.y;
                        key[0][m][i] = codes_f16<KIND>(w0, false);
                        key[0][m][i + 2] = codes_f16<KIND>(w0, true);
                        key[1][m][i] = codes_f16<KIND>(w1, false);
                        key[1][m][i + 2] = codes_f16<KIND>(w1, true);
                    }
            }
#pragma unroll
            for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t x[4];
                    if constexpr (S::kHoldQ) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = held[plane][nt][pair][i];
                    } else {
                        load_q(x, plane, nt, pair);
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int m = 0; m < kMk; ++m) mma16<S::kBf16>(s[m][nt], key[k][m], x[2 * k], x[2 * k + 1]);
                }
        }

        // scores in log2 units, hidden ones -inf
        const int j0 = int(slice * S::kKeys);
        const bool open = there == (S::kKeys == 32 ? 0xffffffffu : 0xffffu) && j0 + S::kKeys - 1 <= all_hi && j0 >= all_lo;
        float vs[kMk][2];
#pragma unroll
        for (int m = 0; m < kMk; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = 16 * m + 8 * i + quad;
                float ks = 1.f;
                if constexpr (S::kEight) {
                    const float* scales = reinterpret_cast<const float*>(here + 2 * S::kHalf);
                    ks = scales[at];
                    vs[m][i] = scales[S::kKeys + at];
                }
                const bool gone = !open && ((there >> at) & 1u) == 0;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = s[m][nt][2 * i + e] * factor[nt][e];
                        if constexpr (S::kEight) v *= ks;
                        if (!open) v = gone || j0 + at > key_hi[nt][e] || j0 + at < key_lo[nt][e] ? -INFINITY : v;
                        s[m][nt][2 * i + e] = v;
                    }
            }
        // references, and the power of two of the values' scales
        float keep[NT][2], down = 1.f;
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) keep[nt][0] = keep[nt][1] = 1.f;
        if constexpr (S::kEight) {
            const uint32_t mine = paged_scale_exponent(reinterpret_cast<const float*>(here + 2 * S::kHalf)[S::kKeys + lane % S::kKeys]);
            const uint32_t top = min(max(__reduce_max_sync(0xffffffffu, mine), 1u), 253u);
            if (top > unit) {                                            // (unit 0: nothing yet, all outputs are zero)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) keep[nt][0] = keep[nt][1] = paged_unit_step(unit, top);
                unit = top;
                moved = true;
            }
            down = __uint_as_float((254u - unit) << 23);
        }
        // (a row's reference is the same in all lanes: a vote tells whether one has to move, and only then its lanes compare their maxima)
        float tops[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                tops[nt][e] = -INFINITY;
#pragma unroll
                for (int m = 0; m < kMk; ++m) tops[nt][e] = fmaxf(tops[nt][e], fmaxf(s[m][nt][e], s[m][nt][2 + e]));
                moved = moved || tops[nt][e] > ref[nt][e] + (kPaLift + kPaStep);           // (-inf before the first visible key)
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = tops[nt][e];
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    if (top > ref[nt][e] + (kPaLift + kPaStep)) {
                        const float next = top - kPaLift, f = exp2_fast(ref[nt][e] - next);
                        l[nt][e] *= f;
                        keep[nt][e] *= f;
                        ref[nt][e] = next;
                    }
                }
#pragma unroll
            for (int j = 0; j < kMo; ++j)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[j][nt][i] *= keep[nt][i & 1];
        }

        // weights, which change sides: pairs of rows of a key become pairs of keys of a row
        uint32_t x[S::kPlanes][kMk][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float at[2] = {ref[nt][0] == -INFINITY ? 0.f : ref[nt][0], ref[nt][1] == -INFINITY ? 0.f : ref[nt][1]};
#pragma unroll
            for (int m = 0; m < kMk; ++m)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float z = s[m][nt][2 * i + e];
                        w[e] = exp2_fast(z - at[e]);
                        l[nt][e] += w[e];
                        // (a hidden key's scale may be anything)
                        if constexpr (S::kEight) w[e] = open || z != -INFINITY ? w[e] * (vs[m][i] * down) : 0.f;
                    }
#pragma unroll
                    for (int plane = 0; plane < S::kPlanes; ++plane) x[plane][m][nt][i] = transposed8x8(take16<S::kBf16>(w[0], w[1]));
                }
        }

        // O^T += V^T P^T
#pragma unroll
        for (int m = 0; m < kMk; ++m) {
            if constexpr (!S::kEight) {
#pragma unroll
                for (int j = 0; j < kMo; ++j) {
                    uint32_t v[4];
                    ldsm4_trans(v, here_at + S::kHalf + S::at(16 * m + (lane & 7) + ((lane >> 4) << 3), 2 * j + ((lane >> 3) & 1)));
#pragma unroll
                    for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16<S::kBf16>(o[j][nt], v, x[plane][m][nt][0], x[plane][m][nt][1]);
                }
            } else {
                // a thread takes 16 (8 for D = 64) neighbouring values of its four keys: its two rows of that many instructions
                constexpr int kWords = D == 64 ? 2 : 4;
#pragma unroll
                for (int part = 0; part < (D == 256 ? 2 : 1); ++part) {
                    uint32_t w[4][kWords];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t key = 16 * m + 2 * tq + (k & 1) + 8 * (k >> 1);
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
                    for (int n = 0; n < kWords; ++n)
#pragma unroll
                        for (int pair = 0; pair < 2; ++pair) {           // values 4 n + 2 pair, + 1 of the four keys
                            uint32_t lo2 = __byte_perm(w[0][n], w[1][n], pair ? 0x7362 : 0x5140), hi2 = __byte_perm(w[2][n], w[3][n], pair ? 0x7362 : 0x5140);
                            if constexpr (KIND == LV_TYPE_I8) {
                                lo2 ^= 0x80808080u;
                                hi2 ^= 0x80808080u;
                            }
                            const uint32_t v[4] = {codes_f16<KIND>(lo2, false), codes_f16<KIND>(lo2, true), codes_f16<KIND>(hi2, false), codes_f16<KIND>(hi2, true)};
#pragma unroll
                            for (int plane = 0; plane < S::kPlanes; ++plane)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) mma16<false>(o[8 * part + 2 * n + pair][nt], v, x[plane][m][nt][0], x[plane][m][nt][1]);
                        }
                }
            }
        }
    }
    cp_async_wait<0>();

    // ---- the four warps meet ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], d);
            if (quad == 0) {
                s_ref[warp][8 * nt + 2 * tq + e] = ref[nt][e];
                s_l[warp][8 * nt + 2 * tq + e] = l[nt][e];
            }
        }
    __syncthreads();                                                     // the rings are empty: their place is the outputs' now
    float* merged = reinterpret_cast<float*>(smem + S::kQ);              // [warp][row][D]
    const float up = S::kEight ? __uint_as_float(max(unit, 1u) << 23) : 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t r = 8 * nt + 2 * tq + e;
            float* to = merged + (warp * S::kRows + r) * D;
            if constexpr (!S::kEight) {
#pragma unroll
                for (int j = 0; j < kMo; ++j) {
                    to[merged_at(r, 16 * j + quad)] = o[j][nt][e];
                    to[merged_at(r, 16 * j + 8 + quad)] = o[j][nt][2 + e];
                }
            } else {
                constexpr int kRun = D == 64 ? 8 : 16;                   // neighbouring values of a thread
#pragma unroll
                for (int j = 0; j < kMo; j += 2)
                    *reinterpret_cast<float4*>(to + merged_at(r, j / 8 * 128 + kRun * quad + 2 * j % kRun)) =
                        make_float4(o[j][nt][e] * up, o[j][nt][2 + e] * up, o[j + 1][nt][e] * up, o[j + 1][nt][2 + e] * up);
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

template <int KIND, int D, bool EXACT, int NT>
static int rows_launch(lv_ctx* ctx, const PagedAttn& p, uint32_t blocks) {
    using S = RowsShape<KIND, D, EXACT, NT>;
    auto* kernel = paged_rows_kernel<KIND, D, EXACT, NT>;
    LV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    LV_CUDA(launch_pdl(ctx, kernel, dim3(p.splits * blocks, p.a.cache.kv_heads, p.a.cache.seqs), dim3(32 * kPrWarps), S::kSmem, p));
    return LV_OK;
}

// rows: of a block, 8, 16, 24 or 32 (heads of more than 128 values: 8 or 16)
template <int KIND, bool EXACT>
static int rows_launch_size(lv_ctx* ctx, const PagedAttn& p, uint32_t rows, uint32_t blocks) {
    if (p.a.cache.dim > 128) return rows <= 8 ? rows_launch<KIND, 256, EXACT, 1>(ctx, p, blocks) : rows_launch<KIND, 256, EXACT, 2>(ctx, p, blocks);
    if (p.a.cache.dim > 64) {
        switch (rows) {
            case 8: return rows_launch<KIND, 128, EXACT, 1>(ctx, p, blocks);
            case 16: return rows_launch<KIND, 128, EXACT, 2>(ctx, p, blocks);
            case 24: return rows_launch<KIND, 128, EXACT, 3>(ctx, p, blocks);
            default: return rows_launch<KIND, 128, EXACT, 4>(ctx, p, blocks);
        }
    }
    switch (rows) {
        case 8: return rows_launch<KIND, 64, EXACT, 1>(ctx, p, blocks);
        case 16: return rows_launch<KIND, 64, EXACT, 2>(ctx, p, blocks);
        case 24: return rows_launch<KIND, 64, EXACT, 3>(ctx, p, blocks);
        default: return rows_launch<KIND, 64, EXACT, 4>(ctx, p, blocks);
    }
}

template <int KIND>
static int rows_launch_kind(lv_ctx* ctx, const PagedAttn& p, uint32_t rows, uint32_t blocks) {
    // f16 caches take two numbers for f16 results too: with one they are off by 4.9e-4 relative to the result instead of its own rounding's 2.0e-4, and two cost 3 to 5 % (one token, 521 keys: 8.75 us
    // against 8.49; 64 sequences: 189 against 181).  8-bit caches, whose codes are off by far more, do not: 142 us against 125 (64 sequences), 65 against 54 (drafts).
    const bool exact = p.a.out_type == LV_TYPE_F32 || (KIND == LV_TYPE_F16 && p.a.out_type == LV_TYPE_F16);
    return exact ? rows_launch_size<KIND, true>(ctx, p, rows, blocks) : rows_launch_size<KIND, false>(ctx, p, rows, blocks);
}

}  // namespace lv

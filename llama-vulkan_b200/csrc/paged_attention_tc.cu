// Attention of many new tokens over a cache in pages, on the tcgen05 tensor cores (16-bit outputs).
//
// A CTA takes up to 256 rows -- (token, query head) pairs of one key/value head -- and walks their keys in steps of 128:
//
//   S = Q K^T          tensor memory, 128 x 128 f32
//   P = 2^(S - r)      a row per thread; 16-bit weights go to tensor memory over the scores that they came from
//   O += P V           P from tensor memory, V as an MN-major operand (its rows are keys)
//
// in two units that take turns: the tensor cores work for one while the other's weights are computed.  With more than 128 rows a unit is a tile of 128 of them, and each
// key and value is fetched once for both; with fewer the units are the even and the odd steps of the same rows, each with its own O, which are added at the end.
// One lane issues a unit's products, in this order: P V, then the next S, so that the scores never overwrite weights that are still to be
// read, and a finished S says that the unit's last P V has finished too.
// Keys and values come by TMA, a box for the rows of a page or for a part of them (the largest power of two that divides the page, at least eight rows: the swizzle's
// pattern): 16-bit rows straight into the operands' swizzle, 8-bit codes into a ring, from which four warps convert them to f16 (exact).  cp.async by the same four
// warps was tried first and kept the load and store unit so busy that every other warp of the CTA waited for it (1142 us against 1084).  Places that no query sees are not
// fetched, or zeroed behind the copy: their weights are zero, but zero times NaN is not.  References, f16 ranges and scales as in paged_attention_rows.cuh.
// Two prompts of 2048 tokens behind 9001 to 16384 keys, bf16, 32/8 heads of 128: 931 us, 876 TFLOP/s of 1681 that a library's large product reaches.  Bound by the chain of a
// unit, not by one pipe: with the softmax left out the copies and products took 775 us, with the products left out the softmax took 744 (947 together then), and the two units hide
// only a part of one behind the other.  Two of 512 behind 4096 to 8192: bf16 165 us, f16 175, int8 399, e4m3 371 (the four warps' conversions).  Without turns at the exponentials: 1003 us.  A quarter of the exponentials by a polynomial on the multipliers: 1003 us with
// turns, for its instructions take the issue slots that the turns have freed.  Steps that one warp issued for both units: 1084 us.
//
// Every wait is bounded; one that gives up sets the error word, and the CTA drains and frees its tensor memory.
#include <cuda.h>

#include "paged_attention.cuh"
#include "tcgen05.cuh"
#include "tmap.h"

namespace lv {

// Warps: eight of the softmax, four that convert or mend what was copied, four of which two issue the products and one the copies.  Registers move from the latter eight to the former: a row's 128 scores are held at a
// time.  512 threads are launched with 128 registers each: (8 x 200 + 8 x 56) x 32 = 512 x 128.
constexpr int kPtSoftmax = 8, kPtHelpers = 4, kPtThreads = 512, kPtStages = 2, kPtRing = 3, kPtManyRegs = 200, kPtFewRegs = 56;
// A wait ends at once where another one has been lost, but not for an index that some earlier kernel found out of range: that was reported, and these sequences are in order.
constexpr uint32_t kPtEnds = ~uint32_t(ERR_BAD_INDEX);

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// two f32 at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ void tmem_load32(uint32_t* u, uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
          "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]),
          "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t* u) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31, %32};"
        ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]),
          "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
          "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* u) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]),
                   "r"(u[13]), "r"(u[14]), "r"(u[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// the largest of three; a NaN among them shows in the sum of the weights
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// V: rows are keys (the K of the product), 64 columns per 128-byte row; groups of eight keys 1024 bytes apart, blocks of 64 columns `block` bytes apart
__device__ __forceinline__ uint64_t values_desc(uint32_t smem_addr, uint32_t block) {
    return uint64_t((smem_addr >> 4) & 0x3fffu) | (uint64_t(block >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

struct TcMeta {                                                          // of a step's keys
    float ks[kPtKeys], vs[kPtKeys];
    uint32_t there[4], exponent[4];
};
struct TcShared {
    TcMeta meta[kPtStages];
    uint64_t k_full[kPtStages], k_empty[kPtStages], v_raw[kPtStages], v_full[kPtStages], v_empty[kPtStages], raw_full[kPtRing], raw_empty[kPtRing], s_full[2], p_full[2][2], o_full[2], q_full, drained[2];
    float factor[kPtRows], ref[128], l[128];                             // of the rows; of the second unit of the same rows
    uint32_t unit, tmem;
};

template <int KIND, int D>
struct TcShape {
    static constexpr bool kEight = KIND == LV_TYPE_I8 || KIND == LV_TYPE_E4M3, kBf16 = KIND == LV_TYPE_BF16;
    static constexpr int kBlocks = D / 64;                               // of 64 columns
    static constexpr uint32_t kBlock = 128 * 128;                        // bytes of 128 rows of one
    static constexpr uint32_t kTile = kBlocks * kBlock;                  // of a query tile, and of a step's keys or values
    static constexpr uint32_t kRaw = kEight ? 128 * D : 0;               // of a step's codes
    // (the keys' barriers are those of even and odd steps in any case: two units that wait for one barrier in turn could take a phase for the next but one)
    // a step's keys are free as soon as its scores are there: one place for them is enough where codes on their way need room
    static constexpr uint32_t kKeyStages = kEight ? 1 : kPtStages;
    // queries (two tiles), keys and values, codes
    static constexpr uint32_t kShared = (2 + kKeyStages + kPtStages) * kTile + kPtRing * kRaw;
    static constexpr size_t kSmem = kShared + sizeof(TcShared);
};

struct TcMaps {
    CUtensorMap k, v;
};

// byte of 16-byte unit u of row r in a tile
__device__ __forceinline__ uint32_t tile_at(uint32_t r, uint32_t u) { return (u >> 3) * (128 * 128) + r * 128 + (((u & 7u) ^ (r & 7u)) << 4); }

template <int KIND, int D>
__global__ void __launch_bounds__(kPtThreads, 1) paged_tc_kernel(const PagedAttn p, const __grid_constant__ TcMaps maps) {
    using S = TcShape<KIND, D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *s_q = smem, *s_k = smem + 2 * S::kTile, *s_v = s_k + S::kKeyStages * S::kTile, *s_raw = s_v + kPtStages * S::kTile;
    TcShared& sh = *reinterpret_cast<TcShared*>(smem + S::kShared);
    const lv_paged_attention_args& a = p.a;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    pdl_wait();
    const uint32_t split = blockIdx.x % p.splits, kv = blockIdx.y;
    PagedSeq q;
    const bool fine = paged_attention_seq(p, blockIdx.z, &q);
    // the last blocks of rows see the most keys: they begin first
    const uint32_t all_rows = q.n * p.group, n_blocks = (all_rows + kPtRows - 1) / kPtRows, back = blockIdx.x / p.splits;
    if (!fine || back >= n_blocks) {
        pdl_launch_dependents();
        return;
    }
    const uint32_t r0 = (n_blocks - 1 - back) * kPtRows, rows = min(uint32_t(kPtRows), all_rows - r0);
    const PagedRange all = paged_range(p, q, r0, r0 + rows - 1);
    const uint64_t begin = uint64_t(all.lo & ~p.align) + uint64_t(split) * p.chunk;        // (steps begin where boxes do)
    if (begin >= all.hi) {
        pdl_launch_dependents();
        return;
    }
    const uint32_t lo = uint32_t(begin), hi = uint32_t(min(uint64_t(all.hi), begin + p.chunk)), steps = (hi - lo + kPtKeys - 1) / kPtKeys;
    // unit w: tile w mod 2 of step w / 2, or (two: false) step w
    const bool two = rows > 128;
    const uint32_t units = two ? 2 * steps : steps;
    auto tile_rows = [&](uint32_t unit) { return two ? (unit ? rows - 128 : 128u) : rows; };
    if (threadIdx.x == 0) {
        if (smem_u32(smem) & 1023u) atomicOr(p.data_err, ERR_BAD_INDEX);      // (the swizzle's rows begin at 1024 bytes; never seen)
        mbar_init(&sh.q_full, kPtSoftmax);
        for (int i = 0; i < kPtStages; ++i) {
            mbar_init(&sh.k_full[i], S::kEight ? kPtHelpers : 1);
            mbar_init(&sh.v_raw[i], 1);
            mbar_init(&sh.v_full[i], kPtHelpers);
            mbar_init(&sh.k_empty[i], two ? 2 : 1);
            mbar_init(&sh.v_empty[i], two ? 2 : 1);
        }
        for (int i = 0; i < kPtRing; ++i) { mbar_init(&sh.raw_full[i], 1); mbar_init(&sh.raw_empty[i], kPtHelpers); }
        for (int i = 0; i < 2; ++i) {
            const uint32_t warps = (tile_rows(i) + 31) / 32;             // those with rows
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i][0], warps);
            mbar_init(&sh.p_full[i][1], warps);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.drained[i], 1);
        }
        fence_mbar_init();
    }
    if (warp == kPtSoftmax + kPtHelpers) {
        tc_alloc(&sh.tmem, 512);
        pdl_launch_dependents();        // (not before: a CTA of the next launch could take the tensor memory that this one needs, and wait for it)
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem);
    const uint32_t tmem_o = tmem + 256;                                  // S of the two units in columns 0 and 128, O in 256 and 384

    if (warp < kPtSoftmax) {
        more_registers<kPtManyRegs>();
        // ---- queries, a warp per sixteenth of the rows at a time, then a row per thread ----------------------
        constexpr int kBatch = 16;
        for (uint32_t i0 = kBatch * warp; i0 < (two ? 256u : 128u); i0 += kBatch * kPtSoftmax) {
            uint4 raw[kBatch];
            float2 turn[kBatch][2];
            const uint32_t d = 4 * lane;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const uint32_t r = r0 + i0 + k, t = q.row0 + r / p.group, h = kv * p.group + r % p.group;
                const bool here = i0 + k < rows && d < c.dim;
                raw[k] = here ? load_raw4(a.q, size_t(t) * a.q_ld + size_t(h) * c.dim + d, a.q_type) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    turn[k][e] = here && a.angles != nullptr && d + 2 * e < 2 * a.angle_pairs ? *reinterpret_cast<const float2*>(a.angles + size_t(t) * a.angle_ld + d + 2 * e) : make_float2(1.f, 0.f);
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                float4 x = unpack_raw4(raw[k], a.q_type);
                if (a.angles != nullptr) x = rotate4(x, turn[k][0], turn[k][1]);
                // (the scale is the scores' factor, in f32: bf16 queries that are not rotated enter as they are)
                float f = 1.f;
                if constexpr (!S::kBf16) {
                    const float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
                    f = paged_row_unit(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))));
                    if (lane == 0) sh.factor[i0 + k] = paged_factor(p.factor, f);
                }
                if (d < D) *reinterpret_cast<uint2*>(s_q + ((i0 + k) >> 7) * S::kTile + tile_at((i0 + k) & 127u, d >> 3) + (d & 4u) * 2) =
                    make_uint2(pack16<S::kBf16>(x.x * f, x.y * f), pack16<S::kBf16>(x.z * f, x.w * f));
            }
        }
        fence_proxy_async();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kPtSoftmax) : "memory");
        if (lane == 0) mbar_arrive(&sh.q_full);
        const uint32_t mine = warp >> 2, quarter = warp & 3, lanes = quarter * 32u << 16;
        const uint32_t base_row = two ? 128 * mine : 0, row = base_row + 32 * quarter + lane, before = q.len - q.n;
        const uint32_t s_at = tmem + lanes + mine * 128, o_at = tmem_o + lanes + mine * 128;
        float ref = -INFINITY, l = 0.f;
        uint32_t unit = 0;
        bool ok = true;
        if (base_row + 32 * quarter < rows) {
            const float row_factor = S::kBf16 ? p.factor : sh.factor[row];
            const uint32_t pos = before + (r0 + min(row, rows - 1)) / p.group;
            const int key_hi = row < rows ? int(pos) - int(lo) : -1, key_lo = int(paged_first_key(pos, a.window)) - int(lo);
            // keys that every row of the warp sees
            const uint32_t first = r0 + base_row + 32 * quarter, last = r0 + min(base_row + 32 * quarter + 31, rows - 1);
            const int warp_hi = int(before + first / p.group) - int(lo), warp_lo = int(paged_first_key(before + last / p.group, a.window)) - int(lo);
            // a unit's turn at the exponentials, which the other one ends with its own (in its warps that have rows); the first is the first unit's
            const uint32_t turns = 32 * ((min(tile_rows(0), 128u) + 31) / 32 + (min(tile_rows(1), 128u) + 31) / 32);
            auto begin_turn = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(2 + mine), "r"(turns) : "memory"); };
            auto end_turn = [&]() { asm volatile("bar.arrive %0, %1;" ::"r"(3 - mine), "r"(turns) : "memory"); };
            auto pass_turn = [&](uint32_t w) { if (w + 1 < units) end_turn(); };          // (behind the last one nobody waits)
            if (mine == 1) end_turn();
            for (uint32_t w = mine; w < units; w += 2) {
                const uint32_t turn = w >> 1, j = two ? turn : w, st = j % kPtStages;
                // (after a lost wait the warp goes through the remaining steps without work: the other unit's wait for it)
                ok = ok && mbar_wait_all(&sh.v_full[st], (j / kPtStages) & 1u, p.err, kPtEnds);
                if (!ok) { begin_turn(); pass_turn(w); continue; }
                const TcMeta& m = sh.meta[st];
                const int j0 = int(j * kPtKeys);
                const uint4 there = *reinterpret_cast<const uint4*>(m.there);
                const bool open = __all_sync(0xffffffffu, (there.x & there.y & there.z & there.w) == 0xffffffffu && j0 + kPtKeys - 1 <= warp_hi && j0 >= warp_lo);
                ok = mbar_wait_all(&sh.s_full[mine], turn & 1u, p.err, kPtEnds);
                if (!ok) { begin_turn(); pass_turn(w); continue; }
                tc_fence_after_sync();
                float2 s[kPtKeys / 2];
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                // half of the keys is looked at while the other is on its way
                tmem_load32(reinterpret_cast<uint32_t*>(s), s_at);
                tmem_load32(reinterpret_cast<uint32_t*>(s) + 32, s_at + 32);
                tc_wait_load();
                tmem_load32(reinterpret_cast<uint32_t*>(s) + 64, s_at + 64);
                tmem_load32(reinterpret_cast<uint32_t*>(s) + 96, s_at + 96);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half == 1) tc_wait_load();
                    if constexpr (S::kEight) {
#pragma unroll
                        for (int i = 32 * half; i < 32 * half + 32; i += 2) {
                            const float4 k = *reinterpret_cast<const float4*>(&m.ks[2 * i]);
                            s[i] = mul2(s[i], make_float2(k.x, k.y));
                            s[i + 1] = mul2(s[i + 1], make_float2(k.z, k.w));
                        }
                    }
                    if (!open) {
                        const uint32_t bits[2] = {half ? there.z : there.x, half ? there.w : there.y};
#pragma unroll
                        for (int i = 32 * half; i < 32 * half + 32; ++i) {
                            const int key = j0 + 2 * i;
                            const uint32_t pair = bits[(i / 16) & 1] >> ((2 * i) & 31);
                            s[i].x = (pair & 1u) != 0 && key <= key_hi && key >= key_lo ? s[i].x : -INFINITY;
                            s[i].y = (pair & 2u) != 0 && key + 1 <= key_hi && key + 1 >= key_lo ? s[i].y : -INFINITY;
                        }
                    }
#pragma unroll
                    for (int i = 32 * half; i < 32 * half + 32; ++i) tops[i & 3] = max3(tops[i & 3], s[i].x, s[i].y);
                }
                float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]);
                top *= row_factor;                                       // (the scale, over a power of two: positive)
                float keep = 1.f;
                bool moved = false;
                if constexpr (S::kEight) {
                    const uint4 e = *reinterpret_cast<const uint4*>(m.exponent);
                    const uint32_t most = min(max(max(e.x, e.y), max(max(e.z, e.w), 1u)), 253u);
                    if (most > unit) {
                        keep = paged_unit_step(unit, most);
                        unit = most;
                        moved = true;
                    }
                }
                if (top > ref + (kPaLift + kPaStep)) {
                    const float next = top - kPaLift, f = exp2_fast(ref - next);
                    l *= f;
                    keep *= f;
                    ref = next;
                    moved = true;
                }
                if (turn != 0 && __any_sync(0xffffffffu, moved)) {       // (S of this step is there, so the unit's last P V has ended)
                    for (uint32_t d = 0; d < c.dim; d += 16) {
                        uint32_t u[16];
                        tc_load16(u, o_at + d);
                        tc_wait_load();
#pragma unroll
                        for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * keep);
                        tmem_store16(o_at + d, u);
                    }
                }
                const float base = ref == -INFINITY ? 0.f : ref, down = S::kEight ? __uint_as_float((254u - unit) << 23) : 1.f;
                const float2 minus = make_float2(-base, -base), factor = make_float2(row_factor, row_factor), downs = make_float2(down, down);
                // weights, half of the keys at a time; they take the first columns of the scores.  The two units take turns at this too: at the same time each would need twice as long
                // for its exponentials, and the tensor cores would wait for both.
                begin_turn();
                float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t u[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 z = s[32 * half + i], x = fma2(z, factor, minus);
                        float2 e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                        sums[i & 1] = add2(sums[i & 1], e);
                        if constexpr (S::kEight) {
                            const float2 v = *reinterpret_cast<const float2*>(&m.vs[64 * half + 2 * i]);
                            e = mul2(e, mul2(v, downs));
                            if (!open) {                                 // (a hidden key's scale may be anything)
                                e.x = z.x != -INFINITY ? e.x : 0.f;
                                e.y = z.y != -INFINITY ? e.y : 0.f;
                            }
                        }
                        u[i] = pack16<S::kBf16>(e.x, e.y);
                    }
                    tmem_store32(s_at + 32 * half, u);
                    tmem_wait_store();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.p_full[mine][half]);
                }
                pass_turn(w);
                l += (sums[0].x + sums[1].x) + (sums[0].y + sums[1].y);
            }
            if (mine < units) ok = ok && mbar_wait_warp_tc(&sh.o_full[mine], 0, p.err, kPtEnds);
        }
        float2 part1 = make_float2(-INFINITY, 0.f);                      // reference and sum of the other unit of the same rows
        uint32_t unit1 = 0;
        if (!two) {
            if (mine == 1) {
                sh.ref[32 * quarter + lane] = ref;
                sh.l[32 * quarter + lane] = l;
                if (warp == 4 && lane == 0) sh.unit = unit;              // (the same in all warps that have rows)
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kPtSoftmax) : "memory");
            if (mine == 0) {
                part1 = make_float2(sh.ref[32 * quarter + lane], sh.l[32 * quarter + lane]);
                unit1 = sh.unit;
            }
        }
        if (!ok && p.splits != 1 && row < rows && (two || mine == 0))    // (a lost wait: the join finds that this part saw nothing)
            p.part_rl[(size_t(q.row0 + (r0 + row) / p.group) * a.heads + kv * p.group + (r0 + row) % p.group) * p.splits + split] = make_float2(-INFINITY, 0.f);
        if (ok && base_row + 32 * quarter < rows && (two || mine == 0)) {
            tc_fence_after_sync();
            const uint32_t t = q.row0 + (r0 + row) / p.group, h = kv * p.group + (r0 + row) % p.group;
            const bool inside = row < rows, whole = p.splits == 1;
            const size_t part = (size_t(t) * a.heads + h) * p.splits + split, to = size_t(t) * a.out_ld + size_t(h) * c.dim;
            const bool none0 = ref == -INFINITY && l == 0.f, none1 = part1.x == -INFINITY && part1.y == 0.f;
            const float sink = whole && inside ? paged_sink(p, h) : -INFINITY, top = fmaxf(fmaxf(ref, part1.x), sink - kPaLift);
            float f0 = ref == -INFINITY ? 0.f : exp2_fast(ref - top), f1 = part1.x == -INFINITY ? 0.f : exp2_fast(part1.x - top);
            float total = (none0 ? 0.f : l * f0) + (none1 ? 0.f : part1.y * f1);
            if (whole) {
                total += paged_sink_weight(sink, top);
                const float g = total == 0.f ? 0.f : 1.f / total;
                f0 *= g;
                f1 *= g;
            } else if (inside) {
                p.part_rl[part] = make_float2(top, total);
            }
            if constexpr (S::kEight) {
                f0 *= __uint_as_float(max(unit, 1u) << 23);
                f1 *= __uint_as_float(max(unit1, 1u) << 23);
            }
            const bool other = !two && units > 1;
            for (uint32_t d = 0; d < c.dim; d += 16) {
                uint32_t u[16], u1[16];
                tc_load16(u, o_at + d);
                if (other) tc_load16(u1, o_at + 128 + d);
                tc_wait_load();
                if (!inside) continue;
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    v[i] = none0 ? 0.f : __uint_as_float(u[i]) * f0;
                    if (other && !none1) v[i] = fmaf(__uint_as_float(u1[i]), f1, v[i]);
                }
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    const float4 x = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]), y = make_float4(v[i + 4], v[i + 5], v[i + 6], v[i + 7]);
                    if (whole) {
                        const uint2 xx = pack_values4(x, a.out_type), yy = pack_values4(y, a.out_type);
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + to + d + i) = make_uint4(xx.x, xx.y, yy.x, yy.y);
                    } else {
                        *reinterpret_cast<float4*>(p.part_o + part * c.dim + d + i) = x;
                        *reinterpret_cast<float4*>(p.part_o + part * c.dim + d + i + 4) = y;
                    }
                }
            }
        }
        tc_fence_before_sync();
    } else if (warp < kPtSoftmax + kPtHelpers) {
        fewer_registers<kPtFewRegs>();
        // ---- what was copied: a warp per 32 rows of every step, a lane per row --------------------------------
        const uint32_t part = warp - kPtSoftmax;
        const uint32_t* table = c.table + size_t(blockIdx.z) * c.table_ld;
        // a row's page is asked for two steps ahead, its scales one
        bool asked = false, next_there = false;
        uint32_t page = 0, in_page = 0, next_row = 0;
        auto ask = [&](uint32_t step) {
            const uint64_t j = uint64_t(lo) + uint64_t(step) * kPtKeys + 32 * part + lane;
            asked = j >= all.lo && j < hi;
            if (!asked) return;
            const uint32_t slot = paged_slot(c, uint32_t(j));
            in_page = uint32_t(j) - slot * c.page_rows;
            page = slot < c.table_ld ? table[slot] : c.pages;
        };
        auto take = [&]() {
            next_there = asked && page < c.pages;
            if (asked && !next_there) atomicOr(p.data_err, ERR_BAD_INDEX);
            next_row = next_there ? (page * c.kv_heads + kv) * c.page_rows + in_page : 0;
        };
        auto publish = [&](uint64_t* bar) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        bool ok = true;
        ask(0);
        take();
        [[maybe_unused]] float ks = 0.f, vs = 0.f;
        if constexpr (S::kEight) {
            if (next_there) { ks = c.k_scale[next_row]; vs = c.v_scale[next_row]; }
        }
        uint32_t there = __ballot_sync(0xffffffffu, next_there);
        ask(1);
        for (uint32_t step = 0; step < steps; ++step) {
            const uint32_t st = step % kPtStages;
            take();                                                      // of the next step
            [[maybe_unused]] float next_ks = 0.f, next_vs = 0.f;
            if constexpr (S::kEight) {
                if (next_there) { next_ks = c.k_scale[next_row]; next_vs = c.v_scale[next_row]; }
            }
            ask(step + 2);
            TcMeta& m = sh.meta[st];
            if constexpr (!S::kEight) {
                ok = mbar_wait_warp(&sh.v_raw[st], (step / kPtStages) & 1u, p.err, kPtEnds);
                if (!ok) break;
                if (there != 0xffffffffu)
                    for (uint32_t r = 0; r < 32; ++r)
                        if (((there >> r) & 1u) == 0 && lane < S::kBlocks * 8) *reinterpret_cast<uint4*>(s_v + st * S::kTile + tile_at(32 * part + r, lane)) = make_uint4(0u, 0u, 0u, 0u);
            } else {
                constexpr uint32_t kUnits = D / 16, kPer = kUnits;       // units of 16 codes of a row, and of a lane
                const uint32_t my_unit = lane % kUnits;
#pragma unroll
                for (uint32_t values = 0; values < 2; ++values) {
                    const uint32_t item = 2 * step + values, slot = item % kPtRing, stages = values ? kPtStages : S::kKeyStages, to_st = step % stages;
                    ok = ok && mbar_wait_warp(&sh.raw_full[slot], (item / kPtRing) & 1u, p.err, kPtEnds);
                    if (step >= stages) ok = ok && mbar_wait_warp(values ? &sh.v_empty[to_st] : &sh.k_empty[(step - stages) & 1u], ((step - stages) >> 1) & 1u, p.err, kPtEnds);
                    if (!ok) break;
                    const uint8_t* from = s_raw + slot * S::kRaw + my_unit * 16;
                    uint8_t* to = (values ? s_v : s_k) + to_st * S::kTile;
#pragma unroll
                    for (int i = 0; i < int(kPer); ++i) {
                        const uint32_t r = (lane + 32 * i) / kUnits;
                        uint4 w = make_uint4(0u, 0u, 0u, 0u);
                        if (((there >> r) & 1u) != 0 && my_unit * 16 < c.dim) w = *reinterpret_cast<const uint4*>(from + (32 * part + r) * c.dim);
                        if constexpr (KIND == LV_TYPE_I8) w = make_uint4(w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u);
                        *reinterpret_cast<uint4*>(to + tile_at(32 * part + r, 2 * my_unit)) =
                            make_uint4(codes_f16<KIND>(w.x, false), codes_f16<KIND>(w.x, true), codes_f16<KIND>(w.y, false), codes_f16<KIND>(w.y, true));
                        *reinterpret_cast<uint4*>(to + tile_at(32 * part + r, 2 * my_unit + 1)) =
                            make_uint4(codes_f16<KIND>(w.z, false), codes_f16<KIND>(w.z, true), codes_f16<KIND>(w.w, false), codes_f16<KIND>(w.w, true));
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.raw_empty[slot]);
                    if (values == 0) publish(&sh.k_full[step & 1u]);
                }
                if (!ok) break;
                m.ks[32 * part + lane] = ks;
                m.vs[32 * part + lane] = vs;
                const uint32_t e = __reduce_max_sync(0xffffffffu, paged_scale_exponent(vs));
                if (lane == 0) m.exponent[part] = e;
            }
            if (lane == 0) m.there[part] = there;
            publish(&sh.v_full[st]);
            there = __ballot_sync(0xffffffffu, next_there);
            if constexpr (S::kEight) { ks = next_ks; vs = next_vs; }
        }
    } else {
        fewer_registers<kPtFewRegs>();
        if (warp == kPtSoftmax + kPtHelpers + 1) {
            // ---- copies: the keys of a step, then its values; a lane per box -----------------------------------------
            const uint32_t* table = c.table + size_t(blockIdx.z) * c.table_ld;
            const uint32_t bytes = S::kEight ? p.box * c.dim : S::kBlocks * p.box * 128;
            uint32_t row = 0, item = 0, page = 0, in_page = 0;
            bool here = false, asked = false;
            auto ask = [&](uint32_t step) {                              // (a step ahead: the table's answer takes as long as a wait)
                const uint64_t j = uint64_t(lo) + uint64_t(step) * kPtKeys + lane * p.box;
                asked = lane * p.box < kPtKeys && j + p.box > all.lo && j < hi;
                if (!asked) return;
                const uint32_t slot = paged_slot(c, uint32_t(j));
                in_page = uint32_t(j) - slot * c.page_rows;
                page = slot < c.table_ld ? table[slot] : c.pages;
            };
            ask(0);
            for (; item < 2 * steps; ++item) {
                const uint32_t step = item >> 1, values = item & 1u, st = step % kPtStages, slot = item % kPtRing;
                if (values == 0) {
                    here = asked && page < c.pages;
                    row = (page * c.kv_heads + kv) * c.page_rows + in_page;
                    ask(step + 1);
                }
                uint64_t* bar = S::kEight ? &sh.raw_full[slot] : values ? &sh.v_raw[st] : &sh.k_full[st];
                if constexpr (S::kEight) {
                    if (item >= kPtRing && !mbar_wait_warp(&sh.raw_empty[slot], (item / kPtRing - 1) & 1u, p.err, kPtEnds)) break;
                } else {
                    if (step >= kPtStages && !mbar_wait_warp(values ? &sh.v_empty[st] : &sh.k_empty[st], (step / kPtStages - 1) & 1u, p.err, kPtEnds)) break;
                }
                const uint32_t n = uint32_t(__popc(__ballot_sync(0xffffffffu, here)));
                if (lane == 0) mbar_expect_tx(bar, n * bytes);
                __syncwarp();
                if (here) {
                    const CUtensorMap* map = values ? &maps.v : &maps.k;
                    if constexpr (S::kEight) {
                        tma_load_2d_plain(s_raw + slot * S::kRaw + lane * bytes, map, 0, int(row), bar);
                    } else {
                        uint8_t* to = (values ? s_v : s_k) + st * S::kTile + lane * p.box * 128;
#pragma unroll
                        for (int block = 0; block < S::kBlocks; ++block) tma_load_2d_plain(to + block * S::kBlock, map, 64 * block, int(row), bar);
                    }
                }
                __syncwarp();
            }
            // (a CTA that gives up leaves when its copies have arrived)
            for (uint32_t i = item - min(item, uint32_t(2 * kPtStages)); i < item; ++i) {
                const uint32_t step = i >> 1, st = step % kPtStages;
                if constexpr (S::kEight) {
                    if (i + kPtRing >= item) mbar_drain(&sh.raw_full[i % kPtRing], (i / kPtRing) & 1u);
                } else {
                    mbar_drain(i & 1u ? &sh.v_raw[st] : &sh.k_full[st], (step / kPtStages) & 1u);
                }
            }
        }
        if (warp & 1) goto meet;
        // ---- products: a warp for each unit (one for both spent 1300 clocks a turn on its waits, as long as the products themselves).  The whole warp waits and counts, one lane
        // issues: values that are the same in all lanes belong in uniform registers, where the instruction wants them, and a reduction tells the compiler which these are.
        constexpr uint32_t kind = (1u << 4) | (S::kBf16 ? (1u << 7) | (1u << 10) : 0u) | (uint32_t(128 >> 4) << 24);
        constexpr uint32_t s_desc = kind | (uint32_t(kPtKeys >> 3) << 17);
        const uint32_t o_desc = kind | (1u << 16) | ((c.dim >> 3) << 17);       // (V is MN-major)
        const uint32_t n = __reduce_max_sync(0xffffffffu, units), both = __reduce_max_sync(0xffffffffu, two ? 1u : 0u), tm = __reduce_max_sync(0xffffffffu, tmem);
        const uint32_t mine = __reduce_max_sync(0xffffffffu, uint32_t(warp - kPtSoftmax - kPtHelpers) / 2);
        const uint64_t q_desc = tc_smem_desc(smem_u32(s_q)) + ((both && mine ? S::kTile : 0u) >> 4), k_desc = tc_smem_desc(smem_u32(s_k)), v_desc = values_desc(smem_u32(s_v), S::kBlock);
        const uint32_t s_at = tm + 128 * mine, o_at = tm + 256 + 128 * mine;
        auto step_of = [&](uint32_t w) { return both ? w >> 1 : w; };
        auto wait_keys = [&](uint32_t w) {
            const uint32_t j = step_of(w);
            return mbar_wait_all(&sh.k_full[j & 1u], (j >> 1) & 1u, p.err, kPtEnds);
        };
        auto keys = [&](uint32_t w) { return k_desc + (((step_of(w) % S::kKeyStages) * S::kTile) >> 4); };
        // (one lane)
        auto scores = [&](uint32_t w, uint64_t kd) {
#pragma unroll
            for (uint32_t k = 0; k < D / 16; ++k) {
                const uint32_t off = (((k >> 2) * S::kBlock) >> 4) + (k & 3u) * 2;
                if (16 * k < c.dim) tc_mma_f16(s_at, q_desc + off, kd + off, s_desc, k != 0);
            }
            tc_commit(&sh.s_full[mine]);
            tc_commit(&sh.k_empty[step_of(w) & 1u]);
        };
        bool ok = mine < n && mbar_wait_all(&sh.q_full, 0, p.err, kPtEnds) && wait_keys(mine);
        if (ok) {
            tc_fence_after_sync();
            const uint64_t kd = keys(mine);
            if (tc_elect()) scores(mine, kd);
            __syncwarp();
        }
        for (uint32_t w = mine; w < n && ok; w += 2) {
            const uint32_t turn = w >> 1, st = step_of(w) % kPtStages;
            const bool more = w + 2 < n;
            // what the products of this turn need beside the weights is waited for first
            ok = mbar_wait_all(&sh.v_full[st], (step_of(w) / kPtStages) & 1u, p.err, kPtEnds) && (!more || wait_keys(w + 2));
            const uint64_t vd = v_desc + ((st * S::kTile) >> 4), kd = keys(w + 2);
            ok = ok && mbar_wait_all(&sh.p_full[mine][0], turn & 1u, p.err, kPtEnds);
            if (!ok) break;
            tc_fence_after_sync();
            if (tc_elect()) {
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)                         // 16 keys: 8 columns of P, two groups of eight rows of V
                    tc_mma_f16_ta(o_at, s_at + 8 * k, vd + 128u * k, o_desc, k != 0 ? 1u : uint32_t(turn != 0));
            }
            __syncwarp();
            ok = mbar_wait_all(&sh.p_full[mine][1], turn & 1u, p.err, kPtEnds);
            if (!ok) break;
            tc_fence_after_sync();
            if (tc_elect()) {
#pragma unroll
                for (uint32_t k = 4; k < 8; ++k) tc_mma_f16_ta(o_at, s_at + 8 * k, vd + 128u * k, o_desc, 1u);
                tc_commit(&sh.v_empty[st]);
                if (more) scores(w + 2, kd);
                else tc_commit(&sh.o_full[mine]);
            }
            __syncwarp();
        }
        if (tc_elect()) tc_commit(&sh.drained[mine]);
        __syncwarp();
        mbar_drain(&sh.drained[mine], 0);
        __syncwarp();
    }
meet:
    __syncthreads();
    if (warp == kPtSoftmax + kPtHelpers) {
        tc_fence_after_sync();
        tc_free(tmem, 512);
    }
}

template <int KIND, int D>
static int tc_launch(lv_ctx* ctx, const PagedAttn& p, uint32_t blocks) {
    auto* kernel = paged_tc_kernel<KIND, D>;
    const size_t smem = TcShape<KIND, D>::kSmem;
    TcMaps maps;
    const uint64_t rows = uint64_t(p.c.pages) * p.c.kv_heads * p.c.page_rows;
    for (int i = 0; i < 2; ++i) {
        CUtensorMap* map = i ? &maps.v : &maps.k;
        const void* base = i ? p.c.v : p.c.k;
        if (TcShape<KIND, D>::kEight) {
            const uint64_t dims[2] = {p.c.dim / 8, rows}, strides[1] = {p.c.dim};
            const uint32_t box[2] = {p.c.dim / 8, p.box};
            if (const int rc = make_tiled_map(map, base, 2, dims, strides, box)) return rc;
        } else if (const int rc = make_bf16_map(map, base, rows, p.c.dim, p.c.dim, p.box)) {
            return rc;
        }
    }
    LV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    LV_CUDA(launch_pdl(ctx, kernel, dim3(p.splits * blocks, p.a.cache.kv_heads, p.a.cache.seqs), dim3(kPtThreads), smem, p, maps));
    return LV_OK;
}

template <int KIND>
static int tc_launch_size(lv_ctx* ctx, const PagedAttn& p, uint32_t blocks) {
    return p.a.cache.dim <= 64 ? tc_launch<KIND, 64>(ctx, p, blocks) : tc_launch<KIND, 128>(ctx, p, blocks);
}

int paged_tc_launch(lv_ctx* ctx, const PagedAttn& p, uint32_t blocks) {
    switch (p.a.cache.type) {
        case LV_TYPE_BF16: return tc_launch_size<LV_TYPE_BF16>(ctx, p, blocks);
        case LV_TYPE_F16: return tc_launch_size<LV_TYPE_F16>(ctx, p, blocks);
        case LV_TYPE_I8: return tc_launch_size<LV_TYPE_I8>(ctx, p, blocks);
        default: return tc_launch_size<LV_TYPE_E4M3>(ctx, p, blocks);
    }
}

}  // namespace lv

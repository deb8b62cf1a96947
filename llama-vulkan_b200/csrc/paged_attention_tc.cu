// Attention of many new tokens over a cache in pages, on the tcgen05 tensor cores (16-bit outputs).
//
// A CTA takes 256 rows -- (token, query head) pairs of one key/value head, in two tiles of 128 -- and walks their keys in steps of 128:
//
//   S = Q K^T          tensor memory, a tile of 128 x 128 f32 per row tile
//   P = 2^(S - r)      a row per thread; 16-bit weights go to tensor memory over the scores that they came from
//   O += P V           P from tensor memory, V as an MN-major operand (its rows are keys)
//
// The two tiles take turns: the tensor cores work for one while the other's weights are computed, and each key and value is fetched once for both.  One lane issues all
// products, in this order for every step: P V of a tile, then S of the tile's next step, so that the scores never overwrite weights that are still to be
// read, and a finished S says that the tile's last P V has finished too.
// Keys and values lie in pages, whose rows four warps fetch: 16-bit rows by 16-byte cp.async straight to their places in the 128-byte swizzle, 8-bit codes through
// registers, converted to f16 on the way (exact).  Rows that no query sees are written as zeros.  References, f16 ranges and scales as in paged_attention.cu.
//
// Every wait is bounded; one that gives up sets the error word, and the CTA drains and frees its tensor memory.
#include <algorithm>

#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace lv {

// Warps: eight of the softmax, four loaders, four of which one issues the products.  Registers move from the latter eight to the former: a row's 128 scores are held at a
// time.  512 threads are launched with 128 registers each: (8 x 176 + 8 x 80) x 32 = 512 x 128.
constexpr int kPtSoftmax = 8, kPtLoaders = 4, kPtThreads = 512, kPtStages = 2, kPtManyRegs = 176, kPtFewRegs = 80;

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

// V: rows are keys (the K of the product), 64 columns per 128-byte row; groups of eight keys 1024 bytes apart, blocks of 64 columns `block` bytes apart
__device__ __forceinline__ uint64_t values_desc(uint32_t smem_addr, uint32_t block) {
    return uint64_t((smem_addr >> 4) & 0x3fffu) | (uint64_t(block >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

template <int KIND, int D>
struct TcShape {
    static constexpr bool kEight = KIND == LV_TYPE_I8 || KIND == LV_TYPE_E4M3, kBf16 = KIND == LV_TYPE_BF16;
    static constexpr int kBlocks = D / 64;                               // of 64 columns
    static constexpr uint32_t kBlock = 128 * 128;                        // bytes of 128 rows of one
    static constexpr uint32_t kTile = kBlocks * kBlock;                  // of a query tile, and of a step's keys or values
    static constexpr size_t kSmem = 1024 + (2 + 2 * kPtStages) * kTile;
};

struct TcMeta {                                                          // of a step's keys
    float ks[kPtKeys], vs[kPtKeys];
    uint32_t there[4], exponent[4];
};

// byte of 16-byte unit u of row r in a tile
__device__ __forceinline__ uint32_t tile_at(uint32_t r, uint32_t u) { return (u >> 3) * (128 * 128) + r * 128 + (((u & 7u) ^ (r & 7u)) << 4); }

template <int KIND, int D>
__global__ void __launch_bounds__(kPtThreads, 1) paged_tc_kernel(const PagedAttn p) {
    using S = TcShape<KIND, D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~uintptr_t(1023));
    uint8_t *s_q = smem, *s_k = smem + 2 * S::kTile, *s_v = s_k + kPtStages * S::kTile;
    __shared__ __align__(16) TcMeta meta[kPtStages];
    __shared__ uint64_t q_full, k_full[kPtStages], k_empty[kPtStages], v_full[kPtStages], v_empty[kPtStages], s_full[2], p_full[2][2], o_full[2], drained;
    __shared__ uint32_t s_tmem;
    const lv_paged_attention_args& a = p.a;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    if (threadIdx.x == 0) {
        mbar_init(&q_full, kPtSoftmax);
        mbar_init(&drained, 1);
        for (int i = 0; i < kPtStages; ++i) { mbar_init(&k_full[i], kPtLoaders); mbar_init(&v_full[i], kPtLoaders); mbar_init(&k_empty[i], 1); mbar_init(&v_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i][0], 4); mbar_init(&p_full[i][1], 4); mbar_init(&o_full[i], 1); }
        fence_mbar_init();
    }
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
    const uint32_t r0 = (n_blocks - 1 - back) * kPtRows, rows = min(uint32_t(kPtRows), all_rows - r0), tiles = rows > 128 ? 2 : 1;
    const PagedRange all = paged_range(p, q, r0, r0 + rows - 1);
    const uint64_t begin = uint64_t(all.lo) + uint64_t(split) * p.chunk;
    if (begin >= all.hi) {
        pdl_launch_dependents();
        return;
    }
    const uint32_t lo = uint32_t(begin), hi = uint32_t(min(uint64_t(all.hi), begin + p.chunk)), steps = (hi - lo + kPtKeys - 1) / kPtKeys;
    if (warp == kPtSoftmax + kPtLoaders) {
        tc_alloc(&s_tmem, 512);
        pdl_launch_dependents();        // (not before: a CTA of the next launch could take the tensor memory that this one needs, and wait for it)
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    const uint32_t tmem_o = tmem + 256;                                  // S of the two tiles in columns 0 and 128, O in 256 and 384

    if (warp < kPtSoftmax) {
        more_registers<kPtManyRegs>();
        // ---- queries, then a row per thread ---------------------------------------------------------
        const uint32_t tile = warp >> 2, quarter = warp & 3, lanes = quarter * 32u << 16;
        float row_factor = 1.f;                                          // of this thread's row
        for (uint32_t i = 0; i < 32; i += 4) {                           // four rows of the warp at a time
            float4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t r = r0 + 32 * warp + i + k, t = q.row0 + r / p.group, h = kv * p.group + r % p.group, d = 4 * lane;
                x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < r0 + rows && d < c.dim) x[k] = load_values4(a.q, size_t(t) * a.q_ld + size_t(h) * c.dim + d, a.q_type);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t r = r0 + 32 * warp + i + k, t = q.row0 + r / p.group, d = 4 * lane, at_row = 32 * quarter + i + k;
                if (a.angles != nullptr && r < r0 + rows && d < c.dim) x[k] = rotate4(x[k], a.angles + size_t(t) * a.angle_ld, d, a.angle_pairs);
                float f = a.scale * kPaLog2e;
                if constexpr (!S::kBf16) {
                    const float u = paged_row_unit(warp_max(fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w)))));
                    if (i + k == uint32_t(lane)) row_factor = f / u;
                    f = u;
                }
                if (d < D) *reinterpret_cast<uint2*>(s_q + tile * S::kTile + tile_at(at_row, d >> 3) + (d & 4u) * 2) =
                    make_uint2(pack16<S::kBf16>(x[k].x * f, x[k].y * f), pack16<S::kBf16>(x[k].z * f, x[k].w * f));
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);
        if (tile < tiles) {
            const uint32_t row = 128 * tile + 32 * quarter + lane, before = q.len - q.n;
            const uint32_t pos = before + (r0 + min(row, rows - 1)) / p.group;
            const int key_hi = row < rows ? int(pos) - int(lo) : -1, key_lo = int(paged_first_key(pos, a.window)) - int(lo);
            // keys that every row of the warp sees
            const uint32_t w0 = r0 + min(128 * tile + 32 * quarter, rows - 1), w1 = r0 + min(128 * tile + 32 * quarter + 31, rows - 1);
            const int warp_hi = int(before + w0 / p.group) - int(lo), warp_lo = int(paged_first_key(before + w1 / p.group, a.window)) - int(lo);
            const uint32_t s_at = tmem + lanes + tile * 128, o_at = tmem_o + lanes + tile * 128;
            float ref = -INFINITY, l = 0.f;
            uint32_t unit = 0;
            bool ok = true;
            for (uint32_t j = 0; j < steps; ++j) {
                const uint32_t st = j % kPtStages;
                // (after a lost wait the warp goes through the remaining steps without work)
                ok = ok && mbar_wait_warp(&v_full[st], (j / kPtStages) & 1u, p.err) && mbar_wait_warp_tc(&s_full[tile], j & 1u, p.err);
                if (!ok) continue;
                tc_fence_after_sync();
                const TcMeta& m = meta[st];
                const int j0 = int(j * kPtKeys);
                float2 s[kPtKeys / 2];
                {
                    uint32_t* u = reinterpret_cast<uint32_t*>(s);
#pragma unroll
                    for (int i = 0; i < kPtKeys; i += 32) tmem_load32(u + i, s_at + i);
                    tc_wait_load();
                }
                const uint4 there = *reinterpret_cast<const uint4*>(m.there);
                const bool open = (there.x & there.y & there.z & there.w) == 0xffffffffu && j0 + kPtKeys - 1 <= warp_hi && j0 >= warp_lo;
                if constexpr (S::kEight) {
#pragma unroll
                    for (int i = 0; i < kPtKeys / 2; i += 2) {
                        const float4 k = *reinterpret_cast<const float4*>(&m.ks[2 * i]);
                        s[i] = mul2(s[i], make_float2(k.x, k.y));
                        s[i + 1] = mul2(s[i + 1], make_float2(k.z, k.w));
                    }
                }
                if (!open) {
                    const uint32_t w[4] = {there.x, there.y, there.z, there.w};
#pragma unroll
                    for (int i = 0; i < kPtKeys / 2; ++i) {
                        const int key = j0 + 2 * i;
                        const uint32_t two = w[i / 16] >> ((2 * i) & 31);
                        s[i].x = (two & 1u) != 0 && key <= key_hi && key >= key_lo ? s[i].x : -INFINITY;
                        s[i].y = (two & 2u) != 0 && key + 1 <= key_hi && key + 1 >= key_lo ? s[i].y : -INFINITY;
                    }
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kPtKeys / 2; ++i) tops[i & 3] = fmaxf(tops[i & 3], fmaxf(s[i].x, s[i].y));
                float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                if constexpr (!S::kBf16) top *= row_factor;              // (the scale over a power of two: positive)
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
                if (j != 0 && __any_sync(0xffffffffu, moved)) {          // (S of this step is there, so P V of the last one has ended)
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
                // weights, half of the keys at a time; they take the first columns of the scores
                float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t u[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float2 z = s[32 * half + i], x = S::kBf16 ? add2(z, minus) : fma2(z, factor, minus);
                        float2 w = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                        sums[i & 1] = add2(sums[i & 1], w);
                        if constexpr (S::kEight) {
                            const float2 v = *reinterpret_cast<const float2*>(&m.vs[64 * half + 2 * i]);
                            w = mul2(w, mul2(v, downs));
                            if (!open) {                                 // (a hidden key's scale may be anything)
                                w.x = z.x != -INFINITY ? w.x : 0.f;
                                w.y = z.y != -INFINITY ? w.y : 0.f;
                            }
                        }
                        u[i] = pack16<S::kBf16>(w.x, w.y);
                    }
                    tmem_store32(s_at + 32 * half, u);
                    tmem_wait_store();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[tile][half]);
                }
                l += (sums[0].x + sums[1].x) + (sums[0].y + sums[1].y);
            }
            ok = ok && mbar_wait_warp_tc(&o_full[tile], 0, p.err);
            if (ok) {
                tc_fence_after_sync();
                const uint32_t t = q.row0 + (r0 + row) / p.group, h = kv * p.group + (r0 + row) % p.group;
                const bool mine = row < rows, whole = p.splits == 1;
                float f = S::kEight ? __uint_as_float(max(unit, 1u) << 23) : 1.f;
                const size_t part = (size_t(t) * a.heads + h) * p.splits + split, to = size_t(t) * a.out_ld + size_t(h) * c.dim;
                if (whole) {
                    const float sink = mine ? paged_sink(p, h) : -INFINITY, top = fmaxf(ref, sink - kPaLift);
                    const float g = ref == -INFINITY ? 0.f : exp2_fast(ref - top), total = fmaf(l, g, paged_sink_weight(sink, top));
                    f = total == 0.f ? 0.f : f * g / total;
                } else if (mine) {
                    p.part_rl[part] = make_float2(ref, l);
                }
                const bool none = ref == -INFINITY && l == 0.f;
                for (uint32_t d = 0; d < c.dim; d += 16) {
                    uint32_t u[16];
                    tc_load16(u, o_at + d);
                    tc_wait_load();
                    if (!mine) continue;
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = none ? 0.f : __uint_as_float(u[i]) * f;
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
        }
    } else if (warp < kPtSoftmax + kPtLoaders) {
        fewer_registers<kPtFewRegs>();
        // ---- keys and values: a warp per 32 rows of every step, a lane looks one up -------------------------
        const uint32_t part = warp - kPtSoftmax;
        const uint32_t* table = c.table + size_t(blockIdx.z) * c.table_ld;
        uint32_t next_row = 0;
        bool next_there = false;
        auto look_up = [&](uint32_t step) {
            const uint64_t j = uint64_t(lo) + uint64_t(step) * kPtKeys + 32 * part + lane;
            next_there = j < hi;
            if (next_there && !paged_row(c, table, uint32_t(j), kv, &next_row)) {
                atomicOr(p.err, ERR_BAD_INDEX);
                next_there = false;
            }
            if (!next_there) next_row = 0;
        };
        auto publish = [&](uint64_t* bar) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto write_meta = [&](uint32_t st, uint32_t there) {
            TcMeta& m = meta[st];
            if constexpr (S::kEight) {
                const float ks = next_there ? c.k_scale[next_row] : 0.f, vs = next_there ? c.v_scale[next_row] : 0.f;
                m.ks[32 * part + lane] = ks;
                m.vs[32 * part + lane] = vs;
                const uint32_t e = __reduce_max_sync(0xffffffffu, paged_scale_exponent(vs));
                if (lane == 0) m.exponent[part] = e;
            }
            if (lane == 0) m.there[part] = there;
        };
        bool ok = true;
        look_up(0);
        if constexpr (!S::kEight) {
            constexpr uint32_t kUnits = D / 8, kPer = kUnits;            // 16-byte units of a row, and of a lane in a step
            const uint32_t row_bytes = c.dim * 2;
            const uint32_t my_unit = lane % kUnits;
            const uint8_t *my_k = static_cast<const uint8_t*>(c.k) + my_unit * 16, *my_v = static_cast<const uint8_t*>(c.v) + my_unit * 16;
            // two tiles (keys, values) a step; a tile is published while the next two are on their way, or before a wait for a place
            uint32_t published = 0;
            auto publish_to = [&](uint32_t end) {
                for (; published < end; ++published) publish(published & 1u ? &v_full[(published >> 1) % kPtStages] : &k_full[(published >> 1) % kPtStages]);
            };
            for (uint32_t item = 0; item < 2 * steps; ++item) {
                const uint32_t step = item >> 1, st = step % kPtStages, values = item & 1u;
                if (step >= kPtStages) {
                    uint64_t* empty = values ? &v_empty[st] : &k_empty[st];
                    const uint32_t phase = (step / kPtStages - 1) & 1u;
                    if (!__any_sync(0xffffffffu, mbar_poll(empty, phase))) {
                        cp_async_wait<0>();
                        publish_to(item);
                    }
                    ok = mbar_wait_warp(empty, phase, p.err);
                    if (!ok) break;
                }
                const uint32_t there = __ballot_sync(0xffffffffu, next_there);
                const uint32_t to = smem_u32((values ? s_v : s_k) + st * S::kTile);
                const uint8_t* from = values ? my_v : my_k;
#pragma unroll
                for (int i = 0; i < int(kPer); ++i) {
                    const uint32_t r = (lane + 32 * i) / kUnits;
                    const uint64_t off = uint64_t(__shfl_sync(0xffffffffu, next_row, int(r))) * row_bytes;
                    const bool here = ((there >> r) & 1u) != 0 && my_unit * 16 < row_bytes;
                    cp_async16_zfill(to + tile_at(32 * part + r, my_unit), here ? from + off : static_cast<const uint8_t*>(c.k), here);
                }
                if (values) {
                    write_meta(st, there);
                    look_up(step + 1);
                }
                cp_async_commit();
                if (item >= 2 && published < item - 1) {
                    cp_async_wait<2>();
                    publish_to(item - 1);
                }
            }
            cp_async_wait<0>();
            if (ok) publish_to(2 * steps);
        } else {
            constexpr uint32_t kUnits = D / 16, kPer = kUnits;           // units of 16 codes
            uint4 code[kPer];
            auto fetch = [&](const void* base) {
                const uint32_t there = __ballot_sync(0xffffffffu, next_there);
#pragma unroll
                for (int i = 0; i < int(kPer); ++i) {
                    const uint32_t at = lane + 32 * i, r = at / kUnits, u = at % kUnits;
                    const uint32_t row = __shfl_sync(0xffffffffu, next_row, int(r));
                    // (codes 0 of int8 are 0x80 here: their sign bits are flipped)
                    code[i] = KIND == LV_TYPE_I8 ? make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u) : make_uint4(0u, 0u, 0u, 0u);
                    if (((there >> r) & 1u) != 0 && u * 16 < c.dim) {
                        const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + uint64_t(row) * c.dim + u * 16));
                        code[i] = KIND == LV_TYPE_I8 ? make_uint4(w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u) : w;
                    }
                }
                return there;
            };
            auto convert = [&](uint8_t* to) {
#pragma unroll
                for (int i = 0; i < int(kPer); ++i) {
                    const uint32_t at = lane + 32 * i, r = at / kUnits, u = at % kUnits;
                    const uint4 w = code[i];
                    *reinterpret_cast<uint4*>(to + tile_at(32 * part + r, 2 * u)) =
                        make_uint4(codes_f16<KIND>(w.x, false), codes_f16<KIND>(w.x, true), codes_f16<KIND>(w.y, false), codes_f16<KIND>(w.y, true));
                    *reinterpret_cast<uint4*>(to + tile_at(32 * part + r, 2 * u + 1)) =
                        make_uint4(codes_f16<KIND>(w.z, false), codes_f16<KIND>(w.z, true), codes_f16<KIND>(w.w, false), codes_f16<KIND>(w.w, true));
                }
            };
            for (uint32_t step = 0; step < steps && ok; ++step) {
                const uint32_t st = step % kPtStages, phase = (step / kPtStages - 1) & 1u;
                const uint32_t there = fetch(c.k);
                ok = step < kPtStages || mbar_wait_warp(&k_empty[st], phase, p.err);
                if (!ok) break;
                convert(s_k + st * S::kTile);
                publish(&k_full[st]);
                fetch(c.v);
                ok = step < kPtStages || mbar_wait_warp(&v_empty[st], phase, p.err);
                if (!ok) break;
                convert(s_v + st * S::kTile);
                write_meta(st, there);
                publish(&v_full[st]);
                look_up(step + 1);
            }
        }
    } else {
        fewer_registers<kPtFewRegs>();
        if (warp != kPtSoftmax + kPtLoaders || lane != 0) goto meet;
        // ---- products ------------------------------------------------------------------------------
        constexpr uint32_t kind = (1u << 4) | (S::kBf16 ? (1u << 7) | (1u << 10) : 0u) | (uint32_t(128 >> 4) << 24);
        const uint32_t s_desc = kind | (uint32_t(kPtKeys >> 3) << 17), o_desc = kind | (1u << 16) | ((c.dim >> 3) << 17);      // (V is MN-major)
        const uint64_t q_desc = tc_smem_desc(smem_u32(s_q)), k_desc = tc_smem_desc(smem_u32(s_k)), v_desc = values_desc(smem_u32(s_v), S::kBlock);
        const uint32_t k_steps = c.dim / 16;
        auto scores = [&](uint32_t tile, uint32_t j) {
            const uint64_t qd = q_desc + ((tile * S::kTile) >> 4), kd = k_desc + (((j % kPtStages) * S::kTile) >> 4);
            for (uint32_t k = 0; k < k_steps; ++k) {
                const uint32_t off = (((k >> 2) * S::kBlock) >> 4) + (k & 3u) * 2;
                tc_mma_f16(tmem + tile * 128, qd + off, kd + off, s_desc, k != 0);
            }
            tc_commit(&s_full[tile]);
            if (tile + 1 == tiles) tc_commit(&k_empty[j % kPtStages]);
        };
        bool ok = mbar_wait(&q_full, 0, p.err) && mbar_wait(&k_full[0], 0, p.err);
        if (ok) {
            tc_fence_after_sync();
            for (uint32_t tile = 0; tile < tiles; ++tile) scores(tile, 0);
        }
        for (uint32_t j = 0; j < steps && ok; ++j) {
            const uint32_t st = j % kPtStages, next = (j + 1) % kPtStages;
            ok = mbar_wait(&v_full[st], (j / kPtStages) & 1u, p.err);
            for (uint32_t tile = 0; tile < tiles && ok; ++tile) {
                const uint64_t vd = v_desc + ((st * S::kTile) >> 4);
                for (uint32_t half = 0; half < 2 && ok; ++half) {
                    ok = mbar_wait(&p_full[tile][half], j & 1u, p.err);
                    if (!ok) break;
                    tc_fence_after_sync();
#pragma unroll
                    for (uint32_t k = 0; k < kPtKeys / 32; ++k)          // 16 keys: 8 columns of P, two groups of eight rows of V
                        tc_mma_f16_ta(tmem_o + tile * 128, tmem + tile * 128 + 32 * half + 8 * k, vd + 128u * (4 * half + k), o_desc, j != 0 || half != 0 || k != 0);
                }
                if (!ok) break;
                if (tile + 1 == tiles) tc_commit(&v_empty[st]);
                if (j + 1 == steps) {
                    tc_commit(&o_full[tile]);
                } else {
                    if (tile == 0) {
                        ok = mbar_wait(&k_full[next], ((j + 1) / kPtStages) & 1u, p.err);
                        if (!ok) break;
                        tc_fence_after_sync();
                    }
                    scores(tile, j + 1);
                }
            }
        }
        tc_commit(&drained);
        mbar_drain(&drained, 0);
    }
meet:
    __syncthreads();
    if (warp == kPtSoftmax + kPtLoaders) {
        tc_fence_after_sync();
        tc_free(tmem, 512);
    }
}

template <int KIND, int D>
static int tc_launch(lv_ctx* ctx, const PagedAttn& p, uint32_t blocks) {
    auto* kernel = paged_tc_kernel<KIND, D>;
    const size_t smem = TcShape<KIND, D>::kSmem;
    LV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    LV_CUDA(launch_pdl(ctx, kernel, dim3(p.splits * blocks, p.a.cache.kv_heads, p.a.cache.seqs), dim3(kPtThreads), smem, p));
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

// Probabilities from logits, and drafted tokens against them.
#include <float.h>
#include <type_traits>

#include "attention_gqa.cuh"
#include "paged.cuh"

namespace lv {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
// a word (two words) into the shared memory of another CTA of the cluster
__device__ __forceinline__ void cluster_store(void* local, uint32_t rank, uint2 v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(v.x), "r"(v.y) : "memory");
}

// Before the first store into another CTA's memory it has to be there: arrive first thing, wait behind the earlier launch.
__device__ __forceinline__ void cluster_here() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_all_here() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// ---- probabilities --------------------------------------------------------------------------------

// out = e^((x - m) / T) / sum: a cluster of up to 16 CTAs takes a row and its CTAs tell one another their maximum and sum once.  Where a CTA's share fits its
// registers (HELD: 8192 values) a value is read, raised and written once; else every thread keeps a running maximum and sum, and values are read (from the L2) and raised a second time.
// 512 rows of 128000: 121 us, 4.3 TB/s of 524 MB; of 128001, off their 16 bytes: 203 (one CTA per row: 418 us; all of a row held in registers, eight groups a thread: 165; every load with its bounds: 125).  5 rows of 32000: 4.4 us, a launch and two meetings (read again: 5.2).
constexpr int kProbThreads = 512, kProbGroups = 4;                       // groups of four values that a thread holds, or has on their way at a time
constexpr uint32_t kProbHeld = kProbThreads * 4 * kProbGroups;           // of a CTA: 8192
constexpr int kProbCluster = 16;

struct Probabilities {
    float* out;
    const float* logits;
    const float* temperature;
    uint32_t out_ld, ld, vocab, each;                                    // each: values of a CTA, a multiple of 4
};

// the first index of the larger value (NaN is smaller than all)
__device__ __forceinline__ void first_max(float& v, uint32_t& i, float w, uint32_t j) {
    if (w > v || (w == v && j < i)) { v = w; i = j; }
}

// VEC: rows are 16-byte aligned; HELD: a CTA's values fit its registers
template <bool VEC, bool HELD>
__global__ void __launch_bounds__(kProbThreads, 3) probabilities_kernel(const Probabilities p) {
    pdl_launch_dependents();
    cluster_here();
    pdl_wait();
    cluster_all_here();
    __shared__ float s_top[kProbThreads / 32], s_sum[kProbThreads / 32];
    __shared__ uint32_t s_at[kProbThreads / 32];
    __shared__ __align__(8) uint2 s_all[2][kProbCluster];                 // {maximum, its index}, {sum}
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x / 32, rank = cluster_rank(), n = cluster_size(), row = blockIdx.x / n;
    const float* x = p.logits + size_t(row) * p.ld;
    float* y = p.out + size_t(row) * p.out_ld;
    const float T = p.temperature ? p.temperature[row] : 1.f;
    // e^(z / T) as a power of two.  Finite and above zero: zero times infinity is NaN, for equal values as well as for what lies behind the end
    const float f = T == 0.f ? 1.f : T > 0.f ? fmaxf(fminf(1.4426950408889634f / T, FLT_MAX), __uint_as_float(1u)) : NAN;
    const uint32_t lo = min(p.vocab, rank * p.each), hi = min(p.vocab, lo + p.each);
    // values i .. i + 3; those behind the end count as -inf.  (Vectors first, the few values behind the last whole one in a branch of their own: the loads of
    // several calls are on their way together.)
    const uint32_t whole_hi = VEC ? lo + (hi - lo) / 4 * 4 : lo;
    auto load4 = [&](uint32_t i) {
        float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (i < whole_hi) return *reinterpret_cast<const float4*>(x + i);
        if (i < hi) v.x = x[i];
        if (i + 1 < hi) v.y = x[i + 1];
        if (i + 2 < hi) v.z = x[i + 2];
        if (i + 3 < hi) v.w = x[i + 3];
        return v;
    };
    auto store4 = [&](uint32_t i, const float4& v) {
        if (i < whole_hi) {
            *reinterpret_cast<float4*>(y + i) = v;
            return;
        }
        if (i < hi) y[i] = v.x;
        if (i + 1 < hi) y[i + 1] = v.y;
        if (i + 2 < hi) y[i + 2] = v.z;
        if (i + 3 < hi) y[i + 3] = v.w;
    };
    constexpr uint32_t kStep = kProbThreads * 4;
    float4 v[kProbGroups];
    float top = -INFINITY, sum = 0.f, base = 0.f;
    uint32_t at = 0xffffffffu;
    auto look = [&](const float4& w, uint32_t i) {
        // (in the order of the indexes: a later value has to be larger)
        if (w.x > top) { top = w.x; at = i; }
        if (w.y > top) { top = w.y; at = i + 1; }
        if (w.z > top) { top = w.z; at = i + 2; }
        if (w.w > top) { top = w.w; at = i + 3; }
        if (at == 0xffffffffu) {                                         // nothing above -inf so far: the first -inf itself (what lies behind the end is nobody's)
            if (w.w == top && i + 3 < hi) at = i + 3;
            if (w.z == top && i + 2 < hi) at = i + 2;
            if (w.y == top && i + 1 < hi) at = i + 1;
            if (w.x == top && i < hi) at = i;
        }
    };
    auto raise4 = [&](const float4& w) { return make_float4(exp2_fast((w.x - base) * f), exp2_fast((w.y - base) * f), exp2_fast((w.z - base) * f), exp2_fast((w.w - base) * f)); };
    const uint32_t mine0 = lo + 4 * threadIdx.x;
    if (T == 0.f) {
        for (uint32_t i = mine0; i < hi; i += kStep) look(load4(i), i);
    } else {
        // a running maximum of each thread; the exponentials of the values held are taken again below the CTA's
        auto take = [&](auto is_whole, uint32_t i0) {                    // whole: no value of the thread's groups is behind the end
            constexpr bool whole = decltype(is_whole)::value;
#pragma unroll
            for (int k = 0; k < kProbGroups; ++k) v[k] = whole ? *reinterpret_cast<const float4*>(x + i0 + k * kStep) : load4(i0 + k * kStep);
            float most = top;
#pragma unroll
            for (int k = 0; k < kProbGroups; ++k) most = fmaxf(fmaxf(most, fmaxf(v[k].x, v[k].y)), fmaxf(v[k].z, v[k].w));
            if constexpr (!HELD) {
                base = most == -INFINITY ? 0.f : most;
                sum *= exp2_fast((top - base) * f);                      // (0 while there is no maximum)
#pragma unroll
                for (int k = 0; k < kProbGroups; ++k) {
                    if (!whole && i0 + k * kStep >= hi) continue;
                    const float4 w = raise4(v[k]);
                    sum += (w.x + w.y) + (w.z + w.w);
                }
            }
            top = most;
        };
        for (uint32_t i0 = mine0; i0 < hi; i0 += kStep * kProbGroups) {
            if (VEC && i0 + (kProbGroups - 1) * kStep < whole_hi) take(std::true_type{}, i0);
            else take(std::false_type{}, i0);
        }
    }
    const float own = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float w = __shfl_xor_sync(0xffffffffu, top, o);
        const uint32_t j = __shfl_xor_sync(0xffffffffu, at, o);
        first_max(top, at, w, j);
    }
    if (lane == 0) { s_top[warp] = top; s_at[warp] = at; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kProbThreads / 32; ++w) first_max(top, at, s_top[w], s_at[w]);
    base = top == -INFINITY ? 0.f : top;
    if (T != 0.f) {
        if constexpr (HELD) {
#pragma unroll
            for (int k = 0; k < kProbGroups; ++k) {
                if (mine0 + k * kStep >= hi) continue;
                v[k] = raise4(v[k]);
                sum += (v[k].x + v[k].y) + (v[k].z + v[k].w);
            }
        } else if (own != -INFINITY) {
            sum *= exp2_fast((own - base) * f);
        }
        sum = warp_sum(sum);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < kProbThreads / 32; ++w) sum += s_sum[w];
    }
    float whole = top, total = 0.f;
    if (threadIdx.x < n) {
        cluster_store(&s_all[0][rank], threadIdx.x, make_uint2(__float_as_uint(top), at));
        cluster_store(&s_all[1][rank], threadIdx.x, make_uint2(__float_as_uint(sum), 0u));
    }
    cluster_sync();
    for (uint32_t r = 0; r < n; ++r) first_max(whole, at, __uint_as_float(s_all[0][r].x), s_all[0][r].y);
    for (uint32_t r = 0; r < n; ++r) {
        const float m = __uint_as_float(s_all[0][r].x), part = __uint_as_float(s_all[1][r].x);
        total += m == -INFINITY ? part : part * exp2_fast((m - whole) * f);   // (without a maximum there is nothing, or NaN)
    }
    if (T == 0.f) {
        if (at == 0xffffffffu) at = 0;
        for (uint32_t i = mine0; i < hi; i += kStep) store4(i, make_float4(i == at, i + 1 == at, i + 2 == at, i + 3 == at));
        return;
    }
    const float g = total == 0.f ? 0.f : (top == -INFINITY ? 1.f : exp2_fast((top - whole) * f)) / total;
    auto give = [&](auto is_whole, uint32_t i0) {
        constexpr bool whole = decltype(is_whole)::value;
        if constexpr (!HELD) {
#pragma unroll
            for (int k = 0; k < kProbGroups; ++k) v[k] = whole ? *reinterpret_cast<const float4*>(x + i0 + k * kStep) : load4(i0 + k * kStep);
#pragma unroll
            for (int k = 0; k < kProbGroups; ++k) v[k] = raise4(v[k]);
        }
#pragma unroll
        for (int k = 0; k < kProbGroups; ++k) {
            const float4 w = make_float4(v[k].x * g, v[k].y * g, v[k].z * g, v[k].w * g);
            if (whole) *reinterpret_cast<float4*>(y + i0 + k * kStep) = w;
            else store4(i0 + k * kStep, w);
        }
    };
    for (uint32_t i0 = mine0; i0 < hi; i0 += kStep * kProbGroups) {
        if (VEC && i0 + (kProbGroups - 1) * kStep < whole_hi) give(std::true_type{}, i0);
        else give(std::false_type{}, i0);
    }
}

// ---- verification ---------------------------------------------------------------------------------

// A cluster of eight CTAs takes a sequence.  Every CTA finds the first rejected draft by itself (two values a draft), then they sum the weights of the one row that
// a token is drawn from, each an eighth of it and every warp a run of neighbours, and tell one another their sums.  The bounds between runs are the same numbers
// for both neighbours and never decrease, and the target is below the last one (pick is at most 1 - 2^-24), so that exactly one run holds it, one with weight; its warp looks through it
// again.  Sums are f64: the first index whose cumulative weight is above
// the target does not depend on the order of the sums but where the two agree to 2^-52.
// 64 sequences with up to 7 drafts, vocabulary 128000: 21.7 us, 3.0 TB/s of 65 MB: two CTAs per SM by their registers, so 1.7 rounds that each wait for look-ups and loads (one CTA per
// sequence: 110 us; 256 threads: 20.7, but 4.65 for one sequence; clusters of four: 21.1 and 4.9).  One
// sequence with 4 drafts: 4.3 us, a launch and its meetings (72 us).
constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32, kVerifyCluster = 8;
constexpr uint32_t kNobody = 0xffffffffu;

template <bool VEC>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const lv_verify_args a, uint32_t* err) {
    pdl_launch_dependents();
    cluster_here();
    pdl_wait();
    cluster_all_here();
    __shared__ double s_before[kVerifyWarps + 1];
    __shared__ __align__(8) uint2 s_all[2][kVerifyCluster];              // the CTAs' sums (of the first and of the second attempt)
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x / 32, rank = cluster_rank(), s = blockIdx.x / kVerifyCluster;
    const uint32_t row0 = a.starts[s], row1 = a.starts[s + 1];
    const float pick = a.pick[s];
    if (row0 > row1 || row1 > a.rows) {
        if (rank == 0 && threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
        return;
    }
    if (row0 == row1) {
        if (rank == 0 && threadIdx.x == 0) a.accepted[s] = 0;
        return;
    }
    // every warp looks at the drafts: no barrier
    const uint32_t n = row1 - row0 - 1;
    uint32_t accepted = n, drafted = kNobody;
    for (uint32_t b = 0; b < n; b += 32) {
        bool bad = false;
        uint32_t d = kNobody;
        if (b + lane < n) {
            const uint32_t r = row0 + b + lane;
            d = a.drafted[r];
            bad = d >= a.vocab;
            if (!bad) {
                const double q = a.draft ? double(a.draft[size_t(r) * a.draft_ld + d]) : 1.0;
                bad = !(double(a.accept[r]) * q < double(a.target[size_t(r) * a.target_ld + d]));
            }
        }
        const uint32_t first = __ballot_sync(0xffffffffu, bad);
        if (first != 0) {
            const int l = __ffs(int(first)) - 1;
            accepted = b + uint32_t(l);
            drafted = __shfl_sync(0xffffffffu, d, l);
            break;
        }
    }
    if (accepted < n && drafted >= a.vocab && rank == 0 && threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
    const uint32_t r = row0 + accepted;
    const float *p = a.target + size_t(r) * a.target_ld, *q = a.draft ? a.draft + size_t(r) * a.draft_ld : nullptr;
    // runs of 128 values: those of this warp
    const uint32_t each = (a.vocab + 128 * kVerifyCluster * kVerifyWarps - 1) / (128 * kVerifyCluster * kVerifyWarps);
    const uint64_t lo = uint64_t(rank * kVerifyWarps + warp) * each * 128;
    const uint32_t whole_hi = VEC ? a.vocab / 4 * 4 : 0;
    auto load4 = [&](const float* x, uint64_t i) {
        if (VEC && i < whole_hi) return *reinterpret_cast<const float4*>(x + i);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < a.vocab) v.x = x[i];
        if (i + 1 < a.vocab) v.y = x[i + 1];
        if (i + 2 < a.vocab) v.z = x[i + 2];
        if (i + 3 < a.vocab) v.w = x[i + 3];
        return v;
    };
    struct Four { double w[4]; };
    auto draft4 = [&](uint64_t i) { return q ? load4(q, i) : make_float4(i == drafted, i + 1 == drafted, i + 2 == drafted, i + 3 == drafted); };
    auto differences = [](const float4& x, const float4& y) {
        Four f = {{double(x.x) - double(y.x), double(x.y) - double(y.y), double(x.z) - double(y.z), double(x.w) - double(y.w)}};
#pragma unroll
        for (int k = 0; k < 4; ++k) f.w[k] = f.w[k] > 0.0 ? f.w[k] : 0.0;
        return f;
    };
    auto weights = [&](uint64_t i, bool rest) { return differences(load4(p, i), rest ? draft4(i) : make_float4(0.f, 0.f, 0.f, 0.f)); };
    bool rest = accepted < n;
    double mine = 0.0, total = 0.0, cta0 = 0.0, cta1 = 0.0;
    for (int attempt = 0;; ++attempt) {
        mine = 0.0;
        uint32_t k = 0;
        if (VEC && lo + 128 * each <= whole_hi) {                        // whole runs: eight loads on their way at a time
            for (; k + 4 <= each; k += 4) {
                float4 x[4], y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t i = lo + 128 * (k + j) + 4 * lane;
                    x[j] = *reinterpret_cast<const float4*>(p + i);
                    y[j] = rest && q ? *reinterpret_cast<const float4*>(q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (rest && !q) y[j] = draft4(lo + 128 * (k + j) + 4 * lane);
                    const Four f = differences(x[j], y[j]);
                    mine += (f.w[0] + f.w[1]) + (f.w[2] + f.w[3]);
                }
            }
        }
        for (; k < each; ++k) {
            const Four f = weights(lo + 128 * k + 4 * lane, rest);
            mine += (f.w[0] + f.w[1]) + (f.w[2] + f.w[3]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (attempt != 0) __syncthreads();
        if (lane == 0) s_before[warp + 1] = mine;
        __syncthreads();
        if (warp == 0) {
            // one after the other: every bound is the one before plus what lies between, so that bounds rise, and stay where a run has no weight
            double run = 0.0;
#pragma unroll
            for (uint32_t w = 0; w < kVerifyWarps; ++w) run += w <= lane ? s_before[w + 1] : 0.0;
            __syncwarp();
            if (lane < kVerifyWarps) s_before[lane + 1] = run;
            if (lane == 0) s_before[0] = 0.0;
            const double sum = __shfl_sync(0xffffffffu, run, kVerifyWarps - 1);
            if (lane < kVerifyCluster) cluster_store(&s_all[attempt][rank], lane, make_uint2(uint32_t(__double2loint(sum)), uint32_t(__double2hiint(sum))));
        }
        cluster_sync();
        total = 0.0;
#pragma unroll
        for (uint32_t c = 0; c < kVerifyCluster; ++c) {
            const uint2 u = s_all[attempt][c];
            if (c == rank) cta0 = total;
            total += __hiloint2double(int(u.y), int(u.x));
            if (c == rank) cta1 = total;
        }
        if (total > 0.0 || !rest) break;
        rest = false;                                                    // nothing is left behind the draft: from the target itself
    }
    const bool drawn = total > 0.0 && total < INFINITY && pick >= 0.f && pick < 1.f;
    if (rank == 0) {
        for (uint32_t i = threadIdx.x; i <= n; i += kVerifyThreads)
            if (i != accepted) a.tokens[row0 + i] = i < accepted ? a.drafted[row0 + i] : kNobody;
        if (threadIdx.x == 0) {
            a.accepted[s] = accepted;
            if (a.lens) {
                const uint32_t len = a.lens[s], gone = n - accepted;
                if (len >= gone) a.lens[s] = len - gone;
                else atomicOr(err, ERR_BAD_INDEX);
            }
            if (!drawn) {
                a.tokens[r] = kNobody;
                atomicOr(err, ERR_BAD_INDEX);
            }
        }
    }
    // the run that holds the target: the last bound of a CTA is the first one of the next (its warps' sums and the CTAs' are added up in order)
    const double target = double(pick) * total;
    const double from = cta0 + s_before[warp], to = warp + 1 == kVerifyWarps ? cta1 : cta0 + s_before[warp + 1];
    if (!drawn || !(from <= target && target < to)) return;
    double run = from;
    uint32_t found = kNobody, fallback = kNobody;
    for (uint32_t k = 0; k < each && found == kNobody; ++k) {
        const uint64_t i = lo + 128 * k + 4 * lane;
        const Four f = weights(i, rest);
        const double sum = (f.w[0] + f.w[1]) + (f.w[2] + f.w[3]);
        double incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= uint32_t(o)) incl += up;
        }
        double cum = run + (incl - sum);
        uint32_t at = kNobody, end = kNobody;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            cum += f.w[j];
            if (f.w[j] > 0.0) {
                end = uint32_t(i) + j;
                if (at == kNobody && cum > target) at = end;
            }
        }
        found = __reduce_min_sync(0xffffffffu, at);
        const uint32_t any = __reduce_max_sync(0xffffffffu, end + 1u);   // (kNobody + 1 is 0)
        if (any != 0) fallback = any - 1u;
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
    // (rounding may leave the target at the very end of the run)
    if (found == kNobody) found = fallback;
    if (lane == 0 && found != kNobody) a.tokens[r] = found;
}

}  // namespace lv

using namespace lv;

extern "C" int lv_probabilities(lv_ctx* ctx, float* out, uint32_t out_ld, const float* logits, uint32_t ld, uint32_t vocab, uint32_t rows, const float* temperature) {
    LV_REQUIRE(out && logits && vocab && out_ld >= vocab && ld >= vocab, "probabilities: bad arguments");
    LV_REQUIRE(vocab <= (1u << 24) && rows < (1u << 27), "probabilities: vocabulary larger than 16777216 or too many rows");
    LV_REQUIRE(out != logits || out_ld == ld, "probabilities: in place, the strides are the same");
    LV_REQUIRE(words_aligned(out, logits, temperature), "probabilities: 32-bit values are 4-byte aligned");
    LV_ENTER(ctx);
    if (!rows) return LV_OK;
    Probabilities p{out, logits, temperature, out_ld, ld, vocab, 0};
    // few rows: as many CTAs as hold the row, down to 2048 values each; many: eight, which read a larger one a second time from the L2.  us with 16 and with 8:
    //   128000 values  5 rows 5.5, 6.5    18  8.7, 12.4    24  12.5, 13.4    30  15.0, 13.2    37  18.7, 13.8
    //    70000         5      5.0, 6.1    16  8.2, 10.6    24  11.3, 10.8    30  12.4, 10.9
    //   200000         5      7.7, 8.7    16 12.7, 17.6    24  19.4, 18.5    30  21.6, 18.8
    // (512 rows of 128000: 127 with eight, 131 with four and four CTAs per SM, on an earlier state)
    const bool few = uint64_t(rows) * 6 <= uint64_t(ctx->sm_count);
    uint32_t n = 1;
    while (n < (few && vocab > 8 * kProbHeld ? uint32_t(kProbCluster) : 8u) && vocab / (2 * n) >= 2048) n *= 2;
    p.each = ((vocab + n - 1) / n + 3) / 4 * 4;
    const bool vec = aligned16(out) && aligned16(logits) && out_ld % 4 == 0 && ld % 4 == 0, held = p.each <= kProbHeld;
    auto* kernel = vec ? (held ? probabilities_kernel<true, true> : probabilities_kernel<true, false>) : (held ? probabilities_kernel<false, true> : probabilities_kernel<false, false>);
    if (n > 8) LV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    LV_CUDA(launch_pdl_cluster(ctx, kernel, dim3(rows * n), dim3(kProbThreads), dim3(n), 0, p));
    return LV_OK;
}

extern "C" int lv_verify_drafts(lv_ctx* ctx, const lv_verify_args* a) {
    LV_REQUIRE(a && a->target && a->drafted && a->starts && a->accept && a->pick && a->tokens && a->accepted, "verification of drafts: null argument");
    LV_REQUIRE(a->vocab && a->vocab <= (1u << 24) && a->target_ld >= a->vocab && (!a->draft || a->draft_ld >= a->vocab), "verification of drafts: bad sizes");
    LV_REQUIRE(a->seqs && a->seqs < (1u << 28) && a->rows < (1u << 31), "verification of drafts: too many rows");
    LV_REQUIRE(words_aligned(a->target, a->draft, a->drafted, a->starts, a->accept, a->pick, a->tokens, a->accepted, a->lens), "verification of drafts: 32-bit values are 4-byte aligned");
    LV_ENTER(ctx);
    const bool vec = aligned16(a->target) && a->target_ld % 4 == 0 && aligned16(a->draft) && (!a->draft || a->draft_ld % 4 == 0);
    LV_CUDA(launch_pdl_cluster(ctx, vec ? verify_kernel<true> : verify_kernel<false>, dim3(a->seqs * kVerifyCluster), dim3(kVerifyThreads), dim3(kVerifyCluster), 0, *a, ctx->data_err()));
    return LV_OK;
}

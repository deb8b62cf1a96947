// Probabilities from logits, and drafted tokens against them.
#include "paged.cuh"

namespace lv {

constexpr int kProbThreads = 1024;

struct Probabilities {
    float* out;
    const float* logits;
    const float* temperature;
    uint32_t out_ld, ld, vocab;
};

// the first index of the larger value (NaN is smaller than all)
__device__ __forceinline__ void first_max(float& v, uint32_t& i, float w, uint32_t j) {
    if (w > v || (w == v && j < i)) { v = w; i = j; }
}

// A CTA per row
__global__ void __launch_bounds__(kProbThreads) probabilities_kernel(const Probabilities p) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float s_f[64];
    __shared__ uint32_t s_i[32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x / 32;
    const float* x = p.logits + size_t(blockIdx.x) * p.ld;
    float* y = p.out + size_t(blockIdx.x) * p.out_ld;
    const float T = p.temperature ? p.temperature[blockIdx.x] : 1.f;
    float top = -INFINITY;
    uint32_t at = 0xffffffffu;
    bool odd = false;
    for (uint32_t i = threadIdx.x; i < p.vocab; i += blockDim.x) {
        const float v = x[i];
        odd = odd || v != v;
        first_max(top, at, v, i);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, top, o);
        const uint32_t j = __shfl_xor_sync(0xffffffffu, at, o);
        first_max(top, at, v, j);
    }
    if (lane == 0) { s_f[warp] = top; s_i[warp] = at; }
    odd = __syncthreads_or(odd);
    for (int w = 0; w < kProbThreads / 32; ++w) first_max(top, at, s_f[w], s_i[w]);
    __syncthreads();
    if (T == 0.f) {
        if (at == 0xffffffffu) at = 0;
        for (uint32_t i = threadIdx.x; i < p.vocab; i += blockDim.x) y[i] = i == at ? 1.f : 0.f;
        return;
    }
    const float f = 1.f / T;
    float sum = 0.f;
    for (uint32_t i = threadIdx.x; i < p.vocab; i += blockDim.x) sum += expf((x[i] - top) * f);
    sum = block_sum(sum, s_f);
    const float g = odd ? NAN : top == -INFINITY ? 0.f : 1.f / sum;
    for (uint32_t i = threadIdx.x; i < p.vocab; i += blockDim.x) y[i] = g == 0.f ? 0.f : expf((x[i] - top) * f) * g;
}

constexpr int kVerifyThreads = 1024;
constexpr uint32_t kNobody = 0xffffffffu;

__device__ __forceinline__ double rest_of(const float* p, const float* q, uint32_t drafted, bool rejected, uint32_t i) {
    double w = p[i];
    if (rejected) w -= q ? double(q[i]) : i == drafted ? 1.0 : 0.0;
    return w > 0.0 ? w : 0.0;
}

// A CTA per sequence
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const lv_verify_args a, uint32_t* err) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ double s_sum[33];
    __shared__ uint32_t s_accepted, s_pick, s_last;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x / 32, s = blockIdx.x;
    const uint32_t row0 = a.starts[s], row1 = a.starts[s + 1];
    if (row0 > row1 || row1 > a.rows) {
        if (threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
        return;
    }
    if (row0 == row1) {
        if (threadIdx.x == 0) a.accepted[s] = 0;
        return;
    }
    const uint32_t n = row1 - row0 - 1;
    if (warp == 0) {
        uint32_t good = n;
        for (uint32_t b = 0; b < n; b += 32) {
            bool bad = false;
            if (b + lane < n) {
                const uint32_t r = row0 + b + lane, d = a.drafted[r];
                if (d >= a.vocab) {
                    atomicOr(err, ERR_BAD_INDEX);
                    bad = true;
                } else {
                    const double q = a.draft ? double(a.draft[size_t(r) * a.draft_ld + d]) : 1.0;
                    bad = !(double(a.accept[r]) * q < double(a.target[size_t(r) * a.target_ld + d]));
                }
            }
            const uint32_t first = __ballot_sync(0xffffffffu, bad);
            if (first != 0) {
                good = b + uint32_t(__ffs(int(first))) - 1;
                break;
            }
        }
        if (lane == 0) { s_accepted = good; s_pick = kNobody; s_last = 0; }
    }
    __syncthreads();
    const uint32_t accepted = s_accepted, r = row0 + accepted;
    const float *p = a.target + size_t(r) * a.target_ld, *q = a.draft ? a.draft + size_t(r) * a.draft_ld : nullptr;
    const uint32_t drafted = accepted < n ? a.drafted[r] : kNobody;
    bool rejected = accepted < n;
    const uint32_t each = (a.vocab + kVerifyThreads - 1) / kVerifyThreads, lo = min(a.vocab, threadIdx.x * each), hi = min(a.vocab, lo + each);
    double mine = 0.0, before = 0.0, total = 0.0;
    for (;;) {
        mine = 0.0;
        for (uint32_t i = lo; i < hi; ++i) mine += rest_of(p, q, drafted, rejected, i);
        double incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= uint32_t(o)) incl += up;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        before = total = 0.0;
        for (uint32_t w = 0; w < kVerifyThreads / 32; ++w) {
            if (w == warp) before = total;
            total += s_sum[w];
        }
        before += incl - mine;
        if (total > 0.0 || !rejected) break;
        rejected = false;
    }
    const double target = double(a.pick[s]) * total;
    if (mine > 0.0) {
        double cum = before;
        uint32_t last = 0;
        bool found = false;
        for (uint32_t i = lo; i < hi; ++i) {
            const double w = rest_of(p, q, drafted, rejected, i);
            if (w > 0.0) last = i + 1;
            cum += w;
            if (cum > target && !found) {
                found = true;
                atomicMin(&s_pick, i);
            }
        }
        atomicMax(&s_last, last);
    }
    __syncthreads();
    uint32_t pick = s_pick;
    if (pick == kNobody && s_last != 0) pick = s_last - 1;
    for (uint32_t i = threadIdx.x; i <= n; i += kVerifyThreads) a.tokens[row0 + i] = i < accepted ? a.drafted[row0 + i] : i == accepted ? pick : kNobody;
    if (threadIdx.x == 0) {
        a.accepted[s] = accepted;
        if (pick == kNobody) atomicOr(err, ERR_BAD_INDEX);
        if (a.lens) a.lens[s] -= n - accepted;
    }
}

}  // namespace lv

using namespace lv;

extern "C" int lv_probabilities(lv_ctx* ctx, float* out, uint32_t out_ld, const float* logits, uint32_t ld, uint32_t vocab, uint32_t rows, const float* temperature) {
    LV_REQUIRE(out && logits && vocab && out_ld >= vocab && ld >= vocab, "probabilities: bad arguments");
    LV_REQUIRE(vocab <= (1u << 24) && rows < (1u << 31), "probabilities: vocabulary larger than 16777216 or too many rows");
    LV_REQUIRE(out != logits || out_ld == ld, "probabilities: in place, the strides are the same");
    LV_ENTER(ctx);
    if (!rows) return LV_OK;
    Probabilities p{out, logits, temperature, out_ld, ld, vocab};
    LV_CUDA(launch_pdl(ctx, probabilities_kernel, dim3(rows), dim3(kProbThreads), 0, p));
    return LV_OK;
}

extern "C" int lv_verify_drafts(lv_ctx* ctx, const lv_verify_args* a) {
    LV_REQUIRE(a && a->target && a->drafted && a->starts && a->accept && a->pick && a->tokens && a->accepted, "verification of drafts: null argument");
    LV_REQUIRE(a->vocab && a->vocab <= (1u << 24) && a->target_ld >= a->vocab && (!a->draft || a->draft_ld >= a->vocab), "verification of drafts: bad sizes");
    LV_REQUIRE(a->seqs && a->rows < (1u << 31), "verification of drafts: too many rows");
    LV_ENTER(ctx);
    LV_CUDA(launch_pdl(ctx, verify_kernel, dim3(a->seqs), dim3(kVerifyThreads), 0, *a, ctx->d_err));
    return LV_OK;
}

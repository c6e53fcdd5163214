// Choice of a token's experts from its router logits: softmax or sigmoid scores, a bias that takes part in the choice
// only, groups of experts, renormalised or plain weights (berth_moe_routing in include/berth_b200.h has the formulas).
#include "exl3_decode.cuh"
#include "route.cuh"

#include <cfloat>
#include <cmath>

namespace berth {
namespace {

struct RouteParams {
    const void* logits;
    long long ld;
    const float* bias;
    int32_t* idx;
    float* w;
    int T, E, k;
    int G, keep, gs;   // groups, groups kept, experts of a group
    int P, q;          // lanes of a group (a power of two), consecutive experts of a lane
    int renorm;
    float scale;
};

// How the choice is ordered: by the logits themselves (no bias, groups ranked by their best: both scores rise with the
// logit), or by sigmoid / softmax scores plus bias.
enum { kByLogit = 0, kSigmoid = 1, kSoftmax = 2 };

// +inf counts as the largest finite logit; NaN stays NaN.
__device__ __forceinline__ float clamp_logit(float v) { return v > FLT_MAX ? FLT_MAX : v; }

template <bool F32>
__device__ __forceinline__ float logit_at(const void* row, int e)
{
    return clamp_logit(F32 ? static_cast<const float*>(row)[e] : __half2float(static_cast<const __half*>(row)[e]));
}

// Order-preserving bits of a double (-0 as +0); NaN: 1, below -inf.  0 is left for "taken".
__device__ __forceinline__ unsigned long long key64(double v)
{
    const unsigned long long b = (unsigned long long) __double_as_longlong(v + 0.0);
    return v != v ? 1ull : ((b >> 63) ? ~b : b | (1ull << 63));
}

__device__ __forceinline__ unsigned long long warp_max64(unsigned long long v)
{
    const unsigned hi = __reduce_max_sync(dq::kFull, unsigned(v >> 32));
    const unsigned lo = __reduce_max_sync(dq::kFull, unsigned(v >> 32) == hi ? unsigned(v) : 0u);
    return (unsigned long long) hi << 32 | lo;
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(dq::kFull, v, off);
    return v;
}
__device__ __forceinline__ float warp_max(float v)   // NaN is ignored
{
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(dq::kFull, v, off));
    return v;
}

// The choice with every score and comparison in 64 bits.  Lane s returns the s-th chosen expert.  The experts of a lane
// are consecutive and rise with the lane, so the first lane and the first of its experts have the lower index of a tie.
template <int PER>
__device__ __noinline__ int choose64(const float (&l)[PER], int cnt, int base, int order, bool top2, const RouteParams& p)
{
    const int lane = threadIdx.x & 31;
    double c[PER];
    double m = -INFINITY, z = 0.0;
    if (order == kSoftmax) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i < cnt) m = fmax(m, double(l[i]));
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) m = fmax(m, __shfl_xor_sync(dq::kFull, m, off));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        c[i] = -INFINITY;
        if (i < cnt) {
            const double v = l[i];
            if (order == kByLogit || v != v || v == -INFINITY) c[i] = v;
            else if (order == kSigmoid) c[i] = 1.0 / (1.0 + exp(-v));
            else {
                c[i] = exp(v - m);
                z += c[i];
            }
        }
    }
    if (order == kSoftmax) {
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) z += __shfl_xor_sync(dq::kFull, z, off);
    }
    unsigned long long key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        key[i] = 0;
        if (i < cnt) {
            if (order == kSoftmax && c[i] > -INFINITY) c[i] /= z;
            if (p.bias && c[i] > -INFINITY) c[i] += double(p.bias[base + i]);
            key[i] = key64(c[i]);
        }
    }
    if (p.keep < p.G) {
        double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i < cnt && c[i] > b2) {
                b2 = c[i] > b1 ? b1 : c[i];
                b1 = c[i] > b1 ? c[i] : b1;
            }
        for (int off = 1; off < p.P; off <<= 1) {
            const double o1 = __shfl_xor_sync(dq::kFull, b1, off), o2 = __shfl_xor_sync(dq::kFull, b2, off);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        }
        const double score = top2 && b2 > -INFINITY ? b1 + b2 : b1;
        const int g = lane / p.P;
        int before = 0;
        for (int j = 0; j < p.G; ++j) {
            const double o = __shfl_sync(dq::kFull, score, j * p.P);
            before += o > score || (o == score && j < g);
        }
        if (before >= p.keep) {
#pragma unroll
            for (int i = 0; i < PER; ++i) key[i] = 0;
        }
    }
    int mine = 0;
    for (int s = 0; s < p.k; ++s) {
        unsigned long long best = 0;
        int best_i = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] > best) { best = key[i]; best_i = i; }
        const unsigned long long top = warp_max64(best);
        const int owner = __ffs(__ballot_sync(dq::kFull, best == top)) - 1;
        const int e = __shfl_sync(dq::kFull, base + best_i, owner);
        if (lane == owner) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i == best_i) key[i] = 0;
        }
        if (lane == s) mine = e;
    }
    return mine;
}

// One warp per token; lane = P lanes per group, q consecutive experts each.
template <int PER, bool F32, int SCORE>   // SCORE: kSigmoid or kSoftmax
__global__ void __launch_bounds__(128) k_moe_route(const RouteParams p, bool by_logit, bool top2)
{
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, t = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (t >= p.T) return;
    const char* row = static_cast<const char*>(p.logits) + size_t(t) * p.ld * (F32 ? 4 : 2);
    const int g = lane / p.P, first = (lane % p.P) * p.q;
    const int cnt = g < p.G ? min(max(p.gs - first, 0), p.q) : 0;
    const int base = g < p.G ? g * p.gs + first : 0;
    float l[PER];
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        l[i] = i < cnt ? logit_at<F32>(row, base + i) : -INFINITY;
        nan |= l[i] != l[i];
    }
    nan = __any_sync(dq::kFull, nan);
    const int mine = choose64<PER>(l, cnt, base, by_logit ? kByLogit : SCORE, top2, p);

    // the weight of this lane's expert, fp32
    const float v = lane < p.k ? logit_at<F32>(row, mine) : -INFINITY;
    float w;
    if (p.renorm) {
        const float m = warp_max(v);
        // relative to the largest of the chosen; a sigmoid far below zero is exp of its logit (within 2^-43)
        if (SCORE == kSoftmax || m < -30.f) w = v > -INFINITY ? expf(v - m) : 0.f;
        else w = 1.f / (1.f + expf(-v));
        if (lane >= p.k) w = 0.f;
        const float sum = warp_sum(w);
        w = sum > 0.f ? w / sum : 0.f;
    } else if (SCORE == kSigmoid) {
        w = 1.f / (1.f + expf(-v));
    } else {
        float m = -INFINITY, z = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = fmaxf(m, l[i]);
        m = warp_max(m);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (l[i] > -INFINITY) z += expf(l[i] - m);
        z = warp_sum(z);
        w = v > -INFINITY ? expf(v - m) / z : 0.f;
    }
    if (lane < p.k) {
        p.idx[size_t(t) * p.k + lane] = mine;
        p.w[size_t(t) * p.k + lane] = nan ? NAN : w * p.scale;
    }
}

template <int PER>
void launch(bool f32, int score, const RouteParams& p, bool by_logit, bool top2, cudaStream_t st)
{
    const dim3 grid((p.T + 3) / 4), block(128);
    auto go = [&](auto kern) { launch_pdl(kern, grid, block, 0, st, "k_moe_route launch", p, by_logit, top2); };
    if (f32) score == kSigmoid ? go(k_moe_route<PER, true, kSigmoid>) : go(k_moe_route<PER, true, kSoftmax>);
    else score == kSigmoid ? go(k_moe_route<PER, false, kSigmoid>) : go(k_moe_route<PER, false, kSoftmax>);
}

}  // namespace

void check_routing(const berth_moe_routing* r, int n_experts, int top_k)
{
    if (r->score != 0 && r->score != 1) throw std::runtime_error("moe route: score must be 0 (softmax) or 1 (sigmoid)");
    if (r->group_score != 0 && r->group_score != 1) throw std::runtime_error("moe route: group_score must be 0 (best) or 1 (sum of two best)");
    if (r->n_group < 1 || r->n_group > 32 || n_experts % r->n_group)
        throw std::runtime_error("moe route: n_group must be in 1..=32 and divide n_experts");
    if (r->topk_group < 1 || r->topk_group > r->n_group) throw std::runtime_error("moe route: topk_group must be in 1..=n_group");
    const int gs = n_experts / r->n_group;
    if (top_k > r->topk_group * gs) throw std::runtime_error("moe route: top_k exceeds the experts of topk_group groups");
    if (r->group_score == 1 && gs < 2) throw std::runtime_error("moe route: the sum of two best needs groups of at least two experts");
    if (!std::isfinite(r->scale)) throw std::runtime_error("moe route: scale must be finite");
}

std::string route_tokens(const void* logits, bool f32, long long ld, const berth_moe_routing& r, int32_t* idx, float* w, int T, int E, int k,
                         cudaStream_t st)
{
    RouteParams p{};
    p.logits = logits; p.ld = ld; p.bias = r.selection_bias; p.idx = idx; p.w = w;
    p.T = T; p.E = E; p.k = k;
    p.G = r.n_group; p.keep = r.topk_group;
    if (p.keep == p.G) p.G = p.keep = 1;   // every group is kept: as one group
    p.gs = E / p.G;
    p.P = 32;
    while (p.P * p.G > 32) p.P >>= 1;
    p.q = (p.gs + p.P - 1) / p.P;
    p.renorm = r.renormalize != 0;
    p.scale = r.scale;
    const bool top2 = p.G > 1 && r.group_score == 1;
    const bool by_logit = !r.selection_bias && !top2;
    const int score = r.score == 1 ? kSigmoid : kSoftmax;
    int per = 1;
    while (per < p.q) per <<= 1;
    switch (per) {
        case 1: launch<1>(f32, score, p, by_logit, top2, st); break;
        case 2: launch<2>(f32, score, p, by_logit, top2, st); break;
        case 4: launch<4>(f32, score, p, by_logit, top2, st); break;
        case 8: launch<8>(f32, score, p, by_logit, top2, st); break;
        case 16: launch<16>(f32, score, p, by_logit, top2, st); break;
        case 32: launch<32>(f32, score, p, by_logit, top2, st); break;
        default: launch<64>(f32, score, p, by_logit, top2, st); break;   // up to 1024 experts: q <= 64
    }
    return "k_moe_route<" + std::to_string(per) + "," + (f32 ? "float" : "half") + "," + (score == kSigmoid ? "sigmoid" : "softmax") + "> grid=" +
           std::to_string((T + 3) / 4);
}

}  // namespace berth

using namespace berth;

extern "C" int berth_moe_route(const void* logits, int logits_fp32, int64_t row_stride, const float* selection_bias, int32_t* topk_idx,
                               float* topk_w, int T, int n_experts, int top_k, int score, int n_group, int topk_group, int group_score,
                               int renormalize, float scale, void* stream)
{
    CallState& st = moe_state();
    return guarded(st, [&] {
        if (!logits || !topk_idx || !topk_w) throw std::runtime_error("moe route: null device pointer");
        if (logits_fp32 != 0 && logits_fp32 != 1) throw std::runtime_error("moe route: logits_fp32 must be 0 or 1");
        if (T < 1) throw std::runtime_error("moe route: T must be positive");
        if (n_experts < 1 || n_experts > 1024) throw std::runtime_error("moe route: n_experts must be in 1..=1024");
        if (top_k < 1 || top_k > 32 || top_k > n_experts) throw std::runtime_error("moe route: top_k must be in 1..=32 and at most n_experts");
        if (row_stride < n_experts && T > 1) throw std::runtime_error("moe route: row_stride is smaller than n_experts");
        const berth_moe_routing r{score, n_group, topk_group, group_score, renormalize, scale, selection_bias};
        check_routing(&r, n_experts, top_k);
        st.launch = route_tokens(logits, logits_fp32 != 0, row_stride, r, topk_idx, topk_w, T, n_experts, top_k, (cudaStream_t) stream);
    });
}

// Choice of a token's experts from its router logits: softmax or sigmoid scores, a bias that takes part in the choice
// only, groups of experts, renormalised or plain weights (berth_moe_routing in include/berth_b200.h has the formulas).
#include "exl3_decode.cuh"
#include "route.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

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

// The choice with every score and comparison in 64 bits.  Lane s returns the s-th chosen expert.  The experts of a lane
// are consecutive and rise with the lane, so the first lane and the first of its experts have the lower index of a tie.
template <int PER>
__device__ __forceinline__ int choose64(const float (&l)[PER], int cnt, int base, int order, bool top2, const RouteParams& p)
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

__device__ __forceinline__ float redux_max(float v) { float r; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float redux_min(float v) { float r; asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float rcp(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// A row whose choice 32 bits cannot tell, or with an infinite or NaN logit: its logits once more, the choice in 64 bits, and what a
// softmax over the row needs.
struct Again {
    int mine;
    bool nan;
    float m, z;
};
template <int PER, bool F32>
__device__ __noinline__ Again choose_again(const char* row, int cnt, int base, int order, bool top2, bool softmax, const RouteParams& p)
{
    float l[PER], m = -INFINITY, z = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        l[i] = i < cnt ? logit_at<F32>(row, base + i) : -INFINITY;
        nan |= l[i] != l[i];
        m = fmaxf(m, l[i]);
    }
    m = redux_max(m);
    if (softmax) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (l[i] > -INFINITY) z += ex2((l[i] - m) * 1.44269504088896341f);
        z = warp_sum(z);
    }
    nan = __any_sync(dq::kFull, nan);
    return Again{choose64<PER>(l, cnt, base, order, top2, p), nan, m, z};
}

// The order of a finite float's bits (-0 as +0).
__device__ __forceinline__ unsigned ordered(float v)
{
    const int b = __float_as_int(v + 0.f);
    return unsigned(b) ^ (unsigned(b >> 31) | 0x80000000u);
}

template <int PER> struct Log2 { static constexpr int v = 1 + Log2<PER / 2>::v; };
template <> struct Log2<1> { static constexpr int v = 0; };

// The two largest of a1 >= a2 and b1 >= b2.
__device__ __forceinline__ void best_two(unsigned& a1, unsigned& a2, unsigned b1, unsigned b2)
{
    a2 = max(min(a1, b1), max(a2, b2));
    a1 = max(a1, b1);
}
// The largest key of a group below its second one, k2 (keys differ).
template <int PER>
__device__ __forceinline__ unsigned third_key(const unsigned (&key)[PER], unsigned k2, int lanes)
{
    unsigned k3 = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) k3 = max(k3, key[i] < k2 ? key[i] : 0u);
    for (int off = 1; off < lanes; off <<= 1) k3 = max(k3, __shfl_xor_sync(dq::kFull, k3, off));
    return k3;
}
// What a softmax under a bias needs in 64 bits: the sum of a finite row's exp(l - m).
template <bool F32>
__device__ __noinline__ double sum64(const void* row, int cnt, int base, double m)
{
    double z = 0.0;
#pragma unroll 1
    for (int i = 0; i < cnt; ++i) z += exp(double(logit_at<F32>(row, base + i)) - m);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) z += __shfl_xor_sync(dq::kFull, z, off);
    return z;
}
// The choice score of expert e in 64 bits (softmax: m and z of the row).
template <bool F32, int ORDER>
__device__ __forceinline__ double score64(const void* row, int e, double m, double z, const RouteParams& p)
{
    const double v = logit_at<F32>(row, e);
    if (ORDER == kByLogit) return v;
    return (ORDER == kSoftmax ? exp(v - m) / z : 1.0 / (1.0 + exp(-v))) + (p.bias ? double(p.bias[e]) : 0.0);
}
// Whether this lane's group is kept, by the scores of the groups' two best experts (keys k1, k2; two lanes of a group or more).
template <bool F32, int ORDER, int LOG_PER>
__device__ __noinline__ bool groups_again(const void* row, unsigned k1, unsigned k2, int log_p, bool top2, double m, double z, const RouteParams& p)
{
    const int lane = threadIdx.x & 31, g = lane >> log_p, member = lane & (p.P - 1);
    double c = -INFINITY;
    const unsigned key = member == 0 ? k1 : k2;
    if (g < p.G && member < 2 && key != 0u) {   // (groups of one expert: no second key)
        const int owner = 31 - int(key >> LOG_PER & 31u);
        c = score64<F32, ORDER>(row, (owner >> log_p) * p.gs + (owner & (p.P - 1)) * p.q + ((1 << LOG_PER) - 1 - int(key & ((1u << LOG_PER) - 1))), m, z, p);
    }
    const double other = __shfl_xor_sync(dq::kFull, c, 1);
    const double worth = __shfl_sync(dq::kFull, top2 ? c + other : fmax(c, other), lane & ~(p.P - 1));
    int before = 0;
    for (int j = 0; j < p.G; ++j) {
        const double o = __shfl_sync(dq::kFull, worth, j << log_p);
        before += o > worth || (o == worth && j < g);
    }
    return before < p.keep;
}

// Blocks of an SM that the registers have to allow, and the grid fills once: eight keys a lane, 16384 tokens, 6: 13.8 us, 8: 14.7 us; two
// keys a lane (64 experts) 8: 7.7 us, 6: 10.3 us.  Softmax scores of 8 and 16 keys a lane, which were not measured apart, keep 36 to 88
// bytes of a thread in local memory under these bounds (64 keys: 12 to 32, all orders).
constexpr int min_blocks(int per) { return per < 8 ? 8 : per == 8 ? 6 : per == 16 ? 4 : 2; }

// One warp per token; lane = P lanes per group, q consecutive experts each.
//
// The choice is made in 32 bits first and repeated in 64 (choose64) where that cannot tell.  An expert's key is its choice score in
// fixed point with its place, (31 - lane, PER - 1 - i), in the lowest bits: keys differ, the larger key is the larger score or of
// equal ones the lower expert, and a round of the choice is one redux over the lanes' heads.  A lane keeps its keys sorted.
//   scores + bias: 2^23 steps (2^22 with 32 experts a lane, 2^21 with 64) over [least bias, 1 + largest bias];
//   fp32 logits by themselves: as many over the 32 below the row's largest;
//   fp16 logits by themselves: the order of their bits, which have room for the place: exact.
// Where two neighbours in the order (the first expert not chosen among them) lie closer than both scores' errors and the steps, the
// k + 1 first are ordered anew in 64 bits, one a lane; so are the groups by their two best experts, where the last one kept and the
// first one dropped lie as close.  The whole choice is repeated where that may not be enough (a third one as close) and for a row that
// has an infinite or NaN logit.
// Errors of c = s + b in units of 2^-24: sigmoid, s (1 - s) (1.5 |l| + 4) for exp and 3 for sum and reciprocal, below 4.5 each;
// softmax, s (2.5 |l - m| + 7) <= 9 S each, S the row's largest, and (2.5 ln E + 6 + PER) |s - s'| for the common 1 / Z, below
// 2 (28 + PER) S for a pair; the sum with the bias, and the bias less the least, half a step of at most the span each.
// Bound: instructions, half of them on the half-rate integer pipe, and their latency: 16384 tokens of 256 experts, 8 groups, 8 chosen
// 13.7 us (17.8 MB would be 2.7), of which 2.5 are a call's least; all of it in 64 bits 57 us.  Sigmoid against
// softmax scores, both under a bias, launches queued ahead: 14.2 and 17.6 us, 8192 tokens of 512 experts 14.8 and 20.1, 16384 of 128 11.6
// and 13.2.
template <int PER, bool F32, int ORDER>
__global__ void __launch_bounds__(128, min_blocks(PER)) k_moe_route(const RouteParams p, bool sigmoid, bool top2, bool wide)
{
    constexpr int kPlace = 5 + Log2<PER>::v, kSteps = 32 - kPlace < 23 ? 32 - kPlace : 23;
    constexpr int kRun = PER < 8 ? PER : 8, kRuns = PER / kRun, kRoom = (kRun + 4) * kRuns;   // a lane's keys: sorted runs, zeros behind each
    constexpr unsigned kMask = (1u << kPlace) - 1, kScore = (1u << kSteps) - 1;
    constexpr bool kSorted = PER <= 32, kExact = ORDER == kByLogit && !F32, kHeldBias = PER <= 16 && ORDER != kByLogit, kAhead = PER <= 16;
    constexpr float kLog2e = 1.44269504088896341f, kUnit = 1.f / (1 << 24), kMagic = 8388608.f;   // 2^23 + n: n in the low bits
    __shared__ __align__(16) unsigned sorted[4][kSorted ? 32 * kRoom : 4];   // every lane's keys
    __shared__ unsigned winners[4][34];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int log_p = 31 - __clz(p.P), g = lane >> log_p, first = (lane & (p.P - 1)) * p.q;
    const int cnt = g < p.G ? min(max(p.gs - first, 0), p.q) : 0;
    const int base = g < p.G ? g * p.gs + first : 0;
    const bool full = __all_sync(dq::kFull, cnt == PER);
    const bool groups = p.keep < p.G;
    auto fetch = [&](int t, float (&l)[PER]) {
        const char* row = static_cast<const char*>(p.logits) + size_t(t) * p.ld * (F32 ? 4 : 2);
        if (PER >= 4 && wide) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                float v[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX};
                if (i < cnt) {
                    if constexpr (F32) {
                        const float4 w = *reinterpret_cast<const float4*>(row + size_t(base + i) * 4);
                        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(row + size_t(base + i) * 2);
                        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
                        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) l[PER >= 4 ? i + j : 0] = v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                l[i] = i < cnt ? (F32 ? reinterpret_cast<const float*>(row)[base + i] : __half2float(reinterpret_cast<const __half*>(row)[base + i])) : -FLT_MAX;
        }
    };

    // the bias and its range
    float bias[kHeldBias ? PER : 1];
    float low = 0.f, span = 1.f;
    if (ORDER != kByLogit && p.bias) {
        float lo = INFINITY, hi = -INFINITY;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float b = i < cnt ? p.bias[base + i] : 0.f;
            if constexpr (kHeldBias) bias[i] = b;
            if (i < cnt) {
                lo = fminf(lo, b);
                hi = fmaxf(hi, b);
                odd |= !(fabsf(b) < 67108864.f);
            }
        }
        low = redux_min(lo);
        span = 1.f + (redux_max(hi) - low);
        if constexpr (kHeldBias) {
#pragma unroll
            for (int i = 0; i < PER; ++i) bias[i] -= low;   // scores from 0 on: the order is the same
        }
        // every row in 64 bits where the sum's rounding there, 2^-53 of the bias, is not small beside a step of the keys: sums that are
        // equal in 64 bits are ties, which the scores less the common bias are not
        if (__any_sync(dq::kFull, odd)) span = INFINITY;
    } else if constexpr (kHeldBias) {
#pragma unroll
        for (int i = 0; i < PER; ++i) bias[i] = 0.f;
    }
    if (ORDER == kByLogit) span = 32.f;
    const bool never = !(span < 1e30f);
    const float scale = ((1 << kSteps) - 4) / span;
    // how close two choice scores, or two groups' scores, may lie before 64 bits decide: their errors, and two steps of each key
    // (softmax: of the row's largest score, once that is known)
    unsigned near = kExact ? 0u : unsigned(ORDER == kByLogit ? 0.f : kUnit * ((ORDER == kSigmoid ? 9.f : 0.f) + 4.f * span) * scale) + 4u;
    const unsigned near_bias = near;

    if constexpr (kSorted) {
        for (int r = 0; r < kRuns; ++r)
            for (int i = 0; i < 4; ++i) sorted[warp][lane * kRoom + r * (kRun + 4) + kRun + i] = 0;   // (read once a round when no key is left)
    }
    const int stride = gridDim.x * 4;
    float next[kAhead ? PER : 1];
    int t = blockIdx.x * 4 + warp;
    if constexpr (kAhead) {
        if (t < p.T) fetch(t, next);
    }
    for (; t < p.T; t += stride) {
        const char* row = static_cast<const char*>(p.logits) + size_t(t) * p.ld * (F32 ? 4 : 2);
        float l[PER], c[PER];
        bool unsure = never;
        if constexpr (kAhead) {
#pragma unroll
            for (int i = 0; i < PER; ++i) l[i] = next[i];
            if (t + stride < p.T) fetch(t + stride, next);
        } else fetch(t, l);
#pragma unroll
        for (int i = 0; i < PER; ++i) unsure |= !(fabsf(l[i]) <= FLT_MAX);

        // ---- choice scores
        float m = 0.f, z = 0.f;
        if (ORDER == kSoftmax || (ORDER == kByLogit && (F32 || !(sigmoid || p.renorm)))) {
            m = l[0];
#pragma unroll
            for (int i = 1; i < PER; ++i) m = fmaxf(m, l[i]);
            m = redux_max(m);
        }
        if (ORDER == kSoftmax || (ORDER == kByLogit && !(sigmoid || p.renorm))) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                c[i] = full || i < cnt ? ex2((l[i] - m) * kLog2e) : 0.f;
                z += c[i];
            }
            z = warp_sum(z);
        }
        const float inv = ORDER == kSoftmax ? rcp(z) : 0.f;
        if constexpr (ORDER == kSoftmax) near = near_bias + unsigned(kUnit * 2.1f * (28 + PER) * inv * scale) + 1u;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (ORDER == kByLogit) c[i] = l[i];
            else if (ORDER == kSigmoid) c[i] = rcp(1.f + ex2(l[i] * -kLog2e));
            else c[i] *= inv;
            if constexpr (kHeldBias) c[i] += bias[i];
            else if (ORDER != kByLogit && p.bias && i < cnt) c[i] += p.bias[base + i] - low;
        }
        if (!full) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i >= cnt) c[i] = -FLT_MAX;
        }

        // ---- keys, largest first
        unsigned key[PER];
        const unsigned place = (31u - lane) << Log2<PER>::v;
        const float shift = ORDER == kByLogit ? kMagic + float((1 << kSteps) - 3) : kMagic + 1.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if constexpr (kExact) {
                key[i] = (ordered(c[i]) & ~kMask) | place | unsigned(PER - 1 - i);
            } else {
                const float n = ORDER == kByLogit ? fmaxf(fmaf(c[i] - m, scale, shift), kMagic) : fmaf(c[i], scale, shift);
                key[i] = __float_as_uint(n) << kPlace | place | unsigned(PER - 1 - i);   // (what the exponent leaves is the same in all)
            }
        }
        if (!full) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (i >= cnt) key[i] = 0;
        }
        if constexpr (kSorted && PER > 1) {
#pragma unroll
            for (int r = 0; r < PER; r += kRun)
#pragma unroll
                for (int span = 2; span <= kRun; span *= 2)      // bitonic, descending; the first step of a span is mirrored
#pragma unroll
                    for (int d = span / 2; d >= 1; d /= 2)
#pragma unroll
                        for (int i = 0; i < kRun; ++i)
                            if (!(i & d)) {
                                const int j = d == span / 2 ? (i | (span - 1)) - (i & (span / 2 - 1)) : i + d;
                                const unsigned hi = max(key[r + i], key[r + j]), lo = min(key[r + i], key[r + j]);
                                key[r + i] = hi;
                                key[r + j] = lo;
                            }
        }
        // ---- groups: the two best keys of each, rounds over the groups' worth
        bool open = true;
        if (groups) {
            unsigned k1 = key[0], k2 = 0;
            if constexpr (kSorted) {
                if constexpr (PER > 1) k2 = key[1];
#pragma unroll
                for (int r = kRun; r < PER; r += kRun) best_two(k1, k2, key[r], key[r + (kRun > 1)]);
            } else {
#pragma unroll
                for (int i = 1; i < PER; ++i) best_two(k1, k2, key[i], 0u);
            }
            for (int off = 1; off < p.P; off <<= 1) best_two(k1, k2, __shfl_xor_sync(dq::kFull, k1, off), __shfl_xor_sync(dq::kFull, k2, off));
            // all lanes of a group hold the same; a sum has room for its group (both hold what the exponent left, the same in all)
            const unsigned worth = !top2 ? k1 : (((k1 >> kPlace) & kScore) + ((k2 >> kPlace) & kScore)) << 5 | (31u - g);
            const int low_bits = top2 ? 5 : kPlace;
            unsigned gkey = g < p.G ? worth : 0u, top = 0;
            open = false;
            for (int s = 0; s < p.keep; ++s) {
                top = __reduce_max_sync(dq::kFull, gkey);
                if (gkey == top) {
                    open = true;
                    gkey = 0;
                }
            }
            const unsigned next_one = __reduce_max_sync(dq::kFull, gkey);
            if (!kExact && (top >> low_bits) - (next_one >> low_bits) <= near * (top2 ? 2 : 1)) {
                // too close for the keys: the groups anew by their two best experts' scores in 64 bits, one a lane, where no group has
                // a third one that could be the second
                unsigned k3 = 0;
                if constexpr (kSorted) k3 = third_key<PER>(key, k2, p.P);
                const bool apart = kSorted && p.P > 1 && (g >= p.G || k3 == 0u || (k2 >> kPlace) - (k3 >> kPlace) > near) &&
                                   (ORDER != kByLogit || g >= p.G || ((k2 >> kPlace) & kScore) > 4u);
                if (__all_sync(dq::kFull, apart) && !__any_sync(dq::kFull, unsure)) open = groups_again<F32, ORDER, Log2<PER>::v>(row, k1, k2, log_p, top2, m, ORDER == kSoftmax ? sum64<F32>(row, cnt, base, m) : 0.0, p);
                else unsure = true;
            }
            if (ORDER == kByLogit && F32) unsure |= (top >> kPlace & kScore) <= 4u;   // (below the 32 of the logits, the steps end)
        }

        unsigned head = open ? key[0] : 0u;
        if constexpr (kSorted) {
            // the keys to shared memory, zeros behind each run: the owner of a round's key reads the next one, instead of moving all up
            unsigned* mine_at = &sorted[warp][lane * kRoom];
            unsigned run[kRuns];
            uint32_t from[kRuns];
#pragma unroll
            for (int r = 0; r < kRuns; ++r) {
                unsigned* at = mine_at + r * (kRun + 4);
                if constexpr (kRun % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < kRun; i += 4)
                        *reinterpret_cast<uint4*>(at + i) = make_uint4(key[r * kRun + i], key[r * kRun + (i + 1) % kRun], key[r * kRun + (i + 2) % kRun], key[r * kRun + (i + 3) % kRun]);
                } else {
#pragma unroll
                    for (int i = 0; i < kRun; ++i) at[i] = key[i];
                }
                run[r] = open ? key[r * kRun] : 0u;
                from[r] = uint32_t(__cvta_generic_to_shared(open ? at : at + kRun));
                head = max(head, run[r]);
            }
            uint32_t to = uint32_t(__cvta_generic_to_shared(winners[warp]));
            for (int s = 0; s < p.k + 2; ++s, to += 4) {
                const unsigned top = __reduce_max_sync(dq::kFull, head);
                head = 0;
#pragma unroll
                for (int r = 0; r < kRuns; ++r) {
                    asm volatile("{\n\t.reg .pred q;\n\t"
                                 "setp.eq.u32 q, %0, %2;\n\t"
                                 "@q st.shared.u32 [%3], %2;\n\t"
                                 "@q add.u32 %1, %1, 4;\n\t"
                                 "@q ld.shared.u32 %0, [%1];\n\t}"
                                 : "+r"(run[r]), "+r"(from[r])
                                 : "r"(top), "r"(to)
                                 : "memory");
                    head = max(head, run[r]);
                }
            }
        } else {
#pragma unroll
            for (int i = 1; i < PER; ++i) head = max(head, open ? key[i] : 0u);
            for (int s = 0; s < p.k + 2; ++s) {
                const unsigned top = __reduce_max_sync(dq::kFull, head);
                if (head == top) {
                    winners[warp][s] = top;
                    unsigned h = 0;
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        key[i] = key[i] == head ? 0u : key[i];
                        h = max(h, key[i]);
                    }
                    head = h;
                }
            }
        }
        __syncwarp();
        const unsigned won = winners[warp][lane], after = winners[warp][lane + 1];   // of lane s <= k: the s-th key, and the next
        const unsigned last = winners[warp][p.k - 1], beyond = winners[warp][p.k + 1];
        __syncwarp();
        const int owner = 31 - int(won >> Log2<PER>::v & 31u);
        int mine = (owner >> log_p) * p.gs + (owner & (p.P - 1)) * p.q + (PER - 1 - int(won & (PER - 1)));
        if constexpr (!kExact) {
            bool close = lane < p.k && after != 0u && (won >> kPlace) - (after >> kPlace) <= near;
            if (ORDER == kByLogit) unsure |= lane < p.k && (won >> kPlace & kScore) <= 4u;
            if (__any_sync(dq::kFull, close)) {
                // neighbours too close for the keys: the k + 1 first anew by their scores in 64 bits, one a lane, where the one
                // behind them cannot be among the k
                const bool apart = p.k < 32 && (beyond == 0u || (last >> kPlace) - (beyond >> kPlace) > near);
                if (apart && !__any_sync(dq::kFull, unsure)) {
                    const bool one = lane < p.k || (lane == p.k && won != 0u);
                    const double sum = ORDER == kSoftmax ? sum64<F32>(row, cnt, base, m) : 0.0;
                    const double c = one ? score64<F32, ORDER>(row, mine, m, sum, p) : -INFINITY;
                    int before = 0;
                    for (int j = 0; j <= p.k; ++j) {
                        const double oc = __shfl_sync(dq::kFull, c, j);
                        const int oe = __shfl_sync(dq::kFull, mine, j);
                        before += oc > c || (oc == c && oe < mine);
                    }
                    if (one) winners[warp][before] = unsigned(mine);
                    __syncwarp();
                    mine = int(winners[warp][lane]);
                    __syncwarp();
                } else unsure = true;
            }
        }
        bool nan = false;
        if (__any_sync(dq::kFull, unsure)) {
            const Again o = choose_again<PER, F32>(row, cnt, base, ORDER, top2, !(sigmoid || p.renorm), p);
            mine = o.mine;
            nan = o.nan;
            m = o.m;
            z = o.z;
        }

        // ---- the weight of this lane's expert
        const float v = lane < p.k ? logit_at<F32>(row, mine) : -INFINITY;
        float w;
        if (p.renorm) {
            const float most = redux_max(v);
            // relative to the largest of the chosen; a sigmoid far below zero is exp of its logit (within 2^-43)
            if (!sigmoid || most < -30.f) w = v > -INFINITY ? expf(v - most) : 0.f;
            else w = __fdividef(1.f, 1.f + expf(-v));
            if (lane >= p.k) w = 0.f;
            float sum = w;
            for (int off = 1; off < p.k; off <<= 1) sum += __shfl_xor_sync(dq::kFull, sum, off);   // (lanes from k on: 0)
            w = sum > 0.f ? __fdividef(w, sum) : 0.f;
        } else if (sigmoid) {
            w = __fdividef(1.f, 1.f + expf(-v));
        } else {
            w = v > -INFINITY ? __fdividef(expf(v - m), z) : 0.f;
        }
        if (lane < p.k) {
            const size_t at = size_t(t) * p.k + lane;
            p.idx[at] = mine;
            p.w[at] = nan ? NAN : w * p.scale;
        }
    }
}

template <int PER>
void launch(bool f32, int order, bool sigmoid, const RouteParams& p, bool top2, bool wide, int blocks, cudaStream_t st)
{
    auto go = [&](auto kern) { launch_pdl(kern, dim3(blocks), dim3(128), 0, st, "k_moe_route launch", p, sigmoid, top2, wide); };
    auto typed = [&](auto f) {
        constexpr bool F = decltype(f)::value;
        if (order == kByLogit) go(k_moe_route<PER, F, kByLogit>);
        else if (order == kSigmoid) go(k_moe_route<PER, F, kSigmoid>);
        else go(k_moe_route<PER, F, kSoftmax>);
    };
    if (f32) typed(std::true_type{});
    else typed(std::false_type{});
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
    check_aligned(r->selection_bias, 4, "moe route: selection_bias");
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
    // four logits per access where every lane's experts begin on a multiple of four of an aligned row
    const int size = f32 ? 4 : 2;
    const bool wide = p.gs % 4 == 0 && p.q % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) | uintptr_t(T > 1 ? ld * size : 0)) % (4 * size) == 0;
    const int blocks = std::min((T + 3) / 4, 148 * min_blocks(per));
    auto go = [&](auto launcher) { launcher(f32, by_logit ? kByLogit : score, score == kSigmoid, p, top2, wide, blocks, st); };
    switch (per) {
        case 1: go(launch<1>); break;
        case 2: go(launch<2>); break;
        case 4: go(launch<4>); break;
        case 8: go(launch<8>); break;
        case 16: go(launch<16>); break;
        case 32: go(launch<32>); break;
        default: go(launch<64>); break;   // up to 1024 experts: q <= 64
    }
    return describe("k_moe_route<", per, ",", f32 ? "float" : "half", ",", score == kSigmoid ? "sigmoid" : "softmax", by_logit ? "" : ",scores", "> grid=", blocks);
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
        if (T < 1 || T > (1 << 30)) throw std::runtime_error("moe route: T must be positive and at most 2^30");
        if (n_experts < 1 || n_experts > 1024) throw std::runtime_error("moe route: n_experts must be in 1..=1024");
        if (top_k < 1 || top_k > 32 || top_k > n_experts) throw std::runtime_error("moe route: top_k must be in 1..=32 and at most n_experts");
        if (row_stride < n_experts && T > 1) throw std::runtime_error("moe route: row_stride is smaller than n_experts");
        check_aligned(logits, logits_fp32 ? 4 : 2, "moe route: logits");
        for (const void* p : {(const void*) topk_idx, (const void*) topk_w}) check_aligned(p, 4, "moe route: a tensor of 32-bit elements");
        const berth_moe_routing r{score, n_group, topk_group, group_score, renormalize, scale, selection_bias};
        check_routing(&r, n_experts, top_k);
        st.launch = route_tokens(logits, logits_fp32 != 0, row_stride, r, topk_idx, topk_w, T, n_experts, top_k, (cudaStream_t) stream);
    });
}

// Log probabilities of given tokens, entropy and the best alternatives of every row of logits.
#include "exl3_decode.cuh"
#include "../../include/berth_b200.h"

#include <algorithm>
#include <cmath>

namespace berth {
namespace {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
constexpr int kMaxTop = 32;

struct LogprobParams {
    const void* logits;
    long long ld;
    const int32_t* tokens;
    float* logprob;
    int32_t* rank;
    float* entropy;
    int32_t* top_idx;
    float* top_logprob;
    int top_n, rows, vocab;
    float inv_temp, scale2;   // scale2 = inv_temp * log2(e)
};

template <bool F32>
__device__ __forceinline__ float value_at(const void* row, int i)
{
    return F32 ? static_cast<const float*>(row)[i] : __half2float(static_cast<const __half*>(row)[i]);
}

// Order of the vocabulary as one number: the larger logit first (-0 as +0, NaN last), then the lower token.  Never 0.
__device__ __forceinline__ unsigned long long order_key(float v, int i)
{
    const unsigned b = __float_as_uint(v + 0.0f);
    const unsigned o = v != v ? 0u : ((b >> 31) ? ~b : b | 0x80000000u);
    return (unsigned long long) o << 32 | (0xffffffffu - unsigned(i));
}
__device__ __forceinline__ float key_value(unsigned long long key)
{
    const unsigned o = unsigned(key >> 32);
    return o == 0u ? NAN : __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* sm, F op)   // 256 threads; every thread gets the result
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v = op(v, __shfl_xor_sync(dq::kFull, v, off));
    __syncthreads();
    if (lane == 0) sm[warp] = v;
    __syncthreads();
    v = sm[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v = op(v, sm[i]);
    return v;
}

// ln p of a logit x in a row of largest logit m and ln of its sum of powers.  The difference is taken before the scale, here
// and in the exponents: a row of the type's lowest value would overflow the product.
__device__ __forceinline__ float logprob_of(float x, float inv_temp, float m, float lnz, bool dead)
{
    if (dead) return -INFINITY;
    return (x - m) * inv_temp - lnz;
}

template <bool F32>
__global__ void __launch_bounds__(256) k_logprobs(const LogprobParams p)
{
    pdl_trigger();
    pdl_wait();
    __shared__ float sf[8];
    __shared__ int si[8];
    __shared__ unsigned long long sk[8];
    const int tid = threadIdx.x;
    const size_t r = blockIdx.x;
    const char* row = static_cast<const char*>(p.logits) + r * p.ld * (F32 ? 4 : 2);
    const int token = p.tokens ? p.tokens[r] : -1;
    const bool real = token >= 0 && token < p.vocab;
    const unsigned long long key = real ? order_key(value_at<F32>(row, token), token) : 0;
    float m = -INFINITY;
    for (int i = tid; i < p.vocab; i += 256) m = fmaxf(m, value_at<F32>(row, i));
    m = block_reduce(m, sf, [](float a, float b) { return fmaxf(a, b); });
    const bool dead = m == -INFINITY;
    if (dead) m = 0.f;
    float z = 0.f, ey = 0.f;
    int before = 0;
    for (int i = tid; i < p.vocab; i += 256) {
        const float x = value_at<F32>(row, i);
        float y = (x - m) * p.scale2;
        y = y < -200.f ? -200.f : y;
        const float e = exp2f(y);
        z += e;
        ey = fmaf(e, y, ey);
        before += order_key(x, i) > key;
    }
    auto add = [](auto a, auto b) { return a + b; };
    z = block_reduce(z, sf, add);
    ey = block_reduce(ey, sf, add);
    before = block_reduce(before, si, add);
    const bool none = dead && z == 0.f;   // masked altogether
    const float log2z = log2f(z);
    if (tid == 0) {
        if (p.logprob) p.logprob[r] = real ? logprob_of(key_value(key), p.inv_temp, m, log2z * kLn2, none) : 0.f;
        if (p.rank) p.rank[r] = real && key >> 32 ? before : -1;
        if (p.entropy) p.entropy[r] = none ? 0.f : (log2z - ey / z) * kLn2;
    }
    unsigned long long last = ~0ull;
    for (int n = 0; n < p.top_n; ++n) {
        unsigned long long best = 0;
        for (int i = tid; i < p.vocab; i += 256) {
            const unsigned long long k = order_key(value_at<F32>(row, i), i);
            if (k < last && k > best) best = k;
        }
        last = block_reduce(best, sk, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        if (tid == 0) {
            p.top_idx[r * p.top_n + n] = int(0xffffffffu - unsigned(last));
            p.top_logprob[r * p.top_n + n] = logprob_of(key_value(last), p.inv_temp, m, log2z * kLn2, none);
        }
    }
}

}  // namespace
}  // namespace berth

using namespace berth;

extern "C" int berth_ops_logprobs(const void* logits, int logits_fp32, int64_t row_stride, const int32_t* tokens, float inv_temp,
                                  float* logprob, int32_t* rank, float* entropy, int32_t* top_idx, float* top_logprob, int top_n,
                                  int rows, int vocab, void* stream)
{
    CallState& st = ops_state();
    return guarded(st, [&] {
        if (!logits) throw std::runtime_error("logprobs: null device pointer");
        if (logits_fp32 != 0 && logits_fp32 != 1) throw std::runtime_error("logprobs: logits_fp32 must be 0 or 1");
        if (rows < 1 || vocab < 1) throw std::runtime_error("logprobs: rows and vocab must be positive");
        if (row_stride < vocab && rows > 1) throw std::runtime_error("logprobs: row_stride is smaller than vocab");
        if (top_n < 0 || top_n > kMaxTop || top_n > vocab) throw std::runtime_error("logprobs: top_n must be in 0..=32 and at most vocab");
        if (top_n > 0 && (!top_idx || !top_logprob)) throw std::runtime_error("logprobs: null device pointer of the alternatives");
        if (!tokens && (logprob || rank)) throw std::runtime_error("logprobs: null tokens with logprob or rank wanted");
        if (!logprob && !rank && !entropy && top_n == 0) throw std::runtime_error("logprobs: every output is null");
        if (!(inv_temp > 0.f && inv_temp <= 1e30f)) throw std::runtime_error("logprobs: inv_temp must be positive and at most 1e30");
        const LogprobParams p{logits, row_stride, logprob || rank ? tokens : nullptr, logprob, rank, entropy, top_idx, top_logprob, top_n, rows, vocab,
                              inv_temp, inv_temp * kLog2e};
        launch_pdl(logits_fp32 ? k_logprobs<true> : k_logprobs<false>, dim3(rows), dim3(256), 0, (cudaStream_t) stream, "logprobs launch", p);
        st.launch = std::string("k_logprobs<") + (logits_fp32 ? "float" : "half") + "> block=256 grid=" + std::to_string(rows);
    });
}

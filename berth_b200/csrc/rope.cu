// Rotary positions of q and k with their per-head RMSNorm, and the host's table of frequencies.
#include "exl3_decode.cuh"
#include "../../include/berth_b200.h"

#include <algorithm>
#include <cmath>
#include <cstdlib>

namespace berth {
namespace {

struct RopeParams {
    berth_rope_rows r[2];   // q, k (heads = 0: none)
    const int32_t* positions;
    const double* inv_freq;
    int tokens, dim, rot, half_rot, interleaved;
    float factor, eps, bias;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float bf16_at(const void* w, int i) { return __uint_as_float(uint32_t(static_cast<const uint16_t*>(w)[i]) << 16); }

// cos and sin of position * inv_freq: the angle in turns in 64 bits, its whole turns dropped (exact), the rest to fp32.
// A position of 10^6 leaves 2^-33 of a turn; in 32 bits it would leave 2^-4.
__device__ __forceinline__ float2 turn(int position, double inv_freq, float factor)
{
    constexpr double kPerTurn = 0.15915494309189533577;   // 1 / (2 pi)
    double t = double(position) * inv_freq * kPerTurn;
    t -= rint(t);
    float s, c;
    sincospif(2.0f * float(t), &s, &c);
    return make_float2(c * factor, s * factor);
}

// One warp per (token, head); a lane reads and writes both elements of its pairs, so y may be x.
template <typename T>
__global__ void __launch_bounds__(128) k_rope(const RopeParams p)
{
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, heads = p.r[0].heads + p.r[1].heads;
    const long long total = (long long) p.tokens * heads;
    for (long long item = (long long) blockIdx.x * 4 + (threadIdx.x >> 5); item < total; item += (long long) gridDim.x * 4) {
        const int t = int(item / heads), hh = int(item % heads);
        const berth_rope_rows& r = p.r[hh >= p.r[0].heads];
        const int h = hh >= p.r[0].heads ? hh - p.r[0].heads : hh;
        const T* x = static_cast<const T*>(r.x) + t * r.x_token + h * r.x_head;
        T* y = static_cast<T*>(r.y) + t * r.y_token + h * r.y_head;
        float rinv = 1.f;
        if (r.norm) {
            float s = 0.f;
            for (int i = lane; i < p.dim; i += 32) { const float v = to_f(x[i]); s = fmaf(v, v, s); }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(dq::kFull, s, off);
            rinv = 1.0f / sqrtf(s / float(p.dim) + p.eps);
        }
        auto in = [&](int i) {
            const float v = to_f(x[i]);
            return r.norm ? v * rinv * (bf16_at(r.norm, i) + p.bias) : v;
        };
        const int pos = p.positions[t];
        for (int i = lane; i < p.half_rot; i += 32) {
            const float2 cs = turn(pos, p.inv_freq[i], p.factor);
            const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + p.half_rot;
            const float xa = in(a), xb = in(b);
            y[a] = from_f<T>(xa * cs.x - xb * cs.y);
            y[b] = from_f<T>(xb * cs.x + xa * cs.y);
        }
        for (int i = p.rot + lane; i < p.dim; i += 32) y[i] = from_f<T>(in(i));
    }
}

// A copy of r with the strides that no element needs set to zero.
berth_rope_rows checked_rows(const berth_rope_rows& r, const char* what, int tokens, int dim)
{
    auto fail = [&](const char* msg) { throw std::runtime_error(std::string("rope: ") + what + ": " + msg); };
    if (!r.x || !r.y) fail("null device pointer");
    if (r.heads < 1 || r.heads > 1024) fail("heads must be in 1..=1024");
    berth_rope_rows c = r;
    if (tokens == 1) c.x_token = c.y_token = 0;
    if (c.heads == 1) c.x_head = c.y_head = 0;
    if ((tokens > 1 && std::llabs(c.y_token) < dim) || (c.heads > 1 && std::llabs(c.y_head) < dim)) fail("the heads of the output overlap");
    if (c.x == c.y && (c.x_token != c.y_token || c.x_head != c.y_head)) fail("an output in place needs the strides of its input");
    return c;
}

}  // namespace
}  // namespace berth

using namespace berth;

extern "C" int berth_ops_rope(const berth_rope_rows* q, const berth_rope_rows* k, const int32_t* positions, const double* inv_freq,
                              int n_tokens, int head_dim, int rot_dim, int interleaved, float attention_factor, float norm_epsilon,
                              float norm_bias, int fp32, void* stream)
{
    CallState& st = ops_state();
    return guarded(st, [&] {
        if (!q || !positions || !inv_freq) throw std::runtime_error("rope: null pointer");
        if (n_tokens < 1) throw std::runtime_error("rope: n_tokens must be positive");
        if (head_dim < 2 || head_dim > 512) throw std::runtime_error("rope: head_dim must be in 2..=512");
        if (rot_dim < 2 || rot_dim % 2 || rot_dim > head_dim) throw std::runtime_error("rope: rot_dim must be positive, even and at most head_dim");
        if (fp32 != 0 && fp32 != 1) throw std::runtime_error("rope: fp32 must be 0 or 1");
        if (!std::isfinite(attention_factor)) throw std::runtime_error("rope: attention_factor must be finite");
        if ((q->norm || (k && k->norm)) && !(norm_epsilon >= 0.f && std::isfinite(norm_epsilon)))
            throw std::runtime_error("rope: norm_epsilon must be finite and not negative");
        RopeParams p{};
        p.r[0] = checked_rows(*q, "q", n_tokens, head_dim);
        if (k) p.r[1] = checked_rows(*k, "k", n_tokens, head_dim);
        p.positions = positions; p.inv_freq = inv_freq; p.tokens = n_tokens; p.dim = head_dim; p.rot = rot_dim; p.half_rot = rot_dim / 2;
        p.interleaved = interleaved != 0; p.factor = attention_factor; p.eps = norm_epsilon; p.bias = norm_bias;
        const long long items = (long long) n_tokens * (p.r[0].heads + p.r[1].heads);
        const int grid = int(std::min<long long>((items + 3) / 4, 148LL * 16));
        launch_pdl(fp32 ? k_rope<float> : k_rope<__half>, dim3(grid), dim3(128), 0, (cudaStream_t) stream, "rope launch", p);
        st.launch = std::string("k_rope<") + (fp32 ? "float" : "half") + "> block=128 grid=" + std::to_string(grid);
    });
}

extern "C" int berth_ops_rope_frequencies(double* inv_freq, int rot_dim, double base, const berth_rope_scaling* scaling, float* attention_factor)
{
    CallState& st = ops_state();
    return guarded(st, [&] {
        if (!inv_freq) throw std::runtime_error("rope frequencies: null pointer");
        if (rot_dim < 2 || rot_dim % 2 || rot_dim > 512) throw std::runtime_error("rope frequencies: rot_dim must be positive, even and at most 512");
        if (!std::isfinite(base) || base <= 1.0) throw std::runtime_error("rope frequencies: base must be finite and above 1");
        const int kind = scaling ? scaling->kind : 0, half = rot_dim / 2;
        if (kind < 0 || kind > 4) throw std::runtime_error("rope frequencies: kind must be in 0..=4");
        const double f = kind ? scaling->factor : 1.0;
        if (kind && (!std::isfinite(f) || f < 1.0)) throw std::runtime_error("rope frequencies: factor must be finite and at least 1");
        const double two_pi = 6.283185307179586476925;
        if (kind == 2) {
            if (rot_dim < 4) throw std::runtime_error("rope frequencies: a scaled base needs rot_dim of at least 4");
            base *= std::pow(f, double(rot_dim) / (rot_dim - 2));
        }
        if (kind >= 3 && !(std::isfinite(scaling->original_context) && scaling->original_context >= 1.0))
            throw std::runtime_error("rope frequencies: original_context must be finite and at least 1");
        double lo = 0.0, hi = 1.0;
        if (kind == 3) {
            if (!(scaling->beta_slow > 0.0 && scaling->beta_fast >= scaling->beta_slow && std::isfinite(scaling->beta_fast)))
                throw std::runtime_error("rope frequencies: beta_fast must be finite and at least beta_slow, which must be positive");
            auto pair_of = [&](double turns) { return rot_dim * std::log(scaling->original_context / (turns * two_pi)) / (2.0 * std::log(base)); };
            lo = std::max(std::floor(pair_of(scaling->beta_fast)), 0.0);
            hi = std::min(std::ceil(pair_of(scaling->beta_slow)), rot_dim - 1.0);
            if (hi - lo < 1e-3) hi = lo + 1e-3;
        }
        if (kind == 4 && !(scaling->low_factor > 0.0 && scaling->high_factor > scaling->low_factor && std::isfinite(scaling->high_factor)))
            throw std::runtime_error("rope frequencies: high_factor must be finite and above low_factor, which must be positive");
        for (int i = 0; i < half; ++i) {
            const double v = std::pow(base, -2.0 * i / rot_dim);
            if (kind == 1) inv_freq[i] = v / f;
            else if (kind == 3) {
                const double ramp = std::min(std::max((i - lo) / (hi - lo), 0.0), 1.0);
                inv_freq[i] = v * (1.0 - ramp) + v / f * ramp;
            } else if (kind == 4) {
                const double turns = scaling->original_context * v / two_pi;
                const double keep = std::min(std::max((turns - scaling->low_factor) / (scaling->high_factor - scaling->low_factor), 0.0), 1.0);
                inv_freq[i] = v * keep + v / f * (1.0 - keep);
            } else inv_freq[i] = v;
        }
        if (attention_factor)
            *attention_factor = kind != 3 ? 1.0f : scaling->attention_factor_override > 0.0 ? float(scaling->attention_factor_override) : float(0.1 * std::log(f) + 1.0);
    });
}

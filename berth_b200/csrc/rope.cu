// Rotary positions of q and k with their per-head RMSNorm, and the host's table of frequencies.
#include "exl3_decode.cuh"
#include "../../include/berth_b200.h"

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>
#include <utility>

namespace berth {
namespace {

struct RopeParams {
    berth_rope_rows r[2];   // q, k (heads = 0: none)
    const int32_t* positions;
    const double* inv_freq;
    int tokens, dim, rot, half_rot, interleaved;
    int lanes, tile;   // lanes of a head (a power of two), tokens of a block (a power of two)
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

// N elements of a head: 16, 8 or 4 bytes in one access (8 fp32 in two).
template <typename T, int N> struct Piece;
template <int N> struct Piece<__half, N> {
    using V = typename std::conditional<N == 8, uint4, typename std::conditional<N == 4, uint2, uint32_t>::type>::type;
    V v;
    __device__ __forceinline__ void load(const __half* p) { v = *reinterpret_cast<const V*>(p); }
    __device__ __forceinline__ void get(float* x) const
    {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store(__half* p, const float* x)
    {
        V v;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<V*>(p) = v;
    }
};
template <int N> struct Piece<float, N> {
    using V = typename std::conditional<N == 1, float, typename std::conditional<N == 2, float2, float4>::type>::type;
    static constexpr int kEach = N < 4 ? N : 4, kParts = N / kEach;
    V v[kParts];
    __device__ __forceinline__ void load(const float* p)
    {
#pragma unroll
        for (int i = 0; i < kParts; ++i) v[i] = reinterpret_cast<const V*>(p)[i];
    }
    __device__ __forceinline__ void get(float* x) const
    {
        const float* e = reinterpret_cast<const float*>(v);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = e[i];
    }
    static __device__ __forceinline__ void store(float* p, const float* x)
    {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            V v;
            float* e = reinterpret_cast<float*>(&v);
#pragma unroll
            for (int j = 0; j < kEach; ++j) e[j] = x[i * kEach + j];
            reinterpret_cast<V*>(p)[i] = v;
        }
    }
};
// N of the norm's weights, bfloat16, at an offset of whole pieces.
template <int N> struct Weights {
    using V = typename std::conditional<N == 1, uint16_t, typename std::conditional<N == 2, uint32_t, typename std::conditional<N == 4, uint2, uint4>::type>::type>::type;
    V v;
    __device__ __forceinline__ void load(const void* w, int at) { v = *reinterpret_cast<const V*>(static_cast<const uint16_t*>(w) + at); }
    __device__ __forceinline__ void scale(float* x, float rinv, float bias) const
    {
        if constexpr (N == 1) {
            x[0] = x[0] * rinv * (__uint_as_float(uint32_t(v) << 16) + bias);
        } else {
            const uint32_t* h = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                x[2 * i] = x[2 * i] * rinv * (__uint_as_float(h[i] << 16) + bias);
                x[2 * i + 1] = x[2 * i + 1] * rinv * (__uint_as_float(h[i] & 0xffff0000u) + bias);
            }
        }
    }
};

constexpr int kThreads = 128, kTable = 2048;   // cos / sin pairs a block holds

// A block takes p.tile tokens: it fills a table of their cos and sin (one thread per pair and token, 64-bit angles), then groups of
// p.lanes lanes walk the heads, each lane sixteen elements of a head.  A group stays with its token, so a lane's eight pairs of cos
// and sin stay in registers.  A lane's sixteen elements are pieces of BYTES, neighbouring lanes' pieces side by side.  kHalf: it holds both
// sides of its pairs, pieces at q and at q + rot / 2 (BYTES: the most of 16, 8 and 4 that rot / 2 is a multiple of); kNeighbours: pairs
// meet in a piece.  (8 consecutive fp32 a lane instead of 4: 4096 tokens of 40 heads of 128 30.6 us, now 28.5; fp16 in pieces of 2
// bytes: 35.9 us, k_rope_any 25.7, but fp32 in pieces of 4 36.4, k_rope_any 42.1.)
enum { kHalf = 0, kNeighbours = 1 };
// NORM kEarly: the norm's weights are on their way during the sum of squares, for grids whose blocks all run at once with the registers
// that it takes (421 tokens of 28 heads of 256 4.8 us, kNorm 5.6; 8192 of 40 of 128, more than run at once, 41 us, kNorm 34).
enum { kPlain = 0, kNorm = 1, kEarly = 2 };
constexpr int early_blocks(int size, int bytes) { return size == 2 && bytes == 16 ? 6 : 5; }   // of an SM
// Blocks of an SM that the registers have to allow (normalised fp16 neighbours left to themselves take 80: 4096 tokens of 40 heads of 128
// 20.8 us, now 18.0).
constexpr int min_blocks(int size, int mode, int bytes, int norm) { return norm == kEarly ? early_blocks(size, bytes) : norm == kNorm && mode == kNeighbours && size == 2 ? 7 : 1; }
template <typename T, int MODE, int BYTES, int NORM>
__global__ void __launch_bounds__(kThreads, min_blocks(sizeof(T), MODE, BYTES, NORM)) k_rope(const RopeParams p)
{
    constexpr int kPiece = BYTES / sizeof(T), kPairs = 8 / kPiece;   // elements of a piece; pairs of pieces of a lane
    // normalised fp16 neighbours: a lane's two pieces are one behind the other, which takes 72 registers instead of 80 (4096 tokens of
    // 40 heads of 128 18.0 us, side by side 20.6; not normalised 16.1, side by side 14.7)
    constexpr bool kTogether = MODE == kNeighbours && NORM != kPlain && sizeof(T) == 2;
    __shared__ __align__(16) float2 table[kTable];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, heads = p.r[0].heads + p.r[1].heads;
    const int group = tid / p.lanes, lane = tid % p.lanes, groups_per_token = kThreads / p.lanes / p.tile;
    const int slot = group / groups_per_token, t0 = blockIdx.x * p.tile, t = t0 + slot;
    // offsets of the pieces, -1 = none.  kHalf: the pairs j * lanes + lane, first those that turn, then what is passed on
    const int turning = p.half_rot / kPiece;
    int at[2][kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
        const int q = j * p.lanes + lane;
        if (MODE == kNeighbours) {
            at[0][j] = kTogether ? 2 * q * kPiece : q * kPiece;
            at[1][j] = kTogether ? at[0][j] + kPiece : (q + kPairs * p.lanes) * kPiece;
        } else if (q < turning) {
            at[0][j] = q * kPiece;
            at[1][j] = at[0][j] + p.half_rot;
        } else {
            at[0][j] = p.rot + 2 * kPiece * (q - turning);
            at[1][j] = at[0][j] + kPiece;
        }
        if (at[0][j] >= p.dim) at[0][j] = -1;
        if (at[1][j] >= p.dim) at[1][j] = -1;
    }

    auto rows_of = [&](int h, const T*& x, T*& y, const void*& norm) {
        const berth_rope_rows& r = p.r[h >= p.r[0].heads];
        const long long hh = h >= p.r[0].heads ? h - p.r[0].heads : h;
        x = static_cast<const T*>(r.x) + t * r.x_token + hh * r.x_head;
        y = static_cast<T*>(r.y) + t * r.y_token + hh * r.y_head;
        norm = r.norm;
    };
    const int step = groups_per_token * gridDim.y;
    int h = blockIdx.y * groups_per_token + group % groups_per_token;
    // pieces of the next heads on their way while one is worked on: two heads (8192 tokens of 40 heads of 128 fp16: 28.6 us, one:
    // 30.2; 4096 fp32: 27.3 us, one: 28.7), one where there is a norm (35.1 us, two: 38.2)
    constexpr int kAhead = NORM != kPlain ? 1 : 2;
    struct Head {
        Piece<T, kPiece> in[2][kPairs];
        T* y;
        const void* norm;
    } ahead[kAhead];
    auto fetch = [&](Head& to, int h) {
        if (t < p.tokens && h < heads) {
            const T* x;
            if constexpr (kAhead == 1) rows_of(h, x, to.y, to.norm);
            else {   // (found again when it is worked on: four registers a head cost more than that)
                T* y;
                const void* norm;
                rows_of(h, x, y, norm);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < kPairs; ++j)
                    if (at[i][j] >= 0) to.in[i][j].load(x + at[i][j]);
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(ahead[i], h + i * step);
    for (int i = tid; i < p.tile * p.half_rot; i += kThreads) {
        const int s = i / p.half_rot;
        if (t0 + s < p.tokens) table[i] = turn(p.positions[t0 + s], p.inv_freq[i - s * p.half_rot], p.factor);
    }
    __syncthreads();
    // a lane's i-th pair, from half_rot on one that does not turn
    auto pair_at = [&](int i) {
        return kTogether ? 8 * lane + i : MODE == kNeighbours ? ((2 * i / kPiece * p.lanes + lane) * kPiece + 2 * i % kPiece) / 2 : (i / kPiece * p.lanes + lane) * kPiece + i % kPiece;
    };
    float2 cs[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (pair_at(i) < p.half_rot) cs[i] = table[slot * p.half_rot + pair_at(i)];
    auto work = [&](Head& now) {
        float v[16];   // first sides, second sides
        const bool live = t < p.tokens && h < heads;
        T* to = nullptr;
        const void* w = nullptr;
        if constexpr (kAhead == 1) {
            to = now.y;
            w = now.norm;
        } else if (live) {
            const T* x;
            rows_of(h, x, to, w);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < kPairs; ++j)
                if (live && at[i][j] >= 0) now.in[i][j].get(v + 8 * i + kPiece * j);
                else {
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) v[8 * i + kPiece * j + e] = 0.f;
                }
        fetch(now, h + kAhead * step);
        h += step;
        if constexpr (NORM != kPlain) {
            Weights<kPiece> weights[2][kPairs];
            if (NORM == kEarly && live && w) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < kPairs; ++j)
                        if (at[i][j] >= 0) weights[i][j].load(w, at[i][j]);
            }
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) s = fmaf(v[j], v[j], s);
            for (int off = p.lanes / 2; off >= 1; off >>= 1) s += __shfl_xor_sync(dq::kFull, s, off);
            if (live && w) {
                const float rinv = rsqrtf(s / float(p.dim) + p.eps);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < kPairs; ++j)
                        if (at[i][j] >= 0) {
                            if (NORM != kEarly) weights[i][j].load(w, at[i][j]);
                            weights[i][j].scale(v + 8 * i + kPiece * j, rinv, p.bias);
                        }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (MODE == kNeighbours ? pair_at(i) >= p.half_rot : i / kPiece * p.lanes + lane >= turning) continue;   // passed on
            float &a = MODE == kNeighbours ? v[2 * i] : v[i], &b = MODE == kNeighbours ? v[2 * i + 1] : v[8 + i];
            const float a0 = a, b0 = b;
            a = a0 * cs[i].x - b0 * cs[i].y;
            b = b0 * cs[i].x + a0 * cs[i].y;
        }
        if (live) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < kPairs; ++j)
                    if (at[i][j] >= 0) Piece<T, kPiece>::store(to + at[i][j], v + 8 * i + kPiece * j);
        }
    };
    // every lane of a warp walks alike, so that the norm's sums meet
    for (int base = blockIdx.y * groups_per_token; base < heads; base += kAhead * step) {
        work(ahead[0]);
        if constexpr (kAhead == 2) {
            if (base + step < heads) work(ahead[1]);
        }
    }
}

// Bound: HBM.  Inputs that change from call to call: 8192 tokens of 40 heads of 128 fp16 as columns of a q/k/v buffer 30.6 us (5.5 TB/s,
// 0.84 of the copy's rate), apart 29.5, normalised 34.5; 4096 fp32 27.6 (6.1 TB/s); 421 tokens of 28 heads of 256, a quarter turned,
// normalised: 4.8 us, one wave of dependent latencies.  (Variants are compared, above and below, by calls on the same buffers, part of which
// the L2 holds: 28.6 us for the first, 31.8 with 256 threads a block.)  Pieces of 4 bytes of fp32 with the weights early keep 48 bytes of a
// thread in local memory (five blocks an SM).

// The same for any part, alignment and stride: a lane holds sixteen consecutive elements and finds the other element of a pair
// in shared memory (pitch 17, so that lanes 16 elements apart meet different banks).  Its cos, signed sin and the places of the other
// elements stay in registers.  Bound: latency, above all of a head's loads, which are asked for only when its turn comes: 4.5 warps a
// scheduler (96 registers, 27 KB) issue in 46 % of the cycles, shared memory's pipe is busy for 44 %, HBM for 29 %.  4096 tokens of 40
// heads of 128 fp16, 42 turned, inputs that change: 27.6 us (k_rope, 44 turned: 22.7), 8192: 51.6; with registers for 4 blocks an SM
// instead of 5 it was 31.5 us instead of 27.1.
template <typename T, bool NORM>
__global__ void __launch_bounds__(kThreads, 5) k_rope_any(const RopeParams p, bool wide)
{
    __shared__ float2 table[kTable + kTable / 16 + kThreads];   // (pitch: half_rot + half_rot / 16 + 1, at most kThreads tokens)
    __shared__ float stage[kThreads * 17];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, heads = p.r[0].heads + p.r[1].heads;
    const int group = tid / p.lanes, lane = tid % p.lanes, groups_per_token = kThreads / p.lanes / p.tile;
    const int slot = group / groups_per_token, t0 = blockIdx.x * p.tile, t = t0 + slot, e0 = 16 * lane;
    const int pitch = p.half_rot + p.half_rot / 16 + 1;
    for (int i = tid; i < p.tile * p.half_rot; i += kThreads) {
        const int s = i / p.half_rot, k = i - s * p.half_rot;
        if (t0 + s < p.tokens) table[s * pitch + k + k / 16] = turn(p.positions[t0 + s], p.inv_freq[k], p.factor);
    }
    __syncthreads();
    float* mine = stage + (tid - lane) * 17;   // the group's head
    // out = v * cos + other * sin, with the sign of the pair's side; the group stays with its token
    float2 cs[16];
    int other_at[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int e = e0 + j;
        const bool second = p.interleaved ? e & 1 : e >= p.half_rot;
        const int k = p.interleaved ? e / 2 : second ? e - p.half_rot : e, o = second ? e - p.half_rot : e + p.half_rot;
        if (e < p.rot) {
            cs[j] = table[slot * pitch + k + k / 16];
            if (!second) cs[j].y = -cs[j].y;
            other_at[j] = o + o / 16;
        }
    }
    const int step = groups_per_token * gridDim.y, h0 = blockIdx.y * groups_per_token;
    for (int base = h0; base < heads; base += step) {
        const int h = base + group % groups_per_token;
        const bool live = t < p.tokens && h < heads;
        const berth_rope_rows& r = p.r[h >= p.r[0].heads];
        const long long hh = h >= p.r[0].heads ? h - p.r[0].heads : h;
        const T* x = static_cast<const T*>(r.x) + t * r.x_token + hh * r.x_head;
        T* y = static_cast<T*>(r.y) + t * r.y_token + hh * r.y_head;
        float v[16];
        if (wide && live && e0 + 16 <= p.dim) {
            Piece<T, 8> a, b;
            a.load(x + e0);
            b.load(x + e0 + 8);
            a.get(v);
            b.get(v + 8);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = live && e0 + j < p.dim ? to_f(x[e0 + j]) : 0.f;
        }
        if constexpr (NORM) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) s = fmaf(v[j], v[j], s);
            for (int off = p.lanes / 2; off >= 1; off >>= 1) s += __shfl_xor_sync(dq::kFull, s, off);
            if (live && r.norm) {
                const float rinv = rsqrtf(s / float(p.dim) + p.eps);
                if (wide && e0 + 16 <= p.dim) {
                    Weights<8> a, b;
                    a.load(r.norm, e0);
                    b.load(r.norm, e0 + 8);
                    a.scale(v, rinv, p.bias);
                    b.scale(v + 8, rinv, p.bias);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (e0 + j < p.dim) v[j] = v[j] * rinv * (bf16_at(r.norm, e0 + j) + p.bias);
                }
            }
        }
        if (p.interleaved) {
#pragma unroll
            for (int j = 0; j < 16; j += 2)
                if (e0 + j < p.rot) {
                    const float a = v[j], b = v[j + 1];
                    v[j] = a * cs[j].x + b * cs[j].y;
                    v[j + 1] = b * cs[j + 1].x + a * cs[j + 1].y;
                }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) mine[lane * 17 + j] = v[j];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (e0 + j < p.rot) v[j] = v[j] * cs[j].x + mine[other_at[j]] * cs[j].y;
            __syncwarp();
        }
        if (!live) continue;
        if (wide && e0 + 16 <= p.dim) {
            Piece<T, 8>::store(y + e0, v);
            Piece<T, 8>::store(y + e0 + 8, v + 8);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (e0 + j < p.dim) y[e0 + j] = from_f<T>(v[j]);
        }
    }
}

// A copy of r with the strides that no element needs set to zero.
berth_rope_rows checked_rows(const berth_rope_rows& r, const char* what, int tokens, int dim, int size)
{
    auto fail = [&](const char* msg) { throw std::runtime_error(std::string("rope: ") + what + ": " + msg); };
    if (!r.x || !r.y) fail("null device pointer");
    if (r.heads < 1 || r.heads > 1024) fail("heads must be in 1..=1024");
    berth_rope_rows c = r;
    if (tokens == 1) c.x_token = c.y_token = 0;
    if (c.heads == 1) c.x_head = c.y_head = 0;
    check_aligned(r.x, size, (std::string("rope: ") + what).c_str());
    check_aligned(r.y, size, (std::string("rope: output of ") + what).c_str());
    check_aligned(r.norm, 2, (std::string("rope: norm of ") + what).c_str());
    // an output's heads lie apart along the smaller of its strides, and all that walks the larger one
    long long a = std::llabs(c.y_head), b = std::llabs(c.y_token), na = c.heads, nb = tokens;
    if (nb > 1 && (na == 1 || b < a)) {
        std::swap(a, b);
        std::swap(na, nb);
    }
    if ((na > 1 && a < dim) || (nb > 1 && b < __int128(na - 1) * a + dim)) fail("the heads of the output overlap");
    if (c.x == c.y && (c.x_token != c.y_token || c.x_head != c.y_head)) fail("an output in place needs the strides of its input");
    return c;
}

// Every row of 16-byte pieces: pointers and strides.
bool wide_rows(const RopeParams& p, int size)
{
    for (const berth_rope_rows& r : p.r) {
        if (r.heads == 0) continue;
        const uintptr_t bits = reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.y) | reinterpret_cast<uintptr_t>(r.norm) |
                               uintptr_t(r.x_token * size) | uintptr_t(r.x_head * size) | uintptr_t(r.y_token * size) | uintptr_t(r.y_head * size);
        if (bits & 15) return false;
    }
    return true;
}

std::string launch_rope(RopeParams p, bool f32, cudaStream_t st)
{
    const int heads = p.r[0].heads + p.r[1].heads;
    const bool wide = wide_rows(p, f32 ? 4 : 2) && p.dim % 8 == 0, norm = p.r[0].norm || p.r[1].norm;
    // bytes of a piece: 16, or the most that half of what turns is a multiple of; 0: k_rope_any
    const int size = f32 ? 4 : 2, half_bytes = p.half_rot * size;
    const int bytes = !wide ? 0 : p.interleaved || half_bytes % 16 == 0 ? 16 : half_bytes % 8 == 0 ? 8 : half_bytes % 4 == 0 ? 4 : 0;
    // lanes of a head: sixteen elements each, of halves both sides of what turns, then what is passed on
    int units = (p.dim + 15) / 16;
    if (bytes && !p.interleaved) {
        const int piece = bytes / size, pairs = p.half_rot / piece + (p.dim - p.rot + 2 * piece - 1) / (2 * piece);
        units = (pairs * piece + 7) / 8;
    }
    p.lanes = 1;
    while (p.lanes < units) p.lanes *= 2;
    const int groups = kThreads / p.lanes;
    // tokens of a block: until every group walks some four heads, or eight where they are normalised (8192 tokens of 40 heads of 128:
    // plain 28.6 us, with eight 28.8; normalised 33.8, with four 35.1), as long as the grid has four blocks an SM
    p.tile = 1;
    while (p.tile < groups && heads * p.tile < (norm ? 8 : 4) * groups && (p.tokens + 2 * p.tile - 1) / (2 * p.tile) >= 148 * 4 && 2 * p.tile * p.half_rot <= kTable)
        p.tile *= 2;
    // few tokens: their heads over several blocks
    const int blocks_x = (p.tokens + p.tile - 1) / p.tile;
    int blocks_y = 1;
    while (blocks_x * blocks_y < 148 * 4 && blocks_y * groups / p.tile < heads) ++blocks_y;
    const dim3 grid(blocks_x, blocks_y);
    const bool early = norm && bytes && blocks_x * blocks_y <= 148 * early_blocks(size, bytes);
    const char* name = "";
    auto go = [&](auto kern, const char* what, auto... more) {
        launch_pdl(kern, grid, dim3(kThreads), 0, st, "rope launch", p, more...);
        name = what;
    };
    auto typed = [&](auto zero) {
        using T = decltype(zero);
        auto pieces = [&](auto mode, auto n, const char* what) {
            constexpr int MODE = decltype(mode)::value, BYTES = decltype(n)::value;
            !norm ? go(k_rope<T, MODE, BYTES, kPlain>, what) : early ? go(k_rope<T, MODE, BYTES, kEarly>, what) : go(k_rope<T, MODE, BYTES, kNorm>, what);
        };
        const std::integral_constant<int, kHalf> halves;
        if (!bytes) norm ? go(k_rope_any<T, true>, "k_rope_any", wide) : go(k_rope_any<T, false>, "k_rope_any", wide);
        else if (p.interleaved) pieces(std::integral_constant<int, kNeighbours>{}, std::integral_constant<int, 16>{}, "k_rope_neighbours");
        else if (bytes == 16) pieces(halves, std::integral_constant<int, 16>{}, "k_rope_half");
        else if (bytes == 8) pieces(halves, std::integral_constant<int, 8>{}, "k_rope_half");
        else pieces(halves, std::integral_constant<int, 4>{}, "k_rope_half");
    };
    if (f32) typed(0.0f);
    else typed(__half{});
    return describe(name, "<", f32 ? "float" : "half", early ? ",norm early" : norm ? ",norm" : "", "> block=", kThreads, " grid=", blocks_x, "x", blocks_y, " tokens=", p.tile,
                    " lanes=", p.lanes, " piece=", bytes);
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
        if (n_tokens < 1 || n_tokens > (1 << 30)) throw std::runtime_error("rope: n_tokens must be positive and at most 2^30");
        if (head_dim < 2 || head_dim > 512) throw std::runtime_error("rope: head_dim must be in 2..=512");
        if (rot_dim < 2 || rot_dim % 2 || rot_dim > head_dim) throw std::runtime_error("rope: rot_dim must be positive, even and at most head_dim");
        if (fp32 != 0 && fp32 != 1) throw std::runtime_error("rope: fp32 must be 0 or 1");
        if (!std::isfinite(attention_factor)) throw std::runtime_error("rope: attention_factor must be finite");
        if ((q->norm || (k && k->norm)) && !(norm_epsilon >= 0.f && std::isfinite(norm_epsilon)))
            throw std::runtime_error("rope: norm_epsilon must be finite and not negative");
        check_aligned(positions, 4, "rope: positions");
        check_aligned(inv_freq, 8, "rope: inv_freq");
        RopeParams p{};
        p.r[0] = checked_rows(*q, "q", n_tokens, head_dim, fp32 ? 4 : 2);
        if (k) p.r[1] = checked_rows(*k, "k", n_tokens, head_dim, fp32 ? 4 : 2);
        p.positions = positions; p.inv_freq = inv_freq; p.tokens = n_tokens; p.dim = head_dim; p.rot = rot_dim; p.half_rot = rot_dim / 2;
        p.interleaved = interleaved != 0; p.factor = attention_factor; p.eps = norm_epsilon; p.bias = norm_bias;
        st.launch = launch_rope(p, fp32 != 0, (cudaStream_t) stream);
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
            if (!std::isfinite(base)) throw std::runtime_error("rope frequencies: the scaled base is out of range");
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
            if (pair_of(scaling->beta_slow) <= 0.0 && pair_of(scaling->beta_fast) < 0.0) lo = -1.0, hi = 0.0;   // not even pair 0 turns more than beta_slow times
            else if (hi - lo < 1e-3) hi = lo + 1e-3;
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

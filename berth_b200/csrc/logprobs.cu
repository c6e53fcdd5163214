// Log probabilities of given tokens, entropy and the best alternatives of every row of logits, in one pass over them.
//
// A row is split over the CTAs of a cluster.  Every thread walks its 16-byte vectors with a running maximum M and the sums
// z = sum 2^y and t = sum 2^y y, y = (x - M) * inv_temp * log2 e: ln p = (x - m) * inv_temp - ln z and the entropy
// ln z - t / z * ln 2 follow from the joined (m, z, t).  A thread adds its vectors' sums, trees of 16 or 32, with the rounding
// kept aside, and joins carry z less the maximum's own 1: a certain row has z = 1 + little, and its entropy is made of that
// little.  (The logits of the maximum's own step, 15 fp32 or 31 fp16, meet its 1 in their tree: up to five roundings of 2^-24, an error
// of 3e-7 in ln p and entropy.)  The rank of a given token is a count of the logits before it, taken in the same walk.
//
// The n best come out of the walk's by-product, the threads' maxima.  The cluster's warps fall into 32 or 64 groups (or give their k
// largest threads each, where there are fewer warps): as many different logits that the row reaches.  At least n logits reach the
// n-th largest of them, tau, and few more do, all of them in threads whose maximum reaches it.  Only those threads' vectors are read
// again, and of those only the steps of the walk in which the warp reached it (well below a percent of the row); what reaches tau
// goes to the first CTA's shared memory, and each finds its place by counting the larger ones.  Rows where too many reach it (equal
// logits, a mask that leaves fewer than n) are scanned once more with a sorted list of 32 per warp instead.
#include "exl3_decode.cuh"
#include "../../include/berth_b200.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace berth {
namespace {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
constexpr int kMaxTop = 32, kMaxCluster = 16, kKeys = 512;
static_assert(kMaxCluster * kMaxTop <= kKeys, "the lists of a cluster share the key buffer");

constexpr int kUnroll = 4, kRingBytes = 2 * kUnroll * 32 * 16;   // vectors of a thread in a step; the ring of a warp

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
__device__ __forceinline__ unsigned order_bits(float v)
{
    const unsigned b = __float_as_uint(v + 0.0f);
    return v != v ? 0u : ((b >> 31) ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(float v, int i)
{
    return (unsigned long long) order_bits(v) << 32 | (0xffffffffu - unsigned(i));
}
__device__ __forceinline__ float key_value(unsigned long long key)
{
    const unsigned o = unsigned(key >> 32);
    return o == 0u ? NAN : __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// Two fp32 lanes of one 64-bit register (one instruction for both).
struct f2 { unsigned long long v; };
__device__ __forceinline__ f2 pack2(float a, float b) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpack2(f2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }

// Cluster plumbing: shared-memory addresses of another CTA of the cluster.
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t peer_addr(const void* p, int cta)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    return r;
}
__device__ __forceinline__ void peer_store(uint32_t a, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void peer_store(uint32_t a, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A part of a row: its maximum m, z = sum 2^y less the 1 of the maximum itself, t = sum 2^y y, y relative to m.  Without the 1,
// fp32 keeps the small rest of a certain row to its own 2^-24.  m = -inf: no logit above it, z = 0 (NaN after a NaN).
struct Part {
    float m, z, t;
};
__device__ __forceinline__ float redux_max(float v) { float r; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
// p, whose maximum is not the one that keeps its 1 out of the sum, relative to the maximum m.
__device__ __forceinline__ Part beside(Part p, float m, float scale2)
{
    if (p.m > -INFINITY) {
        const float d = (p.m - m) * scale2, f = ex2(d), all = 1.f + p.z;
        p.t = f != 0.f ? (p.t + d * all) * f : all * f;   // a factor that vanished leaves 0, or NaN
        p.z = all * f;
    }
    return p;
}
// The N parts of each of the warp's lanes as one, in every lane (the order of the sums is fixed).
template <int N>
__device__ __forceinline__ Part joined(const Part (&p)[N], float scale2)
{
    float m = p[0].m;
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, p[i].m);
    const float mine = m;
    m = redux_max(m);
    bool holds = int(threadIdx.x & 31) == __ffs(__ballot_sync(dq::kFull, mine == m)) - 1;   // the first part with the maximum keeps its 1 out
    Part all{m, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool keeps = holds && p[i].m == m;
        holds = holds && !keeps;
        const Part o = keeps ? p[i] : beside(p[i], m, scale2);
        all.z += o.z;
        all.t += o.t;
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        all.z += __shfl_xor_sync(dq::kFull, all.z, off);
        all.t += __shfl_xor_sync(dq::kFull, all.t, off);
    }
    return all;
}

// 16 bytes of a row: 8 fp16 or 4 fp32.
template <bool F32> struct Vec;
template <> struct Vec<true> {
    static constexpr int N = 4;
    float x[4];
    __device__ __forceinline__ void load(const uint4* a)
    {
        set(__ldcg(a));
    }
    __device__ __forceinline__ void set(const uint4& v)
    {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    __device__ __forceinline__ void clear() { x[0] = x[1] = x[2] = x[3] = -INFINITY; }
    __device__ __forceinline__ f2 pair_plus(int i, float c) const { return add2(pack2(x[2 * i], x[2 * i + 1]), pack2(c, c)); }
    __device__ __forceinline__ float at(int i) const { return x[i]; }
    __device__ __forceinline__ float max_with(float m) const { return max3(max3(m, x[0], x[1]), x[2], x[3]); }
};
template <> struct Vec<false> {
    static constexpr int N = 8;
    __half2 h[4];
    __device__ __forceinline__ void load(const uint4* a)
    {
        set(__ldcg(a));
    }
    __device__ __forceinline__ void set(const uint4& v)
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __half2*>(&w[i]);
    }
    __device__ __forceinline__ void clear() { h[0] = h[1] = h[2] = h[3] = __half2half2(__ushort_as_half(0xfc00)); }
    __device__ __forceinline__ f2 pair_plus(int i, float c) const   // converted and added in one instruction
    {
        float a, b;
        asm("add.f32.f16 %0, %1, %2;" : "=f"(a) : "h"(__half_as_ushort(__low2half(h[i]))), "f"(c));
        asm("add.f32.f16 %0, %1, %2;" : "=f"(b) : "h"(__half_as_ushort(__high2half(h[i]))), "f"(c));
        return pack2(a, b);
    }
    __device__ __forceinline__ float at(int i) const { return (i & 1) ? __high2float(h[i >> 1]) : __low2float(h[i >> 1]); }
    __device__ __forceinline__ float max_with(float m) const
    {
        const __half2 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(m, fmaxf(__low2float(a), __high2float(a)));
    }
};

// The smallest value above v in its type: x > v as x >= above(v), for every x that is not NaN.
__device__ __forceinline__ float above(float v)
{
    const unsigned b = __float_as_uint(v);
    return v == 0.f ? __uint_as_float(1u) : __uint_as_float(v > 0.f ? b + 1 : b - 1);
}
__device__ __forceinline__ __half above(__half v)
{
    const unsigned short b = __half_as_ushort(v);
    const float f = __half2float(v);
    return f == 0.f ? __ushort_as_half(1) : __ushort_as_half(f > 0.f ? (unsigned short) (b + 1) : (unsigned short) (b - 1));
}

// How many of the vectors' logits are >= their vector's threshold.
template <int U>
__device__ __forceinline__ int count_ge(const Vec<true> (&v)[U], const float (&thr)[U])
{
    int c = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) c += v[u].x[i] >= thr[u];
    return c;
}
template <int U>
__device__ __forceinline__ int count_ge(const Vec<false> (&v)[U], const __half (&thr)[U])
{
    __half2 c = __float2half2_rn(0.f);   // up to 4 U in each half: exact
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const __half2 t = __half2half2(thr[u]);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __hadd2(c, __hge2(v[u].h[i], t));
    }
    return int(__low2float(c) + __high2float(c));
}

// A warp's 32 largest keys, lane i the i-th.
__device__ __forceinline__ void insert_key(unsigned long long& list, unsigned long long key)
{
    const int lane = threadIdx.x & 31;
    const int pos = __popc(__ballot_sync(dq::kFull, list > key));
    const unsigned long long up = __shfl_up_sync(dq::kFull, list, 1);
    if (lane == pos) list = key;
    else if (lane > pos) list = up;
}
// Every lane offers one key (0: none); those that belong to the n first are taken in.
__device__ __forceinline__ void offer_keys(unsigned long long& list, unsigned long long key, int n)
{
    for (;;) {
        const unsigned long long floor_key = __shfl_sync(dq::kFull, list, n - 1);
        const unsigned more = __ballot_sync(dq::kFull, key > floor_key);
        if (!more) return;
        const int src = __ffs(more) - 1;
        insert_key(list, __shfl_sync(dq::kFull, key, src));
        if ((threadIdx.x & 31) == src) key = 0;
    }
}
// The 32 largest of two sorted lists, sorted.
__device__ __forceinline__ unsigned long long merge_lists(unsigned long long a, unsigned long long b)
{
    const int lane = threadIdx.x & 31;
    const unsigned long long r = __shfl_sync(dq::kFull, b, 31 - lane);
    unsigned long long v = a > r ? a : r;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const unsigned long long o = __shfl_xor_sync(dq::kFull, v, off);
        v = (lane & off) ? (v < o ? v : o) : (v > o ? v : o);
    }
    return v;
}

template <int WARPS>
struct Shared {
    unsigned long long keys[kKeys];             // first CTA: every CTA's keys that reach tau, or its list; 0 = none
    alignas(16) unsigned long long lists[kKeys / 32][32];   // the warps' lists of the slow way; first CTA: the keys, one behind the other
    float m[kMaxCluster * WARPS], z[kMaxCluster * WARPS], t[kMaxCluster * WARPS];   // first CTA: the parts of the cluster's warps
    int before[kMaxCluster * WARPS];
    float reach[kMaxCluster * WARPS];           // what logits of every warp of the cluster reach
    int cand[WARPS][32];
    unsigned n_own, n_keys, flooded;
    float row_m, row_lnz;
    int none;
};

// The slow way to a CTA's best: its vectors again, 32 sorted keys a warp, merged into sh.lists[0].
template <bool F32, int WARPS>
__device__ __noinline__ void sorted_lists(Shared<WARPS>& sh, const char* row, const uint4* vecs, int head, int nvec, int first, int stride, int single, float tau,
                                          int n)
{
    using V = Vec<F32>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long list = 0;
    offer_keys(list, single >= 0 ? order_key(value_at<F32>(row, single), single) : 0, n);
    for (int base = first - lane; base < nvec; base += stride) {
        const int i = base + lane;
        V w;
        w.clear();
        if (i < nvec) w.load(vecs + i);
#pragma unroll
        for (int e = 0; e < V::N; ++e) offer_keys(list, i < nvec && !(w.at(e) < tau) ? order_key(w.at(e), head + i * V::N + e) : 0, n);
    }
    sh.lists[warp][lane] = list;
    for (int w = WARPS / 2; w >= 1; w >>= 1) {
        __syncthreads();
        if (warp < w) {
            list = merge_lists(list, sh.lists[warp + w][lane]);
            sh.lists[warp][lane] = list;
        }
    }
    __syncthreads();
}

// Vector i of the row belongs to thread i % kThreads of CTA (i / kThreads) % ctas, so that every warp sees all of the
// vocabulary: a threshold taken from the warps' maxima then holds where the likely tokens lie close together.  The walk takes 4
// vectors of a thread at a time, while those of the next step are on their way to shared memory.
// Bound: long rows, instructions (9.9 warp instructions per 32 logits, 67 % of the issue slots) and ex2 (62 % of its pipe) before
// HBM; few rows, the fixed parts of a call (cluster barriers, the dependent reads of the candidates, the join: 4 to 5 us); rows with
// fewer finite logits than alternatives, the scan with sorted lists.
// Inputs that change from call to call: 421 x 248320 fp16, 5 alternatives, 52.4 us (4.0 TB/s), without alternatives 5.5 less; 32 x 248320
// fp32 12.0 us (2.7 TB/s), of which three logits are finite 32; 77 x 100003 fp32 9.1 us (3.4 TB/s); 1 x 248320 fp32, 20 alternatives, 7.9
// us, of which ten are finite 26.  (Variants are compared, here and below, by calls on the same buffers, part of which the L2 holds: the
// first takes 47.5 there.)
template <bool F32, bool RANK, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 32 / WARPS) k_logprobs(const LogprobParams p)
{
    using V = Vec<F32>;
    using E = typename std::conditional<F32, float, __half>::type;
    constexpr int U = kUnroll, kThreads = WARPS * 32;
    __shared__ Shared<WARPS> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int cta, ctas;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    if (cta == 0)
        for (int i = tid; i < kKeys; i += kThreads) sh.keys[i] = 0;
    if (tid == 0) sh.n_own = sh.n_keys = sh.flooded = 0;
    if (ctas > 1) cluster_arrive();             // every CTA has started, and cleared its shared memory, when the wait below ends
    auto sync_all = [&] {
        if (ctas > 1) { cluster_arrive(); cluster_wait(); }
        else __syncthreads();
    };
    pdl_wait();

    const size_t r = blockIdx.x / ctas;
    const char* row = static_cast<const char*>(p.logits) + r * p.ld * sizeof(E);
    // the row as `head` single logits up to a 16-byte boundary, full vectors, and `tail` single logits
    const int head = min(int(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(E)), p.vocab);
    const int nvec = (p.vocab - head) / V::N, tail = p.vocab - head - nvec * V::N;
    const uint4* vecs = reinterpret_cast<const uint4*>(row + head * sizeof(E));
    const int stride = kThreads * ctas, first = cta * kThreads + tid;   // of this thread's vectors
    const int steps = (nvec + stride * U - 1) / (stride * U);
    // a thread copies its vectors to places of its own in the ring and reads nothing else there: no barrier
    extern __shared__ __align__(16) uint4 ring[];   // [2][U][kThreads]
    const uint32_t ring_at = smem_addr(ring + tid);
    const uint4* from = vecs + first;
    auto request = [&](int step) {
        const uint32_t to = ring_at + (step & 1) * (U * kThreads * 16);
        auto copy = [&](int u) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * kThreads * 16), "l"(from + u * stride) : "memory"); };
        if (step + 1 < steps) {
#pragma unroll
            for (int u = 0; u < U; ++u) copy(u);
        } else if (step < steps) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (first + (step * U + u) * stride < nvec) copy(u);
        }
        from += U * stride;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    request(0);
    const int token = RANK ? p.tokens[r] : -1;

    // the first CTA's threads 0..head-1 and 16..16+tail-1 begin with a single logit
    float m = -INFINITY, z = 0.f, z_low = 0.f, t = 0.f;   // z + z_low: the sum with the maximum's 1
    int single = -1, before = 0, token_vec = 0;
    if (cta == 0) {
        if (tid < head) single = tid;
        else if (tid >= 16 && tid < 16 + tail) single = p.vocab - tail + tid - 16;
    }
    if (single >= 0) {
        const float x = value_at<F32>(row, single);
        m = x != x ? -INFINITY : x;
        z = x != x || x == INFINITY ? NAN : (x > -INFINITY ? 1.f : 0.f);
    }
    const bool real = token >= 0 && token < p.vocab;
    unsigned long long token_key = 0;
    E at{}, over{};
    float least = INFINITY;
    if (RANK && real) {
        at = reinterpret_cast<const E*>(row)[token];
        token_vec = token < head ? -1 : (token - head) / V::N;
    }
    // what the count of the logits before the token needs; behind the first step's sums, which do not wait for it
    auto look_at_token = [&] {
        if (!RANK || !real) return;
        over = above(at);
        least = F32 ? float(at) : __half2float(at);
        token_key = order_key(least, token);
        if (single >= 0) before += order_key(value_at<F32>(row, single), single) > token_key;
        // equal logits before the token in its own vector (the walk counts the larger ones there)
        if (cta == 0 && tid >= 32 && tid < 32 + V::N && token_vec >= 0 && token_vec < nvec) {
            const int i = head + token_vec * V::N + tid - 32;
            if (i < token) before += value_at<F32>(row, i) == least;
        }
    };
    float step_max = -INFINITY;   // lane i: the warp's maximum in the steps i, i + 32, ..

    if (steps == 0) look_at_token();
    for (int step = 0; step < steps; ++step) {
        request(step + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].set(ring[((step & 1) * U + u) * kThreads + tid]);
        if (step + 1 == steps) {   // behind the end: adds nothing, and lies behind every token's vector
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (first + (step * U + u) * stride >= nvec) v[u].clear();
        }
        float g = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) g = v[u].max_with(g);
        if (p.top_n > 0) {
            const float w = redux_max(g);
            if (lane == (step & 31)) step_max = fmaxf(step_max, w);
        }
        if (g > m) {
            if (m > -INFINITY) {
                const float d = (m - g) * p.scale2, f = ex2(d);
                t = f != 0.f ? (t + d * (z + z_low)) * f : z * f;
                z *= f;
                z_low *= f;
            }
            m = g;
        }
        const float nref = m > -INFINITY ? -m : 0.f;
        const f2 sc = pack2(p.scale2, p.scale2);
        f2 zs[U], ts[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f2 e[V::N / 2];
#pragma unroll
            for (int i = 0; i < V::N / 2; ++i) {
                float a, b;
                unpack2(mul2(v[u].pair_plus(i, nref), sc), a, b);
                a = max_nan(a, -200.f);   // a masked logit: 2^y is 0 either way, 0 * -inf is not
                b = max_nan(b, -200.f);
                e[i] = pack2(ex2(a), ex2(b));
                ts[u] = i == 0 ? mul2(e[i], pack2(a, b)) : fma2(e[i], pack2(a, b), ts[u]);
            }
            zs[u] = add2(e[0], e[1]);
            if constexpr (V::N == 8) zs[u] = add2(zs[u], add2(e[2], e[3]));
        }
        const f2 z4 = add2(add2(zs[0], zs[1]), add2(zs[2], zs[3])), t4 = add2(add2(ts[0], ts[1]), add2(ts[2], ts[3]));
        float za, zb, ta, tb;
        unpack2(z4, za, zb);
        unpack2(t4, ta, tb);
        za += zb;
        const float sum = z + za, part = sum - z;   // two-sum: z_low takes what sum rounds off
        z_low += (z - (sum - part)) + (za - part);
        z = sum;
        t += ta + tb;
        if (step == 0) look_at_token();
        if (RANK && g >= least) {               // most tokens are likely ones: few steps reach them
            E thr[U];
#pragma unroll
            for (int u = 0; u < U; ++u) thr[u] = first + (step * U + u) * stride < token_vec ? at : over;
            before += count_ge(v, thr);
        }
    }

    // ---- join: the warps leave their parts with the first CTA, and with every CTA what they reach
    const int warps = ctas * WARPS, me = cta * WARPS + warp;
    const Part own = joined({Part{m, m > -INFINITY ? (z - 1.f) + z_low : z, t}}, p.scale2);
    if (RANK) before = __reduce_add_sync(dq::kFull, before);
    // one logit that a warp reaches, or with few warps its k largest threads: lane i the i-th
    const bool many = p.top_n > (warps >= 16 ? 12 : warps == 8 ? 16 : 24);   // 64 groups, or 32 (see tau)
    int k_shift = 0;
    float reach = own.m;
    if (p.top_n > 0 && warps < (many ? 64 : 32)) {
        k_shift = 1;
        while (many ? warps << k_shift < 64 : warps << k_shift < p.top_n) ++k_shift;
        float rest = m, best = own.m;
        for (int i = 1; i < 1 << k_shift; ++i) {
            if (lane == __ffs(__ballot_sync(dq::kFull, rest == best)) - 1) rest = -INFINITY;
            best = redux_max(rest);
            if (lane == i) reach = best;
        }
    }
    const int k_mask = (1 << k_shift) - 1;
    reach = __shfl_sync(dq::kFull, reach, lane & k_mask);
    if (ctas > 1) cluster_wait();
    else __syncthreads();
    if (lane == 0) {
        peer_store(peer_addr(&sh.m[me], 0), __float_as_uint(own.m));
        peer_store(peer_addr(&sh.z[me], 0), __float_as_uint(own.z));
        peer_store(peer_addr(&sh.t[me], 0), __float_as_uint(own.t));
        peer_store(peer_addr(&sh.before[me], 0), unsigned(before));
    }
    if (p.top_n > 0 && lane >> k_shift < ctas) peer_store(peer_addr(&sh.reach[(me << k_shift) + (lane & k_mask)], lane >> k_shift), __float_as_uint(reach));
    sync_all();

    // ---- the candidates for the n best
    if (p.top_n > 0) {
        // up to 32 or 64 different logits that the row reaches, of as many groups of warps or of the warps' largest threads; tau: the
        // n-th of them, the largest that n of them reach (counted by every lane for its own one or two: n rounds of taking the
        // largest, and bisection for a larger n, took longer, 421 x 248320 fp16 48.4 us, now 47.5).  With 32 groups an n of 32
        // would let in all that exceeds the least of them, some 130 logits and now and then 300: 16 rows of 15390 fp32 11.8 us, now 6.5.
        const int values = warps << k_shift;
        float* const reached = reinterpret_cast<float*>(sh.lists[warp]);
        float x = -INFINITY, y = -INFINITY;
        int nx = 0, ny = 0;
        if (many) {
            for (int i = lane; i < values; i += 64) {
                x = fmaxf(x, sh.reach[i]);
                y = fmaxf(y, sh.reach[i + 32]);
            }
            reached[lane + 32] = y;
        } else {
            for (int i = lane; i < values; i += 32) x = fmaxf(x, sh.reach[i]);
        }
        reached[lane] = x;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const float4 o = *reinterpret_cast<const float4*>(reached + i);
            nx += (o.x >= x) + (o.y >= x) + (o.z >= x) + (o.w >= x);
            if (many) ny += (o.x >= y) + (o.y >= y) + (o.z >= y) + (o.w >= y);
        }
        if (many) {
#pragma unroll
            for (int i = 32; i < 64; i += 4) {
                const float4 o = *reinterpret_cast<const float4*>(reached + i);
                nx += (o.x >= x) + (o.y >= x) + (o.z >= x) + (o.w >= x);
                ny += (o.x >= y) + (o.y >= y) + (o.z >= y) + (o.w >= y);
            }
        }
        __syncwarp();
        const float tau = redux_max(fmaxf(nx >= p.top_n ? x : -INFINITY, many && ny >= p.top_n ? y : -INFINITY));

        const int room = kKeys / ctas;
        const uint32_t keys0 = peer_addr(&sh.keys[cta * room], 0);
        auto flood = [&] { for (int i = 0; i < ctas; ++i) peer_store(peer_addr(&sh.flooded, i), 1u); };
        auto push = [&](float x, int i) {
            const unsigned n = atomicAdd(&sh.n_own, 1u);
            if (n < unsigned(room)) peer_store(keys0 + n * 8, order_key(x, i));
            else if (n == unsigned(room)) flood();
        };
        if (tau > -INFINITY) {
            const unsigned has = __ballot_sync(dq::kFull, m >= tau);
            const int n_cand = __popc(has);
            if (m >= tau) sh.cand[warp][__popc(has & ((1u << lane) - 1))] = first;
            __syncwarp();
            if (n_cand <= 16 || steps <= 1) {
                // in the steps in which the warp reached tau, eight threads' four vectors at a time
                for (unsigned in = __ballot_sync(dq::kFull, step_max >= tau); in; in &= in - 1)
                    for (int step = __ffs(in) - 1; step < steps; step += 32)
                        for (int c = lane >> 2; c < n_cand; c += 8) {
                            const int i = sh.cand[warp][c] + (step * U + (lane & 3)) * stride;
                            if (i >= nvec) continue;
                            V w;
                            if (steps <= 2) w.set(ring[((step & 1) * U + (lane & 3)) * kThreads + sh.cand[warp][c] - cta * kThreads]);   // still there
                            else w.load(vecs + i);
                            if (w.max_with(-INFINITY) >= tau) {
#pragma unroll
                                for (int e = 0; e < V::N; ++e)
                                    if (w.at(e) >= tau) push(w.at(e), head + i * V::N + e);
                            }
                        }
                if (single >= 0) {
                    const float y = value_at<F32>(row, single);
                    if (y >= tau) push(y, single);
                }
            } else if (lane == 0) flood();
            sync_all();
        }
        if (tau == -INFINITY || sh.flooded) {
            sorted_lists<F32, WARPS>(sh, row, vecs, head, nvec, first, stride, single, tau, p.top_n);
            for (int i = tid; i < room; i += kThreads) peer_store(keys0 + i * 8, i < p.top_n ? sh.lists[0][i] : 0ull);
            sync_all();
        }
    }
    // the next kernel on the stream comes now: at the start, its blocks took places that this one's later blocks wait for
    // (77 rows of 100003 fp32: 13.1 -> 10.2 us a call, 421 of 32003: 18.8 -> 16.1)
    pdl_trigger();
    if (cta != 0) return;

    // ---- the first CTA writes the row's answers: its last warp joins the parts, and all of them order the keys
    if (warp == WARPS - 1) {
        constexpr int N = kMaxCluster * WARPS / 32;
        Part parts[N];
        int rank = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int w = lane + 32 * i;
            parts[i] = w < warps ? Part{sh.m[w], sh.z[w], sh.t[w]} : Part{-INFINITY, 0.f, 0.f};
            if (RANK && w < warps) rank += sh.before[w];
        }
        const Part all = joined(parts, p.scale2);
        if (RANK) rank = __reduce_add_sync(dq::kFull, rank);
        const bool none = all.m == -INFINITY && all.z == 0.f;   // masked altogether
        const float lnz = log1pf(all.z);
        if (lane == 0) {
            sh.row_m = all.m;
            sh.row_lnz = lnz;
            sh.none = none;
            if (p.entropy) p.entropy[r] = none ? 0.f : lnz - __fdividef(all.t, 1.f + all.z) * kLn2;
            // the difference is taken before the scale: a row of the type's lowest value would overflow the product
            if (RANK && p.logprob) p.logprob[r] = !real ? 0.f : none ? -INFINITY : (least - all.m) * p.inv_temp - lnz;
            if (RANK && p.rank) p.rank[r] = real && token_key >> 32 ? rank : -1;
        }
    }
    if (p.top_n == 0) return;
    unsigned long long* list = &sh.lists[0][0];
    {
        constexpr int kMine = kKeys / kThreads;   // a thread's keys; one warp's lie together in the list, whatever their order
        unsigned long long key[kMine];
        unsigned has[kMine], count = 0, base = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            key[i] = sh.keys[tid + i * kThreads];
            has[i] = __ballot_sync(dq::kFull, key[i] != 0);
            count += __popc(has[i]);
        }
        if (count) {
            if (lane == 0) base = atomicAdd(&sh.n_keys, count);
            base = __shfl_sync(dq::kFull, base, 0);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                if (key[i] != 0) list[base + __popc(has[i] & ((1u << lane) - 1))] = key[i];
                base += __popc(has[i]);
            }
        }
    }
    __syncthreads();
    const int n_keys = int(sh.n_keys), quarter = tid & 3;
    for (int base = 0; base < n_keys; base += kThreads / 4) {   // four threads count the keys before one
        const int k = base + (tid >> 2);
        const unsigned long long key = k < n_keys ? list[k] : 0;
        int place = 0;
#pragma unroll 1
        for (int i = 4 * quarter; i < n_keys; i += 16) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(list + i), b = *reinterpret_cast<const ulonglong2*>(list + i + 2);
            place += (a.x > key) + (i + 1 < n_keys && a.y > key) + (i + 2 < n_keys && b.x > key) + (i + 3 < n_keys && b.y > key);
        }
        place += __shfl_xor_sync(dq::kFull, place, 1);
        place += __shfl_xor_sync(dq::kFull, place, 2);
        if (quarter == 0 && key != 0 && place < p.top_n) {
            p.top_idx[r * p.top_n + place] = int(0xffffffffu - unsigned(key));
            p.top_logprob[r * p.top_n + place] = sh.none ? -INFINITY : (key_value(key) - sh.row_m) * p.inv_temp - sh.row_lnz;
        }
    }
}

template <bool F32, bool RANK, int WARPS>
void launch(const LogprobParams& p, int ctas, cudaStream_t st)
{
    auto kern = k_logprobs<F32, RANK, WARPS>;
    static bool set[kMaxDevices] = {};
    const int dev = current_device();
    if (!set[dev]) {
        cuda_ok(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "logprobs cluster attribute");
        cuda_ok(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, WARPS * kRingBytes), "logprobs smem attribute");
        set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(p.rows) * unsigned(ctas));
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = WARPS * kRingBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(ctas);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cuda_ok(cudaLaunchKernelEx(&cfg, kern, p), "logprobs launch");
}
template <bool F32, bool RANK>
void launch(const LogprobParams& p, int ctas, int warps, cudaStream_t st)
{
    if (warps == 4) launch<F32, RANK, 4>(p, ctas, st);
    else if (warps == 8) launch<F32, RANK, 8>(p, ctas, st);
    else launch<F32, RANK, 16>(p, ctas, st);
}

// How a row is split: CTAs of its cluster and warps of each.  Measured (us, rows x vocabulary, warps/CTAs):
//   as many warps as run at once (4736, of which clusters fill nine tenths), a power of two of them a row, none with less than 1 KB:
//     37 x 187037 fp16 64 warps 7.6, 128 warps 11.3 (4736 of them); 64 x 248320 fp16 64 warps 14.8, 128 warps 21.2; 1 x 5000 fp32 16 warps
//     4.6, 64 warps 5.0; at most 128, above 16 rows 64: 16 x 248320 fp32 8/16 10.6, 16/16 14.6; 32 x 248320 fp32 8/8 12.8, 16/8 13.0;
//   a second wave where the first would leave a quarter of the GPU idle and the parts are long:
//     421 x 248320 fp16 16 warps 48, 8 warps 61; 150 x 250000 fp16 32 warps 26, 16 warps 35; 336 x 37714 fp32 8 warps 13.4, 16 warps 15.7;
//   small CTAs in clusters of up to 8, of 16 for 128 warps: 1 x 32000 fp16 4/8 5.0, 16/2 6.2; 13 x 21619 fp32 8/8 6.3, 4/16 7.2;
//     4 x 248320 fp32 8/16 7.4, 16/8 8.3; one CTA of 8 warps (1 x 2314 fp32 8/1 2.8, 4/2 3.2), and of 16 in a second wave (421 rows 16/1 48,
//     4/4 53; in a first one 160 x 38881 fp32 4/4 13.6, 16/1 16.2).
void row_split(int rows, long long row_bytes, int& ctas, int& warps)
{
    const long long at_once = 148 * 32, limit = rows <= 16 ? 128 : 64;
    long long n = 4;
    while (n < limit && 10 * rows * n * 2 <= 9 * at_once && row_bytes >= n * 2 * 1024) n *= 2;
    if (n < limit && 4 * rows * n <= 3 * at_once && row_bytes > n * 24576) n *= 2;
    if (n < limit && rows > 148 && row_bytes > n * 49152) n *= 2;
    const bool one_wave = 10 * rows * n <= 9 * at_once;
    ctas = n <= 8 || (n == 16 && !one_wave) ? 1 : n == 16 ? 4 : n == 128 ? 16 : 8;
    warps = int(n / ctas);
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
        check_aligned(logits, logits_fp32 ? 4 : 2, "logprobs: logits");
        for (const void* p : {(const void*) tokens, (const void*) logprob, (const void*) rank, (const void*) entropy, (const void*) top_idx, (const void*) top_logprob})
            check_aligned(p, 4, "logprobs: a tensor of 32-bit elements");
        if (rows > (1 << 26)) throw std::runtime_error("logprobs: rows must be at most 2^26");
        const LogprobParams p{logits, row_stride, tokens, logprob, rank, entropy, top_idx, top_logprob, top_n, rows, vocab, inv_temp, inv_temp * kLog2e};
        const bool f32 = logits_fp32 != 0, ranks = logprob || rank;
        int ctas, warps;
        row_split(rows, (long long) vocab * (f32 ? 4 : 2), ctas, warps);
        cudaStream_t cs = (cudaStream_t) stream;
        if (f32) ranks ? launch<true, true>(p, ctas, warps, cs) : launch<true, false>(p, ctas, warps, cs);
        else ranks ? launch<false, true>(p, ctas, warps, cs) : launch<false, false>(p, ctas, warps, cs);
        st.launch = describe("k_logprobs<", f32 ? "float" : "half", ranks ? ",rank" : "", "> block=", warps * 32, " grid=", rows, "x", ctas, " cluster=", ctas);
    });
}

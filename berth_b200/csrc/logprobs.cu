// Log probabilities of given tokens, entropy and the best alternatives of every row of logits, in one pass over them.
//
// A row is split over the CTAs of a cluster.  Every thread walks its 16-byte vectors with a running maximum M and the sums
// z = sum 2^y and t = sum 2^y y, y = (x - M) * inv_temp * log2 e: ln p = (x - m) * inv_temp - ln z and the entropy
// ln z - t / z * ln 2 follow from the joined (m, z, t).  Both sums grow in 64 bits from sums of 32 elements that are added
// as a tree in 32: a certain row has z = 1 + little, and its entropy is made of that little.  The rank of a given token is a
// count of the logits before it, taken in the same walk.
//
// The n best come out of the walk's by-product, the threads' maxima.  The cluster's warps fall into at least n groups; the
// smallest of the groups' maxima is a value that n logits reach, and few more do, all of them in threads whose maximum
// reaches it.  Only those threads' vectors are read again (from L2, a few percent of the row), what reaches the value goes to
// the first CTA's shared memory, and each finds its place by counting the larger ones.  Rows where too many reach it (equal
// logits, a mask that leaves fewer than n) are scanned once more with a sorted list of 32 per warp instead.
#include "exl3_decode.cuh"
#include "../../include/berth_b200.h"

#include <algorithm>
#include <cmath>

namespace berth {
namespace {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
constexpr int kMaxTop = 32, kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 16, kKeys = 512;
static_assert(kMaxCluster * kMaxTop <= kKeys, "the lists of a cluster share the key buffer");

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
__device__ __forceinline__ unsigned peer_add(uint32_t a, unsigned v)
{
    unsigned r;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(a), "r"(v) : "memory");
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Running maximum and sums of a part of a row.
struct Part {
    float m;       // -inf: no logit above it yet
    double z, t;
};
// p brought to the maximum m >= p.m.  A part without a maximum has z = 0 (or NaN, which stays).
__device__ __forceinline__ Part brought_to(Part p, float m, float scale2)
{
    if (p.m > -INFINITY) {
        const float d = (p.m - m) * scale2;
        const double f = ex2(d);
        p.t = f > 0.0 ? (p.t + double(d) * p.z) * f : p.z * f;   // (a factor that vanished leaves 0, or NaN)
        p.z *= f;
    }
    p.m = m;
    return p;
}
template <int LANES>
__device__ __forceinline__ Part joined(Part p, float scale2)   // over groups of LANES lanes
{
    float m = p.m;
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(dq::kFull, m, off));
    p = brought_to(p, m, scale2);
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) {
        p.z += __shfl_xor_sync(dq::kFull, p.z, off);
        p.t += __shfl_xor_sync(dq::kFull, p.t, off);
    }
    return p;
}

// 16 bytes of a row: 8 fp16 or 4 fp32.
template <bool F32> struct Vec;
template <> struct Vec<true> {
    static constexpr int N = 4;
    float x[4];
    __device__ __forceinline__ void load(const uint4* a)
    {
        const uint4 v = __ldcg(a);
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    __device__ __forceinline__ f2 pair(int i) const { return pack2(x[2 * i], x[2 * i + 1]); }
    __device__ __forceinline__ float at(int i) const { return x[i]; }
    __device__ __forceinline__ float max_with(float m) const { return fmaxf(fmaxf(m, fmaxf(x[0], x[1])), fmaxf(x[2], x[3])); }
};
template <> struct Vec<false> {
    static constexpr int N = 8;
    __half2 h[4];
    __device__ __forceinline__ void load(const uint4* a)
    {
        const uint4 v = __ldcg(a);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const __half2*>(&w[i]);
    }
    __device__ __forceinline__ f2 pair(int i) const { const float2 v = __half22float2(h[i]); return pack2(v.x, v.y); }
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

struct Shared {
    unsigned long long keys[kKeys];             // first CTA: keys that reach the threshold, or the CTAs' lists
    unsigned long long lists[kWarps][32];
    Part parts[kWarps], of_cta[kMaxCluster];
    float max1[kMaxCluster * kWarps];           // of every warp of the cluster
    float max2[kWarps];                         // second largest thread of this CTA's warps
    int before[kWarps], before_cta[kMaxCluster];
    int cand[kThreads];
    unsigned n_keys, n_cand, flooded;
};

// U vectors of a thread in flight.  The walk takes 32 logits at a time of either type.
template <bool F32, bool RANK>
__global__ void __launch_bounds__(kThreads, 2) k_logprobs(const LogprobParams p)
{
    using V = Vec<F32>;
    using E = typename std::conditional<F32, float, __half>::type;
    constexpr int U = 32 / V::N;
    __shared__ Shared sh;
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int cta, ctas;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    if (tid == 0) sh.n_keys = sh.n_cand = sh.flooded = 0;
    if (ctas > 1) cluster_arrive();             // every CTA has started, and cleared its counters, when the wait below ends
    pdl_wait();

    const size_t r = blockIdx.x / ctas;
    const char* row = static_cast<const char*>(p.logits) + r * p.ld * sizeof(E);
    // the row as `head` single logits up to a 16-byte boundary, full vectors, and `tail` single logits
    const int head = min(int(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(E)), p.vocab);
    const int nvec = (p.vocab - head) / V::N, tail = p.vocab - head - nvec * V::N;
    const uint4* vecs = reinterpret_cast<const uint4*>(row + head * sizeof(E));
    const int v0 = int((long long) nvec * cta / ctas), v1 = int((long long) nvec * (cta + 1) / ctas);

    int token = -1, before = 0, token_vec = 0;
    bool real = false;
    unsigned long long token_key = 0;
    E at{}, over{};
    if (RANK) {
        token = p.tokens[r];
        real = token >= 0 && token < p.vocab;
        if (real) {
            at = reinterpret_cast<const E*>(row)[token];
            over = above(at);
            token_key = order_key(F32 ? float(at) : __half2float(at), token);
            token_vec = token < head ? -1 : (token - head) / V::N;
        }
    }

    // the first CTA's threads 0..head-1 and 16..16+tail-1 begin with a single logit
    Part own{-INFINITY, 0.0, 0.0};
    int single = -1;
    if (cta == 0) {
        if (tid < head) single = tid;
        else if (tid >= 16 && tid < 16 + tail) single = p.vocab - tail + tid - 16;
    }
    if (single >= 0) {
        const float x = value_at<F32>(row, single);
        own.m = x != x ? -INFINITY : x;
        own.z = x != x ? NAN : (x > -INFINITY ? 1.0 : 0.0);
        if (RANK) before += order_key(x, single) > token_key;
    }
    // equal logits before the token in its own vector (the walk counts the larger ones there)
    if (RANK && real && cta == 0 && tid >= 32 && tid < 32 + V::N && token_vec >= 0) {
        const int i = head + token_vec * V::N + tid - 32;
        if (i < token && token_vec < nvec) before += value_at<F32>(row, i) == key_value(token_key);
    }

    for (int base = v0 + tid; base < v1; base += kThreads * U) {
        V v[U];
        float g = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * kThreads;
            if (i < v1) v[u].load(vecs + i);
            else {   // adds nothing: below every threshold but that of a masked token, which is taken back
                uint4 none = F32 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u) : make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
                memcpy(&v[u], &none, 16);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) g = v[u].max_with(g);
        if (g > own.m) own = brought_to(own, g, p.scale2);
        const float ref = own.m > -INFINITY ? own.m : 0.f;
        const f2 nref = pack2(-ref, -ref), sc = pack2(p.scale2, p.scale2);
        f2 z[U], t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f2 e[V::N / 2];
#pragma unroll
            for (int i = 0; i < V::N / 2; ++i) {
                const f2 y2 = mul2(add2(v[u].pair(i), nref), sc);
                float a, b;
                unpack2(y2, a, b);
                a = a < -200.f ? -200.f : a;      // a masked logit: 2^y is 0 either way, 0 * -inf is not (NaN stays)
                b = b < -200.f ? -200.f : b;
                e[i] = pack2(ex2(a), ex2(b));
                t[u] = i == 0 ? mul2(e[i], pack2(a, b)) : fma2(e[i], pack2(a, b), t[u]);
            }
            z[u] = add2(e[0], e[1]);
            if constexpr (V::N == 8) z[u] = add2(z[u], add2(e[2], e[3]));
        }
#pragma unroll
        for (int w = U / 2; w >= 1; w >>= 1)
#pragma unroll
            for (int u = 0; u < w; ++u) { z[u] = add2(z[u], z[u + w]); t[u] = add2(t[u], t[u + w]); }
        float za, zb, ta, tb;
        unpack2(z[0], za, zb);
        unpack2(t[0], ta, tb);
        own.z += double(za) + double(zb);
        own.t += double(ta) + double(tb);
        if (RANK && real) {
            E thr[U];
#pragma unroll
            for (int u = 0; u < U; ++u) thr[u] = base + u * kThreads < token_vec ? at : over;
            before += count_ge(v, thr);
            if (token_key >> 32 == 0x007fffffu)   // a masked token: the vectors behind the end counted as equal
                for (int u = 0; u < U; ++u)
                    if (base + u * kThreads >= v1 && base + u * kThreads < token_vec) before -= V::N;
        }
    }

    // ---- join: warps, CTA, cluster
    const float mine = own.m;
    Part part = joined<32>(own, p.scale2);
    if (RANK) before = __reduce_add_sync(dq::kFull, before);
    if (p.top_n > kWarps && ctas == 1) {
        const unsigned first = __ffs(__ballot_sync(dq::kFull, mine == part.m)) - 1;   // (a warp without a maximum: -inf == -inf)
        float other = lane == int(first) ? -INFINITY : mine;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) other = fmaxf(other, __shfl_xor_sync(dq::kFull, other, off));
        if (lane == 0) sh.max2[warp] = other;
    }
    if (lane == 0) {
        sh.parts[warp] = part;
        sh.before[warp] = before;
        if (ctas == 1) sh.max1[warp] = part.m;
    }
    if (ctas > 1) cluster_wait();
    __syncthreads();
    if (ctas > 1 && p.top_n > 0 && tid < ctas * kWarps)
        peer_store(peer_addr(&sh.max1[cta * kWarps + (tid & (kWarps - 1))], tid / kWarps), __float_as_uint(sh.parts[tid & (kWarps - 1)].m));
    if (warp == 0) {
        part = lane < kWarps ? sh.parts[lane] : Part{-INFINITY, 0.0, 0.0};
        part = joined<32>(part, p.scale2);
        const int b = RANK ? __reduce_add_sync(dq::kFull, lane < kWarps ? sh.before[lane] : 0) : 0;
        if (ctas == 1) {
            if (lane == 0) { sh.of_cta[0] = part; sh.before_cta[0] = b; }
        } else if (lane == 0) {
            peer_store(peer_addr(&sh.of_cta[cta].m, 0), __float_as_uint(part.m));
            peer_store(peer_addr(&sh.of_cta[cta].z, 0), (unsigned long long) __double_as_longlong(part.z));
            peer_store(peer_addr(&sh.of_cta[cta].t, 0), (unsigned long long) __double_as_longlong(part.t));
            peer_store(peer_addr(&sh.before_cta[cta], 0), unsigned(b));
        }
    }
    if (ctas > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();

    // ---- the candidates for the n best
    if (p.top_n > 0) {
        // at least n groups of warps; tau = the smallest of their maxima
        int groups = 1;
        while (groups < p.top_n) groups <<= 1;
        const int warps = ctas * kWarps;
        float tau = -INFINITY;
        if (groups <= warps) {
            for (int i = lane; i < warps; i += 32) tau = fmaxf(tau, sh.max1[i]);
            if (warps < 32) tau = __shfl_sync(dq::kFull, tau, lane & (kWarps - 1));   // one CTA: 16 warps
            for (int off = groups; off < 32; off <<= 1) tau = fmaxf(tau, __shfl_xor_sync(dq::kFull, tau, off));
        } else {
            tau = sh.max2[lane & (kWarps - 1)];   // one CTA, n > 16: two threads of every warp
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) tau = fminf(tau, __shfl_xor_sync(dq::kFull, tau, off));

        const int per_thread = (v1 - v0 + kThreads - 1) / kThreads;
        const uint32_t keys0 = ctas > 1 ? peer_addr(sh.keys, 0) : smem_addr(sh.keys), n0 = ctas > 1 ? peer_addr(&sh.n_keys, 0) : smem_addr(&sh.n_keys);
        auto push = [&](float x, int i) {
            const unsigned at_key = peer_add(n0, 1u);
            if (at_key < unsigned(kKeys)) peer_store(keys0 + at_key * 8, order_key(x, i));
            else sh.flooded = 1;
        };
        if (tau > -INFINITY) {
            const unsigned has = __ballot_sync(dq::kFull, mine >= tau);
            unsigned at_cand = 0;
            if (lane == 0 && has) at_cand = atomicAdd(&sh.n_cand, __popc(has));
            at_cand = __shfl_sync(dq::kFull, at_cand, 0) + __popc(has & ((1u << lane) - 1));
            if (mine >= tau) sh.cand[at_cand] = tid;
            if (single >= 0) {
                const float x = value_at<F32>(row, single);
                if (x >= tau) push(x, single);
            }
            __syncthreads();
            const int n_cand = int(sh.n_cand);
            if (n_cand <= kThreads / 2) {
                for (int k = tid; k < n_cand * per_thread; k += kThreads) {
                    const int i = v0 + sh.cand[k / per_thread] + (k % per_thread) * kThreads;
                    if (i < v1) {
                        V v;
                        v.load(vecs + i);
                        if (v.max_with(-INFINITY) >= tau) {
#pragma unroll
                            for (int e = 0; e < V::N; ++e)
                                if (v.at(e) >= tau) push(v.at(e), head + i * V::N + e);
                        }
                    }
                }
            } else if (tid == 0) sh.flooded = 1;
            __syncthreads();
            if (ctas > 1) {
                if (tid < ctas && sh.flooded) peer_store(peer_addr(&sh.flooded, tid), 1u);
                cluster_arrive();
                cluster_wait();
            }
        }
        if (tau == -INFINITY || sh.flooded) {
            // the whole part again, 32 sorted keys a warp
            unsigned long long list = 0;
            offer_keys(list, single >= 0 ? order_key(value_at<F32>(row, single), single) : 0, p.top_n);
            for (int base = v0 + warp * 32; base < v1; base += kThreads) {
                const int i = base + lane;
                V v;
                if (i < v1) v.load(vecs + i);
#pragma unroll
                for (int e = 0; e < V::N; ++e) offer_keys(list, i < v1 && !(v.at(e) < tau) ? order_key(v.at(e), head + i * V::N + e) : 0, p.top_n);
            }
            sh.lists[warp][lane] = list;
            for (int w = kWarps / 2; w >= 1; w >>= 1) {
                __syncthreads();
                if (warp < w) {
                    list = merge_lists(list, sh.lists[warp + w][lane]);
                    sh.lists[warp][lane] = list;
                }
            }
            if (warp == 0) {
                if (lane < p.top_n) peer_store(keys0 + (cta * p.top_n + lane) * 8, list);
                if (cta == 0 && lane == 0) sh.n_keys = ctas * p.top_n;
            }
            if (ctas > 1) { cluster_arrive(); cluster_wait(); }
            else __syncthreads();
        }
    }
    if (cta != 0) return;

    // ---- the first CTA writes the row's answers
    part = joined<32>(lane < ctas ? sh.of_cta[lane] : Part{-INFINITY, 0.0, 0.0}, p.scale2);
    const bool none = part.m == -INFINITY && part.z == 0.0;   // masked altogether
    const float m = part.m, lnz = log1pf(float(part.z - 1.0));
    // the difference is taken before the scale: a row of the type's lowest value would overflow the product
    auto logprob_of = [&](float x) { return none ? -INFINITY : (x - m) * p.inv_temp - lnz; };
    if (warp == 0) {
        const int rank = RANK ? __reduce_add_sync(dq::kFull, lane < ctas ? sh.before_cta[lane] : 0) : 0;
        if (lane == 0) {
            if (RANK && p.logprob) p.logprob[r] = real ? logprob_of(key_value(token_key)) : 0.f;
            if (RANK && p.rank) p.rank[r] = real && token_key >> 32 ? rank : -1;
            if (p.entropy) p.entropy[r] = none ? 0.f : lnz - float(part.t / part.z) * kLn2;
        }
    }
    const int n_keys = p.top_n > 0 ? int(sh.n_keys) : 0;
    if (tid < n_keys) {
        const unsigned long long key = sh.keys[tid];
        int place = 0;
        for (int i = 0; i < n_keys; ++i) place += sh.keys[i] > key;
        if (place < p.top_n && key != 0) {
            p.top_idx[r * p.top_n + place] = int(0xffffffffu - unsigned(key));
            p.top_logprob[r * p.top_n + place] = logprob_of(key_value(key));
        }
    }
}

template <bool F32, bool RANK>
void launch(const LogprobParams& p, int ctas, cudaStream_t st)
{
    auto kern = k_logprobs<F32, RANK>;
    static bool set[kMaxDevices] = {};
    const int dev = current_device();
    if (!set[dev]) {
        cuda_ok(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "logprobs cluster attribute");
        set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(p.rows) * unsigned(ctas));
    cfg.blockDim = dim3(kThreads);
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

// CTAs a row is split over.
int row_ctas(int rows, long long row_bytes)
{
    int best = 1;
    double least = 0.0;
    for (int s = 1; s <= kMaxCluster; s *= 2) {
        const long long slots = 296 / s;                       // clusters that run at once (two CTAs an SM)
        const long long waves = (rows + slots - 1) / slots;
        const double t = double(waves) * (3.0 + double(row_bytes) / s / 22e3);   // us: fixed part, then some 22 GB/s... a CTA's share
        if (s == 1 || t < least) { best = s; least = t; }
    }
    return best;
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
        if (rows > (1 << 26)) throw std::runtime_error("logprobs: rows must be at most 2^26");
        const LogprobParams p{logits, row_stride, tokens, logprob, rank, entropy, top_idx, top_logprob, top_n, rows, vocab, inv_temp, inv_temp * kLog2e};
        const bool f32 = logits_fp32 != 0, ranks = logprob || rank;
        const int ctas = row_ctas(rows, (long long) vocab * (f32 ? 4 : 2));
        cudaStream_t cs = (cudaStream_t) stream;
        if (f32) ranks ? launch<true, true>(p, ctas, cs) : launch<true, false>(p, ctas, cs);
        else ranks ? launch<false, true>(p, ctas, cs) : launch<false, false>(p, ctas, cs);
        st.launch = std::string("k_logprobs<") + (f32 ? "float" : "half") + (ranks ? ",rank" : "") + "> block=" + std::to_string(kThreads) + " grid=" +
                    std::to_string(rows) + "x" + std::to_string(ctas) + " cluster=" + std::to_string(ctas);
    });
}

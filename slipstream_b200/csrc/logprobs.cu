// Log probabilities of given tokens, their ranks, the entropy and the largest log probabilities of rows of logits:
//   m = max z, S = sum exp(z - m), T = sum exp(z - m) (z - m);   log p(t) = z_t - m - log S;   entropy = log S - T / S
//   rank = 1 + #{z_j > z_t} + #{j < t : z_j = z_t};   the k largest by (z, lower index first)
//
// One pass over a row: every thread keeps the largest value of its vectors, and S, T relative to it (rescaled when it rises), and counts
// what stands in front of the token.  Masked tokens (z = -inf) add nothing.  The sums of the threads are joined in 64 bits.
//
// The k largest come out of the same pass: a thread knows its largest element.  The k-th largest of the largest elements of 64 or 128
// groups of threads is a bound that at least k elements of the row reach, and hardly more do (24 for k = 20).  Only
// the threads whose largest element reaches it can hold such elements, and only their vectors are looked at again.  Elements are compared
// as (value, index), so no two are equal and ties need no rule of their own; where the values stand so that too many reach the bound,
// the k largest are taken one after the other among the same threads' vectors.
//
// Bound by memory: a row is read once (and about 5 % of it again for k = 20).  A row has a block of 512 threads, or, where rows are few, a
// thread-block cluster of up to 8, which put their results together through shared memory.  A thread's S and T are float32, so beside a
// token that is nearly certain the entropy, a small number, is off by about 1e-7 absolute.
// 1,024 rows of 151,936 in float32: 109 us (5.7 TB/s) without alternatives, 134 with 20 (a block loads nothing while
// it chooses them; the issue slots are 59 % busy); in bfloat16 101 us with 20 for 48 of bytes, bound by the instructions: an exponential,
// four multiply-adds and two comparisons an element.  One row 5.7 us, with 5 alternatives 8.5: launch, the pass of 8 blocks, the join, the choice.

#include "common.cuh"
#include "logprob_calls.h"

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, GROUPS = THREADS / 4, FEW_GROUPS = THREADS / 8, CANDIDATES = 512;
typedef unsigned long long Key;  // value in the upper half, in an order of unsigned integers; the complement of the index below; 0: none

__device__ __forceinline__ Key key_of(float z, int index) {  // z is no NaN
    const uint32_t bits = __float_as_uint(z + 0.f);  // (both zeros are one)
    const uint32_t order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return (Key)order << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t order = (uint32_t)(k >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ int index_of(Key k) { return (int)~(uint32_t)k; }

// The next float32 above z, for z >= up: z > z0; of infinity and NaN NaN, which nothing reaches.
__device__ __forceinline__ float next_above(float z) {
    if (!(z < __uint_as_float(0x7f800000u))) return __uint_as_float(0x7fffffffu);
    const uint32_t bits = __float_as_uint(z + 0.f);
    return __uint_as_float(bits & 0x80000000u ? bits - 1 : bits + 1);
}

// exp(d) for -200 <= d <= 0, as 2^u with u = d log2 e rounded; what was lost, d - u ln 2, comes in behind: p (1 + (d - u ln 2)).
// Without that p is off by up to half a unit of u, 3e-7 at d = -10; so by what ex2.approx is, about 1e-7.  Results below 2^-126 are 0.
constexpr float LOG2_E = 1.442695041f, LN_2 = 0.6931471806f;
__device__ __forceinline__ float exp_of(float d) {
    float p;
    const float u = d * LOG2_E;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(u));
    return fmaf(p, fmaf(u, -LN_2, d), p);
}
// max(d, -200), which keeps a NaN: what is masked counts nothing, and products with it are no NaN.
__device__ __forceinline__ float bounded(float d) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(d), "f"(-200.f));
    return r;
}

template <typename T>
struct Vec {
    static constexpr int G = 16 / (int)sizeof(T);
    static constexpr uint32_t NONE = G == 4 ? 0xff800000u : 0xff80ff80u;  // -inf
    uint4 raw;
    __device__ __forceinline__ float at(int e) const {
        const uint32_t w = G == 4 ? (e == 0 ? raw.x : e == 1 ? raw.y : e == 2 ? raw.z : raw.w)
                                  : (e < 2 ? raw.x : e < 4 ? raw.y : e < 6 ? raw.z : raw.w);
        return G == 4 ? __uint_as_float(w) : __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
    // the largest element that is a number (NaN: none is); of bfloat16 pairs at a time
    __device__ __forceinline__ float largest() const {
        if constexpr (G == 4) {
            return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3)));
        } else {
            const auto pair = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
            const __nv_bfloat162 m = __hmax2(__hmax2(pair(raw.x), pair(raw.y)), __hmax2(pair(raw.z), pair(raw.w)));
            return fmaxf(__low2float(m), __high2float(m));
        }
    }
    // how many elements reach z (which is a T), or exceed it; above: next_above(z)
    __device__ __forceinline__ int reaching(float z, float above, bool exceed) const {
        if constexpr (G == 4) {
            const float limit = exceed ? above : z;
            return (at(0) >= limit) + (at(1) >= limit) + (at(2) >= limit) + (at(3) >= limit);
        } else {
            const auto pair = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
            const __nv_bfloat162 limit = __float2bfloat162_rn(z);
            const auto count = [&](const uint32_t& w) { return exceed ? __hgt2(pair(w), limit) : __hge2(pair(w), limit); };
            const __nv_bfloat162 n = __hadd2(__hadd2(count(raw.x), count(raw.y)), __hadd2(count(raw.z), count(raw.w)));  // (exact: up to 4)
            return (int)(__low2float(n) + __high2float(n));
        }
    }
};

// A row as the block sees it: elements in front of the first whole 16 bytes and behind the last (one a thread, of the first and of the
// last block), and vectors between them, first .. end - 1 of them the block's.
template <typename T>
struct Row {
    const T* z;
    int head, tail_from, vocabulary;  // elements 0 .. head - 1; tail_from .. vocabulary - 1
    int first, end;
    bool has_head, has_tail;
    __device__ __forceinline__ const Vec<T>* vectors() const { return reinterpret_cast<const Vec<T>*>(z + head); }
    __device__ __forceinline__ int index(int v, int e) const { return head + v * Vec<T>::G + e; }
    // f(index, value) of all elements of thread t, dealt out over the lanes of a warp
    template <typename F>
    __device__ __forceinline__ void each_of_thread(int t, int lane, F f) const {
        if (lane == 0) {
            if (has_head && t < head) f(t, to_float(z[t]));
            if (has_tail && tail_from + t < vocabulary) f(tail_from + t, to_float(z[tail_from + t]));
        }
        for (int v = first + t + lane * THREADS; v < end; v += 32 * THREADS) {
            const Vec<T> x = vectors()[v];
#pragma unroll
            for (int e = 0; e < Vec<T>::G; ++e) f(index(v, e), x.at(e));
        }
    }
};

// What a thread has seen: the largest value, where it stands, sums relative to it, and how many elements stand in front of the token.
struct Seen {
    float m, s, t;
    int at;  // the first element of the vectors (or the element of the head or tail) among which it is; -1: nothing yet
    int ahead;
};
constexpr int NOTHING = -1;

__device__ __forceinline__ void raise_to(Seen& a, float m, int at) {
    if (m > a.m || (a.at == NOTHING && m == m)) {
        if (a.s > 0.f) {
            const float d = bounded(a.m - m), f = exp_of(d);
            a.t = f * fmaf(a.s, d, a.t);
            a.s *= f;
        }
        a.m = m;
        a.at = at;
    }
}
__device__ __forceinline__ void add(Seen& a, float z, float m) {
    const float d = bounded(z - m), p = exp_of(d);
    a.s += p;
    a.t = fmaf(p, d, a.t);
}
// The same for pairs: two sums each, an instruction for two elements but for the exponentials.
struct Sums {
    unsigned long long s, t;
};
__device__ __forceinline__ unsigned long long two(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float sum_of(unsigned long long v) {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    return a + b;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void add2(Sums& a, float z0, float z1, unsigned long long minus_m) {
    unsigned long long d;
    float d0, d1, u0, u1, p0, p1;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(two(z0, z1)), "l"(minus_m));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d0), "=f"(d1) : "l"(d));
    d = two(bounded(d0), bounded(d1));
    const unsigned long long u = mul2(d, two(LOG2_E, LOG2_E));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(u0), "=f"(u1) : "l"(u));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p0) : "f"(u0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p1) : "f"(u1));
    const unsigned long long p = two(p0, p1), q = fma2(p, fma2(u, two(-LN_2, -LN_2), d), p);
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.s) : "l"(q));
    a.t = fma2(q, d, a.t);
}
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

struct Part {  // of a block
    double s, t;
    float m;
    int ahead;
};

template <bool TOP>
struct alignas(16) Shared {  // (every array starts on 16 bytes)
    Key groups[TOP ? GROUPS : 2];
    Key found[TOP ? CANDIDATES : 2];
    Key best[TOP ? LOGPROBS_MAX_TOP : 2];  // the block's largest, in order
    Key warp_best[WARPS];
    double sums[2][WARPS];
    Part part;
    Key bound;
    float tops[WARPS];
    int counts[WARPS], chosen[TOP ? THREADS : 4];
    int n_found, n_chosen;
};

// How many of 2 * pairs keys (on 16 bytes, in shared memory) are above `own`: two a read, the same ones for all threads of a warp.
__device__ __forceinline__ int keys_above(const Key* keys, int pairs, Key own) {
    int n = 0;
#pragma unroll 8
    for (int j = 0; j < pairs; ++j) {
        const ulonglong2 k = reinterpret_cast<const ulonglong2*>(keys)[j];
        n += (k.x > own) + (k.y > own);
    }
    return n;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(THREADS, 3)
token_logprobs_kernel(const T* logits, int64_t stride, const void* tokens, int wide, float* __restrict__ out, int vocabulary, int top, int blocks, int* err) {
    constexpr int G = Vec<T>::G, UNROLL = 16 / G;  // vectors on their way: 16 elements
    __shared__ Shared<TOP> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / blocks;
    const int rank = (int)(blockIdx.x - r * blocks);
    pdl_launch_dependents();
    pdl_wait();

    const int64_t given = wide ? ((const int64_t*)tokens)[r] : (int64_t)((const int*)tokens)[r];
    const bool there = given >= 0 && given < vocabulary;
    if (given >= vocabulary && rank == 0 && tid == 0) atomicOr(err, SS_ERR_TOKEN_RANGE);
    const int token = there ? (int)given : -1;

    Row<T> row;
    row.z = logits + r * stride;
    row.vocabulary = vocabulary;
    row.head = min(vocabulary, (int)((16 - ((uintptr_t)row.z & 15)) & 15) / (int)sizeof(T));
    const int n_vec = (vocabulary - row.head) / G, per = (n_vec + blocks - 1) / blocks;
    row.tail_from = row.head + n_vec * G;
    row.first = min(n_vec, rank * per);
    row.end = min(n_vec, row.first + per);
    row.has_head = rank == 0;
    row.has_tail = rank == blocks - 1;

    // all that does not wait for the token is on its way first: a thread's element of the head and of the tail, and its first vectors
    Vec<T> x[UNROLL];
    const auto fetch = [&](int v) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            x[u].raw = make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);
            if (v + u * THREADS < row.end) x[u] = row.vectors()[v + u * THREADS];
        }
    };
    int v = row.first + tid;
    fetch(v);
    const bool in_head = row.has_head && tid < row.head, in_tail = row.has_tail && row.tail_from + tid < vocabulary;
    const float head = in_head ? to_float(row.z[tid]) : 0.f, tail = in_tail ? to_float(row.z[row.tail_from + tid]) : 0.f;
    const float z_token = there ? to_float(row.z[token]) : __uint_as_float(0x7fffffffu);
    const float above = next_above(z_token);
    Seen a = {-INFINITY, 0.f, 0.f, NOTHING, 0};
    const auto one = [&](float z, int i) {
        raise_to(a, z, i);
        add(a, z, reference(a.m));
        a.ahead += z >= (i < token ? z_token : above);
    };
    if (in_head) one(head, tid);
    // vectors: in front of the token equal values count, from its own vector on (whose elements in front of it are looked at below) they do
    // not; a vector behind the block's last is all -inf and counts nothing
    while (v < row.end) {
        float m = x[0].largest();
#pragma unroll
        for (int u = 1; u < UNROLL; ++u) m = fmaxf(m, x[u].largest());
        raise_to(a, m, row.index(v, 0));
        const float ref = reference(a.m);
        const unsigned long long minus = two(-ref, -ref);
        Sums sums = {0, 0};
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int e = 0; e < G; e += 2) add2(sums, x[u].at(e), x[u].at(e + 1), minus);
        a.s += sum_of(sums.s);
        a.t += sum_of(sums.t);
        if (m >= z_token) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                if (v + u * THREADS < row.end) a.ahead += x[u].reaching(z_token, above, row.index(v + u * THREADS, G - 1) >= token);
        }
        v += UNROLL * THREADS;
        fetch(v);
    }
    if (in_tail) one(tail, row.tail_from + tid);
    if (token >= row.head && token < row.tail_from && tid < (token - row.head) % G && row.first <= (token - row.head) / G && (token - row.head) / G < row.end)
        a.ahead += to_float(row.z[token - 1 - tid]) == z_token;

    // the block's sums
    const float warp_m = warp_max(a.m);
    if (lane == 0) sh.tops[warp] = warp_m;
    if (tid == 0) sh.n_found = sh.n_chosen = 0;
    __syncthreads();
    const float block_m = warp_max(lane < WARPS ? sh.tops[lane] : -INFINITY);
    {
        const float d = bounded(a.m - block_m), f = a.m == -INFINITY ? 0.f : exp_of(d);
        double s = (double)(a.s * f), t = a.m == -INFINITY ? s : (double)(f * fmaf(a.s, d, a.t));
        int n = a.ahead;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
            n += __shfl_xor_sync(0xffffffffu, n, o);
        }
        if (lane == 0) { sh.sums[0][warp] = s; sh.sums[1][warp] = t; sh.counts[warp] = n; }
    }

    if constexpr (TOP) {
        // where its largest element stands a thread knows but for its last vectors: what it brings to the bound stands at their last
        // element, so that its own is not behind, and it is chosen as if its own stood at their first
        Key mine = 0, least = 0;
        if (a.at != NOTHING) {
            const bool single = a.at < row.head || a.at >= row.tail_from;
            mine = key_of(a.m, a.at);
            least = key_of(a.m, single ? a.at : a.at + (UNROLL - 1) * THREADS * G + G - 1);  // (which may be none of the row's: it is only a bound)
        }
        const int groups = top <= FEW_GROUPS * 3 / 8 ? FEW_GROUPS : GROUPS, per_group = THREADS / groups;
        Key group = max(least, __shfl_xor_sync(0xffffffffu, least, 1));
        group = max(group, __shfl_xor_sync(0xffffffffu, group, 2));
        if (per_group == 8) group = max(group, __shfl_xor_sync(0xffffffffu, group, 4));
        if (lane % per_group == 0) sh.groups[tid / per_group] = group;
        if (tid == 0) sh.bound = 0;  // fewer than `top` groups have elements: all of them count
        __syncthreads();
        // the place of each group's largest element among them
        if (tid < groups) {
            const Key own = sh.groups[tid];
            if (own && keys_above(sh.groups, groups / 2, own) == top - 1) sh.bound = own;
        }
        __syncthreads();
        const Key limit = sh.bound;
        if (mine && mine >= limit) sh.chosen[atomicAdd(&sh.n_chosen, 1)] = tid;
        __syncthreads();
        const int threads = sh.n_chosen;
        const auto consider = [&](int index, float z) {
            if (z == z) {
                const Key k = key_of(z, index);
                if (k >= limit) {
                    const int at = atomicAdd(&sh.n_found, 1);
                    if (at < CANDIDATES) sh.found[at] = k;
                }
            }
        };
        // the chosen threads' vectors, dealt out to all threads, several on their way at a time
        {
            const int each = (row.end - row.first + THREADS - 1) / THREADS, all = threads * each;
            for (int i = tid; i < all; i += UNROLL * THREADS) {
                Vec<T> x[UNROLL];
                int at[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const int f = i + u * THREADS, owner = f / each;
                    at[u] = f < all ? row.first + sh.chosen[owner] + (f - owner * each) * THREADS : row.end;
                    if (at[u] < row.end) x[u] = row.vectors()[at[u]];
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u)
                    if (at[u] < row.end) {
#pragma unroll
                        for (int e = 0; e < G; ++e) consider(row.index(at[u], e), x[u].at(e));
                    }
            }
            for (int i = tid; i < threads; i += THREADS) {
                const int t = sh.chosen[i];
                if (row.has_head && t < row.head) consider(t, to_float(row.z[t]));
                if (row.has_tail && row.tail_from + t < vocabulary) consider(row.tail_from + t, to_float(row.z[row.tail_from + t]));
            }
        }
        __syncthreads();
        const int n = sh.n_found;
        if (tid < top) sh.best[tid] = 0;
        if (n <= CANDIDATES) {
            if (tid == 0 && n % 2) sh.found[n] = 0;  // (CANDIDATES is even: there is room)
            __syncthreads();
            if (tid < n) {
                const Key own = sh.found[tid];
                const int place = keys_above(sh.found, (n + 1) / 2, own);
                if (place < top) sh.best[place] = own;
            }
        } else {
            Key below = ~(Key)0;
            for (int j = 0; j < top; ++j) {
                Key k = 0;
                for (int i = warp; i < threads; i += WARPS)
                    row.each_of_thread(sh.chosen[i], lane, [&](int index, float z) {
                        if (z == z) {
                            const Key c = key_of(z, index);
                            if (c < below && c > k) k = c;
                        }
                    });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
                __syncthreads();
                if (lane == 0) sh.warp_best[warp] = k;
                __syncthreads();
                k = sh.warp_best[0];
                for (int w = 1; w < WARPS; ++w) k = max(k, sh.warp_best[w]);
                if (tid == 0) sh.best[j] = k;
                below = k;
                if (!k) break;
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        double s = 0, t = 0;
        int n = 0;
        for (int w = 0; w < WARPS; ++w) { s += sh.sums[0][w]; t += sh.sums[1][w]; n += sh.counts[w]; }
        sh.part = {s, t, block_m, n};
    }
    if (blocks > 1) cluster_sync_all();
    else __syncthreads();
    if (rank == 0) {
        auto remote = [&](const void* p, int b) { return ld_cluster_u64((const unsigned long long*)p, (uint32_t)b); };
        float* to = out + r * (3 + 2 * top);
        if (warp == 0) {  // a block a lane
            float m = -INFINITY;
            double s = 0, t = 0;
            int n = 0;
            if (blocks == 1 && lane == 0) {
                m = sh.part.m; s = sh.part.s; t = sh.part.t; n = sh.part.ahead;
            } else if (blocks > 1 && lane < blocks) {
                const unsigned long long word = remote(&sh.part.m, lane);
                m = __uint_as_float((uint32_t)word);
                n = (int)(word >> 32);
                s = __longlong_as_double((long long)remote(&sh.part.s, lane));
                t = __longlong_as_double((long long)remote(&sh.part.t, lane));
            }
            const float high = warp_max(m), d = bounded(m - high);
            if (d != 0.f) {  // (a NaN too: of two infinities)
                const double f = m == -INFINITY ? 0. : (double)exp_of(d);
                t = m == -INFINITY ? s * 0. : f * (t + s * (double)d);
                s *= f;
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) {  // (up to eight blocks; the same bits in all of the first eight lanes)
                s += __shfl_xor_sync(0xffffffffu, s, o);
                t += __shfl_xor_sync(0xffffffffu, t, o);
                n += __shfl_xor_sync(0xffffffffu, n, o);
            }
            if (lane == 0) {
                const double log_s = log(s), ref = (double)reference(high);  // (z - m first: beside a far m log S would be lost)
                to[0] = (float)((double)z_token - ref - log_s);
                to[1] = (float)(log_s - t / s);
                reinterpret_cast<int*>(to)[2] = z_token == z_token ? n + 1 : 0;
                sh.sums[0][0] = ref;
                sh.sums[0][1] = log_s;
            }
        }
        if constexpr (TOP) {
            __syncthreads();
            const float nan = __uint_as_float(0x7fffffffu);
            const double ref = sh.sums[0][0], log_s = sh.sums[0][1];
            const auto write = [&](int place, Key k) {
                to[3 + place] = k ? (float)((double)value_of(k) - ref - log_s) : nan;
                reinterpret_cast<int*>(to)[3 + top + place] = k ? index_of(k) : -1;
            };
            if (blocks == 1) {
                if (tid < top) write(tid, sh.best[tid]);
            } else {
                // (up to 8 * 64 = 512 keys, in `found`; an even number of blocks, so an even number of keys)
                const int all = blocks * top;
                Key own = 0;
                if (tid < all) {
                    const int b = tid / top;
                    own = b ? (Key)remote(&sh.best[tid - b * top], b) : sh.best[tid];
                    sh.found[tid] = own;
                }
                __syncthreads();
                if (tid < all) {
                    int place = keys_above(sh.found, all / 2, own);
                    if (!own)  // (no alternative: behind those that are, in some order)
                        for (int j = 0; j < tid; ++j) place += !sh.found[j];
                    if (place < top) write(place, own);
                }
            }
        }
    }
    if (blocks > 1) cluster_sync_before_exit();
}

template <typename T>
int launch(const LogprobCall& c, int blocks) {
    const dim3 grid((unsigned)(c.rows * blocks));
#define LOGPROBS(TOP) \
    if (blocks > 1) ss_launch_cluster_x(token_logprobs_kernel<T, TOP>, grid, dim3(THREADS), 0, c.stream, blocks, (const T*)c.logits, c.stride, c.tokens, (int)c.wide, c.out, (int)c.vocabulary, (int)c.top, blocks, c.err); \
    else ss_launch(token_logprobs_kernel<T, TOP>, grid, dim3(THREADS), 0, c.stream, (const T*)c.logits, c.stride, c.tokens, (int)c.wide, c.out, (int)c.vocabulary, (int)c.top, blocks, c.err)
    if (c.top) { LOGPROBS(true); } else { LOGPROBS(false); }
#undef LOGPROBS
    return SS_LAUNCH_CHECK();
}

}  // namespace

// stride in elements, of any alignment that the type has.
extern "C" int ss_token_logprobs(const LogprobCall* call) {
    const LogprobCall& c = *call;
    if (c.rows <= 0) return 0;
    if (c.vocabulary < 1 || c.vocabulary > INT32_MAX - 65536 || c.top < 0 || c.top > LOGPROBS_MAX_TOP || c.rows > INT32_MAX / 8) return -2003;
    const uintptr_t size = c.dtype == SS_BF16 ? 2 : 4;
    if ((uintptr_t)c.logits % size || (uintptr_t)c.tokens % (c.wide ? 8 : 4) || (uintptr_t)c.out % 4) return -2004;
    // blocks a row: as many as run at the same time (three an SM), while each has 16 elements a thread or more
    int blocks = 1;
    while (blocks < 8 && c.rows * blocks * 2 <= 3 * (int64_t)ss_sm_count() && c.vocabulary >= blocks * 2 * 16 * THREADS) blocks *= 2;
    return c.dtype == SS_BF16 ? launch<bf16>(c, blocks) : launch<float>(c, blocks);
}

extern "C" void ss_set_pdl(int on) { ss_pdl_flag() = on; }

// Rows of 8-bit integers with one float32 scale each: how activations and weights become such rows, and back.
//
// A row v becomes q and s with q * s near v: a = max |v|, s = a / 127, q = rint(v * (127 / a)), ties to even, so -127 <= q <= 127
// and the largest element keeps its value.  A row of zeros has s = 0.  A row that holds an infinity or NaN has s = NaN and q = 0:
// all that is formed from it is NaN, as it would be without the rounding.  The maximum is taken over the bits of |v| as unsigned
// integers, which order like the values and put NaN on top.
//
// Rows of q start on 16 bytes (their stride is a multiple of 16); what lies between a row's end and the next row is not written.
//
// All kernels are bound by memory: a row is read once, and its results are written from registers.  What a kernel reads may be written
// while it has already been launched (it waits, griddepcontrol.wait), so those pointers are not __restrict__: the loads must not go
// through the read-only path.

#include "int8_calls.h"
#include "tc5.cuh"

namespace {

constexpr uint32_t INF_BITS = 0x7f800000u;
constexpr float MAGIC = 12582912.f;  // 1.5 * 2^23: behind the sum with it, a float's low byte is the rounded integer's

// Four elements from memory: one load of 16 (float32) or 8 bytes (bfloat16) where rows are aligned for it, else one by one,
// the `left` that there are.
template <bool ALIGNED>
__device__ __forceinline__ void load4(const float* p, int left, float (&v)[4]) {
    if (ALIGNED && left >= 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? p[e] : 0.f;
}
template <bool ALIGNED>
__device__ __forceinline__ void load4(const bf16* p, int left, float (&v)[4]) {
    if (ALIGNED && left >= 4) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
        v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? to_float(p[e]) : 0.f;
}

__device__ __forceinline__ uint32_t top_of(uint32_t top, const float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    return top;
}

// Behind a block's last store where the kernel behind was not let go early, so that it starts when every block has ended: it may
// take the results for constant and read them (with plain loads or by TMA) in front of its griddepcontrol.wait, which is what would make
// them visible otherwise.  One thread's fence, behind a barrier, covers the block's stores; the end of a block then waits for them
// (back to values 2,048 x 18,944 18.5 to 19.8 us, 1,531 x 2,051, element by element, 6.1 to 6.9; rounding 21.6 to 21.7 and 4.0 to 4.8; with a
// fence of every thread the pair takes 42.0 instead of 41.5, and 14.3 instead of 11.8).
__device__ __forceinline__ void publish_results() {
    __syncthreads();
    if (threadIdx.x) return;
    __threadfence();
    asm volatile("fence.proxy.async.global;" ::: "memory");
}

// What a row's largest magnitude (its bits) makes of it.
struct RowScale {
    float scale, inverse, before;  // q = rint((v * before) * inverse)
    uint32_t keep;                 // 0: the row's values are written as zeros
};
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
    RowScale r;
    const float a = __uint_as_float(top);
    const bool fine = top < INF_BITS && top > 0;
    r.before = a < 0x1p-100f ? 0x1p64f : 1.f;  // 127 / a stays finite (and the product with `before` is exact)
    r.inverse = fine ? __fdiv_rn(127.f, a * r.before) : 0.f;
    r.scale = top < INF_BITS ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fffffffu);
    r.keep = fine ? 0xffffffffu : 0u;
    return r;
}
__device__ __forceinline__ uint32_t quantize4(const float (&v)[4], const RowScale& r) {
    uint32_t b[4];
    if (r.before == 1.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(__fadd_rn(__fmul_rn(v[e], r.inverse), MAGIC));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(__fadd_rn(__fmul_rn(v[e] * r.before, r.inverse), MAGIC));
    }
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) & r.keep;
}
__device__ __forceinline__ void store4(int8_t* q, int left, uint32_t word) {
    if (left >= 4) {
        *reinterpret_cast<uint32_t*>(q) = word;
        return;
    }
    for (int e = 0; e < left; ++e) q[e] = (int8_t)(word >> (8 * e));
}

// The block's largest `top` and the sum of its `sum`, with one barrier; every thread gets both.
__device__ __forceinline__ void block_top_sum(uint32_t& top, float& sum, uint32_t* tops, float* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    top = __reduce_max_sync(0xffffffffu, top);
    sum = warp_sum(sum);
    if (lane == 0) { tops[warp] = top; sums[warp] = sum; }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? tops[lane] : 0u);
    sum = warp_sum(lane < warps ? sums[lane] : 0.f);
}

// Threads of a block at most where NG vectors of a row stay in a thread's registers.
template <int NG>
constexpr int most_threads() { return NG == 0 || NG > 2 ? 512 : 1024; }

// ---------------------------------------------------------------- rows to int8
//
// A block per row.  NG vectors of 16 bytes a thread stay in registers as they came; NG = 0: rows of any width, read twice.
template <typename T>
struct RawVec {
    static constexpr int G = 16 / (int)sizeof(T);
    uint4 raw;
    template <bool ALIGNED>
    __device__ __forceinline__ void load(const T* p, int left) {
        if (ALIGNED && left >= G) {
            raw = *reinterpret_cast<const uint4*>(p);
            return;
        }
        T t[G];
#pragma unroll
        for (int e = 0; e < G; ++e) t[e] = e < left ? p[e] : from_float<T>(0.f);
        if constexpr (G == 4) {
            raw = make_uint4(__float_as_uint(t[0]), __float_as_uint(t[1]), __float_as_uint(t[2]), __float_as_uint(t[3]));
        } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (uint32_t)__bfloat16_as_ushort(t[2 * e]) | (uint32_t)__bfloat16_as_ushort(t[2 * e + 1]) << 16;
            raw = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w; }
    // bits of the largest magnitude so far: of float32 values, or of bfloat16 values in both halves of the word
    __device__ __forceinline__ uint32_t top(uint32_t t) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            t = G == 4 ? max(t, word(i) & 0x7fffffffu) : __vmaxu2(t, word(i) & 0x7fff7fffu);
        return t;
    }
    static __device__ __forceinline__ uint32_t top_bits(uint32_t t) { return G == 4 ? t : max(t << 16, t & 0xffff0000u); }
    __device__ __forceinline__ void four(int i, float (&v)[4]) const {  // elements 4 i .. 4 i + 3
        if constexpr (G == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(word(e));
        } else {
            v[0] = __uint_as_float(word(2 * i) << 16); v[1] = __uint_as_float(word(2 * i) & 0xffff0000u);
            v[2] = __uint_as_float(word(2 * i + 1) << 16); v[3] = __uint_as_float(word(2 * i + 1) & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void quantize(int8_t* q, int left, const RowScale& r) const {
        float v[4];
        if constexpr (G == 8) {
            uint2 w;
            four(0, v); w.x = quantize4(v, r);
            four(1, v); w.y = quantize4(v, r);
            if (left >= 8) {
                *reinterpret_cast<uint2*>(q) = w;
            } else {
                store4(q, left, w.x);
                store4(q + 4, left - 4, w.y);
            }
        } else {
            four(0, v);
            store4(q, left, quantize4(v, r));
        }
    }
};

template <typename T, bool ALIGNED, int NG>
__global__ void __launch_bounds__(most_threads<NG>())
quantize_rows_kernel(const T* x, int64_t stride, int8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales,
                     int width, int early) {
    using Vec = RawVec<T>;
    constexpr int G = Vec::G;
    __shared__ uint32_t tops[32];
    __shared__ float sums[32];
    if (early) pdl_launch_dependents();
    pdl_wait();
    const T* row = x + (int64_t)blockIdx.x * stride;
    int8_t* out = q + (int64_t)blockIdx.x * q_stride;
    Vec v[NG ? NG : 1];
    uint32_t top = 0;
    float none = 0.f;
    if constexpr (NG > 0) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * blockDim.x) * G;
            v[i].template load<ALIGNED>(row + j, width - j);
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) top = v[i].top(top);
    } else {
        for (int j = threadIdx.x * G; j < width; j += blockDim.x * G) {
            v[0].template load<ALIGNED>(row + j, width - j);
            top = v[0].top(top);
        }
    }
    top = Vec::top_bits(top);
    block_top_sum(top, none, tops, sums);
    const RowScale r = row_scale(top);
    if (threadIdx.x == 0) scales[blockIdx.x] = r.scale;
    if constexpr (NG > 0) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * blockDim.x) * G;
            if (j < width) v[i].quantize(out + j, width - j, r);
        }
    } else {
        for (int j = threadIdx.x * G; j < width; j += blockDim.x * G) {
            v[0].template load<ALIGNED>(row + j, width - j);
            v[0].quantize(out + j, width - j, r);
        }
    }
    if (!early) publish_results();
}

// ---------------------------------------------------------------- add + RMS norm to int8
//
// x = residual + delta, written to residual_out (if there is one); v = x / sqrt(mean(x^2) + eps) * w, as int8 rows.  The norm's
// factor is the same for the whole row, so q is that of x * w, and the factor enters the scale alone: the squares' sum and the
// largest |x * w| are found in one pass with one barrier, and v is never rounded to fewer than its 24 bits.
// The squares' sum does not depend on how many rows there are, whatever shape the launch takes for them: the sums of 32 neighbouring
// groups of four (a warp's, one group a lane) are formed first, then lane l adds sums l, l + 32, ... of the row, then the lanes.
__device__ __forceinline__ float squares_of(const float (&v)[4]) {
    return fmaf(v[3], v[3], fmaf(v[2], v[2], fmaf(v[1], v[1], v[0] * v[0])));
}
// The warp's sums of NG values a thread, sum i to sums[i * stride].  At every level half of the sums that are left go to the other
// half of the lanes (P values in P + log2(32 / P) shuffles, not 5 P); a sum adds the same pairs as warp_sum does.
template <int NG>
__device__ __forceinline__ void warp_sums(const float (&part)[NG], float* sums, int stride) {
    constexpr int P = NG == 1 ? 1 : NG == 2 ? 2 : NG <= 4 ? 4 : NG <= 8 ? 8 : 16, STEP = 32 / P;
    const int lane = threadIdx.x & 31;
    float a[P];
#pragma unroll
    for (int i = 0; i < P; ++i) a[i] = i < NG ? part[i] : 0.f;
    int w = 16;
#pragma unroll
    for (int n = P / 2; n >= 1; n /= 2, w /= 2) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float send = lane & w ? a[i] : a[i + n], keep = lane & w ? a[i + n] : a[i];
            a[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
        }
    }
#pragma unroll
    for (; w >= 1; w /= 2) a[0] += __shfl_xor_sync(0xffffffffu, a[0], w);
    if (lane % STEP == 0 && lane / STEP < NG) sums[lane / STEP * stride] = a[0];
}
__device__ __forceinline__ float sum_of_sums(const float* sums, int width) {
    const int sets = (width + 127) / 128;
    int c = threadIdx.x & 31;
    float total = c < sets ? sums[c] : 0.f;
    for (c += 32; c < sets; c += 32) total += sums[c];
    return warp_sum(total);
}
__device__ __forceinline__ float norm_scale(uint32_t top, float squares, int width, float eps) {
    const float rstd = 1.0f / sqrtf(squares / (float)width + eps);
    return top < INF_BITS ? __fdiv_rn(__uint_as_float(top) * rstd, 127.f) : __uint_as_float(0x7fffffffu);
}

// A block per row; NG groups of four elements a thread stay in registers; NG = 0: rows of any width, read twice.
template <typename T, bool ALIGNED, int NG>
__global__ void __launch_bounds__(most_threads<NG>())
add_rmsnorm_int8_kernel(const float* residual, const T* delta, float* residual_out, const void* __restrict__ weight,
                        int w_f32, int8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int width, float eps) {
    // few rows: the weights do not depend on the kernels in front and are on the way before those are through
    constexpr bool EARLY_W = NG == 1 || NG == 2;
    __shared__ uint32_t tops[32];
    __shared__ float sums[NG ? 32 * NG : 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    float w[EARLY_W ? NG : 1][4], v[NG ? NG : 1][4], part[NG ? NG : 1];
    auto load_w = [&](int j, float (&to)[4]) {
        if (w_f32) load4<ALIGNED>((const float*)weight + j, width - j, to);
        else load4<ALIGNED>((const bf16*)weight + j, width - j, to);
    };
    if constexpr (EARLY_W) {
#pragma unroll
        for (int i = 0; i < NG; ++i) load_w((threadIdx.x + i * blockDim.x) * 4, w[i]);
    }
    pdl_wait();
    const int64_t at = (int64_t)blockIdx.x * width;
    const float* row = residual + at;
    int8_t* out = q + (int64_t)blockIdx.x * q_stride;
    uint32_t top = 0;
    float ss = 0.f;
    auto load_x = [&](int j, bool add, float (&x)[4]) {
        load4<ALIGNED>(row + j, width - j, x);
        if (add) {
            float d[4];
            load4<ALIGNED>(delta + at + j, width - j, d);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __fadd_rn(x[e], d[e]);
        }
    };
    auto store_x = [&](int j, const float (&x)[4]) {
        float* to = residual_out + at + j;
        if (ALIGNED && j + 4 <= width) {
            *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < width) to[e] = x[e];
        }
    };
    if constexpr (NG > 0) {
#pragma unroll
        for (int i = 0; i < NG; ++i) load_x((threadIdx.x + i * blockDim.x) * 4, delta != nullptr, v[i]);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * blockDim.x) * 4;
            if (residual_out && j < width) store_x(j, v[i]);
            float (&wi)[4] = w[EARLY_W ? i : 0];
            if constexpr (!EARLY_W) load_w(j, wi);
            part[i] = squares_of(v[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] *= wi[e];
            top = top_of(top, v[i]);
        }
        warp_sums(part, sums + warp, blockDim.x >> 5);
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) tops[warp] = top;
        __syncthreads();
        top = __reduce_max_sync(0xffffffffu, lane < (blockDim.x >> 5) ? tops[lane] : 0u);
        ss = sum_of_sums(sums, width);
    } else {
        for (int j = threadIdx.x * 4; j < width; j += blockDim.x * 4) {
            load_x(j, delta != nullptr, v[0]);
            if (residual_out) store_x(j, v[0]);
            load_w(j, w[0]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ss = fmaf(v[0][e], v[0][e], ss);
                v[0][e] *= w[0][e];
            }
            top = top_of(top, v[0]);
        }
        block_top_sum(top, ss, tops, sums);
    }
    const RowScale r = row_scale(top);
    if (threadIdx.x == 0) scales[blockIdx.x] = norm_scale(top, ss, width, eps);
    if constexpr (NG > 0) {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * blockDim.x) * 4;
            if (j < width) store4(out + j, width - j, quantize4(v[i], r));
        }
    } else {
        // the sum again: from residual_out where it was written (by this thread), else formed once more
        if (residual_out) row = residual_out + at;
        for (int j = threadIdx.x * 4; j < width; j += blockDim.x * 4) {
            load_x(j, delta != nullptr && !residual_out, v[0]);
            load_w(j, w[0]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[0][e] *= w[0][e];
            store4(out + j, width - j, quantize4(v[0], r));
        }
    }
}

// ---------------------------------------------------------------- many rows
//
// The same two operations for many wide rows: two or three blocks an SM, each taking rows blockIdx.x, + gridDim.x, ... through a ring
// of `stages` rows in shared memory that one thread fills by bulk copies, so that the rows behind are on their way through the two
// passes over this one (with registers alone DRAM was 40 % busy: too few warps fit beside what they hold).  A block's stage is free
// when all its threads have read their part, behind the one barrier a row.  NG vectors a thread; rows of a multiple of 16 bytes that
// start on 16 bytes.  Norm of 4,096 x 3,584 (bfloat16 branch): 29.7 us, 83 % of the measured copy rate, a block per row 36.3;
// 2,048 x 8,192 33.5 and 52.0; rounding 2,048 x 18,944 (bfloat16) 21.7 and 26.1 (four inputs in turn, back to back).  Rows below 16 KB stay with a block per row: a row's
// chain of two passes and a barrier is about 1,500 cycles however narrow it is, and many small blocks hide more of them (norm of
// 4,096 x 896: 10.5 us through a ring, 8.7 so; rounding 4,096 x 3,584: 10.5 and 9.8).
constexpr int RING_THREADS = 256;
constexpr int ring_blocks(int ng) { return ng <= 4 ? 3 : 2; }  // blocks an SM at most

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(s_addr(dst)), "l"(src), "r"(bytes), "r"(s_addr(bar)) : "memory");
}
struct RowRing {
    unsigned char* rows;  // [stages][bytes of a row]
    uint64_t* full;
    int* gave_up;
    int stages;
};
// smem: the rows (16-byte aligned), then the barriers, then the flag
__device__ __forceinline__ RowRing row_ring(unsigned char* smem, int stages, int row_bytes) {
    RowRing r;
    r.rows = smem;
    r.full = reinterpret_cast<uint64_t*>(smem + stages * row_bytes);
    r.gave_up = reinterpret_cast<int*>(r.full + stages);
    r.stages = stages;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&r.full[s], 1);
        *r.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    return r;
}

// Behind a wait that gave up (the block has left its loop at that row): the error word, and a wait for the block's copies in flight,
// the last of the `issued` ones that thread 0 has sent for.
__device__ __forceinline__ void drain_ring(const RowRing& r, int issued, int* err) {
    if (!*(volatile int*)r.gave_up || threadIdx.x) return;
    for (int i = max(0, issued - r.stages); i < issued; ++i) mbar_drain(&r.full[i % r.stages], (i / r.stages) & 1);
    atomicOr(err, SS_ERR_WAIT_LIMIT);
}

template <typename T, int NG>
__global__ void __launch_bounds__(RING_THREADS, ring_blocks(NG))
quantize_ring_kernel(const T* x, int64_t stride, int8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int rows,
                     int width, int stages, int early, int* err) {
    using Vec = RawVec<T>;
    constexpr int G = Vec::G;
    extern __shared__ __align__(128) unsigned char ring_smem[];
    __shared__ uint32_t tops[2][RING_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bytes = width * (int)sizeof(T);
    const RowRing ring = row_ring(ring_smem, stages, bytes);
    if (early) pdl_launch_dependents();
    pdl_wait();
    int issued = 0;  // copies that thread 0 has sent for
    auto fetch = [&](int64_t row, int s) {
        ++issued;
        mbar_expect_tx(&ring.full[s], bytes);
        bulk_load(ring.rows + s * bytes, x + row * stride, bytes, &ring.full[s]);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages && blockIdx.x + (int64_t)s * gridDim.x < rows; ++s) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
    int s = 0, n = 0;
    uint32_t parity = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, ++n) {
        const bool landed = mbar_wait(&ring.full[s], parity, ring.gave_up);
        const T* from = reinterpret_cast<const T*>(ring.rows + s * bytes);
        Vec v[NG];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * RING_THREADS) * G;
            v[i].raw = j < width ? *reinterpret_cast<const uint4*>(from + j) : make_uint4(0, 0, 0, 0);
            top = v[i].top(top);
        }
        top = __reduce_max_sync(0xffffffffu, Vec::top_bits(top));
        if (lane == 0) tops[n & 1][warp] = top;  // (two sets: the next row's are written while slow warps still read these)
        if (!__syncthreads_and(landed)) break;  // nothing of the row is written, nothing more is sent for
        if (threadIdx.x == 0 && row + (int64_t)stages * gridDim.x < rows) fetch(row + (int64_t)stages * gridDim.x, s);
        top = __reduce_max_sync(0xffffffffu, lane < RING_THREADS / 32 ? tops[n & 1][lane] : 0u);
        const RowScale r = row_scale(top);
        if (threadIdx.x == 0) scales[row] = r.scale;
        int8_t* out = q + row * q_stride;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * RING_THREADS) * G;
            if (j < width) v[i].quantize(out + j, width - j, r);
        }
        if (++s == stages) { s = 0; parity ^= 1; }
    }
    drain_ring(ring, issued, err);
    if (!early) publish_results();
}

template <typename T, int NG>
__global__ void __launch_bounds__(RING_THREADS, ring_blocks(NG))
add_rmsnorm_int8_ring_kernel(const float* residual, const T* delta, float* residual_out, const void* __restrict__ weight,
                             int w_f32, int8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int rows, int width, float eps,
                             int stages, int* err) {
    extern __shared__ __align__(128) unsigned char ring_smem[];
    __shared__ uint32_t tops[2][RING_THREADS / 32];
    __shared__ float sums[2][NG * RING_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int x_bytes = width * 4, d_bytes = delta ? width * (int)sizeof(T) : 0, bytes = x_bytes + d_bytes;
    const RowRing ring = row_ring(ring_smem, stages, bytes);
    pdl_launch_dependents();
    float w[NG][4];  // for all rows of the block
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int j = (threadIdx.x + i * RING_THREADS) * 4;
        if (w_f32) load4<true>((const float*)weight + j, width - j, w[i]);
        else load4<true>((const bf16*)weight + j, width - j, w[i]);
    }
    pdl_wait();
    int issued = 0;  // copies that thread 0 has sent for
    auto fetch = [&](int64_t row, int s) {
        ++issued;
        mbar_expect_tx(&ring.full[s], bytes);
        bulk_load(ring.rows + s * bytes, residual + row * width, x_bytes, &ring.full[s]);
        if (d_bytes) bulk_load(ring.rows + s * bytes + x_bytes, delta + row * width, d_bytes, &ring.full[s]);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages && blockIdx.x + (int64_t)s * gridDim.x < rows; ++s) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
    int s = 0, n = 0;
    uint32_t parity = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, ++n) {
        const bool landed = mbar_wait(&ring.full[s], parity, ring.gave_up);
        const float* from = reinterpret_cast<const float*>(ring.rows + s * bytes);
        const T* from_d = reinterpret_cast<const T*>(ring.rows + s * bytes + x_bytes);
        float v[NG][4], part[NG];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * RING_THREADS) * 4;
            if (j < width) {
                load4<true>(from + j, 4, v[i]);
                if (d_bytes) {
                    float d[4];
                    load4<true>(from_d + j, 4, d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[i][e] = __fadd_rn(v[i][e], d[e]);
                }
                if (residual_out && landed) *reinterpret_cast<float4*>(residual_out + row * width + j) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][e] = 0.f;
            }
            part[i] = squares_of(v[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] *= w[i][e];
            top = top_of(top, v[i]);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        warp_sums(part, sums[n & 1] + warp, RING_THREADS / 32);
        if (lane == 0) tops[n & 1][warp] = top;
        if (!__syncthreads_and(landed)) break;  // (of the stream threads have written what they saw land)
        if (threadIdx.x == 0 && row + (int64_t)stages * gridDim.x < rows) fetch(row + (int64_t)stages * gridDim.x, s);
        top = __reduce_max_sync(0xffffffffu, lane < RING_THREADS / 32 ? tops[n & 1][lane] : 0u);
        const float ss = sum_of_sums(sums[n & 1], width);
        const RowScale r = row_scale(top);
        if (threadIdx.x == 0) scales[row] = norm_scale(top, ss, width, eps);
        int8_t* out = q + row * q_stride;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * RING_THREADS) * 4;
            if (j < width) *reinterpret_cast<uint32_t*>(out + j) = quantize4(v[i], r);
        }
        if (++s == stages) { s = 0; parity ^= 1; }
    }
    drain_ring(ring, issued, err);
}

// ---------------------------------------------------------------- int8 rows to values
//
// y = q * s, rounded once.  A row is cut into spans of groups (eight bfloat16 or four float32 elements, where the output's rows
// start on 16 bytes, else one), a block each, four groups a thread, all loaded before the first is written.
constexpr int DEQ_THREADS = 256, DEQ_GROUPS = 4;

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(DEQ_THREADS)
dequantize_rows_kernel(const int8_t* q, int64_t q_stride, const float* scales, T* y, int width,
                       int spans, int early) {
    constexpr int G = ALIGNED ? 16 / (int)sizeof(T) : 1;
    if (early) pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x / spans, first = (blockIdx.x - row * spans) * (int)(blockDim.x * DEQ_GROUPS) + threadIdx.x;
    const float s = scales[row];
    const int8_t* from = q + (int64_t)row * q_stride;
    T* out = y + (int64_t)row * width;
    uint32_t words[DEQ_GROUPS][2];
#pragma unroll
    for (int i = 0; i < DEQ_GROUPS; ++i) {
        const int64_t j = (int64_t)(first + i * blockDim.x) * G;
        if (j < width) {
            if constexpr (G == 8) *reinterpret_cast<uint2*>(words[i]) = *reinterpret_cast<const uint2*>(from + j);
            else if constexpr (G == 4) words[i][0] = *reinterpret_cast<const uint32_t*>(from + j);
            else words[i][0] = (uint32_t)(uint8_t)from[j];
        }
    }
#pragma unroll
    for (int i = 0; i < DEQ_GROUPS; ++i) {
        const int64_t j = (int64_t)(first + i * blockDim.x) * G;
        if (j < width) {
            T v[G];
#pragma unroll
            for (int e = 0; e < G; ++e) v[e] = from_float<T>((float)(int8_t)(words[i][e / 4] >> (8 * (e & 3))) * s);
            if constexpr (ALIGNED) *reinterpret_cast<uint4*>(out + j) = *reinterpret_cast<const uint4*>(v);
            else out[j] = v[0];
        }
    }
    if (!early) publish_results();
}

// ---------------------------------------------------------------- launches

// How a row of `groups` vectors or groups is dealt out: NG a thread (0: the row is read twice) and the threads of a block.  Up to
// two rows an SM leave SMs to spare, so a row gets as many threads as a block holds; many rows run in blocks of up to 256
// threads where that suffices, several of them on an SM.
struct RowShape { int ng, threads; };
inline RowShape row_shape(int groups, int64_t rows) {
    const int sizes[8] = {1, 2, 3, 4, 6, 8, 10, 0};
    const bool few = rows <= 2 * (int64_t)ss_sm_count();
    for (int pass = few ? 1 : 0; pass < 2; ++pass)
        for (int i = 0; i < 7; ++i) {
            const int threads = ((groups + sizes[i] - 1) / sizes[i] + 31) / 32 * 32;
            if (threads <= (pass == 0 ? 256 : sizes[i] > 2 ? 512 : 1024)) return {sizes[i], threads};
        }
    return {0, 512};
}
#define ROW_SHAPES(CASE) switch (shape.ng) { CASE(0); CASE(1); CASE(2); CASE(3); CASE(4); CASE(6); CASE(8); CASE(10); }

// The ring: blocks an SM, and stages of a block's ring (0: the rows are too few, too narrow or too wide).  Three rows in flight a
// block where three blocks share an SM, else two at least; four rows a block at least.
struct RingShape { int blocks, stages; };
constexpr int RING_SMEM = 112 * 1024;  // of a block, two of which share an SM
inline int ring_groups(int vectors) {
    const int ng = (vectors + RING_THREADS - 1) / RING_THREADS;
    return ng <= 4 ? ng : ng <= 6 ? 6 : ng <= 8 ? 8 : ng <= 10 ? 10 : 12;
}
inline RingShape ring_shape(int64_t rows, int64_t row_bytes, int vectors) {
    if (row_bytes < 16384 || vectors > 12 * RING_THREADS || row_bytes % 16) return {0, 0};
    for (int blocks = ring_blocks(ring_groups(vectors)); blocks >= 2; --blocks) {
        const int64_t stages = (224 * 1024 / blocks - 2048) / (row_bytes + 8);
        if (stages >= blocks && rows >= 4 * (int64_t)blocks * ss_sm_count()) return {blocks, (int)stages};
    }
    return {0, 0};
}

template <typename T>
int launch_quantize_ring(const Int8RowsCall& c, RingShape shape) {
    const int vectors = (int)((c.width * sizeof(T) + 15) / 16), blocks = shape.blocks * ss_sm_count(), stages = shape.stages;
    const int smem = (int)(stages * (c.width * sizeof(T) + 8)) + 64;
    int rc = 0;
#define QUANT(NG) case NG: { \
        static SsPerDevice opted; \
        if ((rc = ss_opt_in_smem(quantize_ring_kernel<T, NG>, RING_SMEM, opted))) return rc; \
        ss_launch(quantize_ring_kernel<T, NG>, dim3(blocks), dim3(RING_THREADS), smem, c.stream, (const T*)c.x, c.stride, c.q, c.q_stride, c.scales, (int)c.rows, (int)c.width, stages, (int)c.early, c.err); \
    } break
    switch (ring_groups(vectors)) { QUANT(4); QUANT(6); QUANT(8); QUANT(10); QUANT(12); }
#undef QUANT
    return SS_LAUNCH_CHECK();
}

template <typename T>
int launch_norm_ring(const Int8RowsCall& c, RingShape shape) {
    const int vectors = (int)((c.width + 3) / 4), blocks = shape.blocks * ss_sm_count(), stages = shape.stages;
    const int smem = (int)(stages * (c.width * (4 + (c.delta ? sizeof(T) : 0)) + 8)) + 64;
    int rc = 0;
#define NORM(NG) case NG: { \
        static SsPerDevice opted; \
        if ((rc = ss_opt_in_smem(add_rmsnorm_int8_ring_kernel<T, NG>, RING_SMEM, opted))) return rc; \
        ss_launch(add_rmsnorm_int8_ring_kernel<T, NG>, dim3(blocks), dim3(RING_THREADS), smem, c.stream, (const float*)c.x, (const T*)c.delta, (float*)c.y, c.weight, (int)c.w_f32, c.q, c.q_stride, c.scales, (int)c.rows, (int)c.width, (float)c.eps, stages, c.err); \
    } break
    switch (ring_groups(vectors)) { NORM(2); NORM(3); NORM(4); NORM(6); NORM(8); NORM(10); NORM(12); }
#undef NORM
    return SS_LAUNCH_CHECK();
}

template <typename T, bool ALIGNED>
int launch_quantize(const void* x, int64_t stride, int8_t* q, int64_t q_stride, float* scales, int rows, int width, int early,
                    cudaStream_t stream) {
    constexpr int G = RawVec<T>::G;
    const RowShape shape = row_shape((width + G - 1) / G, rows);
#define QUANT(NG) case NG: ss_launch(quantize_rows_kernel<T, ALIGNED, NG>, dim3(rows), dim3(shape.threads), 0, stream, (const T*)x, stride, q, q_stride, scales, width, early); break
    ROW_SHAPES(QUANT)
#undef QUANT
    return SS_LAUNCH_CHECK();
}

template <typename T, bool ALIGNED>
int launch_norm(const float* residual, const void* delta, float* residual_out, const void* weight, int w_f32, int8_t* q,
                int64_t q_stride, float* scales, int rows, int width, float eps, cudaStream_t stream) {
    const RowShape shape = row_shape((width + 3) / 4, rows);
#define NORM(NG) case NG: ss_launch(add_rmsnorm_int8_kernel<T, ALIGNED, NG>, dim3(rows), dim3(shape.threads), 0, stream, residual, (const T*)delta, residual_out, weight, w_f32, q, q_stride, scales, width, eps); break
    ROW_SHAPES(NORM)
#undef NORM
    return SS_LAUNCH_CHECK();
}

inline bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

static int int8_rows_refused(const Int8RowsCall& c) {
    return c.width <= 0 || c.width > INT8_MAX_WIDTH || c.rows > INT32_MAX || c.q_stride % 16 || !on16(c.q) ? -2003 : 0;
}

// early, here and in the way back: the kernel behind may start at once; it may then have read what it takes for constant before the
// results are written, so only for results that it does not take for that (weights are).
extern "C" int ss_quantize_rows_int8(const Int8RowsCall* call) {
    const Int8RowsCall& c = *call;
    if (c.rows <= 0) return 0;
    if (int rc = int8_rows_refused(c)) return rc;
    const int rows = (int)c.rows, width = (int)c.width, early = (int)c.early;
    const int size = c.dtype == SS_BF16 ? 2 : 4;
    if (on16(c.x) && c.stride * size % 16 == 0) {
        const RingShape shape = ring_shape(c.rows, c.width * size, (int)((c.width * size + 15) / 16));
        if (shape.blocks) return c.dtype == SS_BF16 ? launch_quantize_ring<bf16>(c, shape) : launch_quantize_ring<float>(c, shape);
    }
    if (c.dtype == SS_BF16)
        return on16(c.x) && c.stride % 8 == 0 ? launch_quantize<bf16, true>(c.x, c.stride, c.q, c.q_stride, c.scales, rows, width, early, c.stream)
                                              : launch_quantize<bf16, false>(c.x, c.stride, c.q, c.q_stride, c.scales, rows, width, early, c.stream);
    return on16(c.x) && c.stride % 4 == 0 ? launch_quantize<float, true>(c.x, c.stride, c.q, c.q_stride, c.scales, rows, width, early, c.stream)
                                          : launch_quantize<float, false>(c.x, c.stride, c.q, c.q_stride, c.scales, rows, width, early, c.stream);
}

extern "C" int ss_add_rmsnorm_int8(const Int8RowsCall* call) {
    const Int8RowsCall& c = *call;
    if (c.rows <= 0) return 0;
    if (int rc = int8_rows_refused(c)) return rc;
    const int rows = (int)c.rows, width = (int)c.width, w_f32 = (int)c.w_f32;
    const float* residual = (const float*)c.x;
    const bool aligned = width % 4 == 0 && on16(c.x) && on16(c.delta) && on16(c.y) && on16(c.weight);
    if (aligned && (c.dtype != SS_BF16 || !c.delta || width % 8 == 0)) {
        const RingShape shape = ring_shape(c.rows, c.width * (4 + (!c.delta ? 0 : c.dtype == SS_BF16 ? 2 : 4)), (width + 3) / 4);
        if (shape.blocks) return c.dtype == SS_BF16 ? launch_norm_ring<bf16>(c, shape) : launch_norm_ring<float>(c, shape);
    }
    if (c.dtype == SS_BF16)
        return aligned ? launch_norm<bf16, true>(residual, c.delta, (float*)c.y, c.weight, w_f32, c.q, c.q_stride, c.scales, rows, width, (float)c.eps, c.stream)
                       : launch_norm<bf16, false>(residual, c.delta, (float*)c.y, c.weight, w_f32, c.q, c.q_stride, c.scales, rows, width, (float)c.eps, c.stream);
    return aligned ? launch_norm<float, true>(residual, c.delta, (float*)c.y, c.weight, w_f32, c.q, c.q_stride, c.scales, rows, width, (float)c.eps, c.stream)
                   : launch_norm<float, false>(residual, c.delta, (float*)c.y, c.weight, w_f32, c.q, c.q_stride, c.scales, rows, width, (float)c.eps, c.stream);
}

extern "C" int ss_dequantize_rows_int8(const Int8RowsCall* call) {
    const Int8RowsCall& c = *call;
    if (c.rows <= 0) return 0;
    if (int rc = int8_rows_refused(c)) return rc;
    const int rows = (int)c.rows, width = (int)c.width, g = c.dtype == SS_BF16 ? 8 : 4;
    const bool aligned = on16(c.y) && width % g == 0;
    const int groups = (width + (aligned ? g : 1) - 1) / (aligned ? g : 1);
    int threads = ((groups + DEQ_GROUPS - 1) / DEQ_GROUPS + 31) / 32 * 32;
    threads = threads > DEQ_THREADS ? DEQ_THREADS : threads;
    const int span = threads * DEQ_GROUPS, spans = (groups + span - 1) / span;
    if (c.rows * spans > INT32_MAX) return -2003;
#define DEQ(T, A) ss_launch(dequantize_rows_kernel<T, A>, dim3(rows * spans), dim3(threads), 0, c.stream, c.q, c.q_stride, c.scales, (T*)c.y, width, spans, (int)c.early)
    if (c.dtype == SS_BF16) { if (aligned) DEQ(bf16, true); else DEQ(bf16, false); }
    else { if (aligned) DEQ(float, true); else DEQ(float, false); }
#undef DEQ
    return SS_LAUNCH_CHECK();
}

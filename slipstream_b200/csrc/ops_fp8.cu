// Rows and weights in 8-bit floats with a scale for each block of 128 (fp8.cuh): how they are formed, and the way back.
//
// Rows of q start on 16 bytes (their stride is a multiple of 16); what lies between a row's end and the next row is not written.
//
// All kernels are bound by memory: a value is read once, and the results are written from registers.  What a kernel reads may be
// written while it has already been launched (it waits, griddepcontrol.wait), so those pointers are not __restrict__: the loads must
// not go through the read-only path.

#include "fp8.cuh"
#include "fp8_calls.h"
#include "tc5.cuh"

namespace {

// Elements of a row from memory into registers, V (four or eight) of them: 16 bytes in one load where rows are aligned for it (float32:
// 4, bfloat16: 8 or, for 4, 8 bytes), else one by one, the `left` that there are.
template <int V, bool ALIGNED>
__device__ __forceinline__ void load(const float* p, int left, float (&v)[V]) {
    static_assert(V == 4, "");
    if (ALIGNED && left >= 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? p[e] : 0.f;
}
template <int V, bool ALIGNED>
__device__ __forceinline__ void load(const bf16* p, int left, float (&v)[V]) {
    if (ALIGNED && left >= V) {
        uint32_t w[V / 2];
        if constexpr (V == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
        else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < left ? to_float(p[e]) : 0.f;
}
// 16 bytes of a row as they came.
template <typename T>
struct RawVec {
    static constexpr int V = 16 / (int)sizeof(T);
    uint4 raw;
    template <bool ALIGNED>
    __device__ __forceinline__ void load(const T* p, int left) {
        if (ALIGNED && left >= V) {
            raw = *reinterpret_cast<const uint4*>(p);
            return;
        }
        uint32_t w[4] = {};
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < left) {
                if constexpr (V == 4) w[e] = __float_as_uint(p[e]);
                else w[e / 2] |= (uint32_t)__bfloat16_as_ushort(p[e]) << (16 * (e % 2));
            }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // bits of the largest magnitude: of bfloat16 values pairs at a time
    __device__ __forceinline__ uint32_t top() const {
        if constexpr (V == 4) return max(max(raw.x & 0x7fffffffu, raw.y & 0x7fffffffu), max(raw.z & 0x7fffffffu, raw.w & 0x7fffffffu));
        const uint32_t t = __vmaxu2(__vmaxu2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu), __vmaxu2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu));
        return max(t << 16, t & 0xffff0000u);
    }
    __device__ __forceinline__ void store(uint8_t* q, int left, const Fp8Scale& r) const {
        float v[V];
        values(v);
        if (r.before != 1.f) {  // (very small values)
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] *= r.before;
        }
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            w[i] = fp8_pack4(__fmul_rn(v[4 * i], r.inverse), __fmul_rn(v[4 * i + 1], r.inverse), __fmul_rn(v[4 * i + 2], r.inverse), __fmul_rn(v[4 * i + 3], r.inverse)) & r.keep;
        if (V == 8 && left >= 8) {
            *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[V / 4 - 1]);
            return;
        }
#pragma unroll
        for (int i = 0; i < V / 4; ++i) fp8_store4(q + 4 * i, left - 4 * i, w[i]);
    }
    __device__ __forceinline__ void values(float (&v)[V]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = V == 4 ? __uint_as_float(w[e]) : __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
};
// Behind a block's last store where the kernel behind was not let go early, so that it starts when every block has ended: it may
// take the results for constant and read them (with plain loads or by TMA) in front of its griddepcontrol.wait, which is what would make
// them visible otherwise.  One thread's fence, behind a barrier, covers the block's stores.
__device__ __forceinline__ void publish_results() {
    __syncthreads();
    if (threadIdx.x) return;
    __threadfence();
    asm volatile("fence.proxy.async.global;" ::: "memory");
}

// Rows are dealt out to warps in groups of 32 vectors (128 or 256 columns), `groups` of them a row, all rows in one sequence, of which a
// block of threads takes ROW_WARPS * ROW_GROUPS.  (Fewer than 2^32 of them: launch.)
constexpr int ROW_THREADS = 256, ROW_WARPS = ROW_THREADS / 32, ROW_GROUPS = 4;  // groups a warp
struct Place {
    uint32_t row;
    int column;  // the group's first
};
template <int V>
__device__ __forceinline__ Place place_of(int i, int groups) {  // the i-th group of the warp
    const uint32_t at = blockIdx.x * (uint32_t)(ROW_WARPS * ROW_GROUPS) + i * ROW_WARPS + (threadIdx.x >> 5), row = at / (uint32_t)groups;
    return {row, (int)(at - row * groups) * 32 * V};
}

// ---------------------------------------------------------------- rows to fp8
//
// A lane takes 16 bytes of a row: a block of 128 is 32 lanes of float32 or 16 of bfloat16, whose largest magnitude is found by
// shuffles.  A block of threads takes 32 vectors (128 or 256 columns) of each of 32 rows, a warp four rows, all loaded before the first is
// written; neighbouring blocks take neighbours of the same rows.  The scales of 32 rows stand side by side in memory and are written so.
//
// Bound by instructions as much as by memory: 16 bytes in are 16 values or 8 to take apart, compare, multiply, round and pack.  The largest
// magnitude of bfloat16 pairs at a time, one division a lane (for the group that it leads) and four rows a warp in flight took 4,096 x 3,584
// from 18.8 to 11.5 us (6.7 us of bytes; the issue slots are 65 % busy), 2,048 x 18,944 to 25.6 (17.8), 1,531 x 2,051 in float32 from rows that
// start anywhere to 6.4 (2.4).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(ROW_THREADS)
quantize_rows_kernel(const T* x, int64_t stride, uint8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int64_t scale_row,
                     int64_t scale_block, int64_t rows, int width, unsigned groups, int early) {
    constexpr int V = 16 / (int)sizeof(T), LANES = FP8_BLOCK / V, PER = 32 / LANES, BLOCKS = ROW_GROUPS * PER;
    __shared__ float formed[PER][ROW_WARPS * ROW_GROUPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned down = blockIdx.x / groups;
    const int first = (int)(blockIdx.x - down * groups) * 32 * V, column = first + lane * V, left = width - column;
    const int64_t row0 = (int64_t)down * (ROW_WARPS * ROW_GROUPS) + warp * ROW_GROUPS;
    if (early) pdl_launch_dependents();
    pdl_wait();
    RawVec<T> v[ROW_GROUPS];
#pragma unroll
    for (int i = 0; i < ROW_GROUPS; ++i) {
        const bool in = row0 + i < rows && left > 0;
        v[i].template load<ALIGNED>(x + (in ? (row0 + i) * stride + column : 0), in ? left : 0);
    }
    // The warp holds ROW_GROUPS * PER blocks.  A division takes as long as all that is done with eight elements beside it, so each lane
    // does one: lane b what the values of block b are multiplied by, lane 16 + b its scale.
    const int mine = lane % 16, half = lane / LANES;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < ROW_GROUPS; ++i) {
        uint32_t t = v[i].top();
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
        t = __shfl_sync(0xffffffffu, t, mine % PER * LANES);
        if (mine / PER == i) top = t;
    }
    const Fp8Factor f = fp8_factor(top, lane < 16);
    if (lane >= 16 && mine < BLOCKS) formed[mine % PER][warp * ROW_GROUPS + mine / PER] = f.value;
#pragma unroll
    for (int i = 0; i < ROW_GROUPS; ++i) {
        Fp8Scale r;
        r.inverse = __shfl_sync(0xffffffffu, f.value, i * PER + half);
        r.before = __shfl_sync(0xffffffffu, f.before, i * PER + half);
        r.keep = r.inverse == 0.f ? 0u : 0xffffffffu;
        if (row0 + i < rows && left > 0) v[i].store(q + (row0 + i) * q_stride + column, left, r);
    }
    __syncthreads();
    if (warp < PER && first + warp * FP8_BLOCK < width) {
        const int64_t row = (int64_t)down * (ROW_WARPS * ROW_GROUPS) + lane;
        if (row < rows) scales[row * scale_row + (first / FP8_BLOCK + warp) * scale_block] = formed[warp][lane];
    }
    if (!early) publish_results();
}

// ---------------------------------------------------------------- weights to fp8
//
// A block of threads per 128 x 128 elements, which stay in registers.  Neighbouring blocks take neighbours of the same rows, so that the
// pieces of a row in memory are read at the same time.  Bound by memory: 18,944 x 3,584 bfloat16 35.4 us, 5.8 TB/s.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(ROW_THREADS, sizeof(T) == 2 ? 4 : 3)
quantize_blocks_kernel(const T* x, int64_t stride, uint8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int64_t scale_row,
                       int64_t scale_block, int64_t rows, int width, unsigned across) {
    constexpr int V = 16 / (int)sizeof(T), LANES = FP8_BLOCK / V, AT_ONCE = ROW_THREADS / LANES, N = FP8_BLOCK / AT_ONCE;
    __shared__ uint32_t tops[ROW_WARPS];
    pdl_wait();
    const unsigned down = blockIdx.x / across, right = blockIdx.x - down * across;
    const int64_t r0 = (int64_t)down * FP8_BLOCK + threadIdx.x / LANES;
    const int64_t j = (int64_t)right * FP8_BLOCK + threadIdx.x % LANES * V;
    const int left = (int)min((int64_t)V, max((int64_t)0, width - j));
    RawVec<T> v[N];  // as they came: bfloat16 values take half the registers of float32 ones
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int64_t r = r0 + i * AT_ONCE;
        v[i].template load<ALIGNED>(x + (r < rows && left > 0 ? r * stride + j : 0), r < rows ? left : 0);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, v[i].top());
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, tops[threadIdx.x % ROW_WARPS]);
    const Fp8Scale s = fp8_scale(top);
    if (threadIdx.x == 0) scales[down * scale_row + right * scale_block] = s.scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int64_t r = r0 + i * AT_ONCE;
        if (r < rows && left > 0) v[i].store(q + r * q_stride + j, left, s);
    }
    publish_results();
}

// ---------------------------------------------------------------- add + RMS norm to fp8
//
// x = residual + delta, written to residual_out (if there is one); v = x / sqrt(mean(x^2) + eps) * w, as rows of blocks.  The norm's
// factor is the same for the whole row, so q is that of x * w, and the factor enters the scales alone: a warp, which holds a block of
// 128 (four elements a lane), writes its q at once, and only the scales wait for the row's sum of squares.
// The squares' sum does not depend on how many rows there are, whatever shape the launch takes for them: a block's sum (a warp's) is
// formed first, then lane l adds the sums of blocks l, l + 32, ... of the row, then the lanes.
// Bound by memory, 11 bytes an element with a bfloat16 delta: 4,096 x 3,584 32.0 us (5.1 TB/s; the issue slots are 56 % busy), 4,096 x 8,192 69.5
// (5.3); few rows by the chain of load, sum, barrier, store: 8 x 3,584 2.2 us.
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
// The scale of a block whose largest |x * w| has the bits `top`.
__device__ __forceinline__ float norm_scale(uint32_t top, float rstd) {
    return top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top) * rstd, FP8_TOP) : __uint_as_float(0x7fffffffu);
}

// A block of threads per row; NG groups of four elements a thread, or (NG = 0) rows of any width.  sums: [blocks of the row], then tops.
template <typename T, bool ALIGNED, int NG>
__global__ void __launch_bounds__(1024)
add_rmsnorm_fp8_kernel(const float* residual, const T* delta, float* residual_out, const void* __restrict__ weight, int w_f32,
                       uint8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int64_t scale_row, int64_t scale_block, int width, float eps) {
    extern __shared__ float sums[];
    const int blocks = (width + FP8_BLOCK - 1) / FP8_BLOCK;
    uint32_t* tops = reinterpret_cast<uint32_t*>(sums + blocks);
    const int lane = threadIdx.x & 31;
    pdl_launch_dependents();
    auto load_w = [&](int j, float (&to)[4]) {
        if (w_f32) load<4, ALIGNED>((const float*)weight + j, width - j, to);
        else load<4, ALIGNED>((const bf16*)weight + j, width - j, to);
    };
    float w[NG ? NG : 1][4];  // the weights do not depend on the kernels in front and are on the way before those are through
    if constexpr (NG > 0) {
#pragma unroll
        for (int i = 0; i < NG; ++i) load_w((threadIdx.x + i * blockDim.x) * 4, w[i]);
    }
    pdl_wait();
    const int64_t at = (int64_t)blockIdx.x * width;
    uint8_t* out = q + (int64_t)blockIdx.x * q_stride;
    auto load_x = [&](int j, float (&x)[4], float (&d)[4]) {
        load<4, ALIGNED>(residual + at + j, width - j, x);
        if (delta) load<4, ALIGNED>(delta + at + j, width - j, d);
    };
    auto finish = [&](int j, float (&x)[4], const float (&d)[4], const float (&wi)[4]) {
        if (delta) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __fadd_rn(x[e], d[e]);
        }
        if (residual_out && j < width) {
            float* to = residual_out + at + j;
            if (ALIGNED && j + 4 <= width) {
                *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j + e < width) to[e] = x[e];
            }
        }
        const float squares = warp_sum(squares_of(x));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= wi[e];
        const uint32_t top = __reduce_max_sync(0xffffffffu, fp8_top(0u, x));
        if (lane == 0 && j < width) {
            sums[j / FP8_BLOCK] = squares;
            tops[j / FP8_BLOCK] = top;
        }
        if (j < width) fp8_store4(out + j, width - j, fp8_quantize4(x, fp8_scale(top)));
    };
    float x[NG ? NG : 1][4], d[NG ? NG : 1][4];
    if constexpr (NG > 0) {
#pragma unroll
        for (int i = 0; i < NG; ++i) load_x((threadIdx.x + i * blockDim.x) * 4, x[i], d[i]);
#pragma unroll
        for (int i = 0; i < NG; ++i) finish((threadIdx.x + i * blockDim.x) * 4, x[i], d[i], w[i]);
    } else {
        for (int j0 = 0; j0 < width; j0 += blockDim.x * 4) {  // (whole warps come along)
            const int j = j0 + threadIdx.x * 4;
            load_w(j, w[0]);
            load_x(j, x[0], d[0]);
            finish(j, x[0], d[0], w[0]);
        }
    }
    __syncthreads();
    float total = 0.f;
    for (int b = lane; b < blocks; b += 32) total += sums[b];
    total = warp_sum(total);
    const float rstd = 1.0f / sqrtf(total / (float)width + eps);
    for (int b = threadIdx.x; b < blocks; b += blockDim.x) scales[blockIdx.x * scale_row + b * scale_block] = norm_scale(tops[b], rstd);
}

// Many wide rows: two or three blocks an SM, each taking rows blockIdx.x, + gridDim.x, ... through a ring of `stages` rows in shared
// memory that one thread fills by bulk copies, so that the rows behind are on their way through both passes over this one.  A stage is
// free when all threads have read their part of it, behind the one barrier a row.  NG groups of four a thread; rows of a multiple of 16
// bytes that start on 16 bytes.
constexpr int RING_THREADS = 256;
constexpr int ring_blocks(int ng) { return ng <= 4 ? 3 : 2; }  // blocks an SM at most

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(s_addr(dst)), "l"(src), "r"(bytes), "r"(s_addr(bar)) : "memory");
}

template <typename T, int NG>
__global__ void __launch_bounds__(RING_THREADS, ring_blocks(NG))
add_rmsnorm_fp8_ring_kernel(const float* residual, const T* delta, float* residual_out, const void* __restrict__ weight, int w_f32,
                            uint8_t* __restrict__ q, int64_t q_stride, float* __restrict__ scales, int64_t scale_row, int64_t scale_block, int rows, int width,
                            float eps, int stages, int* err) {
    extern __shared__ __align__(128) unsigned char ring_smem[];
    constexpr int SETS = NG * RING_THREADS / 32;  // blocks of 128 of the widest row
    __shared__ uint32_t tops[2][SETS];            // (two sets: the next row's are written while slow warps still read these)
    __shared__ float sums[2][SETS];
    __shared__ int gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = (width + FP8_BLOCK - 1) / FP8_BLOCK;
    const int x_bytes = width * 4, d_bytes = delta ? width * (int)sizeof(T) : 0, bytes = x_bytes + d_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(ring_smem + stages * bytes);
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    pdl_launch_dependents();
    float w[NG][4];  // for all rows of the block
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int j = (threadIdx.x + i * RING_THREADS) * 4;
        if (w_f32) load<4, true>((const float*)weight + j, width - j, w[i]);
        else load<4, true>((const bf16*)weight + j, width - j, w[i]);
    }
    pdl_wait();
    int issued = 0;  // copies that thread 0 has sent for
    auto fetch = [&](int64_t row, int s) {
        ++issued;
        mbar_expect_tx(&full[s], bytes);
        bulk_load(ring_smem + s * bytes, residual + row * width, x_bytes, &full[s]);
        if (d_bytes) bulk_load(ring_smem + s * bytes + x_bytes, delta + row * width, d_bytes, &full[s]);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages && blockIdx.x + (int64_t)s * gridDim.x < rows; ++s) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
    int s = 0, n = 0;
    uint32_t parity = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, n ^= 1) {
        const bool landed = mbar_wait(&full[s], parity, &gave_up);
        const float* from = reinterpret_cast<const float*>(ring_smem + s * bytes);
        const T* from_d = reinterpret_cast<const T*>(ring_smem + s * bytes + x_bytes);
        float v[NG][4], part[NG];
        uint32_t top[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * RING_THREADS) * 4;
            if (j < width) {
                load<4, true>(from + j, 4, v[i]);
                if (d_bytes) {
                    float d[4];
                    load<4, true>(from_d + j, 4, d);
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
            top[i] = __reduce_max_sync(0xffffffffu, fp8_top(0u, v[i]));
            if (lane == 0) tops[n][i * (RING_THREADS / 32) + warp] = top[i];
        }
        warp_sums(part, &sums[n][warp], RING_THREADS / 32);
        if (!__syncthreads_and(landed)) break;  // nothing more of the row is written, nothing more is sent for
        if (threadIdx.x == 0 && row + (int64_t)stages * gridDim.x < rows) fetch(row + (int64_t)stages * gridDim.x, s);
        float total = 0.f;
        for (int b = lane; b < blocks; b += 32) total += sums[n][b];
        total = warp_sum(total);
        const float rstd = 1.0f / sqrtf(total / (float)width + eps);
        for (int b = threadIdx.x; b < blocks; b += RING_THREADS) scales[row * scale_row + b * scale_block] = norm_scale(tops[n][b], rstd);
        // (a lane a division: lane i what the values of the warp's block i are multiplied by)
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i)
            if (lane == i) mine = top[i];
        const Fp8Factor f = fp8_factor(mine, true);
        uint8_t* out = q + row * q_stride;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int j = (threadIdx.x + i * RING_THREADS) * 4;
            Fp8Scale r;
            r.inverse = __shfl_sync(0xffffffffu, f.value, i);
            r.before = __shfl_sync(0xffffffffu, f.before, i);
            r.keep = r.inverse == 0.f ? 0u : 0xffffffffu;
            if (j < width) *reinterpret_cast<uint32_t*>(out + j) = fp8_quantize4(v[i], r);
        }
        if (++s == stages) { s = 0; parity ^= 1; }
    }
    // behind a wait that gave up: the error word, and a wait for the block's copies in flight, the last of those that thread 0 has sent for
    if (*(volatile int*)&gave_up && threadIdx.x == 0) {
        for (int i = max(0, issued - stages); i < issued; ++i) mbar_drain(&full[i % stages], (i / stages) & 1);
        atomicOr(err, SS_ERR_WAIT_LIMIT);
    }
}

// ---------------------------------------------------------------- fp8 to values
//
// y = q * s, rounded once.  A lane takes eight (bfloat16) or four (float32) elements, side by side where the output's rows start on 16
// bytes, else 32 apart, so that a warp writes whole pieces of a row either way (1,531 x 2,051 to bfloat16, side by side and one by one:
// 22.4 us for 7.9).  Groups are dealt out as in the way there.  Bound by memory: 4,096 x 3,584 to bfloat16 8.4 us (5.2 TB/s), a weight of 18,944 x 3,584
// 33.0 (6.2).
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(ROW_THREADS)
dequantize_kernel(const uint8_t* q, int64_t q_stride, const float* scales, int64_t scale_row, int64_t scale_block, T* __restrict__ y, int64_t rows,
                  int width, int groups, int shift, int early) {
    constexpr int V = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    if (early) pdl_launch_dependents();
    pdl_wait();
    Place p[ROW_GROUPS];
    uint32_t w[ROW_GROUPS][V / 4];
    float s[ROW_GROUPS][ALIGNED ? 1 : (32 * V + FP8_BLOCK - 1) / FP8_BLOCK];
#pragma unroll
    for (int i = 0; i < ROW_GROUPS; ++i) {
        p[i] = place_of<V>(i, groups);
        if (p[i].row >= rows) continue;
        const uint8_t* from = q + p[i].row * q_stride;
        const float* scale = scales + (p[i].row >> shift) * scale_row;
        if constexpr (ALIGNED) {
            p[i].column += lane * V;
            if (p[i].column >= width) continue;
            s[i][0] = scale[p[i].column / FP8_BLOCK * scale_block];
            // (the width is a multiple of V)
            if constexpr (V == 8) *reinterpret_cast<uint2*>(w[i]) = *reinterpret_cast<const uint2*>(from + p[i].column);
            else w[i][0] = *reinterpret_cast<const uint32_t*>(from + p[i].column);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int j = p[i].column + e * 32 + lane;
                if (e % 4 == 0) {
                    w[i][e / 4] = 0;
                    s[i][e / 4] = j - lane < width ? scale[(j - lane) / FP8_BLOCK * scale_block] : 0.f;  // (four times 32 columns: a block)
                }
                if (j < width) w[i][e / 4] |= (uint32_t)from[j] << (8 * (e % 4));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROW_GROUPS; ++i) {
        if (p[i].row >= rows || (ALIGNED && p[i].column >= width)) continue;
        T* to = y + (int64_t)p[i].row * width;
        T v[V];
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            float f[4];
            fp8_values4(w[i][e / 4], f);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[e + k] = from_float<T>(f[k] * s[i][ALIGNED ? 0 : e / 4]);
        }
        if constexpr (ALIGNED) {
            *reinterpret_cast<uint4*>(to + p[i].column) = *reinterpret_cast<const uint4*>(v);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int j = p[i].column + e * 32 + lane;
                if (j < width) to[j] = v[e];
            }
        }
    }
    if (!early) publish_results();
}

// ---------------------------------------------------------------- launches

inline bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int refused(const Fp8RowsCall& c) {
    return c.width <= 0 || c.width > FP8_MAX_WIDTH || c.rows > INT32_MAX || c.q_stride % 16 || !on16(c.q) ? -2003 : 0;
}

// Blocks of threads for `rows` rows of `groups` groups, or 0 where they are too many.
unsigned row_blocks(int64_t rows, int groups) {
    const int64_t n = (rows * groups + ROW_WARPS * ROW_GROUPS - 1) / (ROW_WARPS * ROW_GROUPS);
    return n * ROW_WARPS * ROW_GROUPS > UINT32_MAX ? 0u : (unsigned)n;
}

template <typename T, bool ALIGNED>
int launch_quantize(const Fp8RowsCall& c) {
    const int width = (int)c.width, groups = (int)((c.width + 512 / sizeof(T) - 1) / (512 / sizeof(T)));
    if (c.blocks) {
        const int64_t across = (c.width + FP8_BLOCK - 1) / FP8_BLOCK;
        const int64_t n = across * ((c.rows + FP8_BLOCK - 1) / FP8_BLOCK);
        if (n > INT32_MAX) return -2003;
        ss_launch(quantize_blocks_kernel<T, ALIGNED>, dim3((unsigned)n), dim3(ROW_THREADS), 0, c.stream, (const T*)c.x, c.stride, c.q, c.q_stride, c.scales,
                  c.scale_row, c.scale_block, c.rows, width, (unsigned)across);
    } else {
        const int64_t n = (c.rows + ROW_WARPS * ROW_GROUPS - 1) / (ROW_WARPS * ROW_GROUPS) * groups;
        if (n > INT32_MAX) return -2003;
        ss_launch(quantize_rows_kernel<T, ALIGNED>, dim3((unsigned)n), dim3(ROW_THREADS), 0, c.stream, (const T*)c.x, c.stride, c.q, c.q_stride, c.scales, c.scale_row,
                  c.scale_block, c.rows, width, (unsigned)groups, (int)c.early);
    }
    return SS_LAUNCH_CHECK();
}

// Groups of four of a row: NG a thread and the threads of a block (NG = 0: a loop).
struct RowShape { int ng, threads; };
inline RowShape norm_shape(int width, int64_t rows) {
    const int groups = (width + 3) / 4;
    const bool few = rows <= 2 * (int64_t)ss_sm_count();
    for (int ng : {1, 2, 4}) {
        const int threads = ((groups + ng - 1) / ng + 31) / 32 * 32;
        if (threads <= (few ? 1024 : 512)) return {ng, threads};
    }
    return {0, 512};
}

// The ring: blocks an SM, and stages of a block's ring (0: the rows are too few, too narrow or too wide).  Three rows in flight a
// block where three blocks share an SM, else two at least; four rows a block at least.
struct RingShape { int blocks, stages; };
constexpr int RING_SMEM = 112 * 1024;  // of a block, two of which share an SM
inline int ring_groups(int width) {
    const int ng = (width / 4 + RING_THREADS - 1) / RING_THREADS;
    return ng <= 4 ? ng : ng <= 6 ? 6 : ng <= 8 ? 8 : ng <= 10 ? 10 : 12;
}
inline RingShape ring_shape(const Fp8RowsCall& c) {
    const int64_t bytes = c.width * (4 + (!c.delta ? 0 : c.dtype == SS_BF16 ? 2 : 4));
    if (bytes < 16384 || c.width > 12 * 4 * RING_THREADS || bytes % 16 || (c.delta && c.width * 2 % 16)) return {0, 0};
    for (int blocks = ring_blocks(ring_groups((int)c.width)); blocks >= 2; --blocks) {
        const int64_t stages = (220 * 1024 / blocks - 3 * 1024) / (bytes + 8);
        if (stages >= blocks && c.rows >= 4 * (int64_t)blocks * ss_sm_count()) return {blocks, (int)stages};
    }
    return {0, 0};
}
template <typename T>
int launch_norm_ring(const Fp8RowsCall& c, RingShape shape) {
    const int smem = (int)(shape.stages * (c.width * (4 + (c.delta ? sizeof(T) : 0)) + 8)) + 64;
    int rc = 0;
#define NORM(NG) case NG: { \
        static SsPerDevice opted; \
        if ((rc = ss_opt_in_smem(add_rmsnorm_fp8_ring_kernel<T, NG>, RING_SMEM, opted))) return rc; \
        ss_launch(add_rmsnorm_fp8_ring_kernel<T, NG>, dim3(shape.blocks * ss_sm_count()), dim3(RING_THREADS), smem, c.stream, (const float*)c.x, (const T*)c.delta, (float*)c.y, c.weight, (int)c.w_f32, c.q, c.q_stride, c.scales, c.scale_row, c.scale_block, (int)c.rows, (int)c.width, (float)c.eps, shape.stages, c.err); \
    } break
    switch (ring_groups((int)c.width)) { NORM(2); NORM(3); NORM(4); NORM(6); NORM(8); NORM(10); NORM(12); }
#undef NORM
    return SS_LAUNCH_CHECK();
}

template <typename T, bool ALIGNED>
int launch_norm(const Fp8RowsCall& c) {
    if constexpr (ALIGNED) {
        const RingShape ring = ring_shape(c);
        if (ring.blocks) return launch_norm_ring<T>(c, ring);
    }
    const int width = (int)c.width;
    const RowShape shape = norm_shape(width, c.rows);
    const int64_t smem = (c.width + FP8_BLOCK - 1) / FP8_BLOCK * 8;
    if (smem > 48 * 1024) return -2003;
#define NORM(NG) case NG: ss_launch(add_rmsnorm_fp8_kernel<T, ALIGNED, NG>, dim3((unsigned)c.rows), dim3(shape.threads), (size_t)smem, c.stream, (const float*)c.x, (const T*)c.delta, (float*)c.y, c.weight, (int)c.w_f32, c.q, c.q_stride, c.scales, c.scale_row, c.scale_block, width, (float)c.eps); break
    switch (shape.ng) { NORM(0); NORM(1); NORM(2); NORM(4); }
#undef NORM
    return SS_LAUNCH_CHECK();
}

template <typename T, bool ALIGNED>
int launch_dequantize(const Fp8RowsCall& c) {
    const int groups = (int)((c.width + 512 / sizeof(T) - 1) / (512 / sizeof(T)));
    const unsigned n = row_blocks(c.rows, groups);
    if (!n) return -2003;
    ss_launch(dequantize_kernel<T, ALIGNED>, dim3(n), dim3(ROW_THREADS), 0, c.stream, c.q, c.q_stride, c.scales, c.scale_row, c.scale_block, (T*)c.y, c.rows,
              (int)c.width, groups, c.blocks ? 7 : 0, (int)c.early);
    return SS_LAUNCH_CHECK();
}

}  // namespace

extern "C" int ss_quantize_fp8(const Fp8RowsCall* call) {
    const Fp8RowsCall& c = *call;
    if (c.rows <= 0) return 0;
    if (int rc = refused(c)) return rc;
    const bool aligned = on16(c.x) && c.stride * (c.dtype == SS_BF16 ? 2 : 4) % 16 == 0;
    if (c.dtype == SS_BF16) return aligned ? launch_quantize<bf16, true>(c) : launch_quantize<bf16, false>(c);
    return aligned ? launch_quantize<float, true>(c) : launch_quantize<float, false>(c);
}

extern "C" int ss_add_rmsnorm_fp8(const Fp8RowsCall* call) {
    const Fp8RowsCall& c = *call;
    if (c.rows <= 0) return 0;
    if (int rc = refused(c)) return rc;
    const bool aligned = c.width % 4 == 0 && on16(c.x) && on16(c.delta) && on16(c.y) && on16(c.weight);
    if (c.dtype == SS_BF16) return aligned ? launch_norm<bf16, true>(c) : launch_norm<bf16, false>(c);
    return aligned ? launch_norm<float, true>(c) : launch_norm<float, false>(c);
}

// early, here and in rows of the way there: the kernel behind may start at once; it may then have read what it takes for constant before the results are written, so only for
// results that it does not take for that (weights are).
extern "C" int ss_dequantize_fp8(const Fp8RowsCall* call) {
    const Fp8RowsCall& c = *call;
    if (c.rows <= 0) return 0;
    if (int rc = refused(c)) return rc;
    const bool aligned = on16(c.y) && c.width * (c.dtype == SS_BF16 ? 2 : 4) % 16 == 0;
    if (c.dtype == SS_BF16) return aligned ? launch_dequantize<bf16, true>(c) : launch_dequantize<bf16, false>(c);
    return aligned ? launch_dequantize<float, true>(c) : launch_dequantize<float, false>(c);
}
extern "C" void ss_set_pdl(int on) { ss_pdl_flag() = on; }

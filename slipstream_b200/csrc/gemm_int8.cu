// Matrix product of 8-bit integers on the 5th-generation tensor cores of sm_100a:
//   Y[m, n] = (sum_k X[m, k] * W[n, k]) * x_scale[m] * w_scale[n] (+ bias[n])
// X: activations, one row and one scale a token; W: weights, one row and one scale an output feature; both int8 and K-major.
// The sum is exact: products and additions are 32-bit integers (tcgen05.mma kind::i8; 2^14 K < 2^31 up to K = 131,071, whatever the bytes), so a
// result does not depend on how K is cut, on the kernel or on what else is in the batch.  What follows is float32: the sum is
// converted (one rounding from 2^24 on), multiplied by the token's scale, then by the feature's, then the bias is added, and
// the result is rounded once to the output type.  The gated form pairs the features of a feed-forward's gate and up matrices
// (stacked in runs of 64 rows each) and writes silu(gate) * up.
//
// A row's stage in shared memory is 128 bytes, 128 elements of K, under the 128-byte swizzle; an instruction takes 32 of them.
//
// Every wait on an mbarrier is bounded: after WAIT_LIMIT polls the kernel sets SS_ERR_WAIT_LIMIT in the error word, stops
// waiting everywhere, writes out nothing that it has not formed, waits (with the same limit) for its copies and products in flight,
// frees its tensor memory and returns.
//
// Tensor memory is taken BEHIND griddepcontrol.wait, and the kernel behind is let go only when it has been taken: a kernel
// that takes it before the kernel in front is through, or lets a kernel start that may take it first, can wait for a block
// that waits for it.  Before that wait a block reads only the weights, their scales and the bias, which it takes for constant.

#include <cuda.h>

#include "int8_calls.h"
#include "tc5.cuh"

#define I8_BM 128
#define I8_BK 128       // K elements, and bytes of a row, in a stage
#define I8_THREADS 192
#define I8_MAX_BN 256

struct Int8Args {
    const float* x_scale;  // [tokens]
    const float* w_scale;  // [features]
    const void* bias;      // [features] or null
    void* out;             // [tokens][ldc]
    int* err;
    int64_t ldc;
    int tokens, features, K;
    int out_features;      // columns written: features, or the gated form's (at most features / 2)
    int out_f32, bias_f32, gated;
    int bn;                // few tokens: the tokens of a tile; many tokens: the features of a tile
    int stages, slices;
    int wide_copies;       // the two steps of a stage come in one copy (K is a multiple of 128)
};

__device__ __forceinline__ void i8_load(void* dst, const CUtensorMap* map, int k, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(s_addr(dst)), "l"(map), "r"(s_addr(bar)), "r"(k), "r"(row) : "memory");
}
// weights that are read once a step: the first to leave L2 again
__device__ __forceinline__ void i8_load_once(void* dst, const CUtensorMap* map, int k, int row, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
        ::"r"(s_addr(dst)), "l"(map), "r"(s_addr(bar)), "r"(k), "r"(row), "l"(policy) : "memory");
}
// Two steps of K in one copy: the map's third coordinate counts steps.
__device__ __forceinline__ void i8_load_steps(void* dst, const CUtensorMap* map, int step, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(s_addr(dst)), "l"(map), "r"(s_addr(bar)), "r"(0), "r"(row), "r"(step) : "memory");
}
__device__ __forceinline__ void i8_load_steps_once(void* dst, const CUtensorMap* map, int step, int row, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;"
        ::"r"(s_addr(dst)), "l"(map), "r"(s_addr(bar)), "r"(0), "r"(row), "r"(step), "l"(policy) : "memory");
}
// `rows` rows of the steps of K of stage k, as [step][row][128 bytes]
template <int STEPS, bool ONCE>
__device__ __forceinline__ void i8_load_stage(unsigned char* dst, const CUtensorMap* map, bool wide, int k, int row, int rows, uint64_t* bar, uint64_t policy) {
    if (STEPS == 2 && wide) {
        if (ONCE) i8_load_steps_once(dst, map, 2 * k, row, bar, policy);
        else i8_load_steps(dst, map, 2 * k, row, bar);
        return;
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (ONCE) i8_load_once(dst + i * rows * I8_BK, map, (STEPS * k + i) * I8_BK, row, bar, policy);
        else i8_load(dst + i * rows * I8_BK, map, (STEPS * k + i) * I8_BK, row, bar);
    }
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// Instruction descriptor: D signed 32-bit, A and B signed 8-bit, both K-major.
__device__ __forceinline__ uint32_t i8_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Behind a wait that gave up: the error word, and a wait for the last of the `copies` stages that were sent for, which may still be
// in flight.
__device__ __noinline__ void i8_gave_up(const Int8Args& g, uint64_t* full, int stages, int copies) {
    atomicOr(g.err, SS_ERR_WAIT_LIMIT);
    for (int i = max(0, copies - stages); i < copies; ++i) mbar_drain(&full[i % stages], (i / stages) & 1);
}

// A barrier that is used once a launch, behind a wait that gave up.  (Out of line, as i8_gave_up: in the epilogue's way it cost 0.1 us of
// 13 at 16 x 18,944 x 3,584.)
__device__ __noinline__ void i8_drain(uint64_t* bar) { mbar_drain(bar, 0); }

__device__ __forceinline__ float i8_bias(const Int8Args& g, int f) {
    return g.bias_f32 ? ((const float*)g.bias)[f] : to_float(((const bf16*)g.bias)[f]);
}
// The sum as a result: in this order everywhere, no fused multiply-add, so that both kernels give the same bits.
__device__ __forceinline__ float i8_value(int sum, float xs, float ws, float bias) {
    return __fadd_rn(__fmul_rn(__fmul_rn((float)sum, xs), ws), bias);
}
__device__ __forceinline__ float i8_gate(const Int8Args& g, float gate, float up) {
    return g.out_f32 ? silu_mul<false>(gate, up) : silu_mul<true>(gate, up);
}

// Whether `v` holds in all 128 threads of the few tokens' epilogue; a barrier of theirs.
__device__ __forceinline__ bool i8_epilogue_all(bool v) {
    uint32_t all;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 q, %1, 0;\n"
        "bar.red.and.pred p, 1, 128, q;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(all) : "r"((uint32_t)v) : "memory");
    return all != 0;
}

// Four outputs of a token, `apart` features from one another.
__device__ __forceinline__ void i8_store4(const Int8Args& g, int token, int f, int apart, const float (&v)[4]) {
    const int64_t at = (int64_t)token * g.ldc + f;
    if (apart == 1 && f + 4 <= g.out_features) {
        if (g.out_f32) {
            *reinterpret_cast<float4*>((float*)g.out + at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
            uint2 packed;
            packed.x = *reinterpret_cast<const uint32_t*>(&lo);
            packed.y = *reinterpret_cast<const uint32_t*>(&hi);
            *reinterpret_cast<uint2*>((bf16*)g.out + at) = packed;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (f + e * apart >= g.out_features) break;
        if (g.out_f32) ((float*)g.out)[at + e * apart] = v[e];
        else ((bf16*)g.out)[at + e * apart] = __float2bfloat16_rn(v[e]);
    }
}

// sum at `to` in the shared memory of block `rank` of the cluster += v; four bytes of the transaction that `bar` there counts
__device__ __forceinline__ void i8_add_remote(uint32_t to, uint32_t bar, int v) {
    asm volatile("red.async.relaxed.cluster.shared::cluster.mbarrier::complete_tx::bytes.add.s32 [%0], %1, [%2];"
                 ::"r"(to), "r"(v), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t i8_remote(const void* p, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(s_addr(p)), "r"(rank));
    return remote;
}

// ---------------------------------------------------------------- few tokens: the weights' bytes are the work
//
// The weights are the instruction's A (their rows fill its 128 lanes), the tokens its B (bn of them, a multiple of 16 up to
// 256).  A block forms a tile of 128 features x bn tokens over one slice of K.  The 1 to 8 slices of a tile are a thread-block
// cluster along grid.z: token column c belongs to block c % slices, and every block adds its sums of the column into that
// block's shared memory from its registers (red.async; whole numbers, so in any order), which counts the bytes on a barrier of its
// own.  No block waits for another but for these sums.  Warp 0 (one lane) fetches, warp 1 issues the products, warps 2 to 5
// write the result out.
template <int STEPS>
__global__ void __launch_bounds__(I8_THREADS)
gemm_int8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Int8Args g) {
    extern __shared__ unsigned char smem_raw[];
    const int bn = g.bn, stages = g.stages, n_sl = g.slices;
    constexpr int w_bytes = STEPS * I8_BM * I8_BK;
    const int stage_bytes = w_bytes + STEPS * bn * I8_BK;
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + stages * stage_bytes);
    uint64_t* empty = full + stages;
    uint64_t* acc_ready = empty + stages;
    uint64_t* sums_ready = acc_ready + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_ready + 1);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* xs_s = reinterpret_cast<float*>(full) + 64;  // [256], behind the barriers
    // [own columns][128]: of a cluster's block behind the scales; alone over the ring, when all its stages have been used
    int* sums = n_sl > 1 ? reinterpret_cast<int*>(xs_s + I8_MAX_BN) : reinterpret_cast<int*>(tiles);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t0 = blockIdx.x * bn, f0 = blockIdx.y * I8_BM;  // first token, first feature
    const int live = min(bn, g.tokens - t0);                   // columns that hold tokens
    const int rank = n_sl > 1 ? (int)cluster_rank() : 0;
    const int mine = live > rank ? (live - 1 - rank) / n_sl + 1 : 0;  // columns rank, rank + slices, ...
    const int k_steps = (g.K + I8_BK - 1) / I8_BK, k_total = (k_steps + STEPS - 1) / STEPS;  // stages of K, of all slices
    const int per = (k_total + n_sl - 1) / n_sl;
    const int k_begin = blockIdx.z * per, k_iters = max(0, min(k_total, k_begin + per) - k_begin);
    const int senders = (k_total + per - 1) / per;  // blocks that have any K
    const int ahead = min(stages, k_iters);
    const uint32_t tmem_cols = bn <= 32 ? 32 : bn <= 64 ? 64 : bn <= 128 ? 128 : 256;
    int copies = 0;  // stages that thread 0 has sent for

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(acc_ready, 1);
        mbar_init(sums_ready, 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (n_sl > 1) mbar_expect_tx(sums_ready, (uint32_t)(senders * mine * I8_BM * 4));
        // the weights do not depend on the kernels in front: their first tiles are on the way before those are through
        const uint64_t once = l2_evict_first_policy();
        for (int it = 0; it < ahead; ++it) {
            mbar_expect_tx(&full[it], stage_bytes);
            i8_load_stage<STEPS, true>(tiles + it * stage_bytes, &map_w, g.wide_copies, k_begin + it, f0, I8_BM, &full[it], once);
        }
    } else if (warp >= 2 && n_sl > 1) {
        for (int i = threadIdx.x - 64; i < mine * (I8_BM / 4); i += 128) reinterpret_cast<int4*>(sums)[i] = make_int4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    if (n_sl > 1) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // this block's sums are zero and its barriers stand
        if (warp < 2) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t once = l2_evict_first_policy();
            pdl_wait();
            for (int it = 0; it < ahead; ++it)
                i8_load_stage<STEPS, false>(tiles + it * stage_bytes + w_bytes, &map_x, g.wide_copies, k_begin + it, t0, bn, &full[it], once);
            // (a stage's number and its parity are counted, not divided out: the loops of this thread and of the issuer are what a
            // step takes where its products are small)
            int it = ahead, s = 0;
            uint32_t parity = 0;
            for (; it < k_iters; ++it) {
                if (!mbar_wait(&empty[s], parity, gave_up)) break;
                mbar_expect_tx(&full[s], stage_bytes);
                i8_load_stage<STEPS, true>(tiles + s * stage_bytes, &map_w, g.wide_copies, k_begin + it, f0, I8_BM, &full[s], once);
                i8_load_stage<STEPS, false>(tiles + s * stage_bytes + w_bytes, &map_x, g.wide_copies, k_begin + it, t0, bn, &full[s], once);
                if (++s == stages) { s = 0; parity ^= 1; }
            }
            copies = it;
        }
        __syncwarp();
    } else if (warp == 1) {
        pdl_wait();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_slot)), "r"(tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        pdl_launch_dependents();  // (this warp alone: one call of a block lets the kernel behind go)
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.arrive 2, 160;" ::: "memory");  // the epilogue warps read the slot behind it
        const uint32_t tmem_acc = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
        const uint32_t idesc = i8_idesc(I8_BM, bn);
        const uint64_t w_first = smem_desc(tiles), x_first = smem_desc(tiles + w_bytes);
        const uint32_t stage_step = (uint32_t)stage_bytes >> 4, x_step = (uint32_t)(bn * I8_BK) >> 4;  // of a descriptor's address
        int s = 0;
        uint32_t parity = 0;
        for (int it = 0; it < k_iters; ++it) {
            if (!__all_sync(0xffffffffu, mbar_wait(&full[s], parity, gave_up))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t w_desc = w_first + s * stage_step, x_desc = x_first + s * stage_step;
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < I8_BK / 32; ++kk)  // 32 bytes further along the swizzled row
                    umma_i8(tmem_acc, w_desc + (uint64_t)(kk * 2), x_desc + (uint64_t)(kk * 2), idesc, (it | kk) != 0);
                if (STEPS == 2 && 2 * (k_begin + it) + 1 < k_steps) {
#pragma unroll
                    for (int kk = 0; kk < I8_BK / 32; ++kk)
                        umma_i8(tmem_acc, w_desc + (uint64_t)(I8_BM * I8_BK / 16 + kk * 2), x_desc + (uint64_t)(x_step + kk * 2), idesc, 1);
                }
                umma_commit(&empty[s]);
            }
            __syncwarp();
            if (++s == stages) { s = 0; parity ^= 1; }
        }
        if (elect_one()) umma_commit(acc_ready);
        __syncwarp();
    } else {
        // nor do the scales and the bias of the four features (gated: four pairs) depend on the kernels in front that a lane writes
        // out: neighbours, or, where the output's rows do not start on four elements, one of each quarter of the tile
        const int quarter = warp & 3;
        const int half = g.gated ? lane >> 4 : 0, of = g.gated ? lane & 15 : lane;
        const int apart = (g.ldc & 3) == 0 ? 1 : g.gated ? 16 : 32, fl = apart == 1 ? of * 4 : of;
        float ws[4], bs[4], ws2[4], bs2[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int f = f0 + fl + e * apart, f2 = f + 64;
            ws[e] = f < g.features ? __ldg(g.w_scale + f) : 0.f;
            bs[e] = g.bias && f < g.features ? i8_bias(g, f) : 0.f;
            ws2[e] = g.gated && f2 < g.features ? __ldg(g.w_scale + f2) : 0.f;
            bs2[e] = g.gated && g.bias && f2 < g.features ? i8_bias(g, f2) : 0.f;
        }
        if (n_sl > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        pdl_wait();  // the output may still be in use by the kernels in front, which also wrote the tokens' scales
        for (int i = threadIdx.x - 64; i < live; i += 128) xs_s[i] = g.x_scale[t0 + i];
        asm volatile("bar.sync 2, 160;" ::: "memory");  // the scales are there, and the tensor memory's address
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc = *reinterpret_cast<volatile uint32_t*>(tmem_slot) + ((uint32_t)(quarter * 32) << 16);
        // (the flag, not the wait's result: an issuer that gave up still commits, so that the accumulator can be waited for, and copies may
        // then be landing where the sums would go; a vote over the results cost 0.3 us)
        (void)mbar_wait(acc_ready, 0, gave_up);
        bool ok = !__shfl_sync(0xffffffffu, *gave_up, 0);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (n_sl == 1) {
            for (int c = 0; ok && c < live; c += 16) {
                uint32_t r[16];
                tmem_ld16(acc + c, r);
#pragma unroll
                for (int j = 0; j < 16; ++j) sums[(c + j) * I8_BM + quarter * 32 + lane] = (int)r[j];
            }
            ok = i8_epilogue_all(ok);
        } else {
            if (k_iters > 0) {
                int owner = 0, at = 0;  // of column c: block c % slices, its column c / slices
                for (int c = 0; c < live; c += 16) {
                    // a warp that gave up sends zeros: the bytes that the owners count always arrive, so that none of them leaves with
                    // sums on their way to it (what they write is wrong then; the error word says so)
                    uint32_t r[16] = {};
                    if (ok) tmem_ld16(acc + c, r);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (c + j < live)
                            i8_add_remote(i8_remote(sums + at * I8_BM + quarter * 32 + lane, owner), i8_remote(sums_ready, owner), (int)r[j]);
                        if (++owner == n_sl) { owner = 0; ++at; }
                    }
                }
            }
            if (!mbar_wait(sums_ready, 0, gave_up)) i8_drain(sums_ready);
            ok = !*gave_up;
        }
        // a warp takes a token column (gated: each of its halves one) at a time, a lane four features of it
        for (int i = g.gated ? 2 * quarter + half : quarter; ok && i < mine; i += g.gated ? 8 : 4) {
            const int c = rank + i * n_sl;
            const int* from = sums + i * I8_BM + fl;
            const float xs = xs_s[c];
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = i8_value(from[e * apart], xs, ws[e], bs[e]);
                if (g.gated) v[e] = i8_gate(g, v[e], i8_value(from[e * apart + 64], xs, ws2[e], bs2[e]));
            }
            i8_store4(g, t0 + c, (g.gated ? f0 / 2 : f0) + fl, apart, v);
        }
    }
    if (n_sl > 1) {  // nobody leaves while others may still send to it: each has seen the sums that it owns arrive
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
        asm volatile("barrier.cluster.wait;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*gave_up && threadIdx.x == 0) i8_gave_up(g, full, stages, copies);
    if (warp == 1) {
        if (*gave_up) i8_drain(acc_ready);  // products in flight
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t tmem_acc = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_acc), "r"(tmem_cols));
    }
}

// ---------------------------------------------------------------- many tokens: the tensor cores are the work
//
// A persistent kernel on pairs of SMs (tcgen05.mma.cta_group::2).  A pair walks over tiles of 256 tokens x bn features, token
// tiles fastest.  Block r of the pair fetches tokens r * 128 .. of the tile and half of its features' weights; the leader
// (block 0) issues the products, which leave the tokens of block r in block r's tensor memory.  The accumulator is
// double-buffered (2 x 256 columns): the sixteen epilogue warps of each block write a tile out while the next one is formed.
//   full[s]      in the leader: the bytes of both blocks' copies;     empty[s]     in each block: the products have read the stage
//   acc_full[b]  in each block: the tile's products are through;      acc_empty[b] in the leader: all 32 epilogue warps are
//
// The epilogue has as many warps as registers allow, four of a scheduler's: with eight, which took about 14,000 cycles of latencies for a
// gated tile of 256 x 256, products of short K waited for them.  For the same reason the kernel is compiled for each output type, with
// and without the gate, what a tile's epilogue reads is fetched a tile ahead, and an accumulator is handed back as soon as it
// has been read, not when the outputs have been written.  Gated 4,096 x 896 x 9,728: 70.7 to 39.6 us, 2,048 x 1,536 x 17,920: 66.1 to 44,
// 4,099 x 3,584 x 37,888: 353 to 345 (in a burst).
#define I8_MANY_THREADS 576  // producer, issuer, sixteen epilogue warps

__device__ __forceinline__ uint32_t i8_leader(const void* p) { return s_addr(p) & 0xFEFFFFFFu; }  // same offset in block 0 of the pair

__device__ __forceinline__ void i8_load_pair(void* dst, const CUtensorMap* map, int k, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(s_addr(dst)), "l"(map), "r"(i8_leader(bar)), "r"(k), "r"(row) : "memory");
}
// two steps of K in one copy: the map's third coordinate counts steps
__device__ __forceinline__ void i8_load_pair_steps(void* dst, const CUtensorMap* map, int step, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(s_addr(dst)), "l"(map), "r"(i8_leader(bar)), "r"(0), "r"(row), "r"(step) : "memory");
}
// `rows` rows of the steps of K of stage k, as [step][row][128 bytes]
template <int STEPS>
__device__ __forceinline__ void i8_load_pair_stage(unsigned char* dst, const CUtensorMap* map, bool wide, int k, int row, int rows, uint64_t* bar) {
    if (STEPS == 2 && wide) {
        i8_load_pair_steps(dst, map, 2 * k, row, bar);
        return;
    }
    i8_load_pair(dst, map, STEPS * k * I8_BK, row, bar);
    if (STEPS == 2) i8_load_pair(dst + rows * I8_BK, map, (2 * k + 1) * I8_BK, row, bar);
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void i8_commit_pair(uint64_t* bar) {  // arrives at `bar` in both blocks of the pair
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(s_addr(bar)), "h"((unsigned short)3) : "memory");
}
// A warp is through with what it read of an accumulator (its tcgen05.wait::ld is behind it).  Nothing that it wrote is handed on
// with the arrival, so that need not wait for its stores to global memory, as one with release semantics does.
__device__ __forceinline__ void i8_release_acc(uint64_t* bar) {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
        asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(i8_leader(bar)) : "memory");
}

// 16 columns of the accumulator, or (both) 16 and the 16 that stand 64 behind them
__device__ __forceinline__ void i8_tmem_ld16(uint32_t taddr, bool both, uint32_t (&r)[16], uint32_t (&u)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    if (both) {
        tmem_ld16(taddr + 64, u);  // (waits for both)
        return;
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// 16 sums of a token as values, in place; ws and bs: the features' scales and biases, in shared memory.
__device__ __forceinline__ void i8_values16(uint32_t (&r)[16], float xs, const float* ws, const float* bs) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        const float4 w = *reinterpret_cast<const float4*>(ws + e), b = *reinterpret_cast<const float4*>(bs + e);
        r[e] = __float_as_uint(i8_value((int)r[e], xs, w.x, b.x));
        r[e + 1] = __float_as_uint(i8_value((int)r[e + 1], xs, w.y, b.y));
        r[e + 2] = __float_as_uint(i8_value((int)r[e + 2], xs, w.z, b.z));
        r[e + 3] = __float_as_uint(i8_value((int)r[e + 3], xs, w.w, b.w));
    }
}
// 16 rows of 64 bytes from `stage` to rows of the output that start on P bytes, P bytes a thread; `limit`: the bytes
// of a run that are there.
template <typename P>
__device__ __forceinline__ void i8_copy_run(const unsigned char* stage, unsigned char* out, int64_t pitch, int rows, int limit) {
    constexpr int per_row = 64 / (int)sizeof(P);
    const int lane = threadIdx.x & 31, at = lane % per_row * (int)sizeof(P);
#pragma unroll
    for (int i = 0; i < per_row / 2; ++i) {
        const int r = i * (32 / per_row) + lane / per_row;
        const P v = *reinterpret_cast<const P*>(stage + r * 64 + (((at >> 4) ^ ((r >> 1) & 3)) << 4) + (at & 15));
        if (r < rows && at < limit) *reinterpret_cast<P*>(out + r * pitch + at) = v;
    }
}
// The same for rows of any number of bfloat16 elements, in words: what lies in `stage` of a row that starts between two words begins
// with its second element and has two elements less, which are written elsewhere.  (2,047 x 3,584 x 4,613 to bfloat16: 37.8 us element by
// element, 31.4 so; to float32, where it is the loop above that copies words, 36.8 to 31.6.)
__device__ __forceinline__ void i8_copy_run_odd(const unsigned char* stage, unsigned char* out, int64_t pitch, int rows, int limit) {
    const int lane = threadIdx.x & 31, at = (lane & 15) * 4;
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
        const int r = 2 * i + (lane >> 4);
        const uint32_t v = *reinterpret_cast<const uint32_t*>(stage + r * 64 + (((at >> 4) ^ ((r >> 1) & 3)) << 4) + (at & 15));
        unsigned char* to = out + r * pitch;
        const int odd = (int)((uintptr_t)to & 2), left = min(limit - odd, 64 - 2 * odd) - at;
        to += odd + at;
        if (r >= rows) continue;
        if (left >= 4) *reinterpret_cast<uint32_t*>(to) = v;
        else if (left == 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)v;
    }
}
// A warp's 32 rows of 64 bytes, a row a thread, through 1 KB of shared memory of the warp's own, so that it writes whole
// 64-byte runs of a row instead of 16 bytes of 32 rows at a time (2,048 x 3,584 x 9,472: 49.8 to 46.3 us).  Rows of 64 bytes lie in `stage`
// with their four 16-byte pieces turned by (row / 2) % 4, which keeps both directions free of bank conflicts.
template <typename T, int PIECE>
__device__ __forceinline__ void i8_write_run(const Int8Args& g, unsigned char* stage, const uint32_t (&w)[16], int m0, int f) {
    const int lane = threadIdx.x & 31, size = (int)sizeof(T), row = lane & 15;
    const int64_t pitch = g.ldc * size;
    unsigned char* out = (unsigned char*)g.out + m0 * pitch + (int64_t)f * size;
    const int rows = g.tokens - m0, limit = min(64, (g.out_features - f) * size);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        __syncwarp();
        if (lane >> 4 == h) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint4*>(stage + row * 64 + ((q ^ ((row >> 1) & 3)) << 4)) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        }
        __syncwarp();
        if constexpr (PIECE == 16) i8_copy_run<uint4>(stage, out + 16 * h * pitch, pitch, rows - 16 * h, limit);
        else if constexpr (PIECE == 4) i8_copy_run<uint32_t>(stage, out + 16 * h * pitch, pitch, rows - 16 * h, limit);
        else i8_copy_run_odd(stage, out + 16 * h * pitch, pitch, rows - 16 * h, limit);
    }
}
// A run of 64 bytes (16 or 32 outputs) of each of a warp's 32 tokens, from f on, from the accumulator's columns at `acc` on, whose
// scales and biases are at ws and bs.  `through`: the barrier to arrive at when the accumulator has been read, or null.
template <typename T, int PIECE, bool GATED>
__device__ __forceinline__ void i8_write_outputs(const Int8Args& g, unsigned char* stage, uint32_t acc, float xs, const float* ws, const float* bs, int m0, int f, uint64_t* through) {
    constexpr int PARTS = (int)sizeof(T) == 4 ? 1 : 2;
    uint32_t w[16];
#pragma unroll
    for (int h = 0; h < PARTS; ++h) {
        uint32_t r[16], u[16];
        i8_tmem_ld16(acc + 16 * h, GATED, r, u);
        if (h == PARTS - 1 && through) i8_release_acc(through);
        i8_values16(r, xs, ws + 16 * h, bs + 16 * h);
        if constexpr (GATED) {
            i8_values16(u, xs, ws + 64 + 16 * h, bs + 64 + 16 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(silu_mul<PARTS == 2>(__uint_as_float(r[e]), __uint_as_float(u[e])));
        }
#pragma unroll
        for (int e = 0; e < 16 / PARTS; ++e) {
            if constexpr (PARTS == 1) {
                w[e] = r[e];
            } else {
                const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
                w[8 * h + e] = *reinterpret_cast<const uint32_t*>(&v);
            }
        }
    }
    if constexpr (PIECE == 2) {
        const int m = m0 + (threadIdx.x & 31);
        const int64_t at = (int64_t)m * g.ldc + f;
        if (at & 1) {
            if (m < g.tokens) {
                if (f < g.out_features) ((uint16_t*)g.out)[at] = (uint16_t)w[0];
                if (f + 31 < g.out_features) ((uint16_t*)g.out)[at + 31] = (uint16_t)(w[15] >> 16);
            }
#pragma unroll
            for (int e = 0; e < 15; ++e) w[e] = __funnelshift_r(w[e], w[e + 1], 16);
        }
    }
    i8_write_run<T, PIECE>(g, stage, w, m0, f);
}

// What a block of a pair has sent for and formed, for the other one to read where a wait gave up.
struct I8PairCounts {
    int copies;  // stages that it has sent for
    int tiles;   // leader: accumulators that it has committed
};
// The other block's flag: its waits may go well, for an accumulator that is committed but not formed.
__device__ __noinline__ void i8_tell_pair(volatile int* gave_up) {
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(i8_remote((const void*)gave_up, cluster_rank() ^ 1)), "r"(1) : "memory");
    asm volatile("fence.acq_rel.cluster;" ::: "memory");
}
// Where a wait of either block gave up, both come here: the error word, and a wait for what is in flight to them.  Both blocks' bytes count
// on the leader's barriers (`bytes` a stage, half of them each's), and one may have sent for stages that the other has not: the leader
// arrives for those that it has not sent for itself, and counts the half that nobody sent as landed.
__device__ __noinline__ void i8_pair_gave_up(const Int8Args& g, uint64_t* full, uint64_t* acc_full, int stages, int bytes, const I8PairCounts* counts) {
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        atomicOr(g.err, SS_ERR_WAIT_LIMIT);
        const auto of = [&](uint32_t block, const int* p) {
            int v;
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(i8_remote(p, block)) : "memory");
            return v;
        };
        const int tiles = of(0, &counts->tiles);
        if (rank == 0) {
            const int mine = counts->copies, other = of(1, &counts->copies), all = max(mine, other);
            for (int i = max(0, all - stages); i < all; ++i) {
                uint64_t* bar = &full[i % stages];
                if (i >= mine) mbar_expect_tx(bar, bytes);
                if (i >= min(mine, other))
                    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(s_addr(bar)), "r"(bytes / 2) : "memory");
                mbar_drain(bar, (i / stages) & 1);
            }
        }
        for (int j = max(0, tiles - 2); j < tiles; ++j) mbar_drain(&acc_full[j & 1], (j >> 1) & 1);
    }
    cluster_sync_all();
}

// PIECE: 16, 4 or 2 bytes that the rows of the output start on and are a multiple of.
template <int STEPS, typename T, int PIECE, bool GATED>
__global__ void __launch_bounds__(I8_MANY_THREADS)
gemm_int8_many_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Int8Args g) {
    constexpr int x_bytes = STEPS * I8_BM * I8_BK;
    const int w_rows = g.bn / 2, stages = g.stages, stage_bytes = x_bytes + STEPS * w_rows * I8_BK;  // this block's halves
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + stages * stage_bytes);
    uint64_t* empty = full + stages;
    uint64_t* acc_full = empty + stages;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    I8PairCounts* counts = reinterpret_cast<I8PairCounts*>(tmem_slot + 2);
    float* ws_s = reinterpret_cast<float*>(full) + 64;  // [2][256] scales and [2][256] biases of a tile's features
    float* bs_s = ws_s + 2 * I8_MAX_BN;
    unsigned char* runs = reinterpret_cast<unsigned char*>(bs_s + 2 * I8_MAX_BN);  // 1 KB for each epilogue warp

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();  // 0: the leader
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const int bn = g.bn;  // a multiple of 32
    const int n_m = (g.tokens + 2 * I8_BM - 1) / (2 * I8_BM), n_tiles = n_m * ((g.features + bn - 1) / bn);
    const int k_steps = (g.K + I8_BK - 1) / I8_BK, k_iters = (k_steps + STEPS - 1) / STEPS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 32); }
        *gave_up = 0;
        counts->copies = counts->tiles = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();  // both blocks' barriers exist before either signals the other's
    const int first = min(stages, pair < n_tiles ? k_iters : 0);  // stages of the first tile that are fetched ahead
    const int bytes = 2 * stage_bytes;  // of both blocks
    if (threadIdx.x == 0) {
        // the weights do not depend on the kernels in front: their first tiles are on the way before those are through
#pragma unroll 1
        for (int k = 0; k < first; ++k) {
            if (rank == 0) mbar_expect_tx(&full[k], bytes);
            i8_load_pair_stage<STEPS>(tiles + k * stage_bytes + x_bytes, &map_w, g.wide_copies, k, (pair / n_m) * bn + rank * w_rows, w_rows, &full[k]);
        }
    }
    pdl_wait();
    if (warp == 1) {  // the same warp of both blocks allocates all 512 columns of the pair
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        pdl_launch_dependents();  // (this warp alone: one call of a block lets the kernel behind go)
    } else if (threadIdx.x == 0) {
#pragma unroll 1
        for (int k = 0; k < first; ++k)
            i8_load_pair_stage<STEPS>(tiles + k * stage_bytes, &map_x, g.wide_copies, k, (pair % n_m) * 2 * I8_BM + rank * I8_BM, I8_BM, &full[k]);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();  // the tensor memory of both blocks has been taken
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        int it = 0, s = 0;
        uint32_t parity = 1;  // of the round before the first: the stages are free
        bool ok = true;
#pragma unroll 1
        for (int t = pair; t < n_tiles && ok; t += n_pairs) {
            const int m0 = (t % n_m) * 2 * I8_BM + rank * I8_BM, n0 = (t / n_m) * bn + rank * w_rows;
#pragma unroll 1
            for (int k = 0; k < k_iters; ++k, ++it) {
                if (it >= first) {
                    if (!mbar_wait(&empty[s], parity, gave_up)) { ok = false; break; }
                    if (rank == 0) mbar_expect_tx(&full[s], bytes);
                    unsigned char* x_tile = tiles + s * stage_bytes;
                    i8_load_pair_stage<STEPS>(x_tile, &map_x, g.wide_copies, k, m0, I8_BM, &full[s]);
                    i8_load_pair_stage<STEPS>(x_tile + x_bytes, &map_w, g.wide_copies, k, n0, w_rows, &full[s]);
                }
                if (++s == stages) { s = 0; parity ^= 1; }
            }
        }
        counts->copies = it;
    } else if (warp == 1 && rank == 0) {
        const uint32_t idesc = i8_idesc(2 * I8_BM, bn);
        const uint64_t x_first = smem_desc(tiles), w_first = smem_desc(tiles + x_bytes);
        const uint32_t stage_step = (uint32_t)stage_bytes >> 4;  // of a descriptor's address
        const uint32_t w_step = (uint32_t)(w_rows * I8_BK) >> 4;
        int j = 0, s = 0;
        uint32_t parity = 0;
        bool ok = true;
#pragma unroll 1
        for (int t = pair; t < n_tiles && ok; t += n_pairs, ++j) {
            const int buf = j & 1;
            ok = j < 2 || __all_sync(0xffffffffu, mbar_wait(&acc_empty[buf], ((j >> 1) - 1) & 1, gave_up));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t acc = tmem + buf * I8_MAX_BN;
#pragma unroll 1
            for (int k = 0; ok && k < k_iters; ++k) {
                if (!__all_sync(0xffffffffu, mbar_wait(&full[s], parity, gave_up))) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t x_desc = x_first + s * stage_step, w_desc = w_first + s * stage_step;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < I8_BK / 32; ++kk)
                        umma_i8_pair(acc, x_desc + (uint64_t)(kk * 2), w_desc + (uint64_t)(kk * 2), idesc, (k | kk) != 0);
                    if (STEPS == 2 && 2 * k + 1 < k_steps) {
#pragma unroll
                        for (int kk = 0; kk < I8_BK / 32; ++kk)
                            umma_i8_pair(acc, x_desc + (uint64_t)(I8_BM * I8_BK / 16 + kk * 2), w_desc + (uint64_t)(w_step + kk * 2), idesc, 1);
                    }
                    i8_commit_pair(&empty[s]);
                }
                __syncwarp();
                if (++s == stages) { s = 0; parity ^= 1; }
            }
            if (!ok) i8_tell_pair(gave_up);
            __syncwarp();
            if (elect_one()) i8_commit_pair(&acc_full[buf]);
            __syncwarp();
        }
        if (lane == 0) counts->tiles = j;
    } else if (warp >= 2) {
        // each warp its quarter of the rows, and every fourth run of 64 bytes of them
        const int quarter = warp & 3, part = (warp - 2) >> 2, col = (threadIdx.x - 64) & 255;
        unsigned char* stage = runs + (warp - 2) * 1024;
        constexpr int run = 64 / (int)sizeof(T);
        const int columns = GATED ? bn / 2 : bn;
        // a feature's scale (parts 0 and 1) or bias, and a token's scale: fetched a tile ahead
        const auto feature_value = [&](int t) {
            const int f = (t / n_m) * bn + col;
            if (col >= bn || t >= n_tiles || f >= g.features) return 0.f;
            return part < 2 ? __ldg(g.w_scale + f) : g.bias ? i8_bias(g, f) : 0.f;
        };
        const auto token_scale = [&](int t) {
            const int m = (t % n_m) * 2 * I8_BM + rank * I8_BM + quarter * 32 + lane;
            return t < n_tiles && m < g.tokens ? g.x_scale[m] : 0.f;
        };
        float next_value = feature_value(pair), next_scale = token_scale(pair);
        int j = 0;
#pragma unroll 1
        for (int t = pair; t < n_tiles; t += n_pairs, ++j) {
            const int buf = j & 1, n0 = (t / n_m) * bn, m0 = (t % n_m) * 2 * I8_BM + rank * I8_BM + quarter * 32;
            float* ws = ws_s + buf * I8_MAX_BN;
            float* bs = bs_s + buf * I8_MAX_BN;
            (part < 2 ? ws : bs)[col] = next_value;
            const float xs = next_scale;
            // (a buffer is written again two tiles later, behind the barrier that every warp reaches when it is through with it)
            asm volatile("bar.sync 1, 512;" ::: "memory");
            next_value = feature_value(t + n_pairs);
            next_scale = token_scale(t + n_pairs);
            // (behind a wait that gave up a warp writes nothing but still comes to the barriers, where the others wait for it)
            // (the flag, not the wait's result: an issuer that gave up still commits, so that the accumulator can be waited for)
            (void)mbar_wait(&acc_full[buf], (j >> 1) & 1, gave_up);
            const bool formed = !__shfl_sync(0xffffffffu, *gave_up, 0);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + buf * I8_MAX_BN;
            if (!formed || part * run >= columns) {
                i8_release_acc(&acc_empty[buf]);
                continue;
            }
#pragma unroll 1
            for (int f = part * run; f < columns; f += 4 * run) {
                const int c = GATED ? f / 64 * 128 + f % 64 : f;  // the gate's column; the up's stands 64 behind it
                i8_write_outputs<T, PIECE, GATED>(g, stage, acc + c, xs, ws + c, bs + c, m0, (GATED ? n0 / 2 : n0) + f,
                                                  f + 4 * run < columns ? nullptr : &acc_empty[buf]);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*gave_up && threadIdx.x == 0) i8_tell_pair(gave_up);  // the other block comes along
    cluster_sync_all();  // neither block leaves (or frees tensor memory) while the other may still signal it
    if (*gave_up) i8_pair_gave_up(g, full, acc_full, stages, bytes, counts);
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ---------------------------------------------------------------- host side

typedef CUresult (*I8Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// int8 matrix [rows, K] with row stride ld bytes; box = 128 x box_rows, or, with `steps` (K a multiple of 128), two steps of K:
// the matrix as [K / 128][rows][128], box = 128 x box_rows x 2.
static int i8_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows, bool steps = false) {
    static I8Encode enc = nullptr;
    if (!enc) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return -2001;
        enc = (I8Encode)p;
    }
    cuuint64_t dims[3] = {(cuuint64_t)(steps ? I8_BK : K), (cuuint64_t)rows, (cuuint64_t)(K / I8_BK)};
    cuuint64_t strides[2] = {(cuuint64_t)ld, I8_BK};
    cuuint32_t box[3] = {I8_BK, (cuuint32_t)box_rows, 2};
    cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, steps ? 3 : 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : -2002;
}

#define I8_SMEM_MAX 232448  // 227 KB of a block
#define I8_SMEM_SM 233472   // 228 KB of an SM, 1 KB of it each block's own
#define I8_SMEM_REST 2560   // alignment, barriers, scales

// Only asked about, never launched: blocks of the shape of the kernel for few tokens.  About a kernel that takes tensor memory the
// runtime answers one block an SM, whatever it takes of it; two are resident (11.1 of their 12 warps active on average).
__global__ void __launch_bounds__(I8_THREADS) i8_few_shape() {}

// How many clusters of `n` blocks of the kernel for few tokens run at the same time where the ring is sized for `per_sm` blocks an
// SM (n = 1: blocks).
extern "C" int ss_gemm_int8_resident(int n, int per_sm) {
    static SsPerDevice opted;
    if (n < 1 || n > 8 || per_sm < 1 || ss_opt_in_smem(i8_few_shape, I8_SMEM_MAX, opted)) return 0;
    return ss_resident_clusters(i8_few_shape, I8_THREADS, per_sm > 1 ? I8_SMEM_SM / per_sm - 1024 : I8_SMEM_MAX, n);
}

template <int STEPS, bool GATED, typename T, int PIECE>
static int launch_many(const Int8Call& c, Int8Args& g) {
    CUtensorMap map_x, map_w;
    g.wide_copies = STEPS == 2 && g.K % I8_BK == 0;
    if (int rc = i8_map(&map_x, c.x, g.tokens, g.K, c.ldx, I8_BM, g.wide_copies)) return rc;
    if (int rc = i8_map(&map_w, c.w, g.features, g.K, c.ldw, g.bn / 2, g.wide_copies)) return rc;
    static SsPerDevice opted;
    if (int rc = ss_opt_in_smem(gemm_int8_many_kernel<STEPS, T, PIECE, GATED>, I8_SMEM_MAX, opted)) return rc;
    constexpr int rest = I8_SMEM_REST + 4 * I8_MAX_BN * 4 + 16 * 1024;
    const int stage = STEPS * (I8_BM + g.bn / 2) * I8_BK;
    g.stages = (I8_SMEM_MAX - rest) / stage;
    const int64_t n_tiles = (int64_t)((g.tokens + 255) / 256) * ((g.features + g.bn - 1) / g.bn);
    const int pairs = (int)(n_tiles < ss_sm_count() / 2 ? n_tiles : ss_sm_count() / 2);
    ss_launch_cluster_x(gemm_int8_many_kernel<STEPS, T, PIECE, GATED>, dim3(2 * pairs), dim3(I8_MANY_THREADS), g.stages * stage + rest, c.stream, 2, map_x, map_w, g);
    return SS_LAUNCH_CHECK();
}

// `row`: a number of bytes whose powers of two the rows of the output start on
template <int STEPS, bool GATED>
static int launch_many_as(const Int8Call& c, Int8Args& g, int64_t row) {
    if (g.out_f32) return row % 16 ? launch_many<STEPS, GATED, float, 4>(c, g) : launch_many<STEPS, GATED, float, 16>(c, g);
    return row % 4 ? launch_many<STEPS, GATED, bf16, 2>(c, g) : row % 16 ? launch_many<STEPS, GATED, bf16, 4>(c, g) : launch_many<STEPS, GATED, bf16, 16>(c, g);
}

template <int STEPS>
static int launch_few(const Int8Call& c, Int8Args& g, int per_sm) {
    CUtensorMap map_x, map_w;
    const int bn = g.bn, slices = g.slices;
    g.wide_copies = STEPS == 2 && g.K % I8_BK == 0;
    if (int rc = i8_map(&map_x, c.x, g.tokens, g.K, c.ldx, bn, g.wide_copies)) return rc;
    if (int rc = i8_map(&map_w, c.w, g.features, g.K, c.ldw, I8_BM, g.wide_copies)) return rc;
    static SsPerDevice opted;
    if (int rc = ss_opt_in_smem(gemm_int8_few_kernel<STEPS>, I8_SMEM_MAX, opted)) return rc;
    const int stage = STEPS * (I8_BM + bn) * I8_BK;
    const int rest = I8_SMEM_REST + (slices > 1 ? (bn + slices - 1) / slices * I8_BM * 4 : 0);  // a cluster's blocks: the columns they own
    const int room = per_sm > 1 ? I8_SMEM_SM / per_sm - 1024 : I8_SMEM_MAX;
    int stages = (room - rest) / stage;
    const int needed = slices > 1 ? 2 : (bn * I8_BM * 4 + stage - 1) / stage;  // alone, the ring also holds the sums
    stages = stages < needed ? needed : stages > 12 ? 12 : stages;
    g.stages = stages;
    const int smem = stages * stage + rest;
    if (smem > I8_SMEM_MAX) return -2007;
    const dim3 grid((g.tokens + bn - 1) / bn, (g.features + I8_BM - 1) / I8_BM, slices);
    if (slices > 1) ss_launch_cluster(gemm_int8_few_kernel<STEPS>, grid, dim3(I8_THREADS), smem, c.stream, slices, map_w, map_x, g);
    else ss_launch(gemm_int8_few_kernel<STEPS>, grid, dim3(I8_THREADS), smem, c.stream, map_w, map_x, g);
    return SS_LAUNCH_CHECK();
}

// Row strides are multiples of 16 bytes and bases stand on 16 bytes; K <= 131,071.
// gated: w's rows alternate 64 gate and 64 up features; out_features <= features / 2 columns of silu(gate) * up are written.
// many = 0: bn tokens a tile (a multiple of 16 up to 256), slices 1..8 of K, `per_sm` blocks an SM that the ring is sized for.
// many = 1: bn features a tile (a multiple of 32 up to 256; gated: 128 or 256).
// steps: 1 or 2 steps of K in a stage.
extern "C" int ss_gemm_int8(const Int8Call* call) {
    const Int8Call& c = *call;
    if (c.tokens <= 0 || c.features <= 0 || c.out_features <= 0) return 0;
    if (c.tokens > INT32_MAX - 256 || c.features > INT32_MAX - 256 || c.K <= 0 || c.K > 131071 || c.ldx % 16 || c.ldw % 16 || c.ldx < c.K || c.ldw < c.K) return -2003;
    if (((uintptr_t)c.x & 15) || ((uintptr_t)c.w & 15) || ((uintptr_t)c.out & 15)) return -2004;
    if (c.gated ? (c.features % 128 || c.out_features > c.features / 2) : c.out_features != c.features) return -2005;
    const int bn = (int)c.bn, slices = (int)c.slices, per_sm = (int)c.per_sm;
    if (bn < 16 || bn > I8_MAX_BN || c.steps < 1 || c.steps > 2 || bn % (c.many ? 32 : 16) || (c.many && c.gated && bn % 128)
        || (!c.many && (slices < 1 || slices > 8 || per_sm < 1 || per_sm > 4 || (c.features + I8_BM - 1) / I8_BM > 65535))) return -2006;
    Int8Args g = {};
    g.x_scale = c.x_scale; g.w_scale = c.w_scale; g.bias = c.bias; g.out = c.out; g.err = c.err; g.ldc = c.ldc;
    g.tokens = (int)c.tokens; g.features = (int)c.features; g.K = (int)c.K; g.out_features = (int)c.out_features;
    g.out_f32 = (int)c.out_f32; g.bias_f32 = (int)c.bias_f32; g.gated = (int)c.gated; g.bn = bn; g.slices = slices;
    if (c.many) {
        const int64_t row = (g.ldc | g.out_features) * (g.out_f32 ? 4 : 2);
        if (c.steps == 2) return g.gated ? launch_many_as<2, true>(c, g, row) : launch_many_as<2, false>(c, g, row);
        return g.gated ? launch_many_as<1, true>(c, g, row) : launch_many_as<1, false>(c, g, row);
    }
    return c.steps == 2 ? launch_few<2>(c, g, per_sm) : launch_few<1>(c, g, per_sm);
}

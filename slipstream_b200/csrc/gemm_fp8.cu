// Matrix product of 8-bit floats (e4m3) with a float32 scale for each block of 128, on the 5th-generation tensor cores of sm_100a:
//   Y[m, n] = sum_b x_scale[m, b] * w_scale[n / 128, b] * (sum_{k in block b} X[m, k] * W[n, k]) (+ bias[n])
// X: activations, a scale for each token and 128 elements of K; W: weights, a scale for each 128 features x 128 elements of K; both
// K-major.  The sum over a block is formed by tcgen05.mma (kind::f8f6f4: products exact, added in float32) in tensor memory; the warps of
// the epilogue take it out, multiply it by the product of both scales (rounded once) and add it to their registers with one fused
// multiply-add, block after block of K.  So tensor memory holds a ring of such sums, and the products of the next blocks run meanwhile.
// The bias is added last, and the result is rounded once to the output type.  The gated form pairs the features of a feed-forward's
// gate and up matrices (stacked in runs of 128 rows each) and writes silu(gate) * up, which may be rounded to e4m3 again, with a scale for
// each token and 128 features: those are the features of one tile.
//
// A row's stage in shared memory is 128 bytes, a block of K, under the 128-byte swizzle; an instruction takes 32 of them.
//
// Every wait on an mbarrier is bounded: after WAIT_LIMIT polls the kernel sets SS_ERR_WAIT_LIMIT in the error word, stops
// waiting everywhere, writes out nothing that it has not formed, waits (with the same limit) for its copies and products in flight,
// frees its tensor memory and returns.
//
// Tensor memory is taken BEHIND griddepcontrol.wait, and the kernel behind is let go only when it has been taken: a kernel
// that takes it before the kernel in front is through, or lets a kernel start that may take it first, can wait for a block
// that waits for it.  Before that wait a block reads only the weights, their scales and the bias, which it takes for constant.

#include <cuda.h>

#include "fp8.cuh"
#include "fp8_calls.h"
#include "tc5.cuh"

#define F8_BM 128
#define F8_BK FP8_BLOCK  // K elements, and bytes of a row, in a stage
#define F8_THREADS 320   // few tokens: producer, issuer, eight epilogue warps
#define F8_MAX_BN 256
#define F8_OUT_FP8 2

struct Fp8Args {
    const float* x_scale;
    const float* w_scale;
    int64_t x_row, x_block, w_row, w_block;
    const void* bias;  // [features] or null
    void* out;         // [tokens][ldc]
    float* out_scale;  // [out_features / 128][tokens] where the output is e4m3
    float* parts;      // many tokens, K in slices: [slices][tokens][features up to a multiple of 4]
    int* err;
    int64_t ldc;
    int tokens, features, K;
    int out_features;  // columns written: features, or the gated form's (at most features / 2)
    int out_type, bias_f32;
    int bn;            // few tokens: the tokens of a tile; many tokens: the features of a tile
    int stages, slices;
    int slots, slot_columns;  // of the ring of sums in tensor memory
};

__device__ __forceinline__ void f8_load(void* dst, const CUtensorMap* map, int k, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(s_addr(dst)), "l"(map), "r"(s_addr(bar)), "r"(k), "r"(row) : "memory");
}
// weights that are read once a step: the first to leave L2 again
__device__ __forceinline__ void f8_load_once(void* dst, const CUtensorMap* map, int k, int row, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
        ::"r"(s_addr(dst)), "l"(map), "r"(s_addr(bar)), "r"(k), "r"(row), "l"(policy) : "memory");
}
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// Instruction descriptor: D float32, A and B e4m3, both K-major.
__device__ __forceinline__ uint32_t f8_idesc(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// mbar_wait of a whole warp, the same result in all lanes.  What a warp issues for itself (products, copies) it issues in one elected lane
// behind such waits: where the compiler sees that all lanes go the same way, operands stand in uniform registers; a loop of one lane took
// 0.5 us a block of K, this one 0.26.
__device__ __forceinline__ bool f8_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    for (uint32_t spins = 0; spins < WAIT_POLLS; ++spins) {
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
        if ((spins & 1023u) == 1023u && __any_sync(0xffffffffu, *gave_up)) return false;
    }
    *gave_up = 1;
    return false;
}
// For two barriers: a look at one takes 150 to 290 cycles beside products that read shared memory, at both together hardly more.
__device__ __forceinline__ bool f8_wait(uint64_t* a, uint32_t a_parity, uint64_t* b, uint32_t b_parity, volatile int* gave_up) {
    for (uint32_t spins = 0; spins < WAIT_POLLS; ++spins) {
        const bool first = mbar_try_wait(a, a_parity), second = mbar_try_wait(b, b_parity);
        if (__all_sync(0xffffffffu, first && second)) return true;
        if ((spins & 1023u) == 1023u && __any_sync(0xffffffffu, *gave_up)) return false;
    }
    *gave_up = 1;
    return false;
}
// A look at a barrier that does not wait.  (Where every wait gives up at once, it sees nothing.)
__device__ __forceinline__ uint32_t f8_look(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done) : "r"(s_addr(bar)), "r"(parity) : "memory");
    return WAIT_POLLS ? done : 0;
}

// Behind a wait that gave up: the error word, and a wait for the last of the `copies` stages that were sent for, which may still be
// in flight.
__device__ __noinline__ void f8_gave_up(const Fp8Args& g, uint64_t* full, int stages, int copies) {
    atomicOr(g.err, SS_ERR_WAIT_LIMIT);
    for (int i = max(0, copies - stages); i < copies; ++i) mbar_drain(&full[i % stages], (i / stages) & 1);
}
// ... and for the last of `count` uses of a ring of `n` barriers (sums that were committed).
__device__ __forceinline__ void f8_drain_ring(uint64_t* bars, int n, int count) {
    for (int i = max(0, count - n); i < count; ++i) mbar_drain(&bars[i % n], (i / n) & 1);
}

__device__ __forceinline__ float f8_bias(const Fp8Args& g, int f) {
    return g.bias_f32 ? ((const float*)g.bias)[f] : to_float(((const bf16*)g.bias)[f]);
}
__device__ __forceinline__ float f8_gate(const Fp8Args& g, float gate, float up) {
    return g.out_type == SS_F32 ? silu_mul<false>(gate, up) : silu_mul<true>(gate, up);
}

// Whether `v` holds in all threads of the few tokens' epilogue; a barrier of theirs.
__device__ __forceinline__ bool f8_epilogue_all(bool v) {
    uint32_t all;
    asm volatile(
        "{\n.reg .pred p, q;\nsetp.ne.u32 q, %1, 0;\n"
        "bar.red.and.pred p, 1, 256, q;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(all) : "r"((uint32_t)v) : "memory");
    return all != 0;
}

// Four outputs of a token, `apart` features from one another (float32 or bfloat16).
__device__ __forceinline__ void f8_store4(const Fp8Args& g, int token, int f, int apart, const float (&v)[4]) {
    const int64_t at = (int64_t)token * g.ldc + f;
    if (apart == 1 && f + 4 <= g.out_features) {
        if (g.out_type == SS_F32) {
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
        if (g.out_type == SS_F32) ((float*)g.out)[at + e * apart] = v[e];
        else ((bf16*)g.out)[at + e * apart] = __float2bfloat16_rn(v[e]);
    }
}

// v at `to` in the shared memory of a block of the cluster; four bytes of the transaction that `bar` there counts
__device__ __forceinline__ void f8_send(uint32_t to, uint32_t bar, float v) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(to), "f"(v), "r"(bar) : "memory");
}
// v or-ed into the word at `to`, alike
__device__ __forceinline__ void f8_send_flag(uint32_t to, uint32_t bar, uint32_t v) {
    asm volatile("red.async.relaxed.cluster.shared::cluster.mbarrier::complete_tx::bytes.or.b32 [%0], %1, [%2];" ::"r"(to), "r"(v), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t f8_remote(const void* p, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(s_addr(p)), "r"(rank));
    return remote;
}
// Scales on their way to a thread: four bytes from memory to shared memory, without registers, `FLIGHT` blocks of K ahead of their use, so that
// the loop of the epilogue, which takes about 0.3 us a block of K, does not wait for memory (about 1 us).  A group a
// block; what a thread sent for is there for itself when all but the last FLIGHT - 1 groups are through, for its warp behind __syncwarp.
__device__ __forceinline__ void f8_send_for(float* to, const float* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s_addr(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void f8_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER>
__device__ __forceinline__ void f8_arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

// W columns of tensor memory (8, 16 or 32); the registers hold them behind the wait, through which they pass, so that nothing that reads
// them moves in front of it.
template <int W>
__device__ __forceinline__ void f8_tmem_load(uint32_t taddr, float (&r)[W]) {
    static_assert(W == 8 || W == 16 || W == 32, "");
    if constexpr (W == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]) : "r"(taddr));
    } else if constexpr (W == 16) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
                       "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]) : "r"(taddr));
    } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                     "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
                       "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
                       "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
                       "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]) : "r"(taddr));
    }
}
template <int W>
__device__ __forceinline__ void f8_tmem_wait(float (&r)[W]) {
    if constexpr (W == 8) {
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7])::"memory");
    } else if constexpr (W == 16) {
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                       "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])::"memory");
    } else {
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                       "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                       "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
                       "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])::"memory");
    }
}

// acc = r * f + acc for two elements in one instruction, each rounded as fmaf does.
__device__ __forceinline__ void f8_add2(float (&acc)[2], float r0, float r1, float f) {
    asm("{\n.reg .b64 a, r, f;\nmov.b64 a, {%0, %1};\nmov.b64 r, {%2, %3};\nmov.b64 f, {%4, %4};\nfma.rn.f32x2 a, r, f, a;\nmov.b64 {%0, %1}, a;\n}"
        : "+f"(acc[0]), "+f"(acc[1]) : "f"(r0), "f"(r1), "f"(f));
}

// ---------------------------------------------------------------- few tokens: the weights' bytes are the work
//
// The weights are the instruction's A (their rows fill its 128 lanes), the tokens its B (bn of them, a multiple of 16 up to 256).
// A block forms a tile of 128 features (gated, MT = 2: 128 pairs, the gate's lanes and the up's in columns of their own) x bn
// tokens over one slice of K.  The 1 to 8 slices of a tile are a thread-block cluster along grid.z: token column c belongs to block
// c % slices, and every block sends its sums of the column to that block's shared memory (st.async), which counts the bytes on a
// barrier of its own; the owner adds the slices' sums in their order.  No block waits for another but for these.
// Warp 0 (one lane) fetches, warp 1 issues the products, warps 2 to 9 are the epilogue: two of them for each quarter of the lanes,
// half of the columns each (bn / 2, at most C).
//
// Bound by the weights' bytes where they are many (8 x 3,584 x 37,888 gated to fp8 rows: 22.5 us, 6.1 TB/s, of which L2 holds a part), else by
// what a block of K takes, 0.24 us and 3 ns a token column (a look at a barrier alone takes 150 to 290 cycles): 16 x 18,944 x 3,584,
// in 4 slices of 37 blocks each, 15.9 us for 10.4 of bytes; 1 x 896 x 1,152 4.0.  Two blocks of K a stage and a slot halve
// the looks (64 x 18,944 x 3,584 25.4 to 22.1 us) but leave no room for the next kernel's block beside this one's ring (16 x 3,584 x 4,608
// 6.5 to 8.0), so a stage is one block.
//
// Registers: an SM's scheduler has 16,384 for its warps.  Three warps of one block (ten in all) may have 168 each; two blocks on an SM
// 96, which the sums of up to 64 token columns (gated 32) fit into.
constexpr bool f8_few_shares(int mt, int c) { return mt * c <= 32; }
// Blocks of K that a warp's scales are fetched ahead, and the floats that it needs for them: those, then two sets of factors.
constexpr int f8_few_flight(int mt, int c) { return mt * c <= 32 ? 8 : 4; }
constexpr int f8_few_raw(int mt, int c) { return (c + mt + 3) / 4 * 4; }
constexpr int f8_few_floats(int mt, int c) { return f8_few_flight(mt, c) * f8_few_raw(mt, c) + 2 * mt * c; }

template <int MT, int C>
__global__ void __launch_bounds__(F8_THREADS, f8_few_shares(MT, C) ? 2 : 1)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Args g) {
    extern __shared__ unsigned char smem_raw[];
    constexpr int w_bytes = MT * F8_BM * F8_BK, FL = MT * F8_BM;
    const int bn = g.bn, stages = g.stages, n_sl = g.slices, slots = g.slots;
    const int stage_bytes = w_bytes + bn * F8_BK;
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + stages * stage_bytes);
    uint64_t* empty = full + stages;
    uint64_t* part_full = empty + stages;   // [8]
    uint64_t* part_empty = part_full + 8;   // [8]
    uint64_t* sums_ready = part_empty + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_ready + 1);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* unformed = gave_up + 1;  // of the cluster's sums that were sent here some are not formed
    float* factors = reinterpret_cast<float*>(full) + 128;  // of the eight warps, behind the barriers
    // [senders][own columns][FL]: of a cluster's block behind the factors; alone ([columns][FL]) over the ring, when all its stages have been used
    float* sums = n_sl > 1 ? factors + 8 * f8_few_floats(MT, C) : reinterpret_cast<float*>(tiles);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t0 = blockIdx.x * bn, f0 = blockIdx.y * FL;      // first token, first feature (row of the weight)
    const int live = min(bn, g.tokens - t0);                   // columns that hold tokens
    const int rank = n_sl > 1 ? (int)cluster_rank() : 0;
    const int mine = live > rank ? (live - 1 - rank) / n_sl + 1 : 0;  // columns rank, rank + slices, ...
    const int k_blocks = (g.K + F8_BK - 1) / F8_BK;
    const int per = (k_blocks + n_sl - 1) / n_sl;
    const int k_begin = blockIdx.z * per, k_iters = max(0, min(k_blocks, k_begin + per) - k_begin);
    const int senders = (k_blocks + per - 1) / per;  // blocks that have any K
    const int ahead = min(stages, k_iters);
    const uint32_t tmem_cols = slots * MT * g.slot_columns;
    int copies = 0;  // stages that thread 0 has sent for

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < slots; ++s) { mbar_init(&part_full[s], 1); mbar_init(&part_empty[s], 8); }
        mbar_init(sums_ready, 1);
        *gave_up = *unformed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (n_sl > 1) mbar_expect_tx(sums_ready, (uint32_t)(senders * (mine * FL + 8) * 4));  // (and a flag of each warp)
        // the weights do not depend on the kernels in front: their first tiles are on the way before those are through
        const uint64_t once = l2_evict_first_policy();
        for (int it = 0; it < ahead; ++it) {
            mbar_expect_tx(&full[it], stage_bytes);
            f8_load_once(tiles + it * stage_bytes, &map_w, (k_begin + it) * F8_BK, f0, &full[it], once);
        }
    }
    __syncthreads();
    if (n_sl > 1) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // this block's barriers stand
        if (warp < 2) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }

    if (warp == 0) {
        const uint64_t once = l2_evict_first_policy();
        pdl_wait();
        if (elect_one())
            for (int it = 0; it < ahead; ++it) f8_load(tiles + it * stage_bytes + w_bytes, &map_x, (k_begin + it) * F8_BK, t0, &full[it]);
        __syncwarp();
        int it = ahead, s = 0;
        uint32_t parity = 0;
        for (; it < k_iters; ++it) {
            if (!f8_wait(&empty[s], parity, gave_up)) break;
            if (elect_one()) {
                mbar_expect_tx(&full[s], stage_bytes);
                f8_load_once(tiles + s * stage_bytes, &map_w, (k_begin + it) * F8_BK, f0, &full[s], once);
                f8_load(tiles + s * stage_bytes + w_bytes, &map_x, (k_begin + it) * F8_BK, t0, &full[s]);
            }
            __syncwarp();
            if (++s == stages) { s = 0; parity ^= 1; }
        }
        copies = it;
    } else if (warp == 1) {
        pdl_wait();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_slot)), "r"(tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        pdl_launch_dependents();  // (this warp alone: one call of a block lets the kernel behind go)
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        asm volatile("bar.arrive 2, 288;" ::: "memory");  // the epilogue warps read the slot behind it
        const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
        const uint32_t idesc = f8_idesc(F8_BM, bn);
        const uint64_t w_first = smem_desc(tiles), x_first = smem_desc(tiles + w_bytes);
        const uint32_t stage_step = (uint32_t)stage_bytes >> 4;  // of a descriptor's address
        int s = 0, slot = 0, it = 0;
        uint32_t parity = 0, free_parity = 1;  // (of the round before the first: the slots are free)
        for (; it < k_iters; ++it) {
            if (!f8_wait(&full[s], parity, &part_empty[slot], free_parity, gave_up)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t w_desc = w_first + s * stage_step, x_desc = x_first + s * stage_step;
            const uint32_t acc = tmem + slot * MT * g.slot_columns;
            if (elect_one()) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int kk = 0; kk < F8_BK / 32; ++kk)  // 32 bytes further along the swizzled row
                        umma_f8(acc + m * g.slot_columns, w_desc + (uint64_t)(m * F8_BM * F8_BK / 16 + kk * 2), x_desc + (uint64_t)(kk * 2), idesc, kk != 0);
                umma_commit(&part_full[slot]);
                umma_commit(&empty[s]);
            }
            __syncwarp();
            if (++s == stages) { s = 0; parity ^= 1; }
            if (++slot == slots) { slot = 0; free_parity ^= 1; }
        }
        // (where it gave up: products in flight end before the block does)
        if (it < k_iters) f8_drain_ring(part_full, slots, it);
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2, hc = bn / 2, c0 = half * hc;  // its columns: c0 .. c0 + hc - 1
        constexpr int FLIGHT = f8_few_flight(MT, C), RAW = f8_few_raw(MT, C);
        float* raw = factors + (warp - 2) * f8_few_floats(MT, C);  // [FLIGHT][C of the tokens, MT of the weights]
        float* fac = raw + FLIGHT * RAW;                             // [2][MT][C]
        // nor do the bias of the four features (gated: four pairs) depend on the kernels in front that a lane writes out: neighbours, or,
        // where the output's rows do not start on four elements, one of each quarter of the tile
        const int of0 = f0 / MT;  // first output feature
        const int apart = (g.ldc & 3) == 0 ? 1 : 32, fl = apart == 1 ? lane * 4 : lane;
        float bs[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int f = f0 + m * F8_BM + fl + e * apart;
                bs[m][e] = g.bias && f < g.features ? f8_bias(g, f) : 0.f;
            }
        const float* ws = g.w_scale + (int64_t)(blockIdx.y * MT) * g.w_row + (int64_t)k_begin * g.w_block;
        if (n_sl > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        pdl_wait();  // the output may still be in use by the kernels in front, which also wrote the tokens' scales
        constexpr int XS = (C + 31) / 32, W = C < 16 ? C : MT * C <= 64 ? (C < 32 ? 16 : 32) : 16;
        int sent = 0, sent_at = 0;  // blocks of K whose scales are sent for, and the place of the next
        const auto send_for_scales = [&]() {
            if (sent < k_iters) {
                float* to = raw + sent_at * RAW;
#pragma unroll
                for (int i = 0; i < XS; ++i) {
                    const int c = i * 32 + lane, t = c0 + c;
                    if (c < hc && t < live) f8_send_for(to + c, g.x_scale + (int64_t)(t0 + t) * g.x_row + (int64_t)(k_begin + sent) * g.x_block);
                }
                if (lane < MT) f8_send_for(to + C + lane, ws + lane * g.w_row + (int64_t)sent * g.w_block);
                if (++sent_at == FLIGHT) sent_at = 0;
            }
            f8_group();
            ++sent;
        };
        // (columns without a token keep the zeros that stand there first)
        for (int i = lane; i < FLIGHT * RAW; i += 32) raw[i] = 0.f;
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < FLIGHT - 1; ++i) send_for_scales();
        asm volatile("bar.sync 2, 288;" ::: "memory");  // the tensor memory's address is there
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot) + ((uint32_t)(quarter * 32) << 16) + c0;
        float acc[MT][C];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < C; ++c) acc[m][c] = 0.f;
        int slot = 0, raw_at = 0;
        uint32_t parity = 0;
        bool ok = true;
        for (int it = 0; it < k_iters; ++it) {
            float* f = fac + (it & 1) * MT * C;
            f8_arrived<FLIGHT - 2>();
            __syncwarp();
#pragma unroll
            for (int i = 0; i < XS; ++i)
                if (i * 32 + lane < C) {
#pragma unroll
                    for (int m = 0; m < MT; ++m) f[m * C + i * 32 + lane] = __fmul_rn(raw[raw_at * RAW + i * 32 + lane], raw[raw_at * RAW + C + m]);
                }
            if (++raw_at == FLIGHT) raw_at = 0;
            __syncwarp();
            send_for_scales();  // (into the place that was read a block of K ago)
            if (!f8_wait(&part_full[slot], parity, gave_up)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = tmem + slot * MT * g.slot_columns;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int c = 0; c < C; c += W)
                    if (c < hc) {
                        // (columns from hc on, up to the slot's end, are taken out too and belong to nobody)
                        float r[W];
                        f8_tmem_load<W>(at + m * g.slot_columns + c, r);
                        f8_tmem_wait<W>(r);
#pragma unroll
                        for (int e = 0; e < W; e += 4) {
                            const float4 s4 = *reinterpret_cast<const float4*>(f + m * C + c + e);
                            acc[m][c + e] = fmaf(r[e], s4.x, acc[m][c + e]);
                            acc[m][c + e + 1] = fmaf(r[e + 1], s4.y, acc[m][c + e + 1]);
                            acc[m][c + e + 2] = fmaf(r[e + 2], s4.z, acc[m][c + e + 2]);
                            acc[m][c + e + 3] = fmaf(r[e + 3], s4.w, acc[m][c + e + 3]);
                        }
                    }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&part_empty[slot]);
            if (++slot == slots) { slot = 0; parity ^= 1; }
        }
        f8_arrived<0>();
        // (where a wait gave up, copies may be landing where the sums would go: only the flag says that all is formed)
        ok = ok && !__shfl_sync(0xffffffffu, *gave_up, 0);
        if (n_sl == 1) {
            ok = f8_epilogue_all(ok);  // and every warp has taken its last sums out: the ring is free
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if (ok && c < hc && c0 + c < live) sums[(c0 + c) * FL + m * F8_BM + quarter * 32 + lane] = acc[m][c];
            ok = f8_epilogue_all(ok);
        } else {
            if (k_iters > 0) {
                // a warp that gave up sends what it has: the bytes that the owners count always arrive, so that none of them leaves with
                // sums on their way to it; its flag, which they count too, tells them to write none of it
                const int some = live / n_sl, more = live % n_sl;  // block r owns some (+ 1 where r < more) columns
                int owner = c0 % n_sl, at = c0 / n_sl;             // of column c: block c % slices, its column c / slices
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if (c < hc && c0 + c < live) {
                        const int theirs = some + (owner < more ? 1 : 0);
                        const uint32_t to = f8_remote(sums + (blockIdx.z * theirs + at) * FL + quarter * 32 + lane, owner), bar = f8_remote(sums_ready, owner);
#pragma unroll
                        for (int m = 0; m < MT; ++m) f8_send(to + m * F8_BM * 4, bar, acc[m][c]);
                        if (++owner == n_sl) { owner = 0; ++at; }
                    }
                if (lane < n_sl) f8_send_flag(f8_remote((const void*)unformed, lane), f8_remote(sums_ready, lane), !ok);
            }
            if (!mbar_wait(sums_ready, 0, gave_up)) mbar_drain(sums_ready, 0);
            ok = !*gave_up && !*unformed;
        }
        // a warp takes a token column at a time, a lane four features (gated: pairs) of it
        const int n_sum = n_sl > 1 ? senders : 1;
        for (int i = warp - 2; ok && i < mine; i += 8) {
            const int c = rank + i * n_sl;
            float v[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float* from = sums + i * FL + m * F8_BM + fl + e * apart;
                    float total = *from;
                    for (int s = 1; s < n_sum; ++s) total += from[s * mine * FL];
                    v[m][e] = total + bs[m][e];
                }
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = MT == 2 ? f8_gate(g, v[0][e], v[MT - 1][e]) : v[0][e];
            if (MT == 2 && g.out_type == F8_OUT_FP8) {
                if (of0 >= g.out_features) break;
                const int left = g.out_features - of0 - fl;  // (rows of e4m3 start on 16 bytes: fl = 4 lane)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e >= left) y[e] = 0.f;
                const uint32_t top = __reduce_max_sync(0xffffffffu, fp8_top(0u, y));
                const Fp8Scale r = fp8_scale(top);
                if (lane == 0) g.out_scale[(int64_t)blockIdx.y * g.tokens + t0 + c] = r.scale;
                if (left > 0) fp8_store4((uint8_t*)g.out + (int64_t)(t0 + c) * g.ldc + of0 + fl, left, fp8_quantize4(y, r));
            } else {
                f8_store4(g, t0 + c, of0 + fl, apart, y);
            }
        }
    }
    if (n_sl > 1) {  // nobody leaves while others may still send to it: each has seen the sums that it owns arrive
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
        asm volatile("barrier.cluster.wait;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*gave_up && threadIdx.x == 0) f8_gave_up(g, full, stages, copies);
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols));
    }
}

// ---------------------------------------------------------------- many tokens: the tensor cores are the work
//
// A persistent kernel on pairs of SMs (tcgen05.mma.cta_group::2).  A pair walks over tiles of 256 tokens x bn features, token
// tiles fastest.  Block r of the pair fetches tokens r * 128 .. of the tile and half of its features' weights; the leader
// (block 0) issues the products, which leave the tokens of block r in block r's tensor memory, the sums of one block of K after
// another in a ring of `slots`.  Eight epilogue warps of each block, two for each quarter of the lanes, take the sums of 32 * NC columns each
// out and add them up; the products of the next tile's first blocks of K run while they write a tile out.
//   full[s]       in the leader: the bytes of both blocks' copies;      empty[s]      in each block: the products have read the stage
//   part_full[b]  in each block: the sums of a block of K are formed;   part_empty[b] in the leader: all 16 epilogue warps have them
//
// 256 x 256 outputs x 128 of K take about 0.53 us, the products alone 0.39 (both at 1.9 GHz; the copies keep up), the tensor pipe 0.27.
// Two slots of 256 columns fill the tensor memory, so a period is half of a slot's way round: products, a look at the barrier, the sums
// taken out, their release, another look.  Neither the tensor pipe nor the issue slots (43 % busy) are at a limit; what each part of that
// way takes has not been measured apart.  4,099 x 3,584 x 37,888 gated: 554 to 572 us in a burst, 620 under the power cap, for 330 us at twice the bfloat16 rate;
// 2,047 x 3,581 x 4,613 to float32 60.  The tensor pipe is busy for 46 % of 2,048 tokens.
//
// Few tiles of a long K (256 x 18,944 x 3,584 has 14 of 256 features, and 74 pairs) are cut into slices of K, each a tile of its own whose sums go
// to memory in float32 (they stay in L2), and a second kernel adds them up in order: 54 us in one slice, 31 in five.
//
// Registers: three warps a scheduler are launched with 168 each; the first four warps (producer, issuer, two that do nothing) hand back
// all but 40 of theirs, and the epilogue's have 232: 128 sums and 64 columns on their way.
#define F8_MANY_THREADS 384
#define F8_FLIGHT 4

__device__ __forceinline__ uint32_t f8_leader(const void* p) { return s_addr(p) & 0xFEFFFFFFu; }  // same offset in block 0 of the pair

__device__ __forceinline__ void f8_load_pair(void* dst, const CUtensorMap* map, int k, int row, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(s_addr(dst)), "l"(map), "r"(f8_leader(bar)), "r"(k), "r"(row) : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
        ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void f8_commit_pair(uint64_t* bar) {  // arrives at `bar` in both blocks of the pair
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(s_addr(bar)), "h"((unsigned short)3) : "memory");
}
// A warp is through with what it read of a slot (its tcgen05.wait::ld is behind it).  Nothing that it wrote is handed on
// with the arrival, so that need not wait for its stores to global memory, as one with release semantics does.
__device__ __forceinline__ void f8_release_slot(uint64_t* bar) {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    if ((threadIdx.x & 31) == 0)
        asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(f8_leader(bar)) : "memory");
}
// The two warps that hold the same tokens (quarter: 0 to 3).
__device__ __forceinline__ void f8_quarter_sync(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(2 + quarter) : "memory"); }

// The columns of a part (0 or 1) of the epilogue: its chunk i of 32, of NC.  Gated: chunks of the gate, then those of the up features
// that belong to them.
template <int NC, bool GATED>
__device__ __forceinline__ int f8_column(int part, int i) {
    return GATED ? (i >> 1) * 128 + 64 * part + 32 * (i & 1) : 32 * (NC * part + i);
}

// What a block of a pair has sent for and formed, for the other one to read where a wait gave up.
struct F8PairCounts {
    int x_copies, w_copies;  // stages that it has sent for
    int parts;               // leader: sums that it has committed
};
// The other block's flag: its waits may go well, for a sum that is committed but not formed.
__device__ __noinline__ void f8_tell_pair(volatile int* gave_up) {
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(f8_remote((const void*)gave_up, cluster_rank() ^ 1)), "r"(1) : "memory");
    asm volatile("fence.acq_rel.cluster;" ::: "memory");
}
// Where a wait of either block gave up, both come here: the error word, and a wait for what is in flight to them.  Both blocks' bytes count
// on the leader's barriers (a stage is x_bytes and w_bytes of each), and some may have been sent for that belong to stages of which others
// have not: the leader arrives for those that it has not arrived for, and counts what nobody sent as landed.
template <int x_bytes, int w_bytes>
__device__ __noinline__ void f8_pair_gave_up(const Fp8Args& g, uint64_t* full, uint64_t* part_full, int stages, const F8PairCounts* counts) {
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        atomicOr(g.err, SS_ERR_WAIT_LIMIT);
        const auto of = [&](uint32_t block, const int* p) {
            int v;
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(f8_remote(p, block)) : "memory");
            return v;
        };
        const int parts = of(0, &counts->parts);
        if (rank == 0) {
            const int x0 = counts->x_copies, w0 = counts->w_copies, x1 = of(1, &counts->x_copies), w1 = of(1, &counts->w_copies);
            const int all = max(max(x0, w0), max(x1, w1));
            for (int i = max(0, all - stages); i < all; ++i) {
                uint64_t* bar = &full[i % stages];
                if (i >= x0) mbar_expect_tx(bar, 2 * (x_bytes + w_bytes));
                const int missing = ((i >= x0) + (i >= x1)) * x_bytes + ((i >= w0) + (i >= w1)) * w_bytes;
                if (missing) asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(s_addr(bar)), "r"(missing) : "memory");
                mbar_drain(bar, (i / stages) & 1);
            }
        }
        f8_drain_ring(part_full, g.slots, parts);
    }
    cluster_sync_all();
}

// 16 rows of 64 bytes from `stage` to rows of the output that start on P bytes, P bytes a thread; `limit`: the bytes
// of a run that are there.
template <typename P>
__device__ __forceinline__ void f8_copy_run(const unsigned char* stage, unsigned char* out, int64_t pitch, int rows, int limit) {
    constexpr int per_row = 64 / (int)sizeof(P);
    const int lane = threadIdx.x & 31, at = lane % per_row * (int)sizeof(P);
#pragma unroll
    for (int i = 0; i < per_row / 2; ++i) {
        const int r = i * (32 / per_row) + lane / per_row;
        const P v = *reinterpret_cast<const P*>(stage + r * 64 + (((at >> 4) ^ ((r >> 1) & 3)) << 4) + (at & 15));
        if (r < rows && at < limit) *reinterpret_cast<P*>(out + r * pitch + at) = v;
    }
}
// A warp's 32 rows of 64 bytes, a row a thread, through 1 KB of shared memory of the warp's own, so that it writes whole
// runs of a row instead of 16 bytes of 32 rows at a time.  Rows of 64 bytes lie in `stage` with their four 16-byte pieces turned by
// (row / 2) % 4, which keeps both directions free of bank conflicts.  P: what is written at a time, which the output's rows start on and
// are a multiple of.
template <typename T, typename P>
__device__ __forceinline__ void f8_write_run(const Fp8Args& g, void* to, unsigned char* stage, const uint32_t (&w)[16], int m0, int f) {
    const int lane = threadIdx.x & 31, row = lane & 15, size = (int)sizeof(T);
    const int64_t pitch = g.ldc * size;
    unsigned char* out = (unsigned char*)to + m0 * pitch + (int64_t)f * size;
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
        f8_copy_run<P>(stage, out + 16 * h * pitch, pitch, rows - 16 * h, limit);
    }
}

// T: float, bf16, or (gated) uint8_t, e4m3.  SPLIT: a tile is one of `slices` parts of K, and its sums go to g.parts, [slices][tokens][ldc] in
// float32, where fp8_join_kernel takes them from.  Behind a wait that gave up F8_UNFORMED stands there in their place: a NaN that no
// arithmetic gives (results that are NaN have the bits 0x7fffffff).
#define F8_UNFORMED 0x7fc0beefu
template <int NC, bool GATED, typename T, typename P, bool SPLIT>
__global__ void __launch_bounds__(F8_MANY_THREADS, 1)
gemm_fp8_many_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Fp8Args g) {
    constexpr int bn = 64 * NC, w_rows = bn / 2, x_bytes = F8_BM * F8_BK, stage_bytes = x_bytes + w_rows * F8_BK;  // this block's halves
    static_assert(GATED ? NC == 4 : sizeof(T) > 1, "");
    static_assert(!SPLIT || (!GATED && sizeof(T) == 4), "");
    const int stages = g.stages, slots = g.slots;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + stages * stage_bytes);
    uint64_t* empty = full + stages;
    uint64_t* part_full = empty + stages;  // [8]
    uint64_t* part_empty = part_full + 8;  // [8]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(part_empty + 8);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    F8PairCounts* counts = reinterpret_cast<F8PairCounts*>(tmem_slot + 2);
    uint32_t* tops = reinterpret_cast<uint32_t*>(full) + 128;                   // [2][128 tokens][2 parts]
    float* biases = reinterpret_cast<float*>(tops + 4 * F8_BM);                // [2][256] of a tile's features
    unsigned char* runs = reinterpret_cast<unsigned char*>(biases + 2 * F8_MAX_BN);  // 1 KB for each epilogue warp

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();  // 0: the leader
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const int n_m = (g.tokens + 2 * F8_BM - 1) / (2 * F8_BM), n_out = n_m * ((g.features + bn - 1) / bn), n_tiles = SPLIT ? n_out * g.slices : n_out;
    const int k_blocks = (g.K + F8_BK - 1) / F8_BK, per = SPLIT ? (k_blocks + g.slices - 1) / g.slices : k_blocks;
    // of tile t: its slice, the tile of the output, its first block of K and how many there are (no slice is empty: launch_many)
    const auto slice_of = [&](int t) { return SPLIT ? t / n_out : 0; };
    const auto out_of = [&](int t) { return SPLIT ? t % n_out : t; };
    const auto blocks_of = [&](int t) { return SPLIT ? min(per, k_blocks - slice_of(t) * per) : k_blocks; };
    const int first_k = slice_of(pair) * per;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int s = 0; s < slots; ++s) { mbar_init(&part_full[s], 1); mbar_init(&part_empty[s], 16); }
        *gave_up = 0;
        counts->x_copies = counts->w_copies = counts->parts = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();  // both blocks' barriers exist before either signals the other's
    const int first = min(stages, pair < n_tiles ? blocks_of(pair) : 0);  // stages of the first tile that are fetched ahead
    const int bytes = 2 * stage_bytes;  // of both blocks
    if (threadIdx.x == 0) {
        // the weights do not depend on the kernels in front: their first tiles are on the way before those are through
#pragma unroll 1
        for (int k = 0; k < first; ++k) {
            if (rank == 0) mbar_expect_tx(&full[k], bytes);
            f8_load_pair(tiles + k * stage_bytes + x_bytes, &map_w, (first_k + k) * F8_BK, (out_of(pair) / n_m) * bn + rank * w_rows, &full[k]);
        }
    }
    pdl_wait();
    if (warp == 1) {  // the same warp of both blocks allocates all 512 columns of the pair
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        pdl_launch_dependents();  // (this warp alone: one call of a block lets the kernel behind go)
    } else if (threadIdx.x == 0) {
#pragma unroll 1
        for (int k = 0; k < first; ++k) f8_load_pair(tiles + k * stage_bytes, &map_x, (first_k + k) * F8_BK, (out_of(pair) % n_m) * 2 * F8_BM + rank * F8_BM, &full[k]);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();  // the tensor memory of both blocks has been taken
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        unsigned char* stage = runs + (warp - 4) * 1024;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        int slot = 0, turn = 0, tile = 0;
        uint32_t parity = 0, there = 0;
        bool ok = true;
#pragma unroll 1
        for (int t = pair; t < n_tiles; t += n_pairs) {
            const int n0 = (out_of(t) / n_m) * bn, m0 = (out_of(t) % n_m) * 2 * F8_BM + rank * F8_BM + quarter * 32, m = m0 + lane;
            const int k_iters = blocks_of(t);
            const int64_t k0 = slice_of(t) * per;
            ++tile;
            if (g.bias) {
                const int c = threadIdx.x - 128;
                if (c < bn) biases[(tile & 1) * F8_MAX_BN + c] = n0 + c < g.features ? f8_bias(g, n0 + c) : 0.f;
            }
            float acc[NC][32];
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < 32; ++e) acc[i][e] = 0.f;
            // the scales of a block of K: the token's, and those of the chunks' features (no chunk lies in two blocks;
            // a part's chunks lie in one, gated in two)
            constexpr int NW = GATED ? 2 : 1, PER = NC / NW;
            // Fetched F8_FLIGHT blocks ahead, into registers: a block of K takes about 0.5 us, a load from memory about 1.
            const float* xs = g.x_scale + (int64_t)min(m, g.tokens - 1) * g.x_row + k0 * g.x_block;  // (rows behind the last token are not written)
            const float* ws[NW];
#pragma unroll
            for (int i = 0; i < NW; ++i)
                ws[i] = g.w_scale + (int64_t)min((n0 + f8_column<NC, GATED>(part, i * PER)) / FP8_BLOCK, (g.features - 1) / FP8_BLOCK) * g.w_row + k0 * g.w_block;
            float next_x[F8_FLIGHT], next_w[F8_FLIGHT][NW];
            int fetched = 0;
            const auto fetch_scales = [&](int u) {
                if (fetched >= k_iters) return;
                ++fetched;
                next_x[u] = *xs;
                xs += g.x_block;
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    next_w[u][i] = __ldg(ws[i]);
                    ws[i] += g.w_block;
                }
            };
#pragma unroll
            for (int u = 0; u < F8_FLIGHT; ++u) fetch_scales(u);
            const auto take_sums = [&](int u) {
                if (!__all_sync(0xffffffffu, there) && !f8_wait(&part_full[slot], parity, gave_up)) { ok = false; return; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = lanes + slot * g.slot_columns;
                // 32 columns are on their way while the 32 before them are added
                float r[2][32], f[NW];
                f8_tmem_load<32>(at + f8_column<NC, GATED>(part, 0), r[0]);
#pragma unroll
                for (int i = 0; i < NW; ++i) f[i] = __fmul_rn(next_x[u], next_w[u][i]);
                fetch_scales(u);
                uint64_t* through = &part_empty[slot];
                if (++slot == slots) { slot = 0; parity ^= 1; }
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    f8_tmem_wait<32>(r[i & 1]);
                    if (i + 1 < NC) {
                        f8_tmem_load<32>(at + f8_column<NC, GATED>(part, i + 1), r[(i + 1) & 1]);
                    } else {
                        f8_release_slot(through);
                        there = f8_look(&part_full[slot], parity);  // (the answer is here when the last columns are added)
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) f8_add2(reinterpret_cast<float(&)[2]>(acc[i][e]), r[i & 1][e], r[i & 1][e + 1], f[i / PER]);
                }
            };
#pragma unroll 1
            for (int k = 0; ok && k < k_iters; k += F8_FLIGHT) {
#pragma unroll
                for (int u = 0; u < F8_FLIGHT; ++u)
                    if (ok && k + u < k_iters) take_sums(u);
            }
            // (behind a wait that gave up a warp writes nothing but still comes to the barriers, where the others wait for it)
            // (the flag, not the waits' results: an issuer that gave up has committed what is not formed)
            bool formed = !__shfl_sync(0xffffffffu, *gave_up, 0);
            if (g.bias) {
                // (two sets: a set is written again two tiles later, behind a barrier that all warps reach when they have read it)
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const float* bias = biases + (tile & 1) * F8_MAX_BN;
#pragma unroll
                for (int i = 0; i < NC; ++i)
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 v = *reinterpret_cast<const float4*>(bias + f8_column<NC, GATED>(part, i) + e);
                        acc[i][e] += v.x; acc[i][e + 1] += v.y; acc[i][e + 2] += v.z; acc[i][e + 3] += v.w;
                    }
            }
            const int of0 = GATED ? n0 / 2 : n0;  // first output feature of the tile
            constexpr int NO = GATED ? 2 : NC;
            if constexpr (GATED) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 32; ++e) acc[i][e] = silu_mul<sizeof(T) < 4>(acc[i][e], acc[NC - 2 + i][e]);
            }
            if constexpr (sizeof(T) == 1) {
                const int f = of0 + 64 * part, left = g.out_features - f;
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    if (j >= left) acc[j >> 5][j & 31] = 0.f;
                    top = max(top, __float_as_uint(acc[j >> 5][j & 31]) & 0x7fffffffu);
                }
                // (two sets: a set is written again two tiles later, behind a barrier that both warps reach when they have read it)
                uint32_t* shared_top = tops + turn * 2 * F8_BM + (quarter * 32 + lane) * 2;
                turn ^= 1;
                shared_top[part] = top;
                f8_quarter_sync(quarter);
                formed = !__shfl_sync(0xffffffffu, *gave_up, 0);
                const uint2 all = *reinterpret_cast<const uint2*>(shared_top);
                const Fp8Scale r = fp8_scale(max(all.x, all.y));
                if (!formed || m >= g.tokens || of0 >= g.out_features) continue;
                if (part == 0) g.out_scale[(int64_t)(of0 / FP8_BLOCK) * g.tokens + m] = r.scale;
                uint8_t* to = (uint8_t*)g.out + (int64_t)m * g.ldc + f;
#pragma unroll
                for (int j = 0; j < 64; j += 16) {
                    uint32_t q[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int at = j + 4 * h;
                        const float four[4] = {acc[at >> 5][at & 31], acc[at >> 5][(at & 31) + 1], acc[at >> 5][(at & 31) + 2], acc[at >> 5][(at & 31) + 3]};
                        q[h] = fp8_quantize4(four, r);
                    }
                    if (left >= j + 16) {
                        *reinterpret_cast<uint4*>(to + j) = make_uint4(q[0], q[1], q[2], q[3]);
                    } else {
#pragma unroll
                        for (int h = 0; h < 4; ++h) fp8_store4(to + j + 4 * h, left - j - 4 * h, q[h]);
                    }
                }
            } else {
                if (!formed) {
                    if constexpr (!SPLIT) continue;
#pragma unroll
                    for (int i = 0; i < NC; ++i)
#pragma unroll
                        for (int e = 0; e < 32; ++e) acc[i][e] = __uint_as_float(F8_UNFORMED);
                }
                void* to = SPLIT ? (void*)(g.parts + (int64_t)slice_of(t) * g.tokens * g.ldc) : g.out;
#pragma unroll
                for (int i = 0; i < NO; ++i) {
                    const int f = of0 + f8_column<NC, GATED>(part, i);
                    uint32_t w[16];
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(acc[i][16 * h + e]);
                            f8_write_run<T, P>(g, to, stage, w, m0, f + 16 * h);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(acc[i][2 * e], acc[i][2 * e + 1]);
                            w[e] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        f8_write_run<T, P>(g, to, stage, w, m0, f);
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0 || warp == 2) {  // the tokens' rows, and the weights'
            const bool x = warp == 0;
            const CUtensorMap* map = x ? &map_x : &map_w;
            unsigned char* to = tiles + (x ? 0 : x_bytes);
            int it = 0, s = 0;
            uint32_t parity = 1;  // of the round before the first: the stages are free
            bool ok = true;
#pragma unroll 1
            for (int t = pair; t < n_tiles && ok; t += n_pairs) {
                const int row = x ? (out_of(t) % n_m) * 2 * F8_BM + rank * F8_BM : (out_of(t) / n_m) * bn + rank * w_rows;
                const int k0 = slice_of(t) * per, k_iters = blocks_of(t);
#pragma unroll 1
                for (int k = 0; k < k_iters; ++k, ++it) {
                    if (it >= first) {
                        if (!f8_wait(&empty[s], parity, gave_up)) { ok = false; break; }
                        if (elect_one()) {
                            if (x && rank == 0) mbar_expect_tx(&full[s], bytes);
                            f8_load_pair(to + s * stage_bytes, map, (k0 + k) * F8_BK, row, &full[s]);
                        }
                        __syncwarp();
                    }
                    if (++s == stages) { s = 0; parity ^= 1; }
                }
            }
            if (lane == 0) (x ? counts->x_copies : counts->w_copies) = it;
        } else if (warp == 1 && rank == 0) {
            const uint32_t idesc = f8_idesc(2 * F8_BM, bn);
            const uint64_t x_first = smem_desc(tiles), w_first = smem_desc(tiles + x_bytes);
            int it = 0, s = 0, slot = 0;
            uint32_t parity = 0, free_parity = 1;  // (of the round before the first: the slots are free)
            bool ok = true;
#pragma unroll 1
            for (int t = pair; t < n_tiles && ok; t += n_pairs) {
                const int k_iters = blocks_of(t);
#pragma unroll 1
                for (int k = 0; k < k_iters; ++k, ++it) {
                    if (!f8_wait(&full[s], parity, &part_empty[slot], free_parity, gave_up)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t x_desc = x_first + s * (stage_bytes >> 4), w_desc = w_first + s * (stage_bytes >> 4);
                    const uint32_t acc = tmem + slot * g.slot_columns;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < F8_BK / 32; ++kk) umma_f8_pair(acc, x_desc + (uint64_t)(kk * 2), w_desc + (uint64_t)(kk * 2), idesc, kk != 0);
                        f8_commit_pair(&part_full[slot]);
                        f8_commit_pair(&empty[s]);
                    }
                    __syncwarp();
                    if (++s == stages) { s = 0; parity ^= 1; }
                    if (++slot == slots) { slot = 0; free_parity ^= 1; }
                }
            }
            if (!ok) f8_tell_pair(gave_up);
            if (lane == 0) counts->parts = it;
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*gave_up && threadIdx.x == 0) f8_tell_pair(gave_up);  // the other block comes along
    cluster_sync_all();  // neither block leaves (or frees tensor memory) while the other may still signal it
    if (*gave_up) f8_pair_gave_up<x_bytes, w_rows * F8_BK>(g, full, part_full, stages, counts);
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// The parts of K put together: y = sum over the slices, in their order, + bias, rounded once; a warp takes 128 features of a token, a lane
// four of them.  Where a wait of this product gave up, its parts say which sums are not formed, and nothing is written there.
__global__ void __launch_bounds__(256) fp8_join_kernel(const Fp8Args g, int64_t ldp, int64_t units) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (unit >= units) return;
    const int lane = threadIdx.x & 31, across = (g.features + 127) / 128, token = (int)(unit / across);
    const int apart = (g.ldc & 3) == 0 ? 1 : 32, f = (int)(unit % across) * 128 + (apart == 1 ? lane * 4 : lane);
    if (f >= g.features) return;
    const int64_t plane = g.tokens * ldp;
    const float* p = g.parts + token * ldp + f;
    float v[4] = {};
    bool formed = true;
    const auto add = [&](int e, float part) {
        formed = formed && __float_as_uint(part) != F8_UNFORMED;
        v[e] += part;
    };
    if (apart == 1) {  // (rows of the parts are as long as four elements times some number: those behind the last belong to nobody)
#pragma unroll 4
        for (int s = 0; s < g.slices; ++s) {
            const float4 t = *reinterpret_cast<const float4*>(p + s * plane);
            add(0, t.x); add(1, t.y); add(2, t.z); add(3, t.w);
        }
    } else {
        for (int s = 0; s < g.slices; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (f + 32 * e < g.features) add(e, p[s * plane + 32 * e]);
    }
    if (!formed) return;
    if (g.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f + e * apart < g.features) v[e] += f8_bias(g, f + e * apart);
    }
    f8_store4(g, token, f, apart, v);
}

// ---------------------------------------------------------------- host side

typedef CUresult (*F8Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// e4m3 matrix [rows, K] with row stride ld bytes; box = 128 x box_rows.
static int f8_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows) {
    static F8Encode enc = nullptr;
    if (!enc) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return -2001;
        enc = (F8Encode)p;
    }
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {F8_BK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : -2002;
}

#define F8_SMEM_MAX 232448  // 227 KB of a block
#define F8_SMEM_SM 233472   // 228 KB of an SM, 1 KB of it each block's own
#define F8_SMEM_REST 1536   // alignment, barriers

// Only asked about, never launched: blocks of the shape of the kernel for few tokens.  About a kernel that takes tensor memory the
// runtime answers one block an SM, whatever it takes of it.
__global__ void __launch_bounds__(F8_THREADS) f8_few_shape() {}

// How many clusters of `n` blocks of the kernel for few tokens run at the same time where the ring is sized for `per_sm` blocks an
// SM (n = 1: blocks).
extern "C" int ss_gemm_fp8_resident(int n, int per_sm) {
    static SsPerDevice opted;
    if (n < 1 || n > 8 || per_sm < 1 || ss_opt_in_smem(f8_few_shape, F8_SMEM_MAX, opted)) return 0;
    return ss_resident_clusters(f8_few_shape, F8_THREADS, per_sm > 1 ? F8_SMEM_SM / per_sm - 1024 : F8_SMEM_MAX, n);
}

template <int NC, bool GATED, typename T, typename P, bool SPLIT = false>
static int launch_many(const Fp8Call& c, Fp8Args& g) {
    CUtensorMap map_x, map_w;
    constexpr int bn = 64 * NC;
    if (int rc = f8_map(&map_x, c.x, g.tokens, g.K, c.ldx, F8_BM)) return rc;
    if (int rc = f8_map(&map_w, c.w, g.features, g.K, c.ldw, bn / 2)) return rc;
    static SsPerDevice opted;
    if (int rc = ss_opt_in_smem(gemm_fp8_many_kernel<NC, GATED, T, P, SPLIT>, F8_SMEM_MAX, opted)) return rc;
    // what the warps take of the registers is what the block is launched with: a build with fewer would wait for the rest
    static const int registers = [] {
        cudaFuncAttributes a;
        return cudaFuncGetAttributes(&a, gemm_fp8_many_kernel<NC, GATED, T, P, SPLIT>) == cudaSuccess ? a.numRegs : 0;
    }();
    if (registers * F8_MANY_THREADS < 128 * 40 + 256 * 232) return -2008;
    constexpr int rest = F8_SMEM_REST + 2 * 2 * F8_BM * 4 + 2 * F8_MAX_BN * 4 + 8 * 1024, stage = (F8_BM + bn / 2) * F8_BK;
    g.stages = (F8_SMEM_MAX - rest) / stage;
    if (g.stages > 12) g.stages = 12;
    g.slot_columns = NC == 1 ? 64 : NC == 2 ? 128 : 256;
    g.slots = 512 / g.slot_columns;
    const int64_t n_tiles = (int64_t)((g.tokens + 255) / 256) * ((g.features + bn - 1) / bn) * (SPLIT ? g.slices : 1);
    if (n_tiles > INT32_MAX / 2) return -2003;
    const int pairs = (int)(n_tiles < ss_sm_count() / 2 ? n_tiles : ss_sm_count() / 2);
    ss_launch_cluster_x(gemm_fp8_many_kernel<NC, GATED, T, P, SPLIT>, dim3(2 * pairs), dim3(F8_MANY_THREADS), g.stages * stage + rest, c.stream, 2, map_x, map_w, g);
    return SS_LAUNCH_CHECK();
}

// K in slices: the product to g.parts, then what puts the parts together.
template <int NC>
static int launch_many_split(const Fp8Call& c, Fp8Args& g) {
    const int k_blocks = (g.K + F8_BK - 1) / F8_BK, per = (k_blocks + g.slices - 1) / g.slices;
    g.slices = (k_blocks + per - 1) / per;  // that have any K
    const int64_t ldp = ((int64_t)g.features + 3) & -4, units = (int64_t)g.tokens * ((g.features + 127) / 128), blocks = (units + 7) / 8;
    if (blocks > INT32_MAX) return -2003;
    Fp8Args product = g;
    product.bias = nullptr; product.out = g.parts; product.ldc = ldp; product.out_type = SS_F32; product.out_features = (int)ldp;
    if (int rc = launch_many<NC, false, float, uint4, true>(c, product)) return rc;
    ss_launch(fp8_join_kernel, dim3((unsigned)blocks), dim3(256), 0, c.stream, g, ldp, units);
    return SS_LAUNCH_CHECK();
}

template <int NC, bool GATED>
static int launch_many_as(const Fp8Call& c, Fp8Args& g) {
    if constexpr (GATED)
        if (g.out_type == F8_OUT_FP8) return launch_many<NC, GATED, uint8_t, uint4>(c, g);
    const bool wide = (g.ldc | g.out_features) * (g.out_type == SS_F32 ? 4 : 2) % 16 == 0;
    if (g.out_type == SS_F32) return wide ? launch_many<NC, GATED, float, uint4>(c, g) : launch_many<NC, GATED, float, uint32_t>(c, g);
    return wide ? launch_many<NC, GATED, bf16, uint4>(c, g) : launch_many<NC, GATED, bf16, uint16_t>(c, g);
}

template <int MT, int C>
static int launch_few(const Fp8Call& c, Fp8Args& g, int per_sm) {
    CUtensorMap map_x, map_w;
    const int bn = g.bn, slices = g.slices;
    constexpr int FL = MT * F8_BM;
    if (int rc = f8_map(&map_x, c.x, g.tokens, g.K, c.ldx, bn)) return rc;
    if (int rc = f8_map(&map_w, c.w, g.features, g.K, c.ldw, FL)) return rc;
    static SsPerDevice opted;
    if (int rc = ss_opt_in_smem(gemm_fp8_few_kernel<MT, C>, F8_SMEM_MAX, opted)) return rc;
    const int stage = (FL + bn) * F8_BK;
    const int rest = F8_SMEM_REST + 32 * f8_few_floats(MT, C) + (slices > 1 ? slices * ((bn + slices - 1) / slices) * FL * 4 : 0);  // a cluster's blocks: the sums they own
    g.slot_columns = 2 * C < 32 ? 32 : 2 * C;
    const int tmem = per_sm > 1 ? 256 : 512;
    g.slots = tmem / (MT * g.slot_columns);
    if (g.slots > 4) g.slots = 4;
    if (g.slots < 2) return -2007;
    const int room = per_sm > 1 ? F8_SMEM_SM / per_sm - 1024 : F8_SMEM_MAX;
    int stages = (room - rest) / stage;
    const int needed = slices > 1 ? 2 : (bn * FL * 4 + stage - 1) / stage;  // alone, the ring also holds the sums
    stages = stages < needed ? needed : stages > 12 ? 12 : stages;
    g.stages = stages;
    const int smem = stages * stage + rest;
    if (smem > F8_SMEM_MAX) return -2007;
    const dim3 grid((g.tokens + bn - 1) / bn, (g.features + FL - 1) / FL, slices);
    if (slices > 1) ss_launch_cluster(gemm_fp8_few_kernel<MT, C>, grid, dim3(F8_THREADS), smem, c.stream, slices, map_w, map_x, g);
    else ss_launch(gemm_fp8_few_kernel<MT, C>, grid, dim3(F8_THREADS), smem, c.stream, map_w, map_x, g);
    return SS_LAUNCH_CHECK();
}

// Row strides are multiples of 16 bytes and bases stand on 16 bytes.
// gated: w's rows alternate 128 gate and 128 up features; out_features <= features / 2 columns of silu(gate) * up are written.
// many = 0: bn tokens a tile (a multiple of 16 up to 256, gated 128; ops/fp8.py's own plans go up to 128, gated 64), slices 1..8 of K, `per_sm` blocks an SM that the ring is sized for
// (2: bn up to 64, gated 32).
// many = 1: bn features a tile (64, 128 or 256; gated: 256); not gated, of 128 or 256 features: slices 1..8 of K, with `parts` from 2 on.
extern "C" int ss_gemm_fp8(const Fp8Call* call) {
    const Fp8Call& c = *call;
    if (c.tokens <= 0 || c.features <= 0 || c.out_features <= 0) return 0;
    if (c.tokens > INT32_MAX - 256 || c.features > INT32_MAX - 256 || c.K <= 0 || c.K > INT32_MAX - 256 || c.ldx % 16 || c.ldw % 16 || c.ldx < c.K || c.ldw < c.K) return -2003;
    if (((uintptr_t)c.x & 15) || ((uintptr_t)c.w & 15) || ((uintptr_t)c.out & 15)) return -2004;
    if (c.gated ? (c.features % 256 || c.out_features > c.features / 2) : (c.out_features != c.features || c.out_type == F8_OUT_FP8)) return -2005;
    if (c.out_type == F8_OUT_FP8 && c.ldc % 16) return -2005;
    const int bn = (int)c.bn, slices = (int)c.slices, per_sm = (int)c.per_sm;
    if (bn < 16 || bn > F8_MAX_BN || (c.many ? bn != 64 && bn != 128 && bn != 256 : bn % 16) || (c.many && c.gated && bn != 256)
        || (c.many && (slices < 1 || slices > 8 || (slices > 1 && (c.gated || bn == 64 || !c.parts || ((uintptr_t)c.parts & 15)))))
        || (!c.many && (bn > (c.gated ? 128 : 256) / (per_sm > 1 ? 4 : 1) || slices < 1 || slices > 8 || per_sm < 1 || per_sm > 2
                        || (c.features + F8_BM - 1) / F8_BM > 65535))) return -2006;
    Fp8Args g = {};
    g.x_scale = c.x_scale; g.x_row = c.x_row; g.x_block = c.x_block; g.w_scale = c.w_scale; g.w_row = c.w_row; g.w_block = c.w_block;
    g.parts = c.parts; g.bias = c.bias; g.out = c.out; g.out_scale = c.out_scale; g.err = c.err; g.ldc = c.ldc;
    g.tokens = (int)c.tokens; g.features = (int)c.features; g.K = (int)c.K; g.out_features = (int)c.out_features;
    g.out_type = (int)c.out_type; g.bias_f32 = (int)c.bias_f32; g.bn = bn; g.slices = slices;
    if (c.many) {
        if (c.gated) return launch_many_as<4, true>(c, g);
        if (slices > 1) return bn == 128 ? launch_many_split<2>(c, g) : launch_many_split<4>(c, g);
        return bn == 64 ? launch_many_as<1, false>(c, g) : bn == 128 ? launch_many_as<2, false>(c, g) : launch_many_as<4, false>(c, g);
    }
    if (c.gated)
        return bn <= 16 ? launch_few<2, 8>(c, g, per_sm) : bn <= 32 ? launch_few<2, 16>(c, g, per_sm) : bn <= 64 ? launch_few<2, 32>(c, g, per_sm) : launch_few<2, 64>(c, g, per_sm);
    return bn <= 16 ? launch_few<1, 8>(c, g, per_sm) : bn <= 32 ? launch_few<1, 16>(c, g, per_sm) : bn <= 64 ? launch_few<1, 32>(c, g, per_sm)
         : bn <= 128 ? launch_few<1, 64>(c, g, per_sm) : launch_few<1, 128>(c, g, per_sm);
}

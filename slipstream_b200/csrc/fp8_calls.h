// The arguments of the 8-bit float kernels' entry points, one record a call.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#define FP8_BLOCK 128  // elements that share a scale: of a row, and rows and columns of a weight

// The widest row: its kernels count elements in 32 bits, and a loop of theirs steps over up to 4,096 at a time.
constexpr int64_t FP8_MAX_WIDTH = INT32_MAX - 8192;

// Scales: that of row r (of rows) or of the row's block of 128 (of weights) and of column block b stands at r * scale_row + b * scale_block.
struct Fp8RowsCall {
    const void* x;  // quantize: [rows, width], row stride `stride` elements; dequantize: unused; norm: the stream, [rows, width]
    int64_t stride;
    uint8_t* q;  // [rows, width], row stride q_stride
    int64_t q_stride;
    float* scales;
    int64_t scale_row, scale_block;
    int64_t rows, width, dtype;  // SS_F32 or SS_BF16: of x; of the values; of delta
    int64_t blocks;              // quantize and dequantize: 1, blocks of 128 rows share a scale
    int64_t early;               // quantize (rows) and dequantize: the kernel behind may start at once
    void* y;                     // dequantize: [rows, width]; norm: residual_out or null (may be x)
    const void* delta;           // norm: [rows, width] or null
    const void* weight;
    int64_t w_f32;
    double eps;
    int* err;
    cudaStream_t stream;
};

struct Fp8Call {
    const void* x;  // [tokens, K] e4m3, row stride ldx
    int64_t ldx;
    const float* x_scale;
    int64_t x_row, x_block;
    const void* w;  // [features, K] e4m3, row stride ldw
    int64_t ldw;
    const float* w_scale;
    int64_t w_row, w_block;
    const void* bias;
    int64_t bias_f32;
    void* out;  // [tokens, ldc]
    int64_t ldc, out_type;  // SS_F32, SS_BF16, or 2: e4m3, with
    float* out_scale;       // its scales, [ceil(out_features / 128)][tokens]
    int64_t tokens, features, K, gated, out_features, many, bn, slices, per_sm;
    int* err;
    cudaStream_t stream;
    float* parts;  // many, slices > 1: [slices][tokens][features up to a multiple of 4], on 16 bytes
};

extern "C" {
int ss_quantize_fp8(const Fp8RowsCall* call);
int ss_dequantize_fp8(const Fp8RowsCall* call);
int ss_add_rmsnorm_fp8(const Fp8RowsCall* call);
int ss_gemm_fp8(const Fp8Call* call);
}

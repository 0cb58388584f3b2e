// The arguments of the 8-bit kernels' entry points, one record a call.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

// The widest row: its kernels count elements in 32 bits, and a loop of theirs steps over up to 4,096 at a time.
constexpr int64_t INT8_MAX_WIDTH = INT32_MAX - 8192;

struct Int8RowsCall {
    const void* x;  // quantize: [rows, width], row stride `stride` elements; dequantize: unused; norm: the stream, [rows, width]
    int64_t stride;
    int8_t* q;  // [rows, width], row stride q_stride
    int64_t q_stride;
    float* scales;
    int64_t rows, width, dtype;  // SS_F32 or SS_BF16: of x; of the values; of delta
    int64_t early;               // quantize and dequantize: the kernel behind may start at once
    void* y;                     // dequantize: [rows, width]; norm: residual_out or null (may be x)
    const void* delta;           // norm: [rows, width] or null
    const void* weight;
    int64_t w_f32;
    double eps;
    int* err;
    cudaStream_t stream;
};

struct Int8Call {
    const void* x;  // [tokens, K] int8, row stride ldx
    int64_t ldx;
    const float* x_scale;
    const void* w;  // [features, K] int8, row stride ldw
    int64_t ldw;
    const float* w_scale;
    const void* bias;
    int64_t bias_f32;
    void* out;  // [tokens, ldc]
    int64_t ldc, out_f32, tokens, features, K, gated, out_features, many, bn, slices, per_sm, steps;
    int* err;
    cudaStream_t stream;
};

extern "C" {
int ss_quantize_rows_int8(const Int8RowsCall* call);
int ss_dequantize_rows_int8(const Int8RowsCall* call);
int ss_add_rmsnorm_int8(const Int8RowsCall* call);
int ss_gemm_int8(const Int8Call* call);
}

// The arguments of the log probabilities' entry point.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

constexpr int64_t LOGPROBS_MAX_TOP = 64;

struct LogprobCall {
    const void* logits;  // [rows, vocabulary], row stride `stride` elements
    int64_t stride, rows, vocabulary, dtype;  // SS_F32 or SS_BF16
    const void* tokens;  // [rows]
    int64_t wide;        // 64-bit tokens
    int64_t top;
    float* out;  // [rows][3 + 2 top]: log probability, entropy, rank (int32), the largest log probabilities, their tokens (int32)
    int* err;
    cudaStream_t stream;
};

extern "C" int ss_token_logprobs(const LogprobCall* call);

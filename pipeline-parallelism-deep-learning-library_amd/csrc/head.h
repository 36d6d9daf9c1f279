// Internal interfaces of a language model head's operators: the host's checks and plans (head.cpp)
// and the kernels (quantize_kernels.hip, gemm_blocks_*_kernels.hip, logits_kernels.hip).
//
// Every matrix is given by the address of its first element and a row pitch in elements; extents
// fit 31 bits, and the host has proved that every element lies inside its storage.
#pragma once

#include "lg_internal.h"

namespace lg {

constexpr uint32_t BLOCK_K = 128;  // columns that share a scale
constexpr uint32_t TOP_MAX = 128;  // alternatives of a row, at most

struct QuantizeArgs {
    const void* x;
    int64_t x_pitch;
    uint8_t* q;
    int64_t q_pitch;
    void* s;  // f32, or e8m0 bytes
    int64_t s_pitch;
    uint32_t rows, cols;  // of q; transposed: element (r, c) of x is at x[c * x_pitch + r]
    uint32_t dtype;       // lg_dtype of x
    uint32_t block;       // rows that share a scale: 1 or 128
    bool transposed, e8m0;
};
void launch_quantize_blocks(Context* ctx, hipStream_t s, const QuantizeArgs& args);

struct GemmBlocksArgs {
    const uint8_t* a;  // [m, k] e4m3
    const uint8_t* b;  // [n, k] e4m3
    int64_t a_pitch, b_pitch;
    const void* sa;  // [ceil(m / a_block), ceil(k / 128)], f32 or e8m0
    const void* sb;  // [ceil(n / b_block), ceil(k / 128)]
    int64_t sa_pitch, sb_pitch;
    void* c;
    int64_t c_pitch;
    uint32_t m, n, k;
    uint32_t a_block, b_block;  // 1 or 128
    uint32_t out;               // lg_dtype of c
    float alpha, beta;
    bool e8m0;
};
// One for each type of c, in a file of its own; extents of C below 2^22.
void launch_gemm_blocks_f32(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& args);
void launch_gemm_blocks_f16(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& args);
void launch_gemm_blocks_bf16(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& args);

struct LogprobArgs {
    const void* x;
    int64_t x_pitch;
    uint32_t dtype, rows, cols;
    float temperature;
    const int32_t* tokens;  // or null, with logprobs
    float* logprobs;
    float* entropy;  // or null
    float* stats;    // or null: (max, log of the sum) a row
    int64_t stats_pitch;
    float* top;  // or null, with top_ids
    int32_t* top_ids;
    int64_t top_pitch, ids_pitch;
    uint32_t k;
};
void launch_token_logprobs(lg_ctx* ctx, hipStream_t s, const LogprobArgs& args);

struct LogprobBackArgs {
    const void* x;
    void* dx;
    int64_t x_pitch, dx_pitch;
    uint32_t dtype, rows, cols;
    float temperature;
    const int32_t* tokens;
    const float* stats;
    int64_t stats_pitch;
    const float* entropy;  // with dentropy
    const float* dlogprobs;
    const float* dentropy;  // or null
};
void launch_token_logprobs_backward(lg_ctx* ctx, hipStream_t s, const LogprobBackArgs& args);

struct DistillArgs {
    const void* x;
    void* dx;  // or null
    int64_t x_pitch, dx_pitch;
    uint32_t dtype, rows, cols;
    const int32_t* ids;
    const float* values;
    int64_t ids_pitch, values_pitch;
    uint32_t k;
    const float* weights;  // or null: all one
    float temperature;
    bool normalize;
    float* losses;
};
void launch_distill_grad(lg_ctx* ctx, hipStream_t s, const DistillArgs& args);

}  // namespace lg

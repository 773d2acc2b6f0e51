// Launch interface of what stands around the routed experts of a block: the norm in front of them, the choice of a token's experts, and the
// experts themselves for a few tokens. All launches go to the given stream and read and write this GPU's memory only.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dx {

// ---- root-mean-square norm (norm.cu) -------------------------------------------------------------------------------------------------
constexpr int kNormMaxHidden = 32768;

struct NormArgs {
    const void* x;         // bf16, rows x_stride elements apart, 16-byte aligned
    const void* residual;  // same, or null
    long long x_stride, residual_stride;
    const void* weight;    // bf16 or (weight_f32) fp32 [hidden]
    int weight_f32;
    void* total;           // bf16 [rows, hidden]: x + residual (null without a residual)
    void* y;               // bf16 [rows, hidden], or null
    uint8_t* q;            // e4m3 [rows, hidden], or null
    float* scales;         // fp32 [rows, hidden / 128] of q
    int round_scale;       // powers of two
    long long rows;
    int hidden;            // a multiple of 8; of 128 with q
    float eps;
};
cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t stream);

struct NormBwdArgs {
    const void* total;     // bf16 [rows, hidden]: what was normed
    const void* dy;        // bf16 [rows, hidden]
    const void* dtotal;    // bf16 [rows, hidden] (gradient that reaches the sum past the norm), or null
    long long total_stride, dy_stride, dtotal_stride;
    const void* weight;
    int weight_f32;
    void* dx;              // bf16 [rows, hidden]
    float* partial;        // fp32 [norm_bwd_ctas(), hidden]
    void* dweight;         // [hidden], of the weight's type
    long long rows;
    int hidden;
    float eps;
};
int norm_bwd_ctas(long long rows, int hidden, int num_sms);
cudaError_t launch_rms_norm_bwd(const NormBwdArgs& a, int num_sms, cudaStream_t stream);

// ---- choice of the experts (router.cu) --------------------------------------------------------------------------------------------------
constexpr int kRouterMaxExperts = 1024;
constexpr int kRouterMaxTopk = 32;

struct SelectArgs {
    const void* logits;    // fp32 or (bf16) bf16, rows logits_stride elements apart
    int bf16;
    long long logits_stride;
    int64_t* idx;          // [tokens, topk]
    float* weights;        // [tokens, topk]
    const float* dweights; // backward only: [tokens, topk]
    void* dlogits;         // backward only: [tokens, experts], of the logits' type
    int tokens, experts, topk, renormalize;
};
cudaError_t launch_select_experts(const SelectArgs& a, cudaStream_t stream);
cudaError_t launch_select_experts_bwd(const SelectArgs& a, cudaStream_t stream);

// ---- experts for a few tokens (few_tokens.cu) ---------------------------------------------------------------------------------------------
constexpr int kFewMaxTokens = 32;
constexpr int kFewMaxTopk = 32;
constexpr int kFewMaxExperts = 1024;

struct FewTokensArgs {
    const void* x;            // bf16 [tokens, hidden], rows x_stride elements apart
    long long x_stride;
    const int64_t* idx;       // [tokens, topk]; ids outside [first, first + experts) are skipped
    const float* weights;     // [tokens, topk]
    const void* w13;          // [experts, 2 inter, hidden] = [gate; up], bf16 or (fp8) e4m3
    const void* w2;           // [experts, hidden, inter]
    const float* s13;         // fp8: [experts, 2 inter / 128, hidden / 128]
    const float* s2;          // fp8: [experts, hidden / 128, inter / 128]
    void* scratch;            // few_tokens_scratch() bytes, 256-byte aligned, for this call alone
    void* out;                // bf16 [tokens, hidden]
    int64_t first;
    int tokens, topk, experts, hidden, inter, fp8;
    int* error_flag;          // set where a wait for a copy ran out
    long long wait_limit;     // cycles
};
size_t few_tokens_scratch(const FewTokensArgs& a);
cudaError_t launch_few_tokens(const FewTokensArgs& a, int num_sms, cudaStream_t stream);

}  // namespace dx

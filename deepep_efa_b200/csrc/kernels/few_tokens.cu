// A layer of routed SwiGLU experts for a few tokens, in two launches: out[t] = sum_k weights[t, k] W2[e] (silu(G[e] x[t]) * (U[e] x[t])), e = idx[t, k].
//
// A warp per output value: one of the hidden values of a (token, choice) pair, then one of a token's results.
#include "block_api.h"
#include "launch.cuh"
#include "sigmoid.cuh"

namespace dx {

namespace {

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// sum over this lane's share of row . x; `scale`: one per 128 channels of the row
template <bool kFp8>
__device__ __forceinline__ float row_dot(const void* w, long long row, const float* scale, const __nv_bfloat16* x, int n, int lane) {
    float acc = 0.f;
    for (int i = lane * 8; i < n; i += 256) {
        const int4 xv = *reinterpret_cast<const int4*>(x + i);
        const uint32_t xw[4] = {(uint32_t)xv.x, (uint32_t)xv.y, (uint32_t)xv.z, (uint32_t)xv.w};
        float part = 0.f;
        if constexpr (kFp8) {
            const __nv_fp8_e4m3* p = reinterpret_cast<const __nv_fp8_e4m3*>(w) + row * n + i;
            for (int j = 0; j < 4; ++j) {
                const float2 f = bf16x2_to_f2(xw[j]);
                part = fmaf((float)p[2 * j], f.x, fmaf((float)p[2 * j + 1], f.y, part));
            }
            part *= scale[i >> 7];
        } else {
            const int4 wv = *reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(w) + row * n + i);
            const uint32_t ww[4] = {(uint32_t)wv.x, (uint32_t)wv.y, (uint32_t)wv.z, (uint32_t)wv.w};
            for (int j = 0; j < 4; ++j) {
                const float2 f = bf16x2_to_f2(xw[j]), g = bf16x2_to_f2(ww[j]);
                part = fmaf(g.x, f.x, fmaf(g.y, f.y, part));
            }
        }
        acc += part;
    }
    return warp_add(acc);
}

template <bool kFp8>
__global__ void __launch_bounds__(256) few_up_kernel(const FewTokensArgs a) {
    pdl_wait_predecessor();
    pdl_release_successor();
    const int lane = threadIdx.x & 31, p = blockIdx.y, i = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= a.inter) return;
    const long long e = a.idx[p] - a.first;
    if (a.idx[p] < 0 || e < 0 || e >= a.experts) return;
    const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x) + (p / a.topk) * a.x_stride;
    const long long row = e * 2 * a.inter + i;
    const int kb = a.hidden / 128;
    const float g = row_dot<kFp8>(a.w13, row, a.s13 + row / 128 * kb, x, a.hidden, lane);
    const float u = row_dot<kFp8>(a.w13, row + a.inter, a.s13 + (row + a.inter) / 128 * kb, x, a.hidden, lane);
    if (lane == 0) reinterpret_cast<__nv_bfloat16*>(a.h)[(long long)p * a.inter + i] = __float2bfloat16(silu(g) * u * a.weights[p]);
}

template <bool kFp8>
__global__ void __launch_bounds__(256) few_down_kernel(const FewTokensArgs a) {
    pdl_wait_predecessor();
    pdl_release_successor();
    const int lane = threadIdx.x & 31, t = blockIdx.y, i = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= a.hidden) return;
    float acc = 0.f;
    for (int k = 0; k < a.topk; ++k) {
        const int p = t * a.topk + k;
        const long long e = a.idx[p] - a.first;
        if (a.idx[p] < 0 || e < 0 || e >= a.experts) continue;
        const long long row = e * a.hidden + i;
        acc += row_dot<kFp8>(a.w2, row, a.s2 + row / 128 * (a.inter / 128), reinterpret_cast<const __nv_bfloat16*>(a.h) + (long long)p * a.inter, a.inter, lane);
    }
    if (lane == 0) reinterpret_cast<__nv_bfloat16*>(a.out)[(long long)t * a.hidden + i] = __float2bfloat16(acc);
}

}  // namespace

cudaError_t launch_few_tokens(const FewTokensArgs& a, cudaStream_t stream) {
    if (a.tokens <= 0) return cudaSuccess;
    const int unit = a.fp8 ? 128 : 8;
    if (a.tokens > kFewMaxTokens || a.topk < 1 || a.topk > kFewMaxTopk || a.experts < 1 || a.experts > kFewMaxExperts || a.hidden <= 0 || a.hidden % unit != 0 ||
        a.inter <= 0 || a.inter % unit != 0)
        return cudaErrorInvalidValue;
    const dim3 up((a.inter + 7) / 8, a.tokens * a.topk), down((a.hidden + 7) / 8, a.tokens);
    const cudaError_t e = a.fp8 ? launch_dependent(few_up_kernel<true>, up, 256, 0, stream, a) : launch_dependent(few_up_kernel<false>, up, 256, 0, stream, a);
    if (e != cudaSuccess) return e;
    return a.fp8 ? launch_dependent(few_down_kernel<true>, down, 256, 0, stream, a) : launch_dependent(few_down_kernel<false>, down, 256, 0, stream, a);
}

}  // namespace dx

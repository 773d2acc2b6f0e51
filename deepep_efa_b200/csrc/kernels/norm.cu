// Root-mean-square norm of the residual stream, forward and backward.
//
//   total = x + residual            (rounded to bf16: it is the stream that the next layer adds to, and what the backward pass reads)
//   y     = total * r * weight      with r = 1 / sqrt(mean(total^2) + eps)
//   q, scales                       y in e4m3 with one scale per 128 channels, the rows of an FP8 dispatch. They are made from y in fp32: rounding to
//                                   bf16 first would round twice.
//   dtotal = r (weight dy - total r^2 mean(weight dy total)) + (what reaches the sum past the norm);   dweight = sum over rows of dy total r
//
// Sums are in fp32. Memory bound: a row is read once and stays in registers between its sum and its output. The gradient of the weight goes through one
// partial sum per CTA and is added up in a fixed order, so results do not change from run to run.
#include "block_api.h"
#include "launch.cuh"

namespace dx {

namespace {

__device__ __forceinline__ void unpack8(const int4& v, float (&f)[8]) {
    const uint32_t w[4] = {(uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 p = bf16x2_to_f2(w[j]);
        f[2 * j] = p.x;
        f[2 * j + 1] = p.y;
    }
}
__device__ __forceinline__ int4 pack8(const float (&f)[8]) {
    return make_int4((int)f2_to_bf16x2(f[0], f[1]), (int)f2_to_bf16x2(f[2], f[3]), (int)f2_to_bf16x2(f[4], f[5]), (int)f2_to_bf16x2(f[6], f[7]));
}
template <bool kWide>
__device__ __forceinline__ void load_weight8(const void* w, int chunk, float (&f)[8]) {
    if constexpr (kWide) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(w) + 2 * chunk), b = __ldg(reinterpret_cast<const float4*>(w) + 2 * chunk + 1);
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
        unpack8(ld_cached(reinterpret_cast<const int4*>(w) + chunk), f);
    }
}
__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One row per CTA, C chunks of eight channels per thread.
template <int C, bool kWide>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormArgs a) {
    __shared__ float s_sum[32];
    pdl_wait_predecessor();
    pdl_release_successor();
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, n16 = a.hidden / 8;
    const long long row = blockIdx.x;
    const int4* x = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.x) + row * a.x_stride);
    int4 v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = c * threads + tid;
        v[c] = i < n16 ? ld_once(x + i) : make_int4(0, 0, 0, 0);
    }
    if (a.residual != nullptr) {
        const int4* r = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.residual) + row * a.residual_stride);
        int4* t = reinterpret_cast<int4*>(a.total) + row * n16;
        int4 u[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = c * threads + tid;
            u[c] = i < n16 ? ld_once(r + i) : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = c * threads + tid;
            float f[8], g[8];
            unpack8(v[c], f);
            unpack8(u[c], g);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] += g[j];
            v[c] = pack8(f);
            if (i < n16) t[i] = v[c];
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float f[8];
        unpack8(v[c], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(f[j], f[j], sum);
    }
    sum = warp_add(sum);
    if (lane == 0) s_sum[tid >> 5] = sum;
    __syncthreads();
    sum = warp_add(lane < threads / 32 ? s_sum[lane] : 0.f);
    const float r = rsqrtf(sum / (float)a.hidden + a.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = c * threads + tid;
        const bool in = i < n16;
        float f[8], w[8];
        unpack8(v[c], f);
        load_weight8<kWide>(a.weight, in ? i : 0, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = f[j] * r * w[j];
        if (a.y != nullptr && in) reinterpret_cast<int4*>(a.y)[row * n16 + i] = pack8(f);
        if (a.q != nullptr) {
            // 16 lanes hold the 128 channels of a scale (hidden is a multiple of 128 here, so they are all inside or all outside)
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(f[j]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            float scale, inv;
            fp8_scale_from_amax(amax, a.round_scale != 0, scale, inv);
            if (in) {
                const uint2 p = make_uint2(pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
                reinterpret_cast<uint2*>(a.q)[row * n16 + i] = p;
                if ((lane & 15) == 0) a.scales[row * (n16 / 16) + i / 16] = scale;
            }
        }
    }
}

// A CTA takes every gridDim.x-th row and keeps its share of the weight's gradient in registers.
template <int C, bool kWide>
__global__ void __launch_bounds__(1024) rms_norm_bwd_kernel(const NormBwdArgs a) {
    __shared__ float2 s_sum[2][32];
    pdl_wait_predecessor();
    pdl_release_successor();
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, n16 = a.hidden / 8;
    float dw[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[c][j] = 0.f;
    int parity = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        const int4* t = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.total) + row * a.total_stride);
        const int4* d = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.dy) + row * a.dy_stride);
        int4 tv[C], dv[C], uv[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = c * threads + tid;
            tv[c] = i < n16 ? ld_once(t + i) : make_int4(0, 0, 0, 0);
            dv[c] = i < n16 ? ld_once(d + i) : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < C; ++c) uv[c] = make_int4(0, 0, 0, 0);
        if (a.dtotal != nullptr) {
            const int4* u = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.dtotal) + row * a.dtotal_stride);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int i = c * threads + tid;
                if (i < n16) uv[c] = ld_once(u + i);
            }
        }
        float squares = 0.f, inner = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = c * threads + tid;
            float f[8], g[8], w[8];
            unpack8(tv[c], f);
            unpack8(dv[c], g);
            load_weight8<kWide>(a.weight, i < n16 ? i : 0, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                squares = fmaf(f[j], f[j], squares);
                inner = fmaf(g[j] * w[j], f[j], inner);
            }
        }
        squares = warp_add(squares);
        inner = warp_add(inner);
        if (lane == 0) s_sum[parity][tid >> 5] = make_float2(squares, inner);
        __syncthreads();  // (two buffers: a warp that is a row ahead writes the other one)
        const float2 all = lane < threads / 32 ? s_sum[parity][lane] : make_float2(0.f, 0.f);
        squares = warp_add(all.x);
        inner = warp_add(all.y);
        const float r = rsqrtf(squares / (float)a.hidden + a.eps), back = r * r * (inner / (float)a.hidden);
        int4* o = reinterpret_cast<int4*>(a.dx) + row * n16;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = c * threads + tid;
            float f[8], g[8], w[8], u[8];
            unpack8(tv[c], f);
            unpack8(dv[c], g);
            unpack8(uv[c], u);
            load_weight8<kWide>(a.weight, i < n16 ? i : 0, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                dw[c][j] = fmaf(g[j], f[j] * r, dw[c][j]);
                u[j] = fmaf(r, fmaf(-back, f[j], g[j] * w[j]), u[j]);
            }
            if (i < n16) o[i] = pack8(u);
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = c * threads + tid;
        if (i >= n16) continue;
        float4* p = reinterpret_cast<float4*>(a.partial + (size_t)blockIdx.x * a.hidden) + 2 * i;
        p[0] = make_float4(dw[c][0], dw[c][1], dw[c][2], dw[c][3]);
        p[1] = make_float4(dw[c][4], dw[c][5], dw[c][6], dw[c][7]);
    }
}

// dweight[i] = sum of the CTAs' partial sums, 32 channels per CTA, in a fixed order
template <bool kWide>
__global__ void __launch_bounds__(512) norm_dweight_kernel(const float* __restrict__ partial, void* __restrict__ dweight, int ctas, int hidden) {
    __shared__ float s[16][33];
    pdl_wait_predecessor();
    pdl_release_successor();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (i < hidden)
        for (int c = w; c < ctas; c += 16) sum += partial[(size_t)c * hidden + i];
    s[w][lane] = sum;
    __syncthreads();
    if (w != 0 || i >= hidden) return;
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) sum += s[j][lane];
    if constexpr (kWide)
        reinterpret_cast<float*>(dweight)[i] = sum;
    else
        reinterpret_cast<__nv_bfloat16*>(dweight)[i] = __float2bfloat16(sum);
}

// Chunks of eight channels per thread (1, 2 or 4) and the threads of a row's CTA.
struct Shape {
    int chunks, threads;
};
Shape shape_of(long long rows, int hidden, int num_sms) {
    const int n16 = (hidden + 7) / 8;
    // few rows: as many threads as there are chunks, for the shortest way through a row; many: several rows per SM at a time
    const int most = rows <= num_sms ? 1024 : 256;
    const int chunks = n16 <= most ? 1 : n16 <= 2 * most ? 2 : 4;
    return {chunks, ((n16 + chunks - 1) / chunks + 31) / 32 * 32};
}

template <int C>
cudaError_t norm_forward(const NormArgs& a, int threads, cudaStream_t stream) {
    const dim3 grid((unsigned)a.rows);
    return a.weight_f32 ? launch_dependent(rms_norm_kernel<C, true>, grid, threads, 0, stream, a) : launch_dependent(rms_norm_kernel<C, false>, grid, threads, 0, stream, a);
}
template <int C>
cudaError_t norm_backward(const NormBwdArgs& a, int threads, int ctas, cudaStream_t stream) {
    const dim3 grid((unsigned)ctas);
    return a.weight_f32 ? launch_dependent(rms_norm_bwd_kernel<C, true>, grid, threads, 0, stream, a)
                        : launch_dependent(rms_norm_bwd_kernel<C, false>, grid, threads, 0, stream, a);
}

}  // namespace

cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t stream) {
    if (a.rows <= 0) return cudaSuccess;
    if (a.hidden <= 0 || (a.hidden & 7) != 0 || a.hidden > kNormMaxHidden || a.rows > 0x7fffffffll || (a.q != nullptr && (a.hidden & 127) != 0)) return cudaErrorInvalidValue;
    const Shape s = shape_of(a.rows, a.hidden, 148);
    return s.chunks == 1 ? norm_forward<1>(a, s.threads, stream) : s.chunks == 2 ? norm_forward<2>(a, s.threads, stream) : norm_forward<4>(a, s.threads, stream);
}

int norm_bwd_ctas(long long rows, int hidden, int num_sms) {
    const Shape s = shape_of(num_sms + 1ll, hidden, num_sms);
    const long long most = (long long)num_sms * (s.threads >= 1024 ? 1 : 1024 / s.threads);
    return (int)(rows < most ? rows : most);
}

cudaError_t launch_rms_norm_bwd(const NormBwdArgs& a, int num_sms, cudaStream_t stream) {
    if (a.hidden <= 0 || (a.hidden & 7) != 0 || a.hidden > kNormMaxHidden) return cudaErrorInvalidValue;
    const int ctas = norm_bwd_ctas(a.rows, a.hidden, num_sms);
    if (ctas > 0) {
        const Shape s = shape_of(num_sms + 1ll, a.hidden, num_sms);
        const cudaError_t e = s.chunks == 1   ? norm_backward<1>(a, s.threads, ctas, stream)
                              : s.chunks == 2 ? norm_backward<2>(a, s.threads, ctas, stream)
                                              : norm_backward<4>(a, s.threads, ctas, stream);
        if (e != cudaSuccess) return e;
    }
    const dim3 grid((unsigned)((a.hidden + 31) / 32));
    return a.weight_f32 ? launch_dependent(norm_dweight_kernel<true>, grid, 512, 0, stream, (const float*)a.partial, a.dweight, ctas, a.hidden)
                        : launch_dependent(norm_dweight_kernel<false>, grid, 512, 0, stream, (const float*)a.partial, a.dweight, ctas, a.hidden);
}

}  // namespace dx

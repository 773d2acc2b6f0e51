// Root-mean-square norm of the residual stream, forward and backward.
//
//   total = x + residual            (rounded to bf16: it is the stream that the next layer adds to, and what the backward pass reads)
//   y     = total * r * weight      with r = 1 / sqrt(mean(total^2) + eps)
//   q, scales                       y in e4m3 with one scale per 128 channels, the rows of an FP8 dispatch. They are made from y in fp32: rounding to
//                                   bf16 first would round twice.
//   dtotal = r (weight dy - total r^2 mean(weight dy total)) + (what reaches the sum past the norm);   dweight = sum over rows of dy total r
//
// Sums are in fp32. The squares of a row past some 2^59 are no floats, and its gradient's r^3 is none past 2^42: such rows are multiplied by 2^-80 (exact in bf16, but for what
// is too small to count) and summed again, so a row's size does not matter. Memory bound: a row is read once and stays in registers between its sum and its output. The
// gradient of the weight goes through one partial sum per CTA and is added up in a fixed order, so results do not change from run to run.
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

constexpr float kDown = 8.2718061255302767e-25f;       // 2^-80
constexpr float kLargeSum = 1.2676506002282294e30f;    // 2^100, of a thread's squares in the forward pass
constexpr float kLargeMean = 1.2089258196146292e24f;   // 2^80, of a row's squares in the gradient

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
    // A warp with large values sums their squares times 2^-160 and says so by the sign. (2^-160 itself is no float: factors of 2^-80 one after the other.)
    const bool large = __any_sync(0xffffffffu, sum > kLargeSum);
    if (large) {
        sum = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float f[8];
            unpack8(v[c], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(f[j] * kDown, f[j] * kDown, sum);
        }
    }
    sum = warp_add(sum);
    if (lane == 0) s_sum[tid >> 5] = large ? -sum : sum;
    __syncthreads();
    const float part = lane < threads / 32 ? s_sum[lane] : 0.f;
    sum = warp_add(part < 0.f ? 0.f : part);
    float r = rsqrtf(sum / (float)a.hidden + a.eps);
    if (__any_sync(0xffffffffu, part < 0.f)) r = kDown * rsqrtf((sum * kDown * kDown + warp_add(part < 0.f ? -part : 0.f)) / (float)a.hidden + a.eps * kDown * kDown);
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

// Pairs of fp32 numbers in one register pair: sm_100 adds and multiplies them in one instruction.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair_of(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 of_pair(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void unpack8(const int4& v, f32x2 (&f)[4]) {
    const uint32_t w[4] = {(uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = pair_of(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
}
template <bool kWide>
__device__ __forceinline__ void load_weight8(const void* w, int chunk, f32x2 (&f)[4]) {
    float g[8];
    load_weight8<kWide>(w, chunk, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = pair_of(g[2 * j], g[2 * j + 1]);
}
__device__ __forceinline__ void copy16(uint32_t to, const int4* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

__device__ __forceinline__ int4 scaled_down(const int4& v) {
    float f[8];
    unpack8(v, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= kDown;
    return pack8(f);
}

// A CTA takes every gridDim.x-th row and keeps its share of the weight's gradient in registers, and the weight, where rows are not too wide. A thread copies its own
// chunks of the rows ahead into shared memory and reads them back alone, so that loads stay in flight over a row's sums without a barrier. Chunks past the
// row's end, and a dtotal that is not there, are zeros in shared memory from the start. 8192 x 4096, us: row after row
// straight to registers 62; rows ahead, 16 channels per thread 64; 32 per thread 60; math in pairs, weight kept 43 (its 268 MB at the measured copy rate: 41). In a loop, with the weight's sum behind it, 45.
template <int C, int S, int kMostThreads, bool kWide>
__global__ void __launch_bounds__(kMostThreads) rms_norm_bwd_kernel(const NormBwdArgs a) {
    extern __shared__ __align__(16) uint8_t ahead[];  // [S][three arrays][C * threads chunks of 16 bytes]
    __shared__ float2 s_sum[2][32];
    constexpr bool kKeep = kMostThreads == 256;
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, n16 = a.hidden / 8, pitch = C * threads;
    int4* own = reinterpret_cast<int4*>(ahead) + tid;
    const uint32_t own_at = (uint32_t)__cvta_generic_to_shared(own);
    for (int i = 0; i < S * 3 * C; ++i) own[i * threads] = make_int4(0, 0, 0, 0);
    f32x2 dw[C][4], kept[kKeep ? C : 1][4];
    pdl_wait_predecessor();
    pdl_release_successor();
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) dw[c][j] = 0;
        if constexpr (kKeep) {
            const int i = c * threads + tid;
            load_weight8<kWide>(a.weight, i < n16 ? i : 0, kept[c]);
        }
    }
    auto weight_of = [&](int c, f32x2 (&w)[4]) {
        if constexpr (kKeep) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kept[c][j];
        } else {
            const int i = c * threads + tid;
            load_weight8<kWide>(a.weight, i < n16 ? i : 0, w);
        }
    };
    auto fetch = [&](long long row, int stage) {
        if (row < a.rows) {
            const int4* t = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.total) + row * a.total_stride) + tid;
            const int4* d = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.dy) + row * a.dy_stride) + tid;
            const int4* u = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.dtotal) + row * a.dtotal_stride) + tid;
            const uint32_t to = own_at + stage * 3 * pitch * 16;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (c * threads + tid >= n16) continue;
                copy16(to + c * threads * 16, t + c * threads);
                copy16(to + (pitch + c * threads) * 16, d + c * threads);
                if (a.dtotal != nullptr) copy16(to + (2 * pitch + c * threads) * 16, u + c * threads);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const float per_channel = 1.f / (float)a.hidden;
    int parity = 0, stage = 0;
#pragma unroll
    for (int i = 0; i < S; ++i) fetch(blockIdx.x + (long long)i * gridDim.x, i);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
        const int4* now = own + stage * 3 * pitch;
        f32x2 squares2 = 0, inner2 = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            f32x2 f[4], g[4], w[4];
            unpack8(now[c * threads], f);
            unpack8(now[pitch + c * threads], g);
            weight_of(c, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                squares2 = fma2(f[j], f[j], squares2);
                inner2 = fma2(mul2(g[j], w[j]), f[j], inner2);
            }
        }
        float squares = of_pair(squares2).x + of_pair(squares2).y, inner = of_pair(inner2).x + of_pair(inner2).y;
        auto sum_over_row = [&] {
            squares = warp_add(squares);
            inner = warp_add(inner);
            if (lane == 0) s_sum[parity][tid >> 5] = make_float2(squares, inner);
            __syncthreads();  // (two buffers: a warp that is a row ahead writes the other one)
            squares = inner = 0.f;
            for (int w = 0; w < threads / 32; ++w) {
                const float2 part = s_sum[parity][w];
                squares += part.x;
                inner += part.y;
            }
        };
        sum_over_row();
        int4* o = reinterpret_cast<int4*>(a.dx) + row * n16 + tid;
        if (squares * per_channel > kLargeMean) {  // (the same in all threads)
            squares = inner = 0.f;
#pragma unroll 1
            for (int c = 0; c < C; ++c) {
                float f[8], g[8], w[8];
                unpack8(scaled_down(now[c * threads]), f);
                unpack8(now[pitch + c * threads], g);
                load_weight8<kWide>(a.weight, c * threads + tid < n16 ? c * threads + tid : 0, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    squares = fmaf(f[j], f[j], squares);
                    inner = fmaf(g[j] * w[j], f[j], inner);
                }
            }
            __syncthreads();
            sum_over_row();
            const float r = rsqrtf(fmaf(squares, per_channel, a.eps * kDown * kDown)), back = -(r * r) * (r * (inner * per_channel));
            const f32x2 r2 = pair_of(r, r), back2 = pair_of(back, back), down2 = pair_of(kDown, kDown);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                f32x2 f[4], g[4], w[4], u[4];
                unpack8(scaled_down(now[c * threads]), f);
                unpack8(now[pitch + c * threads], g);
                unpack8(now[2 * pitch + c * threads], u);
                weight_of(c, w);
                uint32_t out[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x2 gr = mul2(g[j], r2);
                    dw[c][j] = fma2(gr, f[j], dw[c][j]);
                    const float2 v = of_pair(fma2(down2, fma2(gr, w[j], mul2(back2, f[j])), u[j]));
                    out[j] = f2_to_bf16x2(v.x, v.y);
                }
                if (c * threads + tid < n16) o[c * threads] = make_int4((int)out[0], (int)out[1], (int)out[2], (int)out[3]);
            }
        } else {
            const float r = rsqrtf(fmaf(squares, per_channel, a.eps)), back = -r * r * r * (inner * per_channel);
            const f32x2 r2 = pair_of(r, r), back2 = pair_of(back, back);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                f32x2 f[4], g[4], w[4], u[4];
                unpack8(now[c * threads], f);
                unpack8(now[pitch + c * threads], g);
                unpack8(now[2 * pitch + c * threads], u);
                weight_of(c, w);
                uint32_t out[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x2 gr = mul2(g[j], r2);
                    dw[c][j] = fma2(gr, f[j], dw[c][j]);
                    const float2 v = of_pair(fma2(gr, w[j], fma2(back2, f[j], u[j])));
                    out[j] = f2_to_bf16x2(v.x, v.y);
                }
                if (c * threads + tid < n16) st_once(o + c * threads, make_int4((int)out[0], (int)out[1], (int)out[2], (int)out[3]));
            }
        }
        fetch(row + (long long)S * gridDim.x, stage);
        stage = stage + 1 == S ? 0 : stage + 1;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = c * threads + tid;
        if (i >= n16) continue;
        float4* p = reinterpret_cast<float4*>(a.partial + (size_t)blockIdx.x * a.hidden) + 2 * i;
        p[0] = make_float4(of_pair(dw[c][0]).x, of_pair(dw[c][0]).y, of_pair(dw[c][1]).x, of_pair(dw[c][1]).y);
        p[1] = make_float4(of_pair(dw[c][2]).x, of_pair(dw[c][2]).y, of_pair(dw[c][3]).x, of_pair(dw[c][3]).y);
    }
}

// dweight[i] = sum of the CTAs' partial sums, 32 channels per CTA, in a fixed order
template <bool kWide>
__global__ void __launch_bounds__(1024) norm_dweight_kernel(const float* __restrict__ partial, void* __restrict__ dweight, int ctas, int hidden) {
    __shared__ float s[32][33];
    pdl_wait_predecessor();
    pdl_release_successor();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float sum = 0.f;
    if (i < hidden) {
#pragma unroll 8
        for (int c = w; c < ctas; c += 32) sum += partial[(size_t)c * hidden + i];
    }
    s[w][lane] = sum;
    __syncthreads();
    if (w != 0 || i >= hidden) return;
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) sum += s[j][lane];
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
    const int chunks = rows <= num_sms ? (n16 <= 1024 ? 1 : n16 <= 2048 ? 2 : 4) : (n16 >= 512 ? 4 : n16 >= 256 ? 2 : 1);
    return {chunks, ((n16 + chunks - 1) / chunks + 31) / 32 * 32};
}

template <int C>
cudaError_t norm_forward(const NormArgs& a, int threads, cudaStream_t stream) {
    const dim3 grid((unsigned)a.rows);
    return a.weight_f32 ? launch_dependent(rms_norm_kernel<C, true>, grid, threads, 0, stream, a) : launch_dependent(rms_norm_kernel<C, false>, grid, threads, 0, stream, a);
}

// The backward pass: rows that a CTA fetches ahead, and CTAs per SM.
struct BwdShape {
    Shape row;
    int stages, per_sm;
    size_t smem;
};
BwdShape bwd_shape_of(int hidden) {
    // Many channels per thread: what a row costs a warp beside its channels (two sums over the CTA, addresses) was two thirds of the instructions with 16 of them. Few of a
    // narrow row, whose CTAs are small enough anyway. us with 8 / 16 / 32 channels: 20000 x 1544 - / 58 / 55, 32768 x 1024 51 / 55 / 53, 70000 x 512 57 / 64 / -; 16384 x 2048 - / 53 / 50.
    // Three rows ahead where six fit an SM: 8192 x 4096 with 4 x 2 / 3 x 3 rows 49.4 / 45.4, 8192 x 5120 with 3 x 2 / 2 x 3 59.8 / 58.7.
    const int n16 = (hidden + 7) / 8, chunks = n16 >= 192 ? 4 : 1;
    BwdShape b;
    b.row = {chunks, ((n16 + chunks - 1) / chunks + 31) / 32 * 32};
    const size_t bytes = (size_t)3 * chunks * b.row.threads * 16, most = 220 * 1024;
    b.stages = 6 * bytes <= most ? 3 : 2 * bytes <= most ? 2 : 1;
    b.smem = b.stages * bytes;
    const int by_smem = (int)(most / (b.smem + 2048)), by_threads = (chunks == 4 ? 512 : 1024) / b.row.threads;
    b.per_sm = by_smem < by_threads ? by_smem : by_threads;
    if (b.per_sm < 1) b.per_sm = 1;
    return b;
}
template <int C, int S, int kMostThreads, bool kWide>
cudaError_t norm_backward_as(const NormBwdArgs& a, const BwdShape& b, int ctas, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(rms_norm_bwd_kernel<C, S, kMostThreads, kWide>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)b.smem);
    return e != cudaSuccess ? e : launch_dependent(rms_norm_bwd_kernel<C, S, kMostThreads, kWide>, dim3((unsigned)ctas), b.row.threads, b.smem, stream, a);
}
template <bool kWide>
cudaError_t norm_backward(const NormBwdArgs& a, const BwdShape& b, int ctas, cudaStream_t stream) {
    if (b.row.chunks == 1) return norm_backward_as<1, 3, 256, kWide>(a, b, ctas, stream);
    if (b.row.threads <= 256) return b.stages == 3 ? norm_backward_as<4, 3, 256, kWide>(a, b, ctas, stream) : norm_backward_as<4, 2, 256, kWide>(a, b, ctas, stream);
    // Two stages fit where a row has at most 576 threads, which leaves each 96 registers (us with 64: 3000 x 9000 111, so 97; 2000 x 16384 82, so 73).
    return b.stages == 2 ? norm_backward_as<4, 2, 576, kWide>(a, b, ctas, stream) : norm_backward_as<4, 1, 1024, kWide>(a, b, ctas, stream);
}

}  // namespace

cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t stream) {
    if (a.rows <= 0) return cudaSuccess;
    if (a.hidden <= 0 || (a.hidden & 7) != 0 || a.hidden > kNormMaxHidden || a.rows > 0x7fffffffll || (a.q != nullptr && (a.hidden & 127) != 0)) return cudaErrorInvalidValue;
    const Shape s = shape_of(a.rows, a.hidden, 148);
    return s.chunks == 1 ? norm_forward<1>(a, s.threads, stream) : s.chunks == 2 ? norm_forward<2>(a, s.threads, stream) : norm_forward<4>(a, s.threads, stream);
}

int norm_bwd_ctas(long long rows, int hidden, int num_sms) {
    const long long most = (long long)num_sms * bwd_shape_of(hidden).per_sm;
    return (int)(rows < most ? rows : most);
}

cudaError_t launch_rms_norm_bwd(const NormBwdArgs& a, int num_sms, cudaStream_t stream) {
    if (a.hidden <= 0 || (a.hidden & 7) != 0 || a.hidden > kNormMaxHidden) return cudaErrorInvalidValue;
    const int ctas = norm_bwd_ctas(a.rows, a.hidden, num_sms);
    if (ctas > 0) {
        const BwdShape b = bwd_shape_of(a.hidden);
        const cudaError_t e = a.weight_f32 ? norm_backward<true>(a, b, ctas, stream) : norm_backward<false>(a, b, ctas, stream);
        if (e != cudaSuccess) return e;
    }
    const dim3 grid((unsigned)((a.hidden + 31) / 32));
    return a.weight_f32 ? launch_dependent(norm_dweight_kernel<true>, grid, 1024, 0, stream, (const float*)a.partial, a.dweight, ctas, a.hidden)
                        : launch_dependent(norm_dweight_kernel<false>, grid, 1024, 0, stream, (const float*)a.partial, a.dweight, ctas, a.hidden);
}

}  // namespace dx

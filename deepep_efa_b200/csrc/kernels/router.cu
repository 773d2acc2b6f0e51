// The choice of a token's experts from its gate logits, and the gradient of the weights that come with it.
//
//   idx      the k largest logits, in falling order, the lowest index first among equals; NaN counts as the largest, as in a sort
//   weights  exp(l_idx - m) / Z, Z over the chosen ones (renormalize) or over all experts
//   dlogits  w_j (g_j - sum_i w_i g_i) at the chosen ones; elsewhere 0, or -p_j sum_i w_i g_i where Z goes over all
// An expert whose logit is -inf is never chosen: where fewer than k are left, the rest of the row is -1 with weight 0, which dispatch skips.
//
// A warp per token, its logits in registers as keys. A round takes the warp's largest key (one redux) and its lowest index (a second one); the lane that held it clears it
// and takes the maximum of the rest. The rounds bound it, not the logits' bytes: 32768 tokens, 8 of 256, 29 us (36.7 MB: 5.6 at the measured copy rate); candidates marked by bits and
// looked through with their places 33.
#include "block_api.h"
#include "launch.cuh"

namespace dx {

namespace {

constexpr int kSelectThreads = 128;
constexpr int kWarps = kSelectThreads / 32;

template <bool kBf16>
__device__ __forceinline__ float load_logit(const void* p, long long i) {
    if constexpr (kBf16)
        return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
    else
        return reinterpret_cast<const float*>(p)[i];
}
// A key whose unsigned order is the order of the values: -0 equals 0, every NaN is the largest.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    if (k == 0xffffffffu) return __uint_as_float(0x7fffffffu);
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kMinusInf = 0x007fffffu;  // order_key(-inf): the smallest of all

__device__ __forceinline__ float warp_add(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// V: logits per lane (experts <= 32 V); expert i is in lane i % 32.
template <int V, bool kBf16>
__global__ void __launch_bounds__(kSelectThreads) select_kernel(const SelectArgs a) {
    pdl_wait_predecessor();
    pdl_release_successor();
    const int lane = threadIdx.x & 31, token = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (token >= a.tokens) return;
    uint32_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int i = j * 32 + lane;
        key[j] = i < a.experts ? order_key(load_logit<kBf16>(a.logits, token * a.logits_stride + i)) : 0;
    }
    uint32_t best = 0;  // of this lane's
    auto look = [&] {
        best = key[0];
#pragma unroll
        for (int j = 1; j < V; ++j) best = max(best, key[j]);
    };
    look();
    uint32_t most = __reduce_max_sync(0xffffffffu, best);
    const float top = key_value(most);
    float z = 0.f;
    if (!a.renormalize) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (key[j] > kMinusInf) z += expf(key_value(key[j]) - top);
    }
    float mine = 0.f;  // lane r: the logit of the r-th choice
    int mine_idx = -1;
    for (int r = 0; r < a.topk && most > kMinusInf; ++r) {  // (the same in all lanes)
        int slot = 0;
        if (best == most) {
#pragma unroll
            for (int j = V - 1; j >= 0; --j)
                if (key[j] == most) slot = j;  // the first of equals
        }
        const int i = (int)__reduce_min_sync(0xffffffffu, best == most ? (uint32_t)(slot * 32 + lane) : 0xffffffffu);
        if (lane == r) {
            mine = key_value(most);
            mine_idx = i;
        }
        if (lane == (i & 31)) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j == slot) key[j] = 0;
            look();
        }
        most = __reduce_max_sync(0xffffffffu, best);
    }
    const float e = mine_idx >= 0 ? expf(mine - top) : 0.f;
    if (a.renormalize) z = e;
    z = warp_add(z);
    if (lane < a.topk) {
        a.idx[(long long)token * a.topk + lane] = mine_idx;
        a.weights[(long long)token * a.topk + lane] = mine_idx >= 0 ? e / z : 0.f;
    }
}

template <int V, bool kBf16>
__global__ void __launch_bounds__(kSelectThreads) select_bwd_kernel(const SelectArgs a) {
    pdl_wait_predecessor();
    pdl_release_successor();
    const int lane = threadIdx.x & 31, token = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (token >= a.tokens) return;
    int idx = -1;
    float w = 0.f, g = 0.f;
    if (lane < a.topk) {
        idx = (int)a.idx[(long long)token * a.topk + lane];
        w = a.weights[(long long)token * a.topk + lane];
        g = a.dweights[(long long)token * a.topk + lane];
    }
    if (idx < 0) w = g = 0.f;
    const float inner = warp_add(w * g);
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = 0.f;
    if (!a.renormalize) {
        float top = -INFINITY, z = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = j * 32 + lane;
            d[j] = i < a.experts ? load_logit<kBf16>(a.logits, token * a.logits_stride + i) : -INFINITY;
            top = fmaxf(top, d[j]);
        }
        top = warp_max(top);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            d[j] = d[j] == -INFINITY ? 0.f : expf(d[j] - top);
            z += d[j];
        }
        z = warp_add(z);
        // (no experts at all: zeros; a NaN among the logits is in Z and so in all entries, those of experts with -inf too)
        const float f = z == 0.f ? 0.f : -inner / z;
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = d[j] == 0.f && z == z ? 0.f : d[j] * f;
    }
    const float at = w * (g - inner);
    for (int r = 0; r < a.topk; ++r) {
        const int i = __shfl_sync(0xffffffffu, idx, r);
        const float v = __shfl_sync(0xffffffffu, at, r);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (i == j * 32 + lane) d[j] = v;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int i = j * 32 + lane;
        if (i >= a.experts) continue;
        if constexpr (kBf16)
            reinterpret_cast<__nv_bfloat16*>(a.dlogits)[(long long)token * a.experts + i] = __float2bfloat16(d[j]);
        else
            reinterpret_cast<float*>(a.dlogits)[(long long)token * a.experts + i] = d[j];
    }
}

template <int V>
cudaError_t select_launch(const SelectArgs& a, bool backward, cudaStream_t stream) {
    const dim3 grid((unsigned)((a.tokens + kWarps - 1) / kWarps));
    if (backward)
        return a.bf16 ? launch_dependent(select_bwd_kernel<V, true>, grid, kSelectThreads, 0, stream, a)
                      : launch_dependent(select_bwd_kernel<V, false>, grid, kSelectThreads, 0, stream, a);
    return a.bf16 ? launch_dependent(select_kernel<V, true>, grid, kSelectThreads, 0, stream, a) : launch_dependent(select_kernel<V, false>, grid, kSelectThreads, 0, stream, a);
}

cudaError_t by_experts(const SelectArgs& a, bool backward, cudaStream_t stream) {
    if (a.tokens <= 0) return cudaSuccess;
    if (a.experts < 1 || a.experts > kRouterMaxExperts || a.topk < 1 || a.topk > kRouterMaxTopk || a.topk > a.experts) return cudaErrorInvalidValue;
    return a.experts <= 64    ? select_launch<2>(a, backward, stream)
           : a.experts <= 256 ? select_launch<8>(a, backward, stream)
                              : select_launch<32>(a, backward, stream);
}

}  // namespace

cudaError_t launch_select_experts(const SelectArgs& a, cudaStream_t stream) { return by_experts(a, false, stream); }
cudaError_t launch_select_experts_bwd(const SelectArgs& a, cudaStream_t stream) { return by_experts(a, true, stream); }

}  // namespace dx

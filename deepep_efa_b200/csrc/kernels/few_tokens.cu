// A layer of routed SwiGLU experts for a few tokens, in two launches:
//
//   h[p]   = weights[p] silu(G[e] x[t]) * (U[e] x[t])      p = (t, k), e = idx[t, k]: rows of G and U against the tokens of their expert
//   out[t] = sum_k W2[e] h[t, k]
//
// Bound by reading the chosen experts' weights once. A work unit is 32 rows of weights (16 of gate and the 16 of up that go with them, or 32 of W2) against the
// selections of one expert, up to eight: the rows are the M operand of mma.sync m16n8k16, the selections its eight columns. (tcgen05 multiplies 128 rows at the
// least and takes both operands in one type: here weights in e4m3 meet activations in bf16, and units of 128 rows leave most SMs without work where a token
// meets eight experts. The tensor cores are idle most of the time either way.)
//
// A warp is a pipeline of its own: it takes every eighth box (128 bytes of each of the unit's rows, 4 KB, one TMA copy with 128-byte swizzle) through a ring
// that only it fills and empties, over the borders of units. So no thread waits for a loader, and the eight partial sums of a unit meet in shared memory. The
// activations' fragments come straight from L2 (a few rows, used by every unit). Since both operands may take the reduction's index in any order as long as they agree, lane t of a
// row's four reads 16 bytes at a time (eight weights in bf16, sixteen in e4m3) and treats them as the fragments of two or four steps; rows are dealt to lanes so
// that a quarter warp reads all 32 banks.
//
// e4m3 becomes bf16 in registers (exactly), and each 128 x 128 block's sum is scaled in fp32. The hidden values are kept as two bf16 numbers, a rounding and
// its remainder, whose products go to the same accumulators: 16 bits of significand for one more mma per step.
//
// The second launch begins while the first one ends (programmatic dependent launch): it plans, fills its rings with weights, and only then waits for h. Its sums per selection
// go to a scratch matrix; the CTA that finishes the last unit of 32 result rows adds them up over the selections of each token, in rising k: no result depends on
// the order of arrival.
#include <cuda.h>

#include "block_api.h"
#include "launch.cuh"
#include "tc_prims.cuh"

namespace dx {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kUnitRows = 32;
constexpr int kBoxBytes = kUnitRows * 128;
constexpr int kStages = 3;
constexpr int kCols = 8;  // selections of a unit
constexpr int kMaxPairs = kFewMaxTokens * kFewMaxTopk;
constexpr int kRedBytes = kWarps * 2 * 32 * 16;

struct Smem {
    uint8_t ring[kWarps][kStages][kBoxBytes];  // 1024-byte aligned: the swizzle goes by address
    union {
        float4 red[kWarps][2][32];  // a unit's partial sums
        int start[kFewMaxExperts];  // while planning: selections per expert, then where they start
    };
    uint16_t pair[kMaxPairs];       // selections t * topk + k in the order of their experts
    uint16_t group_expert[kMaxPairs], group_start[kMaxPairs];  // a unit's columns: up to eight selections of one expert
    uint64_t full[kWarps][kStages];
    int warp_sum[kWarps];
    int num_groups, num_pairs, last, abort;
};
static_assert(sizeof(float4[kWarps][2][32]) == kRedBytes && kRedBytes >= kFewMaxExperts * 4, "");

struct FewParams {
    FewTokensArgs a;
    float* y;       // [tokens * topk, hidden]: W2[e] h[p]
    int* finished;  // [ceil(hidden / 32)]: units done of each 32 result rows
    int* error_flag;
    long long limit;
};

__device__ __forceinline__ void tma_load_box(const CUtensorMap* map, uint32_t bar, uint32_t dst, int c0, int c1, int c2, int c3, bool up) {
    if (up)
        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                     "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c3)
                     : "memory");
}
__device__ __forceinline__ int4 lds128(uint32_t at) {
    int4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four e4m3 numbers as two pairs in bf16, which holds each of them: bytes 0 and 1, bytes 2 and 3.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    uint32_t l, h;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(l), "=r"(h) : "r"(w));
    const float2 fl = __half22float2(*reinterpret_cast<__half2*>(&l)), fh = __half22float2(*reinterpret_cast<__half2*>(&h));
    lo = f2_to_bf16x2(fl.x, fl.y);
    hi = f2_to_bf16x2(fh.x, fh.y);
}
__device__ __forceinline__ int local_expert(const FewTokensArgs& a, int64_t id) {
    const int64_t e = id - a.first;
    return id >= 0 && e >= 0 && e < a.experts ? (int)e : -1;
}

// Lists the selections by expert and cuts each expert's into groups of up to eight. Every CTA does this for itself: at most 1024 ids. The selections of an
// expert that has one group come in any order (a column's result does not depend on its place); those of one that has more are sorted, since all CTAs have to
// cut them alike.
__device__ __forceinline__ void plan(const FewTokensArgs& a, Smem& s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pairs = a.tokens * a.topk;
    int e[kMaxPairs / kThreads];
#pragma unroll
    for (int j = 0; j < kMaxPairs / kThreads; ++j) {
        const int p = j * kThreads + tid;
        e[j] = p < pairs ? local_expert(a, a.idx[p]) : -1;
    }
    for (int i = tid; i < a.experts; i += kThreads) s.start[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMaxPairs / kThreads; ++j)
        if (e[j] >= 0) atomicAdd(&s.start[e[j]], 1);
    __syncthreads();
    // four experts per thread: exclusive sums of selections (low half) and groups (high half)
    constexpr int kEach = kFewMaxExperts / kThreads;
    int n[kEach], sum = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = tid * kEach + j;
        n[j] = i < a.experts ? s.start[i] : 0;
        sum += n[j] + ((n[j] + kCols - 1) / kCols << 16);
    }
    const int incl = warp_incl_scan(sum);
    if (lane == 31) s.warp_sum[warp] = incl;
    __syncthreads();
    int before = incl - sum, total = 0, cut = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.warp_sum[w];
        total += s.warp_sum[w];
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = tid * kEach + j;
        if (i < a.experts) s.start[i] = before & 0xffff;
        int g = before >> 16;
        for (int c = 0; c < n[j]; c += kCols, ++g) {
            s.group_expert[g] = (uint16_t)i;
            s.group_start[g] = (uint16_t)((before & 0xffff) + c);
        }
        before += n[j] + ((n[j] + kCols - 1) / kCols << 16);
        cut |= n[j] > kCols;
    }
    if (tid == 0) {
        s.num_pairs = total & 0xffff;
        s.num_groups = total >> 16;
    }
    cut = __syncthreads_or(cut);
#pragma unroll
    for (int j = 0; j < kMaxPairs / kThreads; ++j)
        if (e[j] >= 0) s.pair[atomicAdd(&s.start[e[j]], 1)] = (uint16_t)(j * kThreads + tid);
    __syncthreads();
    if (!cut) return;
    int to[kMaxPairs / kThreads];
#pragma unroll
    for (int j = 0; j < kMaxPairs / kThreads; ++j) {
        if (e[j] < 0) continue;
        const int begin = e[j] > 0 ? s.start[e[j] - 1] : 0, stop = s.start[e[j]];  // (each has moved on to the end of its own)
        to[j] = begin;
        for (int i = begin; i < stop; ++i) to[j] += s.pair[i] < j * kThreads + tid;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMaxPairs / kThreads; ++j)
        if (e[j] >= 0) s.pair[to[j]] = (uint16_t)(j * kThreads + tid);
    __syncthreads();
}

// kUp: gate and up rows against x; otherwise W2 rows against h.
template <bool kUp, bool kFp8>
__global__ void __launch_bounds__(kThreads, 2) few_kernel(const __grid_constant__ CUtensorMap map, const FewParams p) {
    extern __shared__ uint8_t raw[];
    Smem& s = *reinterpret_cast<Smem*>(raw + ((1024 - (smem_u32(raw) & 1023)) & 1023));
    const FewTokensArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    constexpr int kBoxK = kFp8 ? 128 : 64;
    const int depth = kUp ? a.hidden : a.inter;                           // the reduction
    const int blocks = kUp ? (a.inter + 15) / 16 : (a.hidden + 31) / 32;  // units of one group
    const int boxes = (depth + kBoxK - 1) / kBoxK;

    if (tid < kWarps * kStages) mbar_init(&s.full[0][0] + tid, 1);
    if (tid == 0) {
        s.abort = 0;
        tma_prefetch_desc(&map);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    // What the second launch plans from was there before the first one began (which has waited for it); only h has to be waited for.
    if constexpr (kUp) {
        pdl_wait_predecessor();
        pdl_release_successor();
    }
    plan(a, s);
    const int groups = s.num_groups, units = groups * blocks;
    // Units of this CTA. First launch: dealt out, group by group. Second: neighbours, result rows by result rows, so that a CTA has a part in few of them.
    const int first = kUp ? (int)blockIdx.x : (int)((long long)blockIdx.x * units / gridDim.x);
    const int end = kUp ? units : (int)((long long)(blockIdx.x + 1) * units / gridDim.x);
    const int step = kUp ? (int)gridDim.x : 1;
    auto group_of = [&](int u) { return kUp ? u / blocks : u % groups; };
    auto block_of = [&](int u) { return kUp ? u % blocks : u / groups; };

    // ---- this warp's boxes, in order: number `warp` of the CTA's first unit and every eighth from there
    int pu = first, pj = warp, issued = 0;
    auto issue = [&] {  // the warp's next box, if there is one
        while (pj >= boxes) {
            pj -= boxes;
            pu += step;
        }
        if (pu >= end) return;
        if (lane == 0) {
            const int slot = issued % kStages;
            const uint32_t bar = smem_u32(&s.full[warp][slot]);
            mbar_expect_tx_at(bar, kBoxBytes);
            const int e = s.group_expert[group_of(pu)];
            tma_load_box(&map, bar, smem_u32(s.ring[warp][slot]), pj * kBoxK, block_of(pu) * (kUp ? 16 : 32), 0, e, kUp);
        }
        ++issued;
        pj += kWarps;
    };
    for (int i = 0; i < kStages; ++i) issue();
    if constexpr (!kUp) {
        pdl_wait_predecessor();
        pdl_release_successor();
    } else if (blockIdx.x == 0) {
        for (int i = tid; i < (a.hidden + 31) / 32; i += kThreads) p.finished[i] = 0;
    }

    const int row = (g >> 1) | ((g & 1) << 2);  // of a fragment's eight rows: neighbours in g are four rows apart, on other banks
    const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(a.h);
    const long long plane = (long long)a.tokens * a.topk * a.inter;  // from a rounding to its remainder
    int used = 0, j = warp;
    for (int u = first; u < end; u += step) {
        const int group = group_of(u), block = block_of(u), e = s.group_expert[group], at = s.group_start[group];
        const int stop = group + 1 < groups ? s.group_start[group + 1] : s.num_pairs, n = stop - at;
        const int mine = g < n ? s.pair[at + g] : -1;  // this lane's column
        const __nv_bfloat16* b_row = mine < 0 ? nullptr
                                     : kUp    ? reinterpret_cast<const __nv_bfloat16*>(a.x) + (mine / a.topk) * a.x_stride
                                              : h + (long long)mine * a.inter;
        float acc[2][4] = {};
        for (; j < boxes; j += kWarps) {
            constexpr int kPieces = kFp8 ? 4 : 2;  // of 16 bytes of activations per lane
            int4 b[kPieces], b_lo[kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int k = j * kBoxK + (kFp8 ? (i >> 1) * 64 + t * 16 + (i & 1) * 8 : i * 32 + t * 8);
                const bool in = mine >= 0 && k < depth;
                b[i] = in ? *reinterpret_cast<const int4*>(b_row + k) : make_int4(0, 0, 0, 0);
                if constexpr (!kUp) b_lo[i] = in ? *reinterpret_cast<const int4*>(b_row + plane + k) : make_int4(0, 0, 0, 0);
            }
            float scale[2] = {1.f, 1.f};
            if constexpr (kFp8) {
                const int kb = depth / 128;
                if constexpr (kUp) {
                    const float* sc = a.s13 + ((long long)e * (2 * a.inter / 128) + block * 16 / 128) * kb + j;
                    scale[0] = __ldg(sc);
                    scale[1] = __ldg(sc + (long long)(a.inter / 128) * kb);
                } else {
                    scale[0] = scale[1] = __ldg(a.s2 + ((long long)e * (a.hidden / 128) + block * 32 / 128) * kb + j);
                }
            }
            const int slot = used % kStages;
            mbar_wait(&s.full[warp][slot], (used / kStages) & 1, &s.abort, p.limit);
            const uint32_t base = smem_u32(s.ring[warp][slot]);
            int4 w[2][2][2];  // [16 rows][upper or lower eight][half of the 128 bytes]
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) w[m][r][c] = lds128(base + (m * 16 + r * 8 + row) * 128 + (((c * 4 + t) ^ row) << 4));
            ++used;
            __syncwarp();
            if (!s.abort) issue();
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float part[4] = {};
                float(&d)[4] = kFp8 ? part : acc[m];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t w0[4] = {(uint32_t)w[m][0][c].x, (uint32_t)w[m][0][c].y, (uint32_t)w[m][0][c].z, (uint32_t)w[m][0][c].w};
                    const uint32_t w1[4] = {(uint32_t)w[m][1][c].x, (uint32_t)w[m][1][c].y, (uint32_t)w[m][1][c].z, (uint32_t)w[m][1][c].w};
                    if constexpr (kFp8) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint32_t a0, a1, a2, a3;
                            e4m3x4_to_bf16(w0[q], a0, a2);
                            e4m3x4_to_bf16(w1[q], a1, a3);
                            const int4 &v = b[c * 2 + q / 2], &lo = b_lo[c * 2 + q / 2];
                            mma_bf16(d, a0, a1, a2, a3, (q & 1) ? v.z : v.x, (q & 1) ? v.w : v.y);
                            if constexpr (!kUp) mma_bf16(d, a0, a1, a2, a3, (q & 1) ? lo.z : lo.x, (q & 1) ? lo.w : lo.y);
                        }
                    } else {
                        mma_bf16(d, w0[0], w1[0], w0[1], w1[1], b[c].x, b[c].y);
                        mma_bf16(d, w0[2], w1[2], w0[3], w1[3], b[c].z, b[c].w);
                        if constexpr (!kUp) {
                            mma_bf16(d, w0[0], w1[0], w0[1], w1[1], b_lo[c].x, b_lo[c].y);
                            mma_bf16(d, w0[2], w1[2], w0[3], w1[3], b_lo[c].z, b_lo[c].w);
                        }
                    }
                }
                if constexpr (kFp8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(scale[m], part[i], acc[m][i]);
                }
            }
        }
        j -= boxes;
        // ---- the warps' partial sums: fragment place (lane, i) = row (lane / 4 by `row`, + 8 for i >= 2), column 2 (lane % 4) + i % 2
#pragma unroll
        for (int m = 0; m < 2; ++m) s.red[warp][m][lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
        __syncthreads();
        auto sum = [&](int m, int r, int c) {
            const int from = ((((r & 3) << 1) | ((r >> 2) & 1)) * 4 + (c >> 1)) * 4 + ((r >> 3) << 1) + (c & 1);
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v += reinterpret_cast<const float*>(s.red[w][m])[from];
            return v;
        };
        if constexpr (kUp) {
            const int r = tid & 15, c = tid >> 4, i = block * 16 + r;
            if (c < n && i < a.inter) {
                const int q = s.pair[at + c];
                const float v = silu(sum(0, r, c)) * sum(1, r, c) * a.weights[q];
                const __nv_bfloat16 hi = __float2bfloat16(v);
                __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(a.h) + (long long)q * a.inter + i;
                to[0] = hi;
                to[plane] = __float2bfloat16(v - __bfloat162float(hi));
            }
            __syncthreads();
        } else {
            const int r = tid & 31, c = tid >> 5, i = block * 32 + r;
            if (c < n && i < a.hidden) p.y[(long long)s.pair[at + c] * a.hidden + i] = sum(r >> 4, r & 15, c);
            __syncthreads();
            // the end of this CTA's part in these result rows
            if (u + 1 >= end || block_of(u + 1) != block) {
                const int begun = max(first, block * groups);
                if (tid == 0) {
                    fence_acq_rel_gpu();
                    s.last = atomicAdd(p.finished + block, u + 1 - begun) + u + 1 - begun == groups;
                    fence_acq_rel_gpu();
                }
                __syncthreads();
                if (s.last) {
                    for (int o = tid; o < a.tokens * 32; o += kThreads) {
                        const int tok = o >> 5, col = block * 32 + (o & 31);
                        if (col >= a.hidden) continue;
                        float v = 0.f;
                        for (int k = 0; k < a.topk; ++k) {
                            const int q = tok * a.topk + k;
                            if (local_expert(a, a.idx[q]) >= 0) v += __ldcg(p.y + (long long)q * a.hidden + col);
                        }
                        reinterpret_cast<__nv_bfloat16*>(a.out)[(long long)tok * a.hidden + col] = __float2bfloat16(v);
                    }
                }
                __syncthreads();
            }
        }
    }
    if constexpr (!kUp) {
        if (groups == 0)  // nobody's expert is here
            for (long long i = (long long)blockIdx.x * kThreads + tid; i < (long long)a.tokens * a.hidden; i += (long long)gridDim.x * kThreads)
                reinterpret_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16(0.f);
    }
    if (s.abort) {  // a copy did not come: wait for those in flight, then say so
        for (; used < issued; ++used) {
            const long long t0 = clock64();
            while (!mbar_try_wait(&s.full[warp][used % kStages], (used / kStages) & 1) && clock64() - t0 < p.limit) {}
        }
        if (tid == 0 && p.error_flag != nullptr) atomicExch(p.error_flag, 1);
    }
}

// The weights as boxes of 128 bytes of neighbouring rows: [L, 2, I, H] in boxes of 16 gate and 16 up rows, [L, H, I] in boxes of 32 rows.
bool make_weight_map(CUtensorMap* map, const void* ptr, bool fp8, uint64_t experts, uint64_t halves, uint64_t rows, uint64_t depth) {
    EncodeFn fn = get_encode_fn();
    if (fn == nullptr) return false;
    const uint64_t esz = fp8 ? 1 : 2;
    const bool up = halves == 2;
    const cuuint64_t dims[4] = {depth, rows, up ? halves : experts, experts};
    const cuuint64_t strides[3] = {depth * esz, rows * depth * esz, halves * rows * depth * esz};
    const cuuint32_t box[4] = {(cuuint32_t)(128 / esz), up ? 16u : 32u, up ? 2u : 1u, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, up ? 4 : 3, const_cast<void*>(ptr), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs share an SM");

template <bool kUp, bool kFp8>
cudaError_t launch_half(const FewParams& p, int ctas, cudaStream_t stream) {
    const FewTokensArgs& a = p.a;
    CUtensorMap map;
    if (!make_weight_map(&map, kUp ? a.w13 : a.w2, kFp8, a.experts, kUp ? 2 : 1, kUp ? a.inter : a.hidden, kUp ? a.hidden : a.inter)) return cudaErrorInvalidValue;
    const cudaError_t e = cudaFuncSetAttribute(few_kernel<kUp, kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e != cudaSuccess) return e;
    return launch_dependent(few_kernel<kUp, kFp8>, dim3((unsigned)ctas), kThreads, kSmemBytes, stream, map, p);
}

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t h_bytes(const FewTokensArgs& a) { return aligned((size_t)2 * a.tokens * a.topk * a.inter * 2); }
size_t y_bytes(const FewTokensArgs& a) { return aligned((size_t)a.tokens * a.topk * a.hidden * 4); }

}  // namespace

size_t few_tokens_scratch(const FewTokensArgs& a) { return h_bytes(a) + y_bytes(a) + aligned((size_t)(a.hidden + 31) / 32 * 4); }

cudaError_t launch_few_tokens(const FewTokensArgs& args, int num_sms, cudaStream_t stream) {
    if (args.tokens <= 0) return cudaSuccess;
    const int unit = args.fp8 ? 128 : 8;
    if (args.tokens > kFewMaxTokens || args.topk < 1 || args.topk > kFewMaxTopk || args.experts < 1 || args.experts > kFewMaxExperts || args.hidden <= 0 ||
        args.hidden % unit != 0 || args.inter <= 0 || args.inter % unit != 0)
        return cudaErrorInvalidValue;
    FewParams p{};
    p.a = args;
    p.a.h = args.scratch;
    p.y = reinterpret_cast<float*>(static_cast<char*>(args.scratch) + h_bytes(args));
    p.finished = reinterpret_cast<int*>(static_cast<char*>(args.scratch) + h_bytes(args) + y_bytes(args));
    p.error_flag = args.error_flag;
    p.limit = args.wait_limit;
    const cudaError_t e = args.fp8 ? launch_half<true, true>(p, 2 * num_sms, stream) : launch_half<true, false>(p, 2 * num_sms, stream);
    if (e != cudaSuccess) return e;
    return args.fp8 ? launch_half<false, true>(p, 2 * num_sms, stream) : launch_half<false, false>(p, 2 * num_sms, stream);
}

}  // namespace dx

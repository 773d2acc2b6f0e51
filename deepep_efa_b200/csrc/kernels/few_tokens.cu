// A layer of routed SwiGLU experts for a few tokens, in two launches:
//
//   h[p]   = weights[p] silu(G[e] x[t]) * (U[e] x[t])      p = (t, k), e = idx[t, k]: rows of G and U against the tokens of their expert
//   out[t] = sum_k W2[e] h[t, k]
//
// Bound by reading the chosen experts' weights, as long as an expert has up to eight selections. 32 rows of weights (16 of gate and the 16 of up that go with them, or 32
// of W2) are multiplied with the selections of one expert, up to eight at a time: the rows are the M operand of mma.sync m16n8k16, the selections its eight columns. Past
// eight an expert's boxes are loaded and multiplied again for every eight (32 tokens on 8 experts of 4096 -> 1408, bf16, us: top-2 60, top-8 108, for 42 of reading them
// once; 7168 -> 2048, FP8: 89, 222, 54). (tcgen05 multiplies 128 rows at the least and takes both operands in one type: here weights in e4m3 meet activations of 16 bits, and tiles of 128 rows leave most SMs without work where a token
// meets eight experts. The tensor cores are idle most of the time either way.)
//
// A warp is a pipeline of its own: it takes its share of the boxes (128 bytes of each of 32 rows, 4 KB, one TMA copy with 128-byte swizzle) through a ring that only it
// fills and empties, over the borders of experts. So no thread waits for a loader. The activations' fragments come straight from L2 (a few rows, which every
// CTA reads). Since both operands may take the reduction's index in any order as long as they agree, lane t of a row's four reads 16 bytes at a time (eight
// weights in bf16, sixteen in e4m3) and treats them as the fragments of two or four steps; rows are dealt to lanes so that a quarter warp reads all 32 banks.
//
// First launch: 16 + 16 rows of one expert are a unit, which a team of warps shares; their partial sums meet in shared memory. Second launch: a CTA (or a cluster
// of up to eight, where there are few result rows) has 32 result rows and goes through the experts of all tokens; every warp adds up its own sums per token, which
// meet at the end, in a fixed order. So nothing is exchanged through memory but h, and no result depends on an order of arrival. The second launch begins
// while the first one ends (programmatic dependent launch): it plans, fills its rings with weights, and only then waits for h.
//
// Types: e4m3 becomes fp16 in registers, exactly and with one instruction per pair (bf16 takes four: 8 tokens, FP8, us 447 / 440), and each 128 x 128 block's sum is scaled in
// fp32. Next to it x is fp16 times a power of two per token. h has more bits than bf16, so that its rounding is small beside that of the result: next
// to bf16 weights two bf16 numbers, a rounding and its remainder, whose products go to the same accumulators; next to e4m3 weights fp16 with a power of two per 16 values.
#include <cuda.h>

#include <cuda_fp16.h>

#include <algorithm>

#include "block_api.h"
#include "few_ring.h"
#include "launch.cuh"
#include "tc_prims.cuh"

namespace dx {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kBoxRows = 32;
constexpr int kBoxBytes = kBoxRows * 128;
constexpr int kMostStages = 3;
constexpr int kCols = 8;  // selections that are multiplied at a time
constexpr int kMaxPairs = kFewMaxTokens * kFewMaxTopk;
constexpr int kTeamWarps = 4;  // warps that share a unit of the first launch: its 16 x 8 hidden values are one for each of their threads
static_assert(kTeamWarps * 32 == 16 * kCols, "");

// What a CTA plans by: the selections in the order of their experts, and groups of up to eight of one expert.
struct Plan {
    uint16_t pair[kMaxPairs];  // selection k of token t: t << 5 | k
    uint16_t group_expert[kMaxPairs], group_start[kMaxPairs];
    uint64_t full[kWarps][kMostStages];
    int warp_sum[kWarps];
    uint32_t largest[kFewMaxTokens];  // first launch, e4m3 weights: the largest magnitude of each token, as the bits of a float
    int num_groups, num_pairs, repeated, abort;
};
// In front of it the rings (1024-byte aligned: the swizzle goes by address) and fp32 sums, which while planning hold where experts start: the first launch's partial
// sums of a unit, or the second's per warp, token and row.
__host__ __device__ constexpr size_t ring_bytes(int stages) { return (size_t)kWarps * stages * kBoxBytes; }
__host__ __device__ constexpr size_t sum_bytes(bool up, int tokens) {
    const size_t n = up ? (size_t)kWarps * 2 * 32 * 16 : (size_t)kWarps * tokens * kBoxRows * 4;
    return n < kFewMaxExperts * 4 ? kFewMaxExperts * 4 : n;
}
// Two CTAs fit an SM: 3 x 32 KB of weights on their way in each, or 2 x 32 KB where the sums of more than eight tokens need the room.
__host__ __device__ constexpr int stages_for(bool up, int tokens) { return up || tokens <= 8 ? 3 : 2; }
__host__ __device__ constexpr size_t smem_bytes(bool up, int tokens) {
    return ring_bytes(stages_for(up, tokens)) + sum_bytes(up, tokens) + sizeof(Plan);
}
static_assert(2 * (smem_bytes(true, 1) + 1024) <= 228 * 1024 && 2 * (smem_bytes(false, 8) + 1024) <= 228 * 1024 && 2 * (smem_bytes(false, kFewMaxTokens) + 1024) <= 228 * 1024,
              "two CTAs share an SM");

struct FewParams {
    FewTokensArgs a;
    void* h;         // bf16 weights: [2][tokens * topk, inter] bf16, roundings and remainders; e4m3: [tokens * topk, inter] fp16
    float* h_scale;  // e4m3: [tokens * topk, inter / 16], powers of two
    long long limit;
    int cluster;     // second launch: CTAs that share 32 result rows
};

__device__ __forceinline__ void tma_load_box(const CUtensorMap* map, uint32_t bar, uint32_t dst, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}
__device__ __forceinline__ void tma_load_box(const CUtensorMap* map, uint32_t bar, uint32_t dst, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
                 : "memory");
}
__device__ __forceinline__ int4 lds128(uint32_t at) {
    int4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ float ld_cluster_f32(const float* own, int rank) {
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(own)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
template <bool kHalf>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (kHalf)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four e4m3 numbers as two pairs (bytes 0 and 1, bytes 2 and 3) in fp16, which holds each of them, NaN included.
__device__ __forceinline__ void e4m3x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// A token's activations go from bf16 to fp16 over the power of two at or below the token's largest magnitude: exactly down to 2^-17 of that; what is smaller keeps an
// absolute error of 2^-25 of it.
__device__ __forceinline__ uint32_t exponent_field(uint32_t largest) { return min(max(largest >> 23, 1u), 253u); }
__device__ __forceinline__ uint32_t to_half(uint32_t v, uint32_t under) {
    const __nv_bfloat162 u = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&under));
    const float2 f = __bfloat1622float2(u);
    const __half2 r = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&r);
}
// By all threads, four tokens and four pieces of each at a time, while the first boxes are on their way. (A power of two per box and column instead took no such pass but 38
// of a box's 320 instructions: 1, 8 and 32 tokens, FP8, us 67.4 / 426 / 299, so 64.9 / 415 / 297.)
__device__ __forceinline__ void find_largest(const FewTokensArgs& a, uint32_t* largest) {
    constexpr int V = 4, U = 4;
    const int chunks = a.hidden / 8;
#pragma unroll 1
    for (int t0 = 0; t0 < a.tokens; t0 += V) {
        __nv_bfloat162 most[V];
#pragma unroll
        for (int v = 0; v < V; ++v) most[v] = __float2bfloat162_rn(0.f);
#pragma unroll 1
        for (int i0 = threadIdx.x; i0 < chunks; i0 += kThreads * U) {
            int4 x[V][U];
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const int i = i0 + k * kThreads;
                    x[v][k] = t0 + v < a.tokens && i < chunks ? *(reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(a.x) + (t0 + v) * a.x_stride) + i)
                                                              : make_int4(0, 0, 0, 0);
                }
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const uint32_t w[4] = {(uint32_t)x[v][k].x, (uint32_t)x[v][k].y, (uint32_t)x[v][k].z, (uint32_t)x[v][k].w};
#pragma unroll
                    for (int q = 0; q < 4; ++q) most[v] = __hmax2(most[v], __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[q])));
                }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(__low2float(most[v]), __high2float(most[v]))));
            if (lane_id() == 0 && t0 + v < a.tokens) atomicMax(largest + t0 + v, m);
        }
    }
    __syncthreads();
}
__device__ __forceinline__ uint32_t scale_half2(uint32_t v, __half2 by) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&v), by);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Lists the selections by expert and cuts each expert's into groups of up to eight. Every CTA does this for itself: at most 1024 ids. Where a token names an
// expert twice, the first of the selections stands for both (the first launch adds up their weights). The selections of an expert that has one group come in any order
// (a column's result does not depend on its place); those of one that has more are sorted, since all CTAs have to cut them alike.
__device__ __forceinline__ void make_short_plan(const FewTokensArgs& a, Plan& s) {  // up to 32 selections: one warp, without shared memory in between
    const int lane = lane_id(), pairs = a.tokens * a.topk;
    const int64_t id = lane < pairs ? a.idx[lane] : -1, local = id - a.first;
    const bool here = id >= 0 && local >= 0 && local < a.experts;
    const int token = lane / a.topk;
    const uint32_t before = (1u << lane) - 1, of_token = before & ~((1u << (token * a.topk & 31)) - 1);
    uint32_t same = __match_any_sync(0xffffffffu, here ? (int)local : -1 - lane);
    const bool again = here && (same & of_token) != 0;
    same &= __ballot_sync(0xffffffffu, here && !again);
    const int rank = __popc(same & before), n = __popc(same);
    const bool first = here && !again && rank == 0;
    const int mine = first ? n + (((n + kCols - 1) / kCols) << 16) : 0, incl = warp_incl_scan(mine), total = __shfl_sync(0xffffffffu, incl, 31);
    const int start = __shfl_sync(0xffffffffu, (incl - mine) & 0xffff, same != 0 ? __ffs(same) - 1 : 0);
    if (here && !again) s.pair[start + rank] = (uint16_t)(token << 5 | (lane - token * a.topk));
    if (first) {
        int g = (incl - mine) >> 16;
        for (int c = 0; c < n; c += kCols, ++g) {
            s.group_expert[g] = (uint16_t)local;
            s.group_start[g] = (uint16_t)(start + c);
        }
    }
    const uint32_t repeated = __ballot_sync(0xffffffffu, again);
    if (lane == 0) {
        s.num_pairs = total & 0xffff;
        s.num_groups = total >> 16;
        s.repeated = repeated != 0;
    }
}
__device__ __forceinline__ void make_plan(const FewTokensArgs& a, Plan& s, int* start) {
    if (a.tokens * a.topk <= 32) {
        if (threadIdx.x < 32) make_short_plan(a, s);
        __syncthreads();
        return;
    }
    constexpr int kOwn = kMaxPairs / kThreads, kEach = kFewMaxExperts / kThreads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pairs = a.tokens * a.topk;
    int e[kOwn], repeated = 0;
    auto code = [&](int j) { return (uint16_t)((j * kThreads + tid) / a.topk << 5 | (j * kThreads + tid) % a.topk); };
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int p = j * kThreads + tid;
        e[j] = -1;
        if (p >= pairs) continue;
        const int64_t id = a.idx[p], local = id - a.first;
        if (id < 0 || local < 0 || local >= a.experts) continue;
        e[j] = (int)local;
        int before = 0;
        for (int k = p % a.topk; k > 0; --k) before |= a.idx[p - k] == id;
        if (before) {
            e[j] = -1;
            repeated = 1;
        }
    }
    for (int i = tid; i < a.experts; i += kThreads) start[i] = 0;
    repeated = __syncthreads_or(repeated);
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
        if (e[j] >= 0) atomicAdd(start + e[j], 1);
    __syncthreads();
    // four experts per thread: exclusive sums of selections (low half) and groups (high half)
    int n[kEach], sum = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = tid * kEach + j;
        n[j] = i < a.experts ? start[i] : 0;
        sum += n[j] + (((n[j] + kCols - 1) / kCols) << 16);
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
        if (i < a.experts) start[i] = before & 0xffff;
        int g = before >> 16;
        for (int c = 0; c < n[j]; c += kCols, ++g) {
            s.group_expert[g] = (uint16_t)i;
            s.group_start[g] = (uint16_t)((before & 0xffff) + c);
        }
        before += n[j] + (((n[j] + kCols - 1) / kCols) << 16);
        cut |= n[j] > kCols;
    }
    if (tid == 0) {
        s.num_pairs = total & 0xffff;
        s.num_groups = total >> 16;
        s.repeated = repeated;
    }
    cut = __syncthreads_or(cut);
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
        if (e[j] >= 0) s.pair[atomicAdd(start + e[j], 1)] = code(j);
    __syncthreads();
    if (!cut) return;
    int to[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        if (e[j] < 0) continue;
        const int begin = e[j] > 0 ? start[e[j] - 1] : 0, stop = start[e[j]];  // (each has moved on to the end of its own)
        to[j] = begin;
        for (int i = begin; i < stop; ++i) to[j] += s.pair[i] < code(j);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
        if (e[j] >= 0) s.pair[to[j]] = code(j);
    __syncthreads();
}

__device__ __forceinline__ void start_barriers(const CUtensorMap* map, Plan& s) {
    if (threadIdx.x < kWarps * kMostStages) mbar_init(&s.full[0][0] + threadIdx.x, 1);
    if (threadIdx.x < kFewMaxTokens) s.largest[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        s.abort = 0;
        tma_prefetch_desc(map);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// A warp's ring of boxes.
struct Ring : RingState {
    uint32_t at, bars;
    __device__ __forceinline__ Ring(uint8_t* smem, Plan& s, int warp, int stages_) : RingState(stages_) {
        at = smem_u32(smem) + warp * stages_ * kBoxBytes;
        bars = smem_u32(s.full[warp]);
    }
    __device__ __forceinline__ uint32_t fill_at() const { return at + fill * kBoxBytes; }
    __device__ __forceinline__ uint32_t fill_bar() const { return bars + fill * 8; }
    // Waits for the next box; its place. Where a copy did not come, here or in another warp, it waits (again with a limit) for all that are in flight, and from then
    // on returns at once with a place that holds nothing.
    __device__ __forceinline__ uint32_t next(uint64_t* full, int* abort, long long limit) {
        if (!__all_sync(0xffffffffu, mbar_wait(full + slot, parity, abort, limit)))
            give_up([&](int i, int phase) {
                const long long t0 = clock64();
                while (!mbar_try_wait(full + i, phase) && clock64() - t0 < limit) {}
            });
        const uint32_t box = at + slot * kBoxBytes;
        taken();
        return box;
    }
    __device__ __forceinline__ void report(int* error_flag) const {
        if (!alive && lane_id() == 0 && error_flag != nullptr) atomicExch(error_flag, 1);
    }
};

// A box in registers: [16 rows][upper or lower eight][half of the 128 bytes]
__device__ __forceinline__ void read_box(uint32_t box, int row, int t, int4 (&w)[2][2][2]) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c) w[m][r][c] = lds128(box + (m * 16 + r * 8 + row) * 128 + (((c * 4 + t) ^ row) << 4));
}
// Sixteen rows' products with pieces of eight activations per lane: bf16 weights, e4m3 weights as fp16.
__device__ __forceinline__ void multiply(float (&d)[4], const int4& upper, const int4& lower, const int4& b) {
    mma16<false>(d, upper.x, lower.x, upper.y, lower.y, b.x, b.y);
    mma16<false>(d, upper.z, lower.z, upper.w, lower.w, b.z, b.w);
}
__device__ __forceinline__ void multiply_fp8(float (&d)[4], const int4& upper, const int4& lower, const int4& b0, const int4& b1) {
    const uint32_t u[4] = {(uint32_t)upper.x, (uint32_t)upper.y, (uint32_t)upper.z, (uint32_t)upper.w};
    const uint32_t l[4] = {(uint32_t)lower.x, (uint32_t)lower.y, (uint32_t)lower.z, (uint32_t)lower.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t a0, a1, a2, a3;
        e4m3x4_to_half(u[q], a0, a2);
        e4m3x4_to_half(l[q], a1, a3);
        const int4& b = q < 2 ? b0 : b1;
        mma16<true>(d, a0, a1, a2, a3, (q & 1) ? b.z : b.x, (q & 1) ? b.w : b.y);
    }
}
// Fragment row g of eight is row_of(g): neighbours in g are four rows apart, on other banks.
__device__ __forceinline__ int row_of(int g) { return (g >> 1) | ((g & 1) << 2); }
__device__ __forceinline__ int lane_row_of(int r) { return ((r & 3) << 1) | (r >> 2); }  // its inverse

// ---- first launch: gate and up rows against x ---------------------------------------------------------------------------------------------
template <bool kFp8>
__global__ void __launch_bounds__(kThreads, 2) few_up_kernel(const __grid_constant__ CUtensorMap map, const FewParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const FewTokensArgs& a = p.a;
    constexpr int kStages = stages_for(true, 1), kBoxK = kFp8 ? 128 : 64;
    float4(*red)[2][32] = reinterpret_cast<float4(*)[2][32]>(smem + ring_bytes(kStages));
    Plan& s = *reinterpret_cast<Plan*>(smem + ring_bytes(kStages) + sum_bytes(true, 1));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, row = row_of(g);
    const int blocks = (a.inter + 15) / 16, boxes = (a.hidden + kBoxK - 1) / kBoxK;  // units of one group, boxes of a unit

    start_barriers(&map, s);
    pdl_wait_predecessor();
    pdl_release_successor();
    make_plan(a, s, reinterpret_cast<int*>(red));
    const int groups = s.num_groups, units = groups * blocks;
    // Units are dealt to the teams in turn, group by group, those of an SM last.
    const int team = warp / kTeamWarps, member = warp % kTeamWarps, step = kWarps / kTeamWarps * (int)gridDim.x;
    struct Place {
        int u, group, block;
    };
    const int step_group = step / blocks, step_block = step % blocks;
    auto advance = [&](Place& at) {
        at.u += step;
        at.group += step_group;
        at.block += step_block;
        if (at.block >= blocks) {
            at.block -= blocks;
            ++at.group;
        }
    };
    const int first = team * (int)gridDim.x + (int)blockIdx.x;
    Place now{first, first / blocks, first % blocks}, ahead = now;
    Ring ring(smem, s, warp, kStages);
    int ahead_j = member;  // the warp's boxes: from `member` of the team's first unit on in steps of the team's size
    auto issue = [&] {
        while (ahead_j >= boxes) {
            ahead_j -= boxes;
            advance(ahead);
        }
        if (ahead.u >= units) {
            ahead_j = 0;
            return;
        }
        const int e = s.group_expert[ahead.group];
        if (elect_one()) {
            mbar_expect_tx_at(ring.fill_bar(), kBoxBytes);
            tma_load_box(&map, ring.fill_bar(), ring.fill_at(), ahead_j * kBoxK, ahead.block * 16, 0, e);
        }
        ring.started();
        ahead_j += kTeamWarps;
    };
    for (int i = 0; i < kStages; ++i) issue();
    if constexpr (kFp8) find_largest(a, s.largest);
    auto meet = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kTeamWarps * 32) : "memory"); };

    int j = member;
    for (; now.u < units; advance(now)) {
        const int block = now.block, at = s.group_start[now.group], n = (now.group + 1 < groups ? s.group_start[now.group + 1] : s.num_pairs) - at;
        const int mine = g < n ? s.pair[at + g] : -1;  // this lane's column
        const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x) + (mine >> 5) * a.x_stride;
        const int blocks_k = a.hidden / 128;
        const float* scales = kFp8 ? a.s13 + ((long long)s.group_expert[now.group] * (2 * a.inter / 128) + block * 16 / 128) * blocks_k : nullptr;
        // this thread's hidden value: column `c`, row `r` of the unit
        const int o = member * 32 + lane, r = o & 15, c = o >> 4, code = c < n ? s.pair[at + c] : 0, q = (code >> 5) * a.topk + (code & 31);
        const float first_weight = c < n ? a.weights[q] : 0.f;
        const uint32_t under = (254u - exponent_field(mine >= 0 ? s.largest[mine >> 5] : 0)) << 7, both = under | (under << 16);
        float acc[2][4] = {};
        constexpr int kPieces = kFp8 ? 4 : 2;
        int4 b[kPieces];  // this lane's activations of a box; zeros all along where it has no column
#pragma unroll
        for (int i = 0; i < kPieces; ++i) b[i] = make_int4(0, 0, 0, 0);
        for (; j < boxes; j += kTeamWarps) {
            int4 w[2][2][2];
            if (mine >= 0) {
                const int4* from = reinterpret_cast<const int4*>(x + j * kBoxK + t * (kFp8 ? 16 : 8));
                if constexpr (kFp8) {
                    b[0] = from[0], b[1] = from[1], b[2 % kPieces] = from[8], b[3 % kPieces] = from[9];
                } else {
                    const int k = j * kBoxK + t * 8;
                    b[0] = k < a.hidden ? from[0] : make_int4(0, 0, 0, 0);
                    b[1] = k + 32 < a.hidden ? from[4] : make_int4(0, 0, 0, 0);
                }
            }
            if constexpr (kFp8) {
                const float gate = __ldg(scales + j), up = __ldg(scales + (long long)(a.inter / 128) * blocks_k + j);
                read_box(ring.next(s.full[warp], &s.abort, p.limit), row, t, w);
                __syncwarp();
                if (ring.alive) issue();
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
                    b[i] = make_int4((int)to_half(b[i].x, both), (int)to_half(b[i].y, both), (int)to_half(b[i].z, both), (int)to_half(b[i].w, both));
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    float part[4] = {};
#pragma unroll
                    for (int c = 0; c < 2; ++c) multiply_fp8(part, w[m][0][c], w[m][1][c], b[(2 * c) % kPieces], b[(2 * c + 1) % kPieces]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(m == 0 ? gate : up, part[i], acc[m][i]);
                }
            } else {
                read_box(ring.next(s.full[warp], &s.abort, p.limit), row, t, w);
                __syncwarp();
                if (ring.alive) issue();
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int c = 0; c < 2; ++c) multiply(acc[m], w[m][0][c], w[m][1][c], b[c]);
            }
        }
        j -= boxes;
        // the warps' partial sums: place (lane, i) of a fragment is row row_of(lane / 4), + 8 for i >= 2, column 2 (lane % 4) + i % 2
#pragma unroll
        for (int m = 0; m < 2; ++m) red[warp][m][lane] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
        meet();
        if (c < n) {
            const int i = block * 16 + r, from = (lane_row_of(r & 7) * 4 + (c >> 1)) * 4 + ((r >> 3) << 1) + (c & 1);
            float gate = 0.f, up = 0.f;
#pragma unroll
            for (int w = 0; w < kTeamWarps; ++w) {
                gate += reinterpret_cast<const float*>(red[team * kTeamWarps + w][0])[from];
                up += reinterpret_cast<const float*>(red[team * kTeamWarps + w][1])[from];
            }
            if constexpr (kFp8) {
                const float power = __uint_as_float(exponent_field(s.largest[code >> 5]) << 23);
                gate *= power;
                up *= power;
            }
            float weight = first_weight;
            if (s.repeated)
                for (int z = q + 1; z < ((code >> 5) + 1) * a.topk; ++z)
                    if (a.idx[z] == a.idx[q]) weight += a.weights[z];
            const float v = silu(gate) * up * weight;
            const long long to = (long long)q * a.inter + i;
            if constexpr (kFp8) {
                // sixteen lanes have the sixteen values of a scale: the power of two at or below the largest (of zeros the smallest there is, so that they do not count
                // in the box's, which is the largest of eight; of infinities the largest, next to which finite values stay finite)
                float most = fabsf(v);
#pragma unroll
                for (int x16 = 8; x16 > 0; x16 >>= 1) most = fmaxf(most, __shfl_xor_sync((lane & 16) ? 0xffff0000u : 0xffffu, most, x16));
                const uint32_t field = exponent_field(__float_as_uint(most));
                reinterpret_cast<__half*>(p.h)[to] = __float2half(v * __uint_as_float((254u - field) << 23));
                if (r == 0) p.h_scale[to / 16] = __uint_as_float(field << 23);
            } else if (i < a.inter) {
                // an infinity has no remainder (and infinity - infinity is NaN); a finite value that would round to one is cut off instead
                __nv_bfloat16 hi = __float2bfloat16(v);
                float rest = v - __bfloat162float(hi);
                if (fabsf(rest) == INFINITY) hi = __float2bfloat16_rz(v), rest = v - __bfloat162float(hi);
                if (fabsf(v) == INFINITY) rest = 0.f;
                reinterpret_cast<__nv_bfloat16*>(p.h)[to] = hi;
                reinterpret_cast<__nv_bfloat16*>(p.h)[to + (long long)a.tokens * a.topk * a.inter] = __float2bfloat16(rest);
            }
        }
        meet();
    }
    ring.report(a.error_flag);
}

// ---- second launch: W2 rows against h ---------------------------------------------------------------------------------------------------
template <bool kFp8>
__global__ void __launch_bounds__(kThreads, 2) few_down_kernel(const __grid_constant__ CUtensorMap map, const FewParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const FewTokensArgs& a = p.a;
    constexpr int kBoxK = kFp8 ? 128 : 64;
    const int stages = stages_for(false, a.tokens);
    float* sums = reinterpret_cast<float*>(smem + ring_bytes(stages));
    Plan& s = *reinterpret_cast<Plan*>(smem + ring_bytes(stages) + sum_bytes(false, a.tokens));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, row = row_of(g);
    const int tile = (int)blockIdx.x / p.cluster, rank = (int)blockIdx.x % p.cluster, boxes = (a.inter + kBoxK - 1) / kBoxK;

    start_barriers(&map, s);
    // What this launch plans from was there before the first one began (which has waited for it); only h has to be waited for.
    make_plan(a, s, reinterpret_cast<int*>(sums));
    const int groups = s.num_groups;
    const long long all = (long long)groups * boxes;
    // this warp's boxes: an equal share of the groups' boxes, laid out one after the other
    const int share = rank * kWarps + warp, shares = p.cluster * kWarps, first = (int)(all * share / shares), end = (int)(all * (share + 1) / shares);
    struct Place {
        int b, group, j;
    };
    auto advance = [&](Place& at) {
        ++at.b;
        if (++at.j == boxes) {
            at.j = 0;
            ++at.group;
        }
    };
    Place now{first, first / boxes, first % boxes}, ahead = now;
    Ring ring(smem, s, warp, stages);
    auto issue = [&] {
        if (ahead.b >= end) return;
        const int e = s.group_expert[ahead.group];
        if (elect_one()) {
            mbar_expect_tx_at(ring.fill_bar(), kBoxBytes);
            tma_load_box(&map, ring.fill_bar(), ring.fill_at(), ahead.j * kBoxK, tile * kBoxRows, e);
        }
        ring.started();
        advance(ahead);
    };
    for (int i = 0; i < stages; ++i) issue();
    // this warp's sums, [tokens][32 rows], the rows of a token turned by 8 per token so that four tokens' fragments are on different banks
    float* mine_sums = sums + warp * a.tokens * kBoxRows;
    for (int i = lane; i < a.tokens * kBoxRows; i += 32) mine_sums[i] = 0.f;
    pdl_wait_predecessor();
    pdl_release_successor();

    float acc[2][4] = {};
    int group = -1, at = 0, n = 0, mine = -1;
    auto flush = [&] {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (2 * t + i >= n) continue;
            const int token = s.pair[at + 2 * t + i] >> 5;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r) mine_sums[token * kBoxRows + ((m * 16 + r * 8 + row + 8 * token) & 31)] += acc[m][2 * r + i];
        }
        // Columns without a selection too: zeros times a weight (or a scale) that is no number are NaN, which the next group's selection in that column would get.
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
    };
    const float* scales = nullptr;
    int4 b[4];           // this lane's activations of a box, zeros all along where it has no column: four pieces of fp16, or [half of the box][rounding, remainder] in bf16
    float hs[2];         // the powers of two of the two halves
    for (; now.b < end; advance(now)) {
        if (now.group != group) {
            if (group >= 0) flush();
            group = now.group;
            at = s.group_start[group];
            n = (group + 1 < groups ? s.group_start[group + 1] : s.num_pairs) - at;
            mine = g < n ? (s.pair[at + g] >> 5) * a.topk + (s.pair[at + g] & 31) : -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = make_int4(0, 0, 0, 0);
            hs[0] = hs[1] = 1.f;
            if constexpr (kFp8) scales = a.s2 + ((long long)s.group_expert[group] * (a.hidden / 128) + tile * kBoxRows / 128) * (a.inter / 128);
        }
        int4 w[2][2][2];
        if constexpr (kFp8) {
            const float scale = __ldg(scales + now.j);
            if (mine >= 0) {
                const int4* h = reinterpret_cast<const int4*>(reinterpret_cast<const __half*>(p.h) + (long long)mine * a.inter + now.j * kBoxK + t * 16);
                b[0] = h[0], b[1] = h[1], b[2] = h[8], b[3] = h[9];
                const float* f = p.h_scale + (long long)mine * (a.inter / 16) + now.j * 8 + t;
                hs[0] = f[0], hs[1] = f[4];
            }
            read_box(ring.next(s.full[warp], &s.abort, p.limit), row, t, w);
            __syncwarp();
            if (ring.alive) issue();
            // one power of two for the box's 128 values of a column: the largest of its eight
            float top = fmaxf(hs[0], hs[1]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float under = __uint_as_float((254u << 23) - __float_as_uint(top));
            const __half2 by[2] = {__float2half2_rn(hs[0] * under), __float2half2_rn(hs[1] * under)};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                b[i] = make_int4((int)scale_half2(b[i].x, by[i / 2]), (int)scale_half2(b[i].y, by[i / 2]), (int)scale_half2(b[i].z, by[i / 2]), (int)scale_half2(b[i].w, by[i / 2]));
            const float col[2] = {scale * __shfl_sync(0xffffffffu, top, 8 * t), scale * __shfl_sync(0xffffffffu, top, 8 * t + 4)};  // columns 2 t and 2 t + 1
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float part[4] = {};
#pragma unroll
                for (int c = 0; c < 2; ++c) multiply_fp8(part, w[m][0][c], w[m][1][c], b[2 * c], b[2 * c + 1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(col[i & 1], part[i], acc[m][i]);
            }
        } else {
            if (mine >= 0) {
                const int k = now.j * kBoxK + t * 8;
                const int4* from = reinterpret_cast<const int4*>(reinterpret_cast<const __nv_bfloat16*>(p.h) + (long long)mine * a.inter + k);
                const long long plane = (long long)a.tokens * a.topk * a.inter / 8;
                const int4 none = make_int4(0, 0, 0, 0);
                b[0] = k < a.inter ? from[0] : none, b[1] = k < a.inter ? from[plane] : none;
                b[2] = k + 32 < a.inter ? from[4] : none, b[3] = k + 32 < a.inter ? from[4 + plane] : none;
            }
            read_box(ring.next(s.full[warp], &s.abort, p.limit), row, t, w);
            __syncwarp();
            if (ring.alive) issue();
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    multiply(acc[m], w[m][0][c], w[m][1][c], b[2 * c]);
                    multiply(acc[m], w[m][0][c], w[m][1][c], b[2 * c + 1]);
                }
        }
    }
    if (group >= 0) flush();
    ring.report(a.error_flag);
    __syncthreads();
    // the warps' sums, in order, and then the cluster's
    const int outputs = a.tokens * kBoxRows;
    auto store = [&](int o, float v) {
        const int token = o / kBoxRows, i = tile * kBoxRows + ((o - 8 * token) & 31);
        if (i < a.hidden) reinterpret_cast<__nv_bfloat16*>(a.out)[(long long)token * a.hidden + i] = __float2bfloat16(v);
    };
    for (int o = tid; o < outputs; o += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += sums[w * outputs + o];
        if (p.cluster == 1)
            store(o, v);
        else
            sums[o] = v;  // (this thread's alone until the cluster meets)
    }
    if (p.cluster == 1) return;
    cluster_sync();
    for (int o = rank * kThreads + tid; o < outputs; o += p.cluster * kThreads) {
        float v = 0.f;
        for (int c = 0; c < p.cluster; ++c) v += ld_cluster_f32(sums + o, c);
        store(o, v);
    }
    cluster_sync();  // (nobody leaves while its sums are read)
}

// The weights as boxes of 128 bytes of neighbouring rows: [L, 2, I, H] in boxes of 16 gate and 16 up rows, [L, H, I] in boxes of 32 rows.
bool make_weight_map(CUtensorMap* map, const void* ptr, bool fp8, bool up, uint64_t experts, uint64_t rows, uint64_t depth) {
    EncodeFn fn = get_encode_fn();
    if (fn == nullptr) return false;
    const uint64_t esz = fp8 ? 1 : 2;
    const cuuint64_t dims[4] = {depth, rows, up ? 2 : experts, experts};
    const cuuint64_t strides[3] = {depth * esz, rows * depth * esz, 2 * rows * depth * esz};
    const cuuint32_t box[4] = {(cuuint32_t)(128 / esz), up ? 16u : 32u, up ? 2u : 1u, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return fn(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, up ? 4 : 3, const_cast<void*>(ptr), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kFp8>
cudaError_t launch_both(FewParams& p, int num_sms, cudaStream_t stream) {
    const FewTokensArgs& a = p.a;
    CUtensorMap up, down;
    if (!make_weight_map(&up, a.w13, kFp8, true, a.experts, a.inter, a.hidden) || !make_weight_map(&down, a.w2, kFp8, false, a.experts, a.hidden, a.inter))
        return cudaErrorInvalidValue;
    const size_t up_smem = smem_bytes(true, 1), down_smem = smem_bytes(false, a.tokens);
    constexpr size_t most_down = std::max(smem_bytes(false, 8), smem_bytes(false, kFewMaxTokens));
    cudaError_t e = cudaFuncSetAttribute(few_up_kernel<kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)up_smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(few_down_kernel<kFp8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_down);
    // No more CTAs than there can be units for: beside fewer than two per SM the second launch finds room at once.
    const long long units = (long long)std::min(a.tokens * a.topk, a.experts + a.tokens * a.topk / kCols) * ((a.inter + 15) / 16), teams = kWarps / kTeamWarps;
    const int up_ctas = (int)std::min<long long>(2 * num_sms, (units + teams - 1) / teams);
    if (e == cudaSuccess) e = launch_dependent(few_up_kernel<kFp8>, dim3((unsigned)up_ctas), kThreads, up_smem, stream, up, p);
    if (e != cudaSuccess) return e;
    // As many CTAs as two per SM hold, but no more than leave a warp three boxes, which it has on their way before h is there: past that a larger cluster only has more to
    // wait for (3 tokens, 16 experts of 1032 -> 648, bf16, us: 8 CTAs per cluster 11.1, 4 9.8).
    const int tiles = (a.hidden + kBoxRows - 1) / kBoxRows;
    const long long boxes = (long long)std::min(a.tokens * a.topk, a.experts) * ((a.inter + (kFp8 ? 127 : 63)) / (kFp8 ? 128 : 64));
    p.cluster = 1;
    while (p.cluster < 8 && tiles * p.cluster * 2 <= 2 * num_sms && boxes > 3 * kWarps * p.cluster) p.cluster *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * p.cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = down_smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, few_down_kernel<kFp8>, down, p);
}

size_t h_bytes(const FewTokensArgs& a) { return ((size_t)a.tokens * a.topk * a.inter * (a.fp8 ? 2 : 4) + 255) / 256 * 256; }

}  // namespace

size_t few_tokens_scratch(const FewTokensArgs& a) { return h_bytes(a) + (a.fp8 ? (size_t)a.tokens * a.topk * (a.inter / 16) * 4 : 0); }

cudaError_t launch_few_tokens(const FewTokensArgs& a, int num_sms, cudaStream_t stream) {
    if (a.tokens <= 0) return cudaSuccess;
    const int unit = a.fp8 ? 128 : 8;
    if (a.tokens > kFewMaxTokens || a.topk < 1 || a.topk > kFewMaxTopk || a.experts < 1 || a.experts > kFewMaxExperts || a.hidden <= 0 || a.hidden % unit != 0 ||
        a.inter <= 0 || a.inter % unit != 0)
        return cudaErrorInvalidValue;
    FewParams p{};
    p.a = a;
    p.h = a.scratch;
    p.h_scale = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + h_bytes(a));
    p.limit = a.wait_limit;
    return a.fp8 ? launch_both<true>(p, num_sms, stream) : launch_both<false>(p, num_sms, stream);
}

}  // namespace dx

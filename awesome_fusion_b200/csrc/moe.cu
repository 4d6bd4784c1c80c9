// Router and weighted sum of a mixture-of-experts layer (afb_moe_route_launch, afb_moe_combine_launch).  The reference has no counterpart:
// its GEMM serves dense layers (bfAintBGemm.cc:36-217).
//
// Route.  A warp takes a token: every lane holds the logits of experts lane, lane + 32, ... as integers that order like the floats, the
// largest is found top_k times by two warp reductions (value, then lowest index).  exp and sums in fp32.
//   Few pairs: one CTA does it all; the rank of a pair among those of its expert is counted in shared memory.  What bounds it is latency.
//   Many: the tokens are cut into blocks; a first kernel picks and counts, per block and expert; in a second one every block adds up the
//   counts of the blocks before it and places its pairs, in order.  No atomic decides an order, so the plan is the same in every run.
// Combine.  A thread owns eight channels of a token and has the rows of eight picks on their way at once; HBM-bound for many tokens.
// Measured: route of 4099 tokens, 128 experts in fp32, top 8: 14.3 us (its 2.6 MB take 0.4 us): two launches' latency, the picks' chains of reductions, and every
// block of the second kernel adds up all 129 blocks' counts.
// Combine of those, 4096 channels: 54 us, 5.9 TB/s; of 5 tokens 4 us, the host's call.
#include <cuda_bf16.h>
#include "afb_internal.h"

namespace afb {
namespace {

constexpr int kRouteThreads = 1024, kRouteWarps = kRouteThreads / 32;
// Up to here one CTA: two tokens a warp, ranks counted pair against pair (221 tokens of 108 experts, one pick: 22.5 us in one CTA).
constexpr uint32_t kOneBlockTokens = 64, kOneBlockPairs = 512;
constexpr uint32_t kMaxBlocks = 256;       // of the two-kernel form: every block reads all blocks' counts
constexpr uint32_t kMinBlockTokens = 32;   // one per warp

struct RouteParams {
    const void* logits;
    int32_t *ids, *offsets, *row_pair, *pair_row;
    float* weights;
    int32_t* counts;          // [blocks][experts]
    uint32_t tokens, experts, ld, top_k, block_tokens, blocks;
    bool f32, renormalize;
};

// Integers that order like the floats; 0 for what is masked (-inf, NaN).  -0 and 0 are the same.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k); }
// exp(x - largest); both may be +inf
__device__ __forceinline__ float weight_of(float x, float largest) { return x == largest ? 1.f : expf(x - largest); }

// The picks of token t by one warp: lane j < top_k gets the j-th pick and its weight.
template <int NV>   // logits per lane
__device__ __forceinline__ void pick_token(const RouteParams& p, uint32_t t, uint32_t lane, int32_t& id, float& weight) {
    uint32_t key[NV];
    const size_t base = (size_t)t * p.ld;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t e = lane + 32u * i;
        key[i] = 0u;
        if (e < p.experts) {
            const float x = p.f32 ? reinterpret_cast<const float*>(p.logits)[base + e]
                                  : __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p.logits)[base + e] << 16);
            key[i] = order_key(x);
        }
    }
    uint32_t mine = 0u;
    float largest = 0.f, all = 0.f;
    id = -1;
    for (uint32_t j = 0; j < p.top_k; ++j) {
        uint32_t best = 0u, at = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (key[i] > best) { best = key[i]; at = lane + 32u * i; }
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0u) break;
        const uint32_t winner = __reduce_min_sync(0xffffffffu, best == most ? at : 0xffffffffu);
        if (j == 0) {
            largest = key_value(most);
            if (!p.renormalize) {
#pragma unroll
                for (int i = 0; i < NV; ++i) all += key[i] ? weight_of(key_value(key[i]), largest) : 0.f;
            }
        }
        if (lane == j) { id = (int32_t)winner; mine = most; }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (winner == lane + 32u * i) key[i] = 0u;
    }
    weight = id >= 0 ? weight_of(key_value(mine), largest) : 0.f;
    if (p.renormalize) all = weight;
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (id >= 0) weight /= all;
}

// offsets[e] = counts before e: an exclusive scan of `count[0 .. experts)` into `start`, by warp 0; start[experts] = their sum.
__device__ __forceinline__ void scan_experts(const int32_t* count, int32_t* start, uint32_t experts, uint32_t lane) {
    int32_t before = 0;
    for (uint32_t e0 = 0; e0 < experts; e0 += 32) {
        const uint32_t e = e0 + lane;
        const int32_t c = e < experts ? count[e] : 0;
        int32_t s = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= (uint32_t)o) s += y;
        }
        if (e < experts) start[e] = before + s - c;
        before += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) start[experts] = before;
}

template <int NV>
__global__ void __launch_bounds__(kRouteThreads) route_one_kernel(const RouteParams p) {
    __shared__ int32_t s_id[kOneBlockPairs];
    __shared__ int32_t s_count[AFB_MOE_MAX_EXPERTS], s_start[AFB_MOE_MAX_EXPERTS + 1];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, pairs = p.tokens * p.top_k;
    for (uint32_t e = tid; e < p.experts; e += kRouteThreads) s_count[e] = 0;
    __syncthreads();
    for (uint32_t t = warp; t < p.tokens; t += kRouteWarps) {
        int32_t id; float w;
        pick_token<NV>(p, t, lane, id, w);
        if (lane < p.top_k) {
            const uint32_t i = t * p.top_k + lane;
            s_id[i] = id;
            p.ids[i] = id;
            p.weights[i] = w;
            if (id >= 0) atomicAdd(&s_count[id], 1);   // a count: its order does not matter
        }
    }
    __syncthreads();
    if (warp == 0) scan_experts(s_count, s_start, p.experts, lane);
    __syncthreads();
    for (uint32_t e = tid; e <= p.experts; e += kRouteThreads) p.offsets[e] = s_start[e];
    const uint32_t rows = (uint32_t)s_start[p.experts];
    for (uint32_t i = tid; i < pairs; i += kRouteThreads) {
        const int32_t id = s_id[i];
        int32_t row = -1;
        if (id >= 0) {
            row = s_start[id];
            for (uint32_t j = 0; j < i; ++j) row += s_id[j] == id;
            p.row_pair[row] = (int32_t)i;
        }
        p.pair_row[i] = row;
        if (i >= rows) p.row_pair[i] = -1;
    }
}

// Picks and counts of one block of tokens.
template <int NV>
__global__ void __launch_bounds__(kRouteThreads) route_pick_kernel(const RouteParams p) {
    __shared__ int32_t s_count[AFB_MOE_MAX_EXPERTS];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the second kernel waits for this one's end before it reads
    for (uint32_t e = tid; e < p.experts; e += kRouteThreads) s_count[e] = 0;
    __syncthreads();
    const uint32_t t0 = blockIdx.x * p.block_tokens, t1 = min(p.tokens, t0 + p.block_tokens);
    for (uint32_t t = t0 + warp; t < t1; t += kRouteWarps) {
        int32_t id; float w;
        pick_token<NV>(p, t, lane, id, w);
        if (lane < p.top_k) {
            const size_t i = (size_t)t * p.top_k + lane;
            p.ids[i] = id;
            p.weights[i] = w;
            if (id >= 0) atomicAdd(&s_count[id], 1);
        }
    }
    __syncthreads();
    for (uint32_t e = tid; e < p.experts; e += kRouteThreads) p.counts[(size_t)blockIdx.x * p.experts + e] = s_count[e];
}

// Places of one block's pairs: shared memory holds, per expert, the rows of all blocks (then their scan), of the blocks before this one, and
// per warp the counts of its run of pairs (then the next free row of each).
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteParams p) {
    extern __shared__ int32_t smem[];
    int32_t *s_all = smem, *s_before = smem + p.experts, *s_start = s_before + p.experts, *s_next = s_start + p.experts + 1;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (uint32_t i = tid; i < 2 * p.experts; i += kRouteThreads) smem[i] = 0;
    for (uint32_t i = tid; i < kRouteWarps * p.experts; i += kRouteThreads) s_next[i] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // this block's pairs in runs, one per warp; the first 32 of a run are fetched once, ahead of the counts
    const size_t i0 = (size_t)blockIdx.x * p.block_tokens * p.top_k;
    const uint32_t mine = (uint32_t)(min(p.tokens, (blockIdx.x + 1) * p.block_tokens) - blockIdx.x * p.block_tokens) * p.top_k;
    const uint32_t run = (mine + kRouteWarps - 1) / kRouteWarps, r0 = min(mine, warp * run), r1 = min(mine, r0 + run);
    auto id_at = [&](uint32_t r) { return r < r1 ? __ldcg(p.ids + i0 + r) : -1; };
    const int32_t first_id = id_at(r0 + lane);
    // counts of all blocks: the threads of one expert (or of one of its stretches) take every `parts`-th block
    const uint32_t parts = p.experts >= kRouteThreads ? 1u : kRouteThreads / p.experts;
    for (uint32_t e = tid % min(p.experts, (uint32_t)kRouteThreads); e < p.experts; e += kRouteThreads) {
        const uint32_t part = p.experts >= kRouteThreads ? 0u : tid / p.experts;
        if (part >= parts) break;
        int32_t all = 0, before = 0;
#pragma unroll 16
        for (uint32_t b = part; b < p.blocks; b += parts) {
            const int32_t c = __ldcg(p.counts + (size_t)b * p.experts + e);
            all += c;
            before += b < blockIdx.x ? c : 0;
        }
        atomicAdd(&s_all[e], all);
        atomicAdd(&s_before[e], before);
    }
    int32_t* next = s_next + warp * p.experts;
    for (uint32_t r = r0 + lane; r < r1; r += 32) {
        const int32_t id = r < r0 + 32 ? first_id : id_at(r);
        if (id >= 0) atomicAdd(&next[id], 1);
    }
    __syncthreads();
    if (warp == 0) scan_experts(s_all, s_start, p.experts, lane);
    __syncthreads();
    for (uint32_t e = tid; e < p.experts; e += kRouteThreads) {
        int32_t row = s_start[e] + s_before[e], c[kRouteWarps];
#pragma unroll
        for (int w = 0; w < kRouteWarps; ++w) c[w] = s_next[w * p.experts + e];
#pragma unroll
        for (int w = 0; w < kRouteWarps; ++w) { s_next[w * p.experts + e] = row; row += c[w]; }
    }
    if (blockIdx.x == 0)
        for (uint32_t e = tid; e <= p.experts; e += kRouteThreads) p.offsets[e] = s_start[e];
    __syncthreads();
    const uint32_t rows = (uint32_t)s_start[p.experts];
    for (uint32_t r = r0; r < r1; r += 32) {
        const bool there = r + lane < r1;
        const int32_t id = r == r0 ? first_id : id_at(r + lane);
        const uint32_t same = __match_any_sync(0xffffffffu, id), below = same & ((1u << lane) - 1u);
        int32_t row = -1;
        if (id >= 0) row = next[id] + __popc(below);
        __syncwarp();
        if (id >= 0 && below == 0) next[id] += __popc(same);
        __syncwarp();
        if (there) {
            const size_t i = i0 + r + lane;
            p.pair_row[i] = row;
            if (row >= 0) p.row_pair[row] = (int32_t)i;
            if (i >= rows) p.row_pair[i] = -1;
        }
    }
}

__global__ void clear_offsets_kernel(int32_t* offsets, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) offsets[i] = 0;
}

bool one_block(uint32_t tokens, uint32_t top_k) { return tokens <= kOneBlockTokens && tokens * top_k <= kOneBlockPairs; }

// Blocks of the two-kernel form: at most kMaxBlocks, of a multiple of kMinBlockTokens tokens.
uint32_t route_block_tokens(uint32_t tokens) {
    const uint32_t least = (tokens + kMaxBlocks - 1) / kMaxBlocks;
    return (least + kMinBlockTokens - 1) / kMinBlockTokens * kMinBlockTokens;
}

template <int NV>
int launch_route(const RouteParams& p, DeviceCtx* ctx, cudaStream_t s) {
    if (one_block(p.tokens, p.top_k)) {
        route_one_kernel<NV><<<1, kRouteThreads, 0, s>>>(p);
        count_launch();
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? AFB_OK : cuda_fail(e);
    }
    const size_t smem = ((size_t)(3 + kRouteWarps) * p.experts + 1) * sizeof(int32_t);
    static DeviceOnce attr_set;
    if (!attr_set.done(ctx->device)) {
        const cudaError_t e = cudaFuncSetAttribute(route_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)(((3 + kRouteWarps) * AFB_MOE_MAX_EXPERTS + 1) * sizeof(int32_t)));
        if (e != cudaSuccess) return cuda_fail(e);
        attr_set.mark(ctx->device);
    }
    route_pick_kernel<NV><<<p.blocks, kRouteThreads, 0, s>>>(p);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.blocks); cfg.blockDim = dim3(kRouteThreads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, route_place_kernel, p);
    count_launch(2);
    return e == cudaSuccess ? AFB_OK : cuda_fail(e);
}

struct CombineParams {
    uint16_t* out;
    const uint16_t *y, *residual;
    const float* weights;
    const int32_t* pair_row;
    uint32_t tokens, top_k, rows, n, ld_out, ld_y, ld_residual;
};

__device__ __forceinline__ void add_pair(uint32_t v, float w, float& lo, float& hi) {
    lo = fmaf(w, __uint_as_float(v << 16), lo);
    hi = fmaf(w, __uint_as_float(v & 0xffff0000u), hi);
}

constexpr int kCombineThreads = 128;

// VEC = 8 channels per thread where everything is 16-byte aligned, else 1.
template <int VEC>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const CombineParams p) {
    constexpr uint32_t kPicks = 8;   // in flight at once
    const uint32_t c = (blockIdx.x * kCombineThreads + threadIdx.x) * VEC;
    if (c >= p.n) return;
    for (uint32_t t = blockIdx.y; t < p.tokens; t += gridDim.y) {
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
        const size_t pair0 = (size_t)t * p.top_k;
        for (uint32_t j0 = 0; j0 < p.top_k; j0 += kPicks) {
            uint4 v[kPicks];
            uint16_t h[kPicks];
            float w[kPicks];
            bool there[kPicks];
#pragma unroll
            for (uint32_t j = 0; j < kPicks; ++j) {
                const uint32_t row = j0 + j < p.top_k ? (uint32_t)__ldg(p.pair_row + pair0 + j0 + j) : 0xffffffffu;
                there[j] = row < p.rows;
                w[j] = there[j] ? __ldg(p.weights + pair0 + j0 + j) : 0.f;
                v[j] = make_uint4(0u, 0u, 0u, 0u);
                h[j] = 0;
                if (there[j]) {
                    const uint16_t* src = p.y + (size_t)row * p.ld_y + c;
                    if (VEC == 8) v[j] = __ldcs(reinterpret_cast<const uint4*>(src));
                    else h[j] = *src;
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < kPicks; ++j) {
                if (!there[j]) continue;
                if constexpr (VEC == 8) {
                    add_pair(v[j].x, w[j], sum[0], sum[1]); add_pair(v[j].y, w[j], sum[2], sum[3]);
                    add_pair(v[j].z, w[j], sum[4], sum[5]); add_pair(v[j].w, w[j], sum[6], sum[7]);
                } else {
                    sum[0] = fmaf(w[j], __uint_as_float((uint32_t)h[j] << 16), sum[0]);
                }
            }
        }
        uint16_t* dst = p.out + (size_t)t * p.ld_out + c;
        if constexpr (VEC == 8) {
            if (p.residual) {
                const uint4 r = *reinterpret_cast<const uint4*>(p.residual + (size_t)t * p.ld_residual + c);
                add_pair(r.x, 1.f, sum[0], sum[1]); add_pair(r.y, 1.f, sum[2], sum[3]);
                add_pair(r.z, 1.f, sum[4], sum[5]); add_pair(r.w, 1.f, sum[6], sum[7]);
            }
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(sum[2 * i], sum[2 * i + 1]);
                o[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
            if (p.residual) sum[0] += __uint_as_float((uint32_t)p.residual[(size_t)t * p.ld_residual + c] << 16);
            *dst = __bfloat16_as_ushort(__float2bfloat16_rn(sum[0]));
        }
    }
}

}  // namespace
}  // namespace afb

using namespace afb;

extern "C" int afb_moe_route_workspace(uint32_t tokens, uint32_t experts, uint64_t* bytes) {
    if (!bytes || experts == 0 || experts > AFB_MOE_MAX_EXPERTS) return AFB_ERR_BAD_ARG;
    if (tokens >> 31) return AFB_ERR_TOO_LARGE;   // no route has as many; the block sizes below would leave 32 bits
    // also for sizes that one CTA takes: top_k decides, and it is not asked for here
    const uint64_t blocks = tokens ? (tokens + route_block_tokens(tokens) - 1) / route_block_tokens(tokens) : 0;
    *bytes = one_block(tokens, experts < AFB_MOE_MAX_TOP_K ? experts : AFB_MOE_MAX_TOP_K) ? 0 : blocks * experts * sizeof(int32_t);
    return AFB_OK;
}

extern "C" int afb_moe_route_launch(const afb_moe_route_args* a, void* stream) {
    if (!a || a->reserved != 0 || !a->ptr_offsets || (uintptr_t)a->ptr_offsets % 4) return AFB_ERR_BAD_ARG;
    if (a->experts == 0 || a->experts > AFB_MOE_MAX_EXPERTS || a->top_k == 0 || a->top_k > a->experts || a->top_k > AFB_MOE_MAX_TOP_K) return AFB_ERR_BAD_ARG;
    if (a->logits_f32 > 1 || a->renormalize > 1 || a->ld_logits < a->experts) return AFB_ERR_BAD_ARG;
    if (((uint64_t)a->tokens * a->top_k) >> 31) return AFB_ERR_TOO_LARGE;
    uint64_t need = 0;
    if (a->tokens) {
        for (const void* ptr : {(const void*)a->ptr_ids, (const void*)a->ptr_weights, (const void*)a->ptr_row_pair, (const void*)a->ptr_pair_row})
            if (!ptr || (uintptr_t)ptr % 4) return AFB_ERR_BAD_ARG;
        if (!a->ptr_logits || (uintptr_t)a->ptr_logits % (a->logits_f32 ? 4 : 2)) return AFB_ERR_BAD_ARG;
        afb_moe_route_workspace(a->tokens, a->experts, &need);
        if (!one_block(a->tokens, a->top_k) && (!a->ptr_workspace || (uintptr_t)a->ptr_workspace % 4 || a->workspace_bytes < need)) return AFB_ERR_BAD_ARG;
    }
    DeviceCtx* ctx = current_ctx();
    if (!ctx) return AFB_ERR_NOT_INIT;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->tokens == 0) {
        clear_offsets_kernel<<<1, 256, 0, s>>>(a->ptr_offsets, a->experts + 1);
        count_launch();
        const cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? AFB_OK : cuda_fail(e);
    }
    RouteParams p{};
    p.logits = a->ptr_logits;
    p.ids = a->ptr_ids; p.offsets = a->ptr_offsets; p.row_pair = a->ptr_row_pair; p.pair_row = a->ptr_pair_row;
    p.weights = a->ptr_weights;
    p.counts = reinterpret_cast<int32_t*>(a->ptr_workspace);
    p.tokens = a->tokens; p.experts = a->experts; p.ld = a->ld_logits; p.top_k = a->top_k;
    p.block_tokens = route_block_tokens(a->tokens);
    p.blocks = (a->tokens + p.block_tokens - 1) / p.block_tokens;
    p.f32 = a->logits_f32 != 0; p.renormalize = a->renormalize != 0;
    if (p.experts <= 64) return launch_route<2>(p, ctx, s);
    if (p.experts <= 128) return launch_route<4>(p, ctx, s);
    if (p.experts <= 256) return launch_route<8>(p, ctx, s);
    return launch_route<32>(p, ctx, s);
}

extern "C" int afb_moe_combine_launch(const afb_moe_combine_args* a, void* stream) {
    if (!a || a->reserved != 0 || a->top_k == 0 || a->n == 0) return AFB_ERR_BAD_ARG;
    if (a->n >> 31 || a->tokens >> 31) return AFB_ERR_TOO_LARGE;   // the blocks' stride over the tokens stays in 32 bits
    if (a->tokens == 0) return AFB_OK;
    if (!a->ptr_out || !a->ptr_weights || !a->ptr_pair_row || (a->rows && !a->ptr_y)) return AFB_ERR_BAD_ARG;
    if ((uintptr_t)a->ptr_out % 2 || (uintptr_t)a->ptr_y % 2 || (uintptr_t)a->ptr_residual % 2 || (uintptr_t)a->ptr_weights % 4 || (uintptr_t)a->ptr_pair_row % 4) return AFB_ERR_BAD_ARG;
    if (a->ld_out < a->n || a->ld_y < a->n || (a->ptr_residual && a->ld_residual < a->n)) return AFB_ERR_BAD_ARG;
    if (a->ptr_out == a->ptr_y) return AFB_ERR_BAD_ARG;
    if (a->ptr_residual == a->ptr_out && a->ld_residual != a->ld_out) return AFB_ERR_BAD_ARG;   // in place means element by element
    if (!current_ctx()) return AFB_ERR_NOT_INIT;
    CombineParams p{};
    p.out = reinterpret_cast<uint16_t*>(a->ptr_out);
    p.y = reinterpret_cast<const uint16_t*>(a->ptr_y); p.residual = reinterpret_cast<const uint16_t*>(a->ptr_residual);
    p.weights = a->ptr_weights; p.pair_row = a->ptr_pair_row;
    p.tokens = a->tokens; p.top_k = a->top_k; p.rows = a->rows; p.n = a->n;
    p.ld_out = a->ld_out; p.ld_y = a->ld_y; p.ld_residual = a->ld_residual;
    const bool wide = a->n % 8 == 0 && a->ld_out % 8 == 0 && a->ld_y % 8 == 0 && (!a->ptr_residual || a->ld_residual % 8 == 0) &&
                      (((uintptr_t)a->ptr_out | (uintptr_t)a->ptr_y | (uintptr_t)a->ptr_residual) % 16) == 0;
    const uint32_t per_block = kCombineThreads * (wide ? 8 : 1);
    const dim3 grid((a->n + per_block - 1) / per_block, a->tokens < 65535u ? a->tokens : 65535u);
    if (wide) combine_kernel<8><<<grid, kCombineThreads, 0, (cudaStream_t)stream>>>(p);
    else combine_kernel<1><<<grid, kCombineThreads, 0, (cudaStream_t)stream>>>(p);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? AFB_OK : cuda_fail(e);
}

extern "C" int afb_moe_abi_sizes(uint32_t sizes[3]) {
    if (!sizes) return AFB_ERR_BAD_ARG;
    sizes[0] = sizeof(afb_moe_route_args); sizes[1] = sizeof(afb_expert_gemm_args); sizes[2] = sizeof(afb_moe_combine_args);
    return AFB_OK;
}

// Products grouped by expert, few rows per expert (afb_expert_gemm_launch): each expert's weights are read once and multiply the handful of
// rows that picked it.  Reference counterpart of the product itself: bf16gemm_kernel_gfx90a.s:410-489; it has no experts.
//
//   D[n, r] = sum_k W[e][n,k] * A[row(r),k],   16 channels x 8 rows per mma.sync.m16n8k16, the channels as the row operand
//
// A cluster of S CTAs (1 to 8) owns 128 channels of one expert and up to 8 * MT of its rows; each CTA has a stretch of K, each of its eight
// warps 16 channels.  A lane reads the 16 bytes of its two channels (16 or 32 consecutive k) straight into registers, four chunks ahead,
// and unpacks them there (dequant.cuh).  The rows of A are staged in shared memory once per pass, in the order of k that the
// unpack yields: a dot product does not care.  Group scales multiply the fp32 sum of a chunk, which lies in one group (HALF: in two, int4 in
// groups of 64; a lane's 16 bytes are then 8 of each).  The CTAs of a cluster add their fp32 sums through distributed shared memory in the
// order of k: no workspace, no counter, the same bits in every run.
#include <cooperative_groups.h>
#include "dequant.cuh"
#include "decode_common.cuh"
#include "expert_common.cuh"

namespace afb {
namespace {

constexpr int kAhead = 4;             // chunks of weights in registers
constexpr uint32_t kFewChannels = 128;
constexpr uint32_t kSumPitch = 132;   // floats per row of the CTA's sums: 16-byte rows, banks shifted by 4

template <bool HALF> struct Chunk {
    uint4 wa, wb;
    float sa[HALF ? 2 : 1], sb[HALF ? 2 : 1];
    uint32_t za[HALF ? 2 : 1], zb[HALF ? 2 : 1];   // the unpack's addends, where there are zero-points
};

__device__ __forceinline__ uint4 ldg_weights(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ldg_weights8(const uint8_t* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

template <int BITS, int MT, bool GROUPED, bool HALF>
__global__ void __launch_bounds__(kThreads, MT == 4 ? 1 : 2)
expert_few_kernel(const ExpertParams p, const uint32_t split, const uint32_t pass_chunks, const uint32_t row_bytes) {
    constexpr uint32_t CH = BITS == 8 ? 64 : 128, LK = CH / 4, AV = LK / 8;   // k per chunk; k per lane; 16-byte pieces of A per lane
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t s_act = (uint32_t)__cvta_generic_to_shared(smem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    const uint32_t rank = blockIdx.x % split, unit = blockIdx.x / split;   // the CTAs of a cluster are consecutive
    ExpertTile t;
    if (!find_tile(p, unit / p.n_blocks, 1, lane, t)) return;              // the whole cluster alike
    const uint32_t n0 = unit % p.n_blocks * kFewChannels;

    const uint32_t row_a = n0 + warp * 16 + g, row_b = row_a + 8;
    const bool ok_a = row_a < p.n, ok_b = row_b < p.n;
    const size_t chan_a = (size_t)t.expert * p.n + (ok_a ? row_a : 0), chan_b = (size_t)t.expert * p.n + (ok_b ? row_b : 0);
    const uint32_t chunks = p.k / CH, c0 = (uint32_t)((uint64_t)chunks * rank / split), nch = (uint32_t)((uint64_t)chunks * (rank + 1) / split) - c0;
    const uint8_t* pa = p.b + chan_a * p.ldb_bytes + (size_t)c0 * 64 + tig * (HALF ? 8 : 16);
    const uint8_t* pb = p.b + chan_b * p.ldb_bytes + (size_t)c0 * 64 + tig * (HALF ? 8 : 16);
    const uint32_t groups_per_row = GROUPED ? p.k >> p.group_shift : 0;
    const uint32_t flip = BITS == 8 ? flip8(p.enc) : flip4(p.enc);
    uint32_t add_a = unpack_add(BITS, 0), add_b = add_a;
    const bool has_zero = p.zero != nullptr;
    auto zero_add = [&](size_t i) { return unpack_add(BITS, BITS == 8 ? decode_zero8(p.zero[i], p.enc) : decode_zero4(p.zero[i], p.enc)); };
    if (!GROUPED && has_zero) { add_a = zero_add(chan_a); add_b = zero_add(chan_b); }

    auto load = [&](Chunk<HALF>& q, uint32_t c) {   // chunk c of this CTA's stretch
        if (HALF) {
            const uint2 a0 = ldg_weights8(pa + (size_t)c * 64), a1 = ldg_weights8(pa + (size_t)c * 64 + 32);
            const uint2 b0 = ldg_weights8(pb + (size_t)c * 64), b1 = ldg_weights8(pb + (size_t)c * 64 + 32);
            q.wa = make_uint4(a0.x, a0.y, a1.x, a1.y); q.wb = make_uint4(b0.x, b0.y, b1.x, b1.y);
        } else {
            q.wa = ldg_weights(pa + (size_t)c * 64); q.wb = ldg_weights(pb + (size_t)c * 64);
        }
        if (GROUPED) {
#pragma unroll
            for (int h = 0; h < (HALF ? 2 : 1); ++h) {
                const uint32_t grp = ((c0 + c) * CH + h * (CH / 2)) >> p.group_shift;
                const size_t ia = chan_a * groups_per_row + grp, ib = chan_b * groups_per_row + grp;
                q.sa[h] = load_scale(p.scale, ia, p.scale_dtype); q.sb[h] = load_scale(p.scale, ib, p.scale_dtype);
                if (has_zero) { q.za[h] = zero_add(ia); q.zb[h] = zero_add(ib); }
            }
        }
    };
    Chunk<HALF> q[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) if ((uint32_t)u < nch) load(q[u], u);

    // B operand: lane (g, tig) reads row g's k of lane tig.  Rows behind the last one read row 0; their columns of D are never stored.
    uint32_t act_base[MT], act_off[AV];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) act_base[mt] = s_act + (mt * 8 + g < t.rows ? mt * 8 + g : 0) * row_bytes;
    // 16-byte pieces of a chunk; int4 with whole groups: bit 3 of the piece flips bit 1, else lanes 0 and 2 of a quad share a bank
    constexpr bool kSwizzle = BITS == 4 && !HALF;
#pragma unroll
    for (uint32_t v = 0; v < AV; ++v) {
        const uint32_t piece = HALF ? (v / 2) * 8 + tig * 2 + (v & 1) : tig * AV + v;
        act_off[v] = (kSwizzle ? swz_piece(piece) : piece) * 16;
    }
    float acc[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[mt][e] = 0.f;

    auto consume = [&](const Chunk<HALF>& q, uint32_t coff) {   // coff: byte offset of the chunk in a staged row
        const uint32_t wa[4] = {q.wa.x, q.wa.y, q.wa.z, q.wa.w}, wb[4] = {q.wb.x, q.wb.y, q.wb.z, q.wb.w};
        float part[MT][4];
        if (GROUPED) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[mt][e] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int h = HALF ? j / 2 : 0;
            const uint32_t aa = GROUPED && has_zero ? q.za[h] : add_a, ab = GROUPED && has_zero ? q.zb[h] : add_b;
            uint32_t fa[4], fb[4];
            if (BITS == 8) {
                s8x4_to_bf16(wa[j], flip, kSel8Strided02, kSel8Strided13, kMulByte, aa, fa[0], fa[1]);
                s8x4_to_bf16(wb[j], flip, kSel8Strided02, kSel8Strided13, kMulByte, ab, fb[0], fb[1]);
            } else {
                s4x8_to_bf16_strided(wa[j], flip, aa, fa);
                s4x8_to_bf16_strided(wb[j], flip, ab, fb);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                if (mt * 8 >= (int)t.rows && mt > 0) break;
                float (&d)[4] = GROUPED ? part[mt] : acc[mt];
                if (BITS == 8) {
                    const uint4 x = lds128(act_base[mt] + coff + act_off[j / 2]);   // two words' worth: the compiler reads it once
                    if (j % 2 == 0) mma_bf16(d, fa[0], fb[0], fa[1], fb[1], x.x, x.y);
                    else            mma_bf16(d, fa[0], fb[0], fa[1], fb[1], x.z, x.w);
                } else {
                    const uint4 x = lds128(act_base[mt] + coff + act_off[j]);
                    mma_bf16(d, fa[0], fb[0], fa[1], fb[1], x.x, x.y);
                    mma_bf16(d, fa[2], fb[2], fa[3], fb[3], x.z, x.w);
                }
            }
            if (GROUPED && (j == 3 || (HALF && j == 1))) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    acc[mt][0] = fmaf(q.sa[h], part[mt][0], acc[mt][0]); acc[mt][1] = fmaf(q.sa[h], part[mt][1], acc[mt][1]);
                    acc[mt][2] = fmaf(q.sb[h], part[mt][2], acc[mt][2]); acc[mt][3] = fmaf(q.sb[h], part[mt][3], acc[mt][3]);
                    if (HALF) part[mt][0] = part[mt][1] = part[mt][2] = part[mt][3] = 0.f;
                }
            }
        }
    };

    // threads per row of A when staging: all 256 for one row, 32 for eight and more
    const uint32_t per_row = t.rows >= 5 ? 32u : t.rows >= 3 ? 64u : t.rows == 2 ? 128u : 256u;
    for (uint32_t p0 = 0; p0 < nch; p0 += pass_chunks) {
        const uint32_t in_pass = min(pass_chunks, nch - p0);
        if (p0) __syncthreads();   // the previous pass has been consumed by every warp
        const uint32_t pieces = in_pass * (CH / 8);
        for (uint32_t r = tid / per_row; r < t.rows; r += kThreads / per_row) {
            const uint32_t src_row = source_row(p, t.row0 + r);
            const uint16_t* src = p.a + (size_t)src_row * p.lda + (size_t)(c0 + p0) * CH;
            const bool there = src_row < p.a_rows;
#pragma unroll 4
            for (uint32_t pc = tid % per_row; pc < pieces; pc += per_row) {
                const uint4 v = there ? ldg_act(src + (size_t)pc * 8) : make_uint4(0u, 0u, 0u, 0u);
                uint4 o;
                if (p.packed) {           // pre-packed weights unpack to consecutive k
                    o = v;
                } else if (BITS == 8) {   // {k0,k2},{k1,k3},{k4,k6},{k5,k7}
                    o.x = prmt(v.x, v.y, 0x5410u); o.y = prmt(v.x, v.y, 0x7632u);
                    o.z = prmt(v.z, v.w, 0x5410u); o.w = prmt(v.z, v.w, 0x7632u);
                } else {                  // {k0,k4},{k1,k5},{k2,k6},{k3,k7}
                    o.x = prmt(v.x, v.z, 0x5410u); o.y = prmt(v.x, v.z, 0x7632u);
                    o.z = prmt(v.y, v.w, 0x5410u); o.w = prmt(v.y, v.w, 0x7632u);
                }
                *reinterpret_cast<uint4*>(smem + r * row_bytes + (kSwizzle ? swz_piece(pc) : pc) * 16) = o;
            }
        }
        __syncthreads();
        for (uint32_t i = 0; i < in_pass; i += kAhead) {   // pass_chunks is a multiple of kAhead: chunk p0 + i is in q[0]
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (i + u >= in_pass) break;
                consume(q[u], (i + u) * (CH * 2));
                if (p0 + i + u + kAhead < nch) load(q[u], p0 + i + u + kAhead);
            }
        }
    }

    // ---- the sums meet in shared memory: [row][channel] of every CTA, added up in the order of the ranks
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (mt * 8 + 2 * tig + (e & 1) < t.rows)
                sums[(mt * 8 + 2 * tig + (e & 1)) * kSumPitch + warp * 16 + g + (e >> 1) * 8] = acc[mt][e];
    namespace cg = cooperative_groups;
    if (split > 1) cg::this_cluster().sync(); else __syncthreads();
    const uint32_t vecs = t.rows * (kFewChannels / 4);
    for (uint32_t v = rank * kThreads + tid; v < vecs; v += split * kThreads) {
        const uint32_t r = v / (kFewChannels / 4), ch = v % (kFewChannels / 4) * 4, nn = n0 + ch;
        if (nn >= p.n) continue;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (split == 1) {
            x = *reinterpret_cast<const float4*>(sums + r * kSumPitch + ch);
        } else {
            for (uint32_t c = 0; c < split; ++c) {
                const float4 y = *reinterpret_cast<const float4*>(cg::this_cluster().map_shared_rank(sums, c) + r * kSumPitch + ch);
                x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
            }
        }
        float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (GROUPED) f[e] *= kUnpackInverse;
            else f[e] = nn + e < p.n ? unscaled(f[e], load_scale(p.scale, (size_t)t.expert * p.n + nn + e, p.scale_dtype)) : 0.f;
        }
        if (p.gated) {
            uint16_t* dst = p.c + (size_t)(t.row0 + r) * p.ldc + nn / 2;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (nn + 2 * e < p.n) dst[e] = __bfloat16_as_ushort(__float2bfloat16_rn((p.silu ? silu(f[2 * e]) : f[2 * e]) * f[2 * e + 1]));
        } else {
            uint16_t* dst = p.c + (size_t)(t.row0 + r) * p.ldc + nn;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (nn + e < p.n) dst[e] = __bfloat16_as_ushort(__float2bfloat16_rn(p.silu ? silu(f[e]) : f[e]));
        }
    }
    if (split > 1) cg::this_cluster().sync();   // no CTA leaves while another reads its sums
}

template <int BITS, int MT, bool GROUPED, bool HALF>
int launch_cfg(const ExpertParams& p, uint32_t split, DeviceCtx* ctx, cudaStream_t s) {
    auto kern = expert_few_kernel<BITS, MT, GROUPED, HALF>;
    constexpr uint32_t CH = BITS == 8 ? 64 : 128;
    // rows of A in shared memory: 32 KiB (48 from 16 rows on) for two CTAs per SM and more
    const uint32_t most = MT == 4 ? 96 * 1024 : MT == 2 ? 64 * 1024 : 32 * 1024;
    const uint32_t chunks = (p.k / CH + split - 1) / split;
    uint32_t pass = (most / p.tile_rows - 16) / (CH * 2) / kAhead * kAhead;
    const uint32_t whole = (chunks + kAhead - 1) / kAhead * kAhead;
    if (pass > whole) pass = whole;
    const uint32_t row_bytes = pass * CH * 2 + 16;   // + 16: consecutive rows lie in different banks
    uint32_t bytes = p.tile_rows * row_bytes;
    if (bytes < p.tile_rows * kSumPitch * 4) bytes = p.tile_rows * kSumPitch * 4;
    static DeviceOnce attr_set;
    if (!attr_set.done(ctx->device)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024 + 1024);
        if (e != cudaSuccess) return cuda_fail(e);
        attr_set.mark(ctx->device);
    }
    const uint64_t grid = expert_tiles(p.m, p.experts, p.tile_rows) * p.n_blocks * split;
    if (grid >> 31) return AFB_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)grid); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = bytes; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, split, pass, row_bytes);
    count_launch();
    return e == cudaSuccess ? AFB_OK : cuda_fail(e);
}

template <int MT>
int launch_rows(const ExpertParams& p, uint32_t bits, uint32_t group, uint32_t split, DeviceCtx* ctx, cudaStream_t s) {
    if (bits == 8) return group ? launch_cfg<8, MT, true, false>(p, split, ctx, s) : launch_cfg<8, MT, false, false>(p, split, ctx, s);
    if (group == 64) return launch_cfg<4, MT, true, true>(p, split, ctx, s);
    return group ? launch_cfg<4, MT, true, false>(p, split, ctx, s) : launch_cfg<4, MT, false, false>(p, split, ctx, s);
}

}  // namespace

int launch_expert_few(const ExpertParams& q, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s) {
    ExpertParams p = q;
    p.n_blocks = (p.n + kFewChannels - 1) / kFewChannels;
    const uint32_t mean = (p.m + p.experts - 1) / p.experts;   // rows per expert
    const uint32_t mt = mean <= 2 ? 1 : mean <= 12 ? 2 : 4;
    p.tile_rows = 8 * mt;
    // stretches of K: enough CTAs for two waves of two per SM, at least four chunks each
    const uint32_t chunks = p.k / (bits == 8 ? 64 : 128);
    const uint64_t ctas = expert_tiles(p.m, p.experts, p.tile_rows) * p.n_blocks;
    uint32_t split = 1;
    while (split < 8 && ctas * split < 4ull * ctx->sm_count && chunks >= split * 2 * kAhead) split *= 2;
    return mt == 1 ? launch_rows<1>(p, bits, group, split, ctx, s) : mt == 2 ? launch_rows<2>(p, bits, group, split, ctx, s)
                                                                             : launch_rows<4>(p, bits, group, split, ctx, s);
}

}  // namespace afb

using namespace afb;

extern "C" int afb_expert_gemm_launch(const afb_expert_gemm_args* x, void* stream) {
    if (!x || x->reserved != 0 || x->gated > 1 || x->activation > AFB_ACT_SILU) return AFB_ERR_BAD_ARG;
    const afb_gemm_args& a = x->gemm;
    if (x->experts == 0 || x->experts > AFB_MOE_MAX_EXPERTS || x->top_k == 0 || (a.m && !x->ptr_row_pair && x->top_k != 1)) return AFB_ERR_BAD_ARG;
    if (!x->ptr_offsets || (uintptr_t)x->ptr_offsets % 4 || (uintptr_t)x->ptr_row_pair % 4) return AFB_ERR_BAD_ARG;
    if (a.n == 0 || a.k == 0 || (x->gated && (a.n & 1u))) return AFB_ERR_BAD_ARG;
    const uint32_t n_out = x->gated ? a.n / 2 : a.n;
    if (a.reserved != 0 || a.reserved2 != 0 || (a.b_bits != 8 && a.b_bits != 4) || a.b_encoding > 1 || a.b_layout > 2 || a.scale_dtype > 1 || a.variant > 3) return AFB_ERR_BAD_ARG;
    if (a.lda < a.k || a.ldb < a.k || a.ldc < n_out || (a.group_size && a.k % a.group_size)) return AFB_ERR_BAD_ARG;
    if (!a.ptr_b || !a.ptr_scale || (uintptr_t)a.ptr_scale % (a.scale_dtype == AFB_SCALE_BF16 ? 2 : 4) || (uintptr_t)a.ptr_c % 2 || (uintptr_t)a.ptr_a % 2) return AFB_ERR_BAD_ARG;
    if (a.m && (!a.ptr_c || (x->a_rows && !a.ptr_a))) return AFB_ERR_BAD_ARG;
    if (a.m && !x->ptr_row_pair && x->a_rows < a.m) return AFB_ERR_BAD_ARG;
    if (a.flags || a.variant == AFB_VARIANT_NAIVE || a.b_layout == AFB_LAYOUT_ROW) return AFB_ERR_UNSUPPORTED;
    if (a.k % (a.b_bits == 8 ? 64u : 128u) || a.lda % 8 || ((uint64_t)a.ldb * a.b_bits / 8) % 16) return AFB_ERR_UNSUPPORTED;
    if ((uintptr_t)a.ptr_a % 16 || (uintptr_t)a.ptr_b % 16) return AFB_ERR_UNSUPPORTED;
    if (a.group_size && (a.group_size < 64 || (a.group_size & (a.group_size - 1)))) return AFB_ERR_UNSUPPORTED;
    if (a.m >> 31 || x->a_rows >> 31 || ((uint64_t)x->experts * a.n) >> 31) return AFB_ERR_TOO_LARGE;
    DeviceCtx* ctx = current_ctx();
    if (!ctx) return AFB_ERR_NOT_INIT;
    if (a.m == 0) return AFB_OK;
    ExpertParams p{};
    p.c = reinterpret_cast<uint16_t*>(a.ptr_c);
    p.a = reinterpret_cast<const uint16_t*>(a.ptr_a);
    p.b = reinterpret_cast<const uint8_t*>(a.ptr_b);
    p.scale = a.ptr_scale;
    p.zero = reinterpret_cast<const uint8_t*>(a.ptr_zero);
    p.offsets = x->ptr_offsets; p.row_pair = x->ptr_row_pair;
    p.m = a.m; p.n = a.n; p.n_out = n_out; p.k = a.k; p.lda = a.lda; p.ldc = a.ldc;
    p.ldb_bytes = (size_t)a.ldb * a.b_bits / 8;
    p.experts = x->experts; p.top_k = x->top_k; p.a_rows = x->a_rows;
    p.enc = a.b_encoding; p.scale_dtype = a.scale_dtype; p.packed = a.b_layout == AFB_LAYOUT_COL_PACKED ? 1u : 0u;
    for (uint32_t g = a.group_size; g > 1; g >>= 1) ++p.group_shift;
    p.gated = x->gated; p.silu = x->activation == AFB_ACT_SILU ? 1u : 0u;
    const bool many = a.variant == AFB_VARIANT_PREFILL || (a.variant == AFB_VARIANT_AUTO && (uint64_t)a.m > 24ull * x->experts);
    if (many && x->a_rows) return launch_expert_many(p, a.b_bits, a.group_size, ctx, (cudaStream_t)stream);
    return launch_expert_few(p, a.b_bits, a.group_size, ctx, (cudaStream_t)stream);
}

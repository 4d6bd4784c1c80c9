// Products grouped by expert, few rows per expert (afb_expert_gemm_launch): each expert's weights are read once and multiply the handful of
// rows that picked it.  Reference counterpart of the product itself: bf16gemm_kernel_gfx90a.s:410-489; it has no experts.
//
//   D[n, r] = sum_k W[e][n,k] * A[row(r),k],   16 channels x 8 rows per mma.sync.m16n8k16, the channels as the row operand
//
// One CTA per SM walks tiles of 128 channels of one expert x up to 8 * MT of its rows; the weights of the next tiles are on their way while
// one is worked on, in a ring of kStages stages of 128 bytes of k (256 int4, 128 int8):
//
//   warps 0-15   32 channels each; four warps share a stage, the four fours take every fourth stage.  A lane reads 16 bytes of four channels and
//                32 bytes of a row of A per 16 (int8) or 32 (int4) k of its own, unpacks the weights in registers (dequant.cuh) and feeds mma.sync: the
//                four lanes of a quad hold different k.  At the end of a tile the fours' sums meet in shared memory.
//   warps 16-19  the rows of A, 16-byte copies that report to the stage's barrier by themselves; warp 16 also the raw weights by TMA, two boxes of 128
//                channels x 64 bytes: rows of 64 bytes are read without bank conflicts as they lie
//
// Group scales multiply the fp32 sum of 64 bytes of k, which lie in one group (HALF: in two, int4 in groups of 64; a lane's 16 bytes are then 8 of each).
// No workspace, no counter, the same bits in every run.
//
// What bounds it.  int8 per channel: HBM (32 rows on 8 experts of 22016 x 4096, gated: 114 to 140 us with the experts' shares of the rows, 5.2 to 6.3 TB/s).  int4 in groups:
// instructions, 650 to 780 per warp and stage of 4 KB, four warps a scheduler at 0.55 of the issue slots (8 rows on 8 experts of 2048 x 4096: 14 us, 2.4 TB/s
// from L2; 16 rows each on 64 experts: 133 us, where the form for many rows takes 112).
#include "dequant.cuh"
#include "decode_common.cuh"
#include "expert_common.cuh"
#include "stream_common.cuh"

namespace afb {
namespace {

constexpr int kFewWarps = 16, kLoadWarps = 4, kFewThreads = 32 * (kFewWarps + kLoadWarps);   // 640: launched with 96 registers a thread
constexpr uint32_t kRegsWork = 112, kRegsLoad = 32;
constexpr uint32_t kRegsAll = 32 * kFewWarps * kRegsWork + 32 * kLoadWarps * kRegsLoad;
static_assert(kRegsAll <= 96 * kFewThreads, "shares of the registers");
constexpr uint32_t kWays = 4, kStages = 8;     // kStages: a multiple of kWays, so that a warp meets every phase of the stages that it meets
constexpr uint32_t kHalfBytes = kCh * 64;      // a box of weights
constexpr uint32_t kSumPitch = kCh + 4;        // floats per row of a way's sums
constexpr int kOffBars = 0, kOffStage = 256;   // two barriers per stage, the abort flag
static_assert(kLoadWarps % 2 == 0 && kStages % kWays == 0 && 16 * kStages + 8 <= kOffStage, "ring");

struct FewParams {
    ExpertParams x;
    uint32_t stages_per_tile;   // along K
    uint32_t off_sums, off_table;
    uint32_t c_vec;             // four results of a row (gated: two) in one store
    int32_t* status;
};

__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// The unpack's addend for a zero-point byte: -(the byte as an unsigned weight) * 2^-6, by the unpack's own multiply-add.
template <int BITS> __device__ __forceinline__ uint32_t zero_addend(uint32_t zbyte, uint32_t flip) {
    const uint32_t u = (zbyte ^ flip) & (BITS == 8 ? 0xffu : 0xfu);
    return bf16x2_fma(u * 0x00010001u, kMulByte | 0x80008000u, 0u);
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
// Place of 16-byte piece `pc` of a row of A: the eight lanes that read at once hold two rows and, of int4, pieces 4 apart.
__device__ __forceinline__ uint32_t act_place(uint32_t row, uint32_t pc) { return pc ^ (((pc >> 3) & 1u) << 1) ^ (row & 1u); }

template <int N> struct Tiles { static constexpr int value = N; };

// PACKED (int4 only): the unpack of the pre-packed order, 9 instructions per 8 weights, with constants instead of registers; otherwise either order, 10.
template <int BITS, int MT, bool GROUPED, bool HALF, bool PACKED>
__global__ void __launch_bounds__(kFewThreads, 1)
expert_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const FewParams p) {
    constexpr uint32_t CH = BITS == 8 ? 64 : 128, LK = CH / 4, AV = LK / 8;   // k per 64 bytes; of them per lane; 16-byte pieces of A per lane
    constexpr uint32_t kRowBytes = 2 * CH * 2;                                // of A per stage
    constexpr uint32_t kStageAct = 8 * MT * kRowBytes, kStageAll = 2 * kHalfBytes + kStageAct;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t base = ptx::smem_u32(smem);
    const ExpertParams& x = p.x;
    auto full = [&](uint32_t s) { return base + kOffBars + 8u * s; };
    auto empty = [&](uint32_t s) { return base + kOffBars + 8u * (kStages + s); };
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + 16 * kStages);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const ExpertTable table(smem + p.off_table, x.experts);

    if (warp == kFewWarps) {
        if (lane == 0) {
            for (uint32_t s = 0; s < kStages; ++s) { ptx::mbar_init(full(s), 1 + 32 * kLoadWarps); ptx::mbar_init(empty(s), kWays); }
            *abort_flag = 0;
            ptx::fence_mbar_init();
            ptx::prefetch_tmap(&tmap_w);
        }
        __syncwarp();
    } else if (warp == 0) {
        table.build(x, lane);
    }
    __syncthreads();
    auto give_up = [&](int where, uint32_t a, uint32_t b) {
        if (!*abort_flag) { report_timeout(p.status, where, (int)a, (int)b); *abort_flag = 1; }
    };
    const uint32_t tiles = table.strips() * x.n_blocks, ns = p.stages_per_tile;
    ExpertStrip t;

    if (warp >= kFewWarps) {
        ptx::regs_down<kRegsLoad>();
        // ======================= weights and rows of A =======================
        constexpr uint32_t kPieces = kRowBytes / 16, kRowsAtOnce = 32 / kPieces, kTurn = kLoadWarps * kRowsAtOnce;   // of one warp's copy; of all warps'
        const uint32_t r0 = (warp - kFewWarps) * kRowsAtOnce + lane / kPieces, piece = lane % kPieces;
        // the halves of a stage one after the other: the pieces of 64 bytes of weights, for every row
        const uint32_t half = piece / (kPieces / 2), pc = piece % (kPieces / 2);
        const uint32_t dst = 2 * kHalfBytes + half * (kStageAct / 2) + r0 * (kRowBytes / 2) + act_place(r0, pc) * 16u;   // kTurn rows on: the same place
        Ring r{0, 0};
        uint32_t issued = 0, parity = 0;
        bool ok = true;
        for (uint32_t i = blockIdx.x; ok && i < tiles; i += gridDim.x) {
            table.tile<1>(x, i, t);
            const int y = (int)(t.expert * x.n + t.block * kCh);
            const uint16_t* src[8 * MT / kTurn];   // of this lane's piece of the next stage
            uint32_t size[8 * MT / kTurn];         // bytes that there are of it; the rest is zeros
#pragma unroll
            for (uint32_t j = 0; j < 8 * MT / kTurn; ++j) {
                const uint32_t row = r0 + j * kTurn < t.rows ? source_row(x, t.row0 + r0 + j * kTurn) : 0xffffffffu;
                size[j] = row < x.a_rows ? 16u : 0u;
                src[j] = x.a + (size[j] ? (size_t)row * x.lda : 0) + piece * 8u;
            }
            for (uint32_t kb = 0; kb < ns; ++kb) {
                if (!warp_wait(empty(r.i), r.phase ^ 1u, abort_flag)) { give_up(71, i, kb); ok = false; break; }
                const uint32_t stage = base + kOffStage + r.i * kStageAll;
                if (warp == kFewWarps && ptx::elect_one()) {
                    ptx::mbar_arrive_expect_tx(full(r.i), 2 * kHalfBytes);
                    ptx::tma_load_2d(stage, &tmap_w, (int)(kb * 128u), y, full(r.i));
                    ptx::tma_load_2d(stage + kHalfBytes, &tmap_w, (int)(kb * 128u + 64u), y, full(r.i));
                }
                __syncwarp();
                const bool inside = kb * (2 * CH) + piece * 8u < x.k;   // the last stage may have but one half
#pragma unroll
                for (uint32_t j = 0; j < 8 * MT / kTurn; ++j) {
                    if (r0 + j * kTurn >= t.rows) break;   // the columns of D of the rows behind the last one are never stored
                    cp_async16_or_zero(stage + dst + j * (kTurn * kRowBytes / 2), inside ? src[j] : x.a, inside ? size[j] : 0u);
                    src[j] += 2 * CH;
                }
                cp_async_arrive(full(r.i));
                issued |= 1u << r.i; parity = (parity & ~(1u << r.i)) | (r.phase << r.i);
                r.step(1, kStages);
            }
        }
        cp_async_wait_all();   // never leave with a copy still writing this CTA's shared memory
        for (uint32_t s = 0; s < kStages; ++s)
            if (issued & (1u << s)) ptx::mbar_wait(full(s), (parity >> s) & 1u);
    } else {
        // ======================= 32 channels x one of the ways =======================
        ptx::regs_up<kRegsWork>();
        const uint32_t cg = warp & 3u, way = warp >> 2, g = lane >> 2, tig = lane & 3;
        const uint32_t flip = BITS == 8 ? flip8(x.enc) : flip4(x.enc);
        const uint32_t sel0 = x.packed ? kSel8Strided02 : kSel8Natural01, sel1 = x.packed ? kSel8Strided13 : kSel8Natural23;
        const Nibbles nib = nibbles(x.packed != 0);
        const bool has_zero = x.zero != nullptr, half_scale = x.scale_dtype == AFB_SCALE_BF16;
        const uint32_t groups_per_row = GROUPED ? x.k >> x.group_shift : 0;
        constexpr int kGroupsPer = GROUPED ? (HALF ? 4 : 2) : 1;   // scale groups of a stage, at most
        uint32_t act_off[AV];
#pragma unroll
        for (uint32_t v = 0; v < AV; ++v) act_off[v] = act_place(g, HALF ? (v / 2) * 8 + tig * 2 + (v & 1) : tig * AV + v) * 16u + g * (kRowBytes / 2);   // eight rows on: the same place
        const uint32_t raw_off = (cg * 32 + g) * 64 + tig * (HALF ? 8 : 16);
        float* sums = reinterpret_cast<float*>(smem + p.off_sums);
        uint32_t before = 0;   // stages of the tiles walked so far
        bool ok = true;
        for (uint32_t i = blockIdx.x; i < tiles; i += gridDim.x) {
            table.tile<1>(x, i, t);
            const uint32_t n0 = t.block * kCh;
            const bool two = MT > 1 && t.rows > 8;   // eight rows or less take one instruction where there could be two
            uint32_t chan[4];      // rows of B of this lane's channels: 8 apart
#pragma unroll
            for (int j = 0; j < 4; ++j) chan[j] = t.expert * x.n + min(n0 + cg * 32 + j * 8 + g, x.n - 1);
            uint32_t add[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) add[j] = !GROUPED && has_zero ? zero_addend<BITS>(x.zero[chan[j]], flip) : unpack_add(BITS, 0);
            // scales and zero-points of this warp's next stage, as they are stored: fetched when it is done with the one before, converted (which
            // waits for them) when they are used
            uint32_t sc[kGroupsPer][4], zp[kGroupsPer][4];
            const size_t tile0 = ((size_t)t.expert * x.n + n0) * groups_per_row;   // the offsets inside a tile fit 32 bits
            const uint16_t* scale16 = reinterpret_cast<const uint16_t*>(x.scale) + tile0;
            const uint32_t* scale32 = reinterpret_cast<const uint32_t*>(x.scale) + tile0;
            uint32_t at0[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) at0[j] = (chan[j] - t.expert * x.n - n0) * groups_per_row;
            auto load_scales = [&](uint32_t kb) {
                if constexpr (!GROUPED) return;
                if (kb >= ns) return;
#pragma unroll
                for (int q = 0; q < kGroupsPer; ++q) {
                    const uint32_t k = kb * (2 * CH) + q * (2 * CH / kGroupsPer);
                    if (k >= x.k) break;
                    const uint32_t grp = k >> x.group_shift;
                    if (half_scale) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[q][j] = scale16[at0[j] + grp];
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[q][j] = scale32[at0[j] + grp];
                    }
                    if (has_zero) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) zp[q][j] = x.zero[tile0 + at0[j] + grp];
                    }
                }
            };
            auto scale_of = [&](uint32_t raw) { return __uint_as_float(half_scale ? raw << 16 : raw); };
            float acc[2][MT][4];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int nt = 0; nt < MT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[m][nt][e] = 0.f;
            // One stage: NT tiles of 8 rows.
            auto work = [&](auto tiles_of_rows, uint32_t kb, uint32_t at) {
                constexpr int NT = decltype(tiles_of_rows)::value;
                const uint32_t stage = base + kOffStage + at * kStageAll;
#pragma unroll
                for (int c = 0; c < 2; ++c) {   // 64 bytes of k
                    if (c == 1 && kb * (2 * CH) + CH >= x.k) break;
                    const uint32_t raw = stage + c * kHalfBytes + raw_off, act = stage + 2 * kHalfBytes + c * (kStageAct / 2);
                    uint32_t w[4][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (HALF) {
                            const uint2 lo = lds64(raw + j * 512), hi = lds64(raw + j * 512 + 32);
                            w[j][0] = lo.x; w[j][1] = lo.y; w[j][2] = hi.x; w[j][3] = hi.y;
                        } else {
                            const uint4 v = lds128(raw + j * 512);
                            w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
                        }
                    }
                    float part[2][NT][4];
                    uint4 b[NT];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {   // words of the 16 bytes
                        const int grp = !GROUPED ? 0 : HALF ? 2 * c + q / 2 : c;
                        if (GROUPED && has_zero && (q == 0 || (HALF && q == 2))) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) add[j] = zero_addend<BITS>(zp[grp][j], flip);
                        }
                        if (BITS == 4 || q % 2 == 0) {
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) b[nt] = lds128(act + act_off[BITS == 4 ? q : q / 2] + nt * (8 * kRowBytes / 2));
                        }
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            uint32_t fa[4], fb[4];
                            const uint32_t aa = add[2 * m], ab = add[2 * m + 1];
                            if (BITS == 8) {
                                s8x4_to_bf16(w[2 * m][q], flip, sel0, sel1, kMulByte, aa, fa[0], fa[1]);
                                s8x4_to_bf16(w[2 * m + 1][q], flip, sel0, sel1, kMulByte, ab, fb[0], fb[1]);
                            } else {
                                if constexpr (PACKED) {
                                    s4x8_to_bf16_strided(w[2 * m][q], flip, aa, fa);
                                    s4x8_to_bf16_strided(w[2 * m + 1][q], flip, ab, fb);
                                } else {
                                    s4x8_to_bf16(w[2 * m][q], flip, nib, nib.mul[0], nib.mul[1], aa, fa);
                                    s4x8_to_bf16(w[2 * m + 1][q], flip, nib, nib.mul[0], nib.mul[1], ab, fb);
                                }
                            }
                            const bool first = GROUPED && (q == 0 || (HALF && q == 2)), last = GROUPED && (q == 3 || (HALF && q == 1));
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (BITS == 8) {
                                    const uint32_t b0 = q % 2 == 0 ? b[nt].x : b[nt].z, b1 = q % 2 == 0 ? b[nt].y : b[nt].w;
                                    if (!GROUPED) mma_bf16(acc[m][nt], fa[0], fb[0], fa[1], fb[1], b0, b1);
                                    else if (first) mma_bf16_first(part[m][nt], fa[0], fb[0], fa[1], fb[1], b0, b1);
                                    else mma_bf16(part[m][nt], fa[0], fb[0], fa[1], fb[1], b0, b1);
                                } else {
                                    if (!GROUPED) mma_bf16(acc[m][nt], fa[0], fb[0], fa[1], fb[1], b[nt].x, b[nt].y);
                                    else if (first) mma_bf16_first(part[m][nt], fa[0], fb[0], fa[1], fb[1], b[nt].x, b[nt].y);
                                    else mma_bf16(part[m][nt], fa[0], fb[0], fa[1], fb[1], b[nt].x, b[nt].y);
                                    mma_bf16(GROUPED ? part[m][nt] : acc[m][nt], fa[2], fb[2], fa[3], fb[3], b[nt].z, b[nt].w);
                                }
                                if (last) {
                                    const float sa = scale_of(sc[grp][2 * m]), sb = scale_of(sc[grp][2 * m + 1]);
                                    acc[m][nt][0] = fmaf(sa, part[m][nt][0], acc[m][nt][0]); acc[m][nt][1] = fmaf(sa, part[m][nt][1], acc[m][nt][1]);
                                    acc[m][nt][2] = fmaf(sb, part[m][nt][2], acc[m][nt][2]); acc[m][nt][3] = fmaf(sb, part[m][nt][3], acc[m][nt][3]);
                                }
                            }
                        }
                    }
                }
            };
            uint32_t kb = (way - before) & (kWays - 1);
            Ring r;
            r.set(before + kb, kStages);
            load_scales(kb);
            for (; kb < ns; kb += kWays) {
                ok = ok && warp_wait(full(r.i), r.phase, abort_flag);
                if (!ok) { give_up(73, i, kb); break; }
                if (MT > 1 && two) work(Tiles<MT>(), kb, r.i); else work(Tiles<1>(), kb, r.i);
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(empty(r.i));
                load_scales(kb + kWays);
                r.step(kWays, kStages);
            }
            before += ns;
            // ---- the ways' sums meet: [way][row][channel], added in the order of the ways.  (Also after an abort: the barriers count all warps.)
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int nt = 0; nt < MT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sums[(way * (8 * MT) + nt * 8 + 2 * tig + (e & 1)) * kSumPitch + cg * 32 + m * 16 + (e >> 1) * 8 + g] = acc[m][nt][e];
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kFewWarps) : "memory");
            const uint32_t row = tid / (kCh / 4), ch = tid % (kCh / 4) * 4, nn = n0 + ch;
            if (row < t.rows && nn < x.n) {
                float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t wy = 0; wy < kWays; ++wy) {
                    const float4 y = *reinterpret_cast<const float4*>(sums + (wy * (8 * MT) + row) * kSumPitch + ch);
                    f[0] += y.x; f[1] += y.y; f[2] += y.z; f[3] += y.w;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (GROUPED) f[e] *= kUnpackInverse;
                    else f[e] = nn + e < x.n ? unscaled(f[e], load_scale(x.scale, (size_t)t.expert * x.n + nn + e, x.scale_dtype)) : 0.f;
                }
                const int n_here = x.gated ? 2 : 4;
                uint32_t o[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float lo = x.silu ? silu(f[2 * e]) : f[2 * e], hi = f[2 * e + 1];
                    if (x.gated) {
                        f[e] = lo * hi;   // f[1] has been read
                    } else {
                        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, x.silu ? silu(hi) : hi);
                        o[e] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                }
                if (x.gated) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]);
                    o[0] = *reinterpret_cast<const uint32_t*>(&v);
                }
                const uint32_t col = x.gated ? nn / 2 : nn;
                uint16_t* dst = x.c + (size_t)(t.row0 + row) * x.ldc + col;
                if (p.c_vec && col + n_here <= x.n_out) {
                    if (x.gated) *reinterpret_cast<uint32_t*>(dst) = o[0];
                    else *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < n_here && col + e < x.n_out) dst[e] = (uint16_t)(o[e / 2] >> (e % 2 * 16));
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kFewWarps) : "memory");
        }
    }
}

template <int BITS, int MT, bool GROUPED, bool HALF, bool PACKED = false>
int launch_cfg(const CUtensorMap& tw, const FewParams& q, DeviceCtx* ctx, cudaStream_t s) {
    auto kern = expert_few_kernel<BITS, MT, GROUPED, HALF, PACKED>;
    FewParams p = q;
    p.off_sums = kOffStage + kStages * (2 * kHalfBytes + 8 * MT * (BITS == 8 ? 256 : 512));
    p.off_table = p.off_sums + kWays * 8 * MT * kSumPitch * sizeof(float);
    const uint32_t bytes = p.off_table + ExpertTable::bytes(p.x.experts);
    if (bytes > 232448) return AFB_ERR_UNSUPPORTED;   // the caller has seen to it
    static DeviceOnce attr_set;
    if (!attr_set.done(ctx->device)) {
        cudaFuncAttributes attr;
        cudaError_t e = cudaFuncGetAttributes(&attr, kern);
        if (e != cudaSuccess) return cuda_fail(e);
        if ((uint32_t)(attr.numRegs * kFewThreads) < kRegsAll) return AFB_ERR_UNSUPPORTED;   // the shares come out of what the block is launched with
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (e != cudaSuccess) return cuda_fail(e);
        attr_set.mark(ctx->device);
    }
    const uint64_t tiles = expert_tiles(p.x.m, p.x.experts, p.x.tile_rows) * p.x.n_blocks;
    if (tiles >> 31) return AFB_ERR_TOO_LARGE;
    const uint32_t grid = tiles < (uint64_t)ctx->sm_count ? (uint32_t)tiles : (uint32_t)ctx->sm_count;
    kern<<<grid, kFewThreads, bytes, s>>>(tw, p);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? AFB_OK : cuda_fail(e);
}

template <int MT>
int launch_rows(const CUtensorMap& tw, const FewParams& p, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s) {
    if (bits == 8) return group ? launch_cfg<8, MT, true, false>(tw, p, ctx, s) : launch_cfg<8, MT, false, false>(tw, p, ctx, s);
    if (p.x.packed) {
        if (group == 64) return launch_cfg<4, MT, true, true, true>(tw, p, ctx, s);
        return group ? launch_cfg<4, MT, true, false, true>(tw, p, ctx, s) : launch_cfg<4, MT, false, false, true>(tw, p, ctx, s);
    }
    if (group == 64) return launch_cfg<4, MT, true, true>(tw, p, ctx, s);
    return group ? launch_cfg<4, MT, true, false>(tw, p, ctx, s) : launch_cfg<4, MT, false, false>(tw, p, ctx, s);
}

}  // namespace

int launch_expert_few(const ExpertParams& q, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s) {
    FewParams p{};
    p.x = q;
    p.x.set_blocks((q.n + kCh - 1) / kCh);
    p.stages_per_tile = (uint32_t)(((uint64_t)q.k * bits / 8 + 127) / 128);
    p.c_vec = q.ldc % 4 == 0 && (uintptr_t)q.c % 8 == 0;
    p.status = ctx->status;
    // tiles of 8 rows where few experts have more; of int4 also where the table of many experts leaves no room for the rows of 16
    const bool small = (uint64_t)q.m <= 3ull * q.experts || (bits == 4 && q.experts > 128);
    p.x.tile_rows = small ? 8 : 16;
    CUtensorMap tw;
    const int rc = tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, q.b, (uint64_t)q.k * bits / 8, (uint64_t)q.experts * q.n, q.ldb_bytes, 64, kCh, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc) return rc;
    return small ? launch_rows<1>(tw, p, bits, group, ctx, s) : launch_rows<2>(tw, p, bits, group, ctx, s);
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
    if (a.m && (!a.ptr_c || !a.ptr_a || !x->a_rows)) return AFB_ERR_BAD_ARG;
    if (a.m && !x->ptr_row_pair && x->a_rows < a.m) return AFB_ERR_BAD_ARG;
    if (a.flags || a.variant == AFB_VARIANT_NAIVE || a.b_layout == AFB_LAYOUT_ROW) return AFB_ERR_UNSUPPORTED;
    if (a.k % (a.b_bits == 8 ? 64u : 128u) || a.lda % 8 || ((uint64_t)a.ldb * a.b_bits / 8) % 16) return AFB_ERR_UNSUPPORTED;
    if ((uintptr_t)a.ptr_a % 16 || (uintptr_t)a.ptr_b % 16) return AFB_ERR_UNSUPPORTED;
    if (a.group_size && (a.group_size < 64 || (a.group_size & (a.group_size - 1)))) return AFB_ERR_UNSUPPORTED;
    if (a.k >> 24 || a.m >> 31 || x->a_rows >> 31 || ((uint64_t)x->experts * a.n) >> 31) return AFB_ERR_TOO_LARGE;
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
    // Which form is the faster one, by the mean of the rows per expert (us, few / many; their own numbers of rows spread around it):
    //   64 experts of 2048 x 4096 gated, int4 group-128: 8 rows 86 / 97, 12: 110 / 112, 16: 133 / 112, 24: 165 / 126;  int8: 4: 82 / 80, 8: 102 / 92
    //   8 of 11008 x 4096, int4 group-128: 12: 74 / 85, 16: 88 / 85, 24: 121 / 85;  int8: 4: 82 / 80, 12: 88 / 80
    //   16 of 4096 x 2816, int4 group-64: 8: 50 / 54, 12: 59 / 54, 24: 80 / 56;  128 of 1536 x 2048, int8 group-128: 4: 72 / 81, 8: 92 / 87
    // One threshold per width: between 8 and 12 int4 in groups of 64, between 4 and 8 int8 in groups take the slower form by a tenth at most.  m is the host's bound of the
    // pairs: those of padded tokens count.
    const bool many = a.variant == AFB_VARIANT_PREFILL || (a.variant == AFB_VARIANT_AUTO && (uint64_t)a.m > (a.b_bits == 8 ? 4ull : 12ull) * x->experts);
    if (many) {
        bool done = false;
        const int rc = launch_expert_many(p, a.b_bits, a.group_size, ctx, (cudaStream_t)stream, &done);
        if (done) return rc;
    }
    return launch_expert_few(p, a.b_bits, a.group_size, ctx, (cudaStream_t)stream);
}

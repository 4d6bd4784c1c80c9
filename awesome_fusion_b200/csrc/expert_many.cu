// Products grouped by expert, many rows per expert (afb_expert_gemm_launch): two SMs on one tile, as in the pair form of the dense product
// (pair.cu; reference counterpart of the product: bf16gemm_kernel_gfx90a.s:184-636, which has no experts).
//
// D[n, r] = sum_k W[e][n,k] * A[row(r),k] with the unpacked weights as the tensor-memory operand.  A cluster of two CTAs owns 256 channels of
// one expert x one strip of its rows: each unpacks its own 128 channels into its own tensor memory, each gathers half of the strip's rows of A, and
// one tcgen05.mma.cta_group::2 reads both halves.  An expert's rows are cut into strips of equal height, a multiple of 32.
//
//   warp 0        TMA: raw weight blocks, 128 channels x 128 bytes, 128-byte swizzle
//   warp 2        rank 0: tcgen05.mma 256 x height x 16 (low strips: with warp 3, every second step each, into an accumulator each);  rank 1: reports
//                 to rank 0 that its half of a step is complete
//   warps 4-11    epilogue, two per lane quarter: accumulator -> registers -> (accumulator free) -> shared memory -> C
//   then          converters: four groups of four warps; group g takes every fourth step of k (KS = 128 or 64 wide)
//   last four     the rows of A: 16-byte copies to shared memory, written in the 128-byte swizzle.  (A TMA gather of four rows takes 65 cycles of
//                 the issuing warp, which has to make every lane's row numbers uniform first: 4200 cycles per step of 256 rows.)
//
// The sum over all of K stays in the accumulator.  Scales per channel multiply it in the end.  Scales per group go into the weights, and there bf16 has no
// room for them: a weight of 4 bits times a scale of 8 has up to 12 significant ones, and a rounding to 8 costs as much accuracy as the rounding of the
// result.  So these products are made in fp16, with 11: int4 without zero-points exactly (|q| <= 8 has three significant bits), with them and int8 off by
// 2^-11 at most.  What fp16 lacks is range, so a kernel ahead of this one gives every row of A a power of two that brings its largest value below 2^15 (what is
// below 2^-28 of it loses bits: 2^-39 of the largest at most), and finds one for every channel's scales (below 2^-20 of the largest they lose bits); the
// epilogue takes both out again.  (Tried before: sums of each group in accumulators of their own, scaled and added in fp32 registers, which is exact, too:
// 1650 cycles per step of 128 rows, the chain from accumulator to registers and back; 2048 tokens, 64 experts of 2048 x 4096 int4: 516 us.)
//
// Every role walks the same tiles (ExpertTable): worker, worker + workers, ...
//
// What bounds it.  Strips of 256 rows: the tensor pipe, under the power limit (8192 rows on 8 experts of 22016 x 4096 int8, gated: 1047 us = 1.41 PFLOP/s), and per tile
// the drain of the only accumulator (2000 to 3000 cycles); where they are lower than that the hand-offs (16384 rows on 64 experts of 2048 x 4096 int4 group-128: 274 us
// = 1.0 PFLOP/s).  Strips up to 64: int4 in groups by instructions, 0.66 of the issue slots (1024 rows: 114 us; a group of converters needs 2600 cycles for a
// step, four of them at a time); int8 per channel by HBM (103 us, 5.2 TB/s of weights).
#include <cuda_fp16.h>
#include "dequant.cuh"
#include "expert_common.cuh"
#include "stream_common.cuh"

namespace afb {
namespace {

constexpr int kFirstEpi = 4, kEpiWarps = 8, kFirstConv = kFirstEpi + kEpiWarps, kLoadWarps = 4;
// Groups of converters.  Four: a group's chain (wait, load, unpack, tcgen05.st, arrive) is what a step waits for where strips are low (1024 rows on 64 experts of
// 2048 x 4096 int4: 141 us with four, 153 with two), and int4 in groups where they are high (16384 rows: 273 with four, 284 with two); int8 does not mind (8192 rows on 8
// experts: 1056, 1062).  Six, with four other warps less: slower, the rows of A then come from one warp (1024 rows: 134 where four groups take 115).
constexpr int kConvGroups = 4, kFirstLoad = kFirstConv + 4 * kConvGroups, kManyThreads = 32 * (kFirstLoad + kLoadWarps);   // 1024: launched with 64 registers a thread
// Registers a thread of each role.  HEAVY: converters of int4 in groups, which hold the words, the scales and the results of a step; with 56 they go to
// local memory and back 13 times a step (1024 rows: 123 us; with 64: 119; int8 per channel, which needs no more than 56, 109 and 111).
struct Shares { uint32_t ctrl, epi, conv, load; };
__host__ __device__ constexpr Shares shares(bool heavy) { return heavy ? Shares{32, 96, 64, 32} : Shares{40, 104, 56, 40}; }
__host__ __device__ constexpr uint32_t regs_all(bool heavy) {
    const Shares r = shares(heavy);
    return 128 * r.ctrl + 32 * kEpiWarps * r.epi + 128 * kConvGroups * r.conv + 32 * kLoadWarps * r.load;
}
static_assert(regs_all(false) <= 64u * kManyThreads && regs_all(true) <= 64u * kManyThreads, "shares of the registers");
constexpr int kMaxRaw = 12, kMaxSlots = 8, kMaxAcc = 2;   // kMaxAcc: one accumulator per issuer
__host__ __device__ constexpr uint32_t slots(int ks, bool low) { return ks == 128 && !low ? 4 : 6; }   // steps under way, in 256 columns at most (low strips: 384)
constexpr uint32_t kTmemCols = 512;
constexpr int kBars = 2 * (kMaxRaw + kMaxSlots + kMaxAcc);
constexpr int kOffMisc = kBars * 8, kOffOut = 1024;
constexpr int kOutBytes = 16 * 32 * 2;   // one block of the result: 16 rows x 32 channels; two per epilogue warp
constexpr int kOffTable = kOffOut + kEpiWarps * 2 * kOutBytes;
static_assert(kOffMisc + 16 <= kOffOut, "shared memory layout");
constexpr uint32_t kUnit = 32;           // rows: 16 per epilogue warp

struct ManyParams {
    ExpertParams x;
    uint32_t steps;           // along K
    uint32_t raw_stages;
    uint32_t slot_first;      // converters wait for their slot before they wait for their raw block
    uint32_t off_raw;         // behind the table
    uint32_t c_vec;           // 16-byte stores of C
    const float* row_factor;    // group scales: see PrepareParams
    const float* channel_mult;
    int32_t* status;
};

// Two fp16 values at a time.
__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t f16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t f16_dup(float v) { return (uint32_t)__half_as_ushort(__float2half_rn(v)) * 0x00010001u; }
// The largest power of two that is not above v, as its exponent; 0 for v = 0, infinity and NaN.
__device__ __forceinline__ int exponent_of(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    if (u == 0u || u >= 0x7f800000u) return 0;
    return u >= 0x00800000u ? (int)(u >> 23) - 127 : -118 - __clz((int)u);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127
// The factor that brings values of up to 2^(e + 1) below 2^15.
__device__ __forceinline__ int headroom(int e) { return min(14 - e, 126); }

// Group scales: the rows of A as fp16 with a power of two of their own, and the power of two of each channel's scales.  The first blocks take 256 channels each (of
// experts that have rows), the others rows, with `row_threads` threads each, so that a row is held in registers between the search for its
// largest value and the conversion: up to kHeld pieces of 16 bytes a thread, 16384 k with a block's 256 threads.
struct PrepareParams {
    ExpertParams x;
    uint16_t* a;          // [a_rows, k]
    float* row_factor;    // what a row's products have to be multiplied by
    float* channel_mult;  // [experts * n] what a channel's scales are multiplied by
    uint32_t channel_blocks, row_threads;
};
constexpr int kPrepareThreads = 256, kHeld = 8;
__device__ __forceinline__ uint32_t largest_finite(const uint4& v, uint32_t most) {   // as the bits of its absolute value
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t a = (w[i] >> (16 * h)) & 0x7fffu;
            if (a < 0x7f80u) most = max(most, a);   // infinities and NaN stay what they are
        }
    return most;
}
__device__ __forceinline__ uint4 to_f16(const uint4& v, float mult) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(__uint_as_float(w[i] << 16) * mult, __uint_as_float(w[i] & 0xffff0000u) * mult);
        o[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}
__global__ void __launch_bounds__(kPrepareThreads) expert_prepare_kernel(const PrepareParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the product's kernel sets up meanwhile; what this one writes it waits for
    if (blockIdx.x >= p.channel_blocks) {
        __shared__ uint32_t s_most[kPrepareThreads / 32];
        const uint32_t per = p.row_threads, t = threadIdx.x % per, pieces = p.x.k / 8;
        const uint64_t row = (uint64_t)(blockIdx.x - p.channel_blocks) * (kPrepareThreads / per) + threadIdx.x / per;
        const bool there = row < p.x.a_rows;
        const uint4* src = reinterpret_cast<const uint4*>(p.x.a + (there ? row : 0) * p.x.lda);
        uint4* dst = reinterpret_cast<uint4*>(p.a + row * p.x.k);
        uint4 held[kHeld];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t c = i * per + t;
            held[i] = c < pieces ? src[c] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) most = largest_finite(held[i], most);
        for (uint32_t c = kHeld * per + t; c < pieces; c += per) most = largest_finite(src[c], most);
        most = __reduce_max_sync(0xffffffffu, most);
        if (per > 32) {
            if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
            __syncthreads();
            for (uint32_t w = 0; w < per / 32; ++w) most = max(most, s_most[threadIdx.x / per * (per / 32) + w]);
        }
        if (!there) return;
        const int e = headroom(exponent_of(__uint_as_float(most << 16)));
        const float mult = power_of_two(e);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t c = i * per + t;
            if (c < pieces) dst[c] = to_f16(held[i], mult);
        }
        for (uint32_t c = kHeld * per + t; c < pieces; c += per) dst[c] = to_f16(src[c], mult);
        if (t == 0) p.row_factor[row] = power_of_two(-e);
        return;
    }
    const uint32_t chan = blockIdx.x * kPrepareThreads + threadIdx.x;
    if (chan >= p.x.experts * p.x.n) return;
    const uint32_t expert = chan / p.x.n, groups = p.x.k >> p.x.group_shift;
    if (clamp_offset(__ldg(p.x.offsets + expert + 1), p.x.m) <= clamp_offset(__ldg(p.x.offsets + expert), p.x.m)) return;
    float largest = 0.f;
    if (p.x.scale_dtype == AFB_SCALE_BF16 && groups % 8 == 0 && (uintptr_t)p.x.scale % 16 == 0) {
        const uint4* src = reinterpret_cast<const uint4*>(p.x.scale) + (size_t)chan * (groups / 8);
        uint32_t most = 0;
#pragma unroll 4
        for (uint32_t g = 0; g < groups / 8; ++g) most = largest_finite(src[g], most);
        largest = __uint_as_float(most << 16);
    } else {
#pragma unroll 8
        for (uint32_t g = 0; g < groups; ++g) {
            const size_t at = (size_t)chan * groups + g;
            const float s = fabsf(p.x.scale_dtype == AFB_SCALE_BF16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p.x.scale)[at] << 16)
                                                                    : reinterpret_cast<const float*>(p.x.scale)[at]);
            if (s < INFINITY) largest = fmaxf(largest, s);
        }
    }
    p.channel_mult[chan] = power_of_two(headroom(exponent_of(largest)));
}

struct Strip : ExpertStrip { uint32_t n0; };   // n0: of this CTA's 128 channels

template <int BITS, bool GROUPED, int KS, bool LOW>
__global__ void __launch_bounds__(kManyThreads, 1)
expert_many_kernel(const __grid_constant__ CUtensorMap tmap_w, const ManyParams p) {
    constexpr uint32_t SPB = (BITS == 8 ? 128 : 256) / KS;   // steps per raw block
    constexpr uint32_t kSlotCols = KS / 2;                   // TMEM columns of a step's weights
    constexpr uint32_t kSlots = slots(KS, LOW);
    constexpr Shares kShares = shares(BITS == 4 && GROUPED);
    constexpr uint32_t kIssuers = LOW ? 2 : 1;
    static_assert(!LOW || (KS == 128 && kConvGroups % 2 == 0 && kSlots % 2 == 0), "a slot's steps are one issuer's");
    extern __shared__ uint8_t smem_raw_base[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw_base) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw_base + (smem_base - ptx::smem_u32(smem_raw_base));
    auto bar = [&](uint32_t i) { return smem_base + 8u * i; };
    auto raw_full = [&](uint32_t s) { return bar(s); };
    auto raw_empty = [&](uint32_t s) { return bar(kMaxRaw + s); };
    auto step_full = [&](uint32_t s) { return bar(2 * kMaxRaw + s); };                // weights in TMEM, activations in shared memory; rank 0: of both CTAs
    auto step_empty = [&](uint32_t s) { return bar(2 * kMaxRaw + kMaxSlots + s); };   // the MMAs of the step are done with both
    auto acc_full = [&](uint32_t s) { return bar(2 * (kMaxRaw + kMaxSlots) + s); };
    auto acc_empty = [&](uint32_t s) { return bar(2 * (kMaxRaw + kMaxSlots) + kMaxAcc + s); };   // rank 0: of both CTAs
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(smem_gen + kOffMisc);   // TMEM base, abort flag
    volatile uint32_t* abort_flag = misc + 1;
    const ExpertTable table(smem_gen + kOffTable, p.x.experts);
    const uint32_t act_stride = p.x.tile_rows * KS;   // bytes of one CTA's half of a step, at most
    const uint32_t off_act = p.off_raw + p.raw_stages * kRawBytes;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_rank(), worker = blockIdx.x >> 1, workers = gridDim.x >> 1;

    if (warp == 0 && lane == 0) {
        for (uint32_t s = 0; s < p.raw_stages; ++s) { ptx::mbar_init(raw_full(s), 1); ptx::mbar_init(raw_empty(s), 4 * SPB); }
        for (uint32_t s = 0; s < kSlots; ++s) { ptx::mbar_init(step_full(s), 4 + 32 * kLoadWarps + (rank == 0 ? 1 : 0)); ptx::mbar_init(step_empty(s), 1); }
        for (uint32_t s = 0; s < kIssuers; ++s) { ptx::mbar_init(acc_full(s), 1); ptx::mbar_init(acc_empty(s), 2 * kEpiWarps); }
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::prefetch_tmap(&tmap_w);
    }
    if (warp == 2) {
        ptx::tmem_alloc_pair(ptx::smem_u32(const_cast<uint32_t*>(misc)), kTmemCols);
        ptx::tmem_relinquish_pair();
    }
    if (warp == 3) table.build(p.x, lane);
    __syncwarp();
    ptx::tc_fence_before_sync();
    __syncthreads();       // the table
    ptx::cluster_arrive();
    ptx::cluster_wait();   // both CTAs' barriers are there
    ptx::tc_fence_after_sync();
    if (GROUPED && warp >= kFirstEpi) asm volatile("griddepcontrol.wait;" ::: "memory");   // the warps before these touch weights only
    constexpr uint32_t tmem_base = 0;   // all 512 columns are this CTA's: the allocation starts at column 0
    const uint32_t slot_base = tmem_base + kTmemCols - kSlots * kSlotCols;   // accumulators from column 0, slots at the end
    const uint32_t acc_cols = p.x.tile_rows;

    auto give_up = [&](int where, uint32_t a, uint32_t b) {
        if (!*abort_flag) { report_timeout(p.status, where, (int)a, (int)b); *abort_flag = 1; }
    };
    const uint32_t tiles = table.strips() * p.x.n_blocks;   // < 2^31, the launcher sees to it
    uint32_t t = worker;   // every role of both CTAs walks the same list of tiles
    auto next = [&](Strip& s) {
        if (t >= tiles) return false;
        table.tile<kUnit>(p.x, t, s);
        s.n0 = (2 * s.block + rank) * kCh;
        t += workers;
        return true;
    };
    Strip x;
    const uint32_t ns = p.steps;

    // Warps 0 to 3 run their loops as whole warps and elect a lane for the asynchronous instructions only (stream.cu).
    if (warp < kFirstEpi) {
        ptx::regs_down<kShares.ctrl>();
        Ring r{0, 0};
        uint32_t issued = 0, parity = 0;
        bool ok = true;
        if (warp == 0) {
            // ======================= TMA: raw weights =======================
            const uint32_t blocks = (ns + SPB - 1) / SPB;
            while (ok && next(x)) {
                const int y = (int)(x.expert * p.x.n + x.n0);
                for (uint32_t kb = 0; kb < blocks; ++kb) {
                    if (!warp_wait(raw_empty(r.i), r.phase ^ 1u, abort_flag)) { give_up(61, x.expert, kb); ok = false; break; }
                    if (ptx::elect_one()) {
                        ptx::mbar_arrive_expect_tx(raw_full(r.i), kRawBytes);
                        ptx::tma_load_2d(smem_base + p.off_raw + r.i * kRawBytes, &tmap_w, (int)(kb * 128u), y, raw_full(r.i));
                    }
                    issued |= 1u << r.i; parity = (parity & ~(1u << r.i)) | (r.phase << r.i);
                    r.step(1, p.raw_stages);
                }
            }
            for (uint32_t s = 0; s < p.raw_stages; ++s)   // never leave with a bulk copy still writing this CTA's shared memory
                if (issued & (1u << s)) ptx::mbar_wait(raw_full(s), (parity >> s) & 1u);
        } else if (rank == 0 && (uint32_t)warp - 2 < kIssuers) {
            // ======================= MMA issuer(s) =======================
            const uint32_t who = (uint32_t)warp - 2;
            const uint64_t desc0 = ptx::umma_desc_kmajor_sw128(smem_base + off_act);
            r.i = who;
            uint32_t acc_phase = 0;
            uint32_t before = 0, g = who;   // steps of the tiles walked so far; this warp's next step, counted over all tiles
            bool ready = false;
            while (ok && next(x)) {
                const uint32_t idesc = GROUPED ? ptx::umma_idesc_f16_f32(2 * kCh, x.height) : ptx::umma_idesc_bf16_f32(2 * kCh, x.height), slab_d = x.height * 64u >> 4;
                const uint32_t td = tmem_base + who * acc_cols, acc_done = acc_full(who), first = g;
                if (!warp_wait(acc_empty(who), acc_phase ^ 1u, abort_flag)) { give_up(63, x.expert, 0); break; }
                for (; g < before + ns; g += kIssuers) {
                    if (!__all_sync(0xffffffffu, ready) && !warp_wait(step_full(r.i), r.phase, abort_flag)) { give_up(64, x.expert, g); ok = false; break; }
                    ptx::fence_proxy_async_smem();
                    ptx::tc_fence_after_sync();
                    const uint32_t ta = slot_base + r.i * kSlotCols, done = step_empty(r.i);
                    const uint64_t db = desc0 + r.i * (act_stride >> 4);
                    r.step(kIssuers, kSlots);
                    ready = ptx::mbar_test_wait(step_full(r.i), r.phase);   // of the next step: the answer is back when this one has been issued
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int j = 0; j < KS / 16; ++j)
                            ptx::umma_bf16_ts_pair(td, ta + 8 * j, db + (uint32_t)(j / 4) * slab_d + 2u * (j % 4), idesc, g > first || j > 0 ? 1u : 0u);   // kind::f16: the types are the descriptor's
                        ptx::umma_commit_pair(done);
                        if (g + kIssuers >= before + ns) ptx::umma_commit_pair(acc_done);
                    }
                }
                before += ns;
                acc_phase ^= 1u;
            }
        } else if (warp == 2) {
            // ======================= rank 1: reports its half of each step =======================
            while (ok && next(x)) {
                for (uint32_t l = 0; l < ns; ++l) {
                    if (!warp_wait(step_full(r.i), r.phase, abort_flag)) { give_up(65, x.expert, l); ok = false; break; }
                    ptx::fence_proxy_async_smem();
                    ptx::tc_fence_after_sync();
                    ptx::tc_fence_before_sync();
                    if (ptx::elect_one()) ptx::mbar_arrive_remote(step_full(r.i), 0);
                    r.step(1, kSlots);
                }
            }
        }
    } else if (warp >= kFirstConv && warp < kFirstLoad) {
        // ======================= converters =======================
        ptx::regs_down<kShares.conv>();
        const uint32_t g = (uint32_t)(warp - kFirstConv) >> 2, quarter = (uint32_t)warp & 3u;
        const uint32_t ch = quarter * 32 + lane;
        const uint32_t flip = BITS == 8 ? flip8(p.x.enc) : flip4(p.x.enc);
        const uint32_t sel0 = p.x.packed ? kSel8Strided02 : kSel8Natural01, sel1 = p.x.packed ? kSel8Strided13 : kSel8Natural23;
        const Nibbles nib = nibbles(p.x.packed != 0);
        const bool has_zero = p.x.zero != nullptr;
        const uint32_t groups_per_row = GROUPED ? p.x.k >> p.x.group_shift : 0;
        const bool half_scale = p.x.scale_dtype == AFB_SCALE_BF16, two_groups = GROUPED && p.x.group_shift < 7;
        auto zero_of = [&](size_t i) { return BITS == 8 ? decode_zero8(p.x.zero[i], p.x.enc) : decode_zero4(p.x.zero[i], p.x.enc); };
        // bf16: weight * 2^-6 in one step (dequant.cuh).  fp16: an unsigned weight u, zero-extended, is u * 2^-24; fma makes (u - 128 - zero) * 2^-9 of it,
        // exactly, and a multiplication by the channel's scale, at most 2^15, rounds once.
        constexpr uint32_t kByteF16 = 0x78007800u, kHighF16 = 0x68006800u, kPairF16 = 0x68007800u;   // 2^15, 2^11, 2^11 and 2^15
        auto add_of = [&](int zero) { return GROUPED ? f16_dup((float)(-(BITS == 8 ? 128 : 8) - zero) * 0x1p-9f) : unpack_add(BITS, zero); };
        const uint32_t mul0 = BITS == 8 ? (GROUPED ? kByteF16 : kMulByte) : !GROUPED ? nib.mul[0] : p.x.packed ? kByteF16 : kPairF16;
        const uint32_t mul1 = BITS == 8 ? mul0 : !GROUPED ? nib.mul[1] : p.x.packed ? kHighF16 : kPairF16;
        auto unpack2 = [&](uint32_t v, uint32_t mul, uint32_t add, uint32_t sc) { return GROUPED ? f16x2_mul(f16x2_fma(v, mul, add), sc) : bf16x2_fma(v, mul, add); };
        uint32_t add[KS / 64];
#pragma unroll
        for (int h = 0; h < KS / 64; ++h) add[h] = add_of(0);
        const uint32_t row = p.off_raw + ch * 128 + ((ch & 7u) << 4),   // its first 16 bytes in the swizzle; piece i is 16 * i away, by xor
                       lanes = (quarter * 32u) << 16;
        uint32_t steps_before = 0, blocks_before = 0;   // of the tiles walked so far
        bool ok = true;
        while (ok && next(x)) {
            const uint32_t nn = x.n0 + ch;
            const size_t chan = (size_t)x.expert * p.x.n + (nn < p.x.n ? nn : 0);
            if (!GROUPED && has_zero) {
#pragma unroll
                for (int h = 0; h < KS / 64; ++h) add[h] = add_of(zero_of(chan));
            }
            const float mult = GROUPED ? p.channel_mult[chan] : 1.f;
            // scales and zero-points of this group's next step, of each 64 k that have their own, as they are stored
            const char* scales = GROUPED ? reinterpret_cast<const char*>(p.x.scale) + chan * groups_per_row * (half_scale ? 2 : 4) : nullptr;
            const uint8_t* zeros = GROUPED && has_zero ? p.x.zero + chan * groups_per_row : nullptr;
            uint32_t sc_nxt[KS / 64] = {}, z_nxt[KS / 64] = {};
            auto load_group = [&](uint32_t l) {
                if constexpr (GROUPED) {
                    if (l >= ns) return;
#pragma unroll
                    for (int h = 0; h < KS / 64; ++h) {
                        if (h && !two_groups) break;
                        const uint32_t i = (l * KS + h * 64) >> p.x.group_shift;
                        sc_nxt[h] = half_scale ? reinterpret_cast<const uint16_t*>(scales)[i] : reinterpret_cast<const uint32_t*>(scales)[i];
                        if (has_zero) z_nxt[h] = zeros[i];
                    }
                }
            };
            uint32_t l = (g - steps_before) & (kConvGroups - 1);
            Ring rr, rs;
            rr.set(blocks_before + l / SPB, p.raw_stages);
            rs.set(steps_before + l, kSlots);
            load_group(l);
            for (; l < ns; l += kConvGroups) {
                const uint32_t sub = l % SPB;
                uint32_t sc[KS / 64] = {};
                if (GROUPED) {
#pragma unroll
                    for (int h = 0; h < KS / 64; ++h) {
                        if (h && !two_groups) { sc[h] = sc[0]; add[h] = add[0]; break; }
                        sc[h] = f16_dup(__uint_as_float(half_scale ? sc_nxt[h] << 16 : sc_nxt[h]) * mult);
                        if (has_zero) add[h] = add_of(BITS == 8 ? decode_zero8(z_nxt[h], p.x.enc) : decode_zero4(z_nxt[h], p.x.enc));
                    }
                    load_group(l + kConvGroups);
                }
                if (p.slot_first && !warp_wait(step_empty(rs.i), rs.phase ^ 1u, abort_flag)) { give_up(66, x.expert, l); ok = false; break; }
                if (!warp_wait(raw_full(rr.i), rr.phase, abort_flag)) { give_up(67, x.expert, l); ok = false; break; }
                const uint32_t raw = smem_base + row + rr.i * kRawBytes, slot = slot_base + lanes + rs.i * kSlotCols;
                // KS / 64 times: the raw words of 64 k (of int4 the whole step's) first, then 32 k at a time
                constexpr int kWords = BITS == 8 ? 16 : KS / 8, kPieces = BITS == 8 ? KS / 64 : 1, kPerStore = BITS == 8 ? 8 : 4;
#pragma unroll
                for (int h = 0; h < kPieces; ++h) {
                    uint32_t w[kWords];
#pragma unroll
                    for (int i = 0; i < kWords / 4; ++i) {
                        const uint32_t at = (raw ^ (sub * (kPieces * kWords * 4))) ^ ((h * (kWords / 4) + i) << 4);
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3]) : "r"(at));
                    }
#pragma unroll
                    for (int q = 0; q < kWords / kPerStore; ++q) {
                        uint32_t o[16];
                        const int k64 = BITS == 8 ? h : q / 2;   // which 64 k of the step
#pragma unroll
                        for (int j = 0; j < kPerStore; ++j) {
                            const uint32_t v = w[q * kPerStore + j];
                            if (BITS == 8) {
                                const uint32_t t8 = v ^ flip;
                                o[2 * j] = unpack2(prmt(t8, 0u, sel0), mul0, add[k64], sc[k64]);
                                o[2 * j + 1] = unpack2(prmt(t8, 0u, sel1), mul0, add[k64], sc[k64]);
                            } else {   // s4x8_to_bf16's steps
                                const uint32_t e = lop3_and_xor(v, 0x0f0f0f0fu, flip & 0x0f0f0f0fu), d = lop3_and_xor(v, 0xf0f0f0f0u, flip & 0xf0f0f0f0u);
#pragma unroll
                                for (int i = 0; i < 4; ++i) o[4 * j + i] = unpack2(prmt(e, d, nib.sel[i]), i % 2 ? mul1 : mul0, add[k64], sc[k64]);
                            }
                        }
                        if (h == 0 && q == 0) {
                            if (!p.slot_first && !warp_wait(step_empty(rs.i), rs.phase ^ 1u, abort_flag)) { give_up(66, x.expert, l); ok = false; break; }
                            ptx::tc_fence_after_sync();
                        }
                        ptx::tmem_st_32x16(slot + (h * (kWords / kPerStore) + q) * 16, o);
                    }
                    if (!ok) break;
                }
                if (!ok) break;
                ptx::tmem_st_wait();
                ptx::tc_fence_before_sync();
                __syncwarp();   // every lane's weights are in tensor memory
                if (lane == 0) {
                    ptx::mbar_arrive(step_full(rs.i));
                    const uint32_t left = ns - (l - sub);   // steps of this block and all after it
                    ptx::mbar_arrive_count(raw_empty(rr.i), left < SPB && sub + 1 == left ? 1 + SPB - left : 1u);   // a short last block: for its missing steps, too
                }
                rr.step((sub + kConvGroups) / SPB, p.raw_stages);   // of this group's next step
                rs.step(kConvGroups, kSlots);
            }
            steps_before += ns;
            blocks_before += (ns + SPB - 1) / SPB;
        }
    } else if (warp >= kFirstLoad) {
        // ======================= rows of A =======================
        // All four warps copy a step together.  The copies report themselves when they are complete, so the warps run ahead as far as there are slots.  They are these
        // threads' writes, and tcgen05.mma reads shared memory through the asynchronous proxy: the issuers (rank 1: the reporter) fence between the two once they
        // have waited.  (Waited for and reported by the warps, one to three steps later: 16384 rows on 64 experts of int4 299 us, 8192 rows of int8 1128; now 287 and
        // 1072.)  A lane copies 16 bytes of rows 16 * i + 4 * (which loader) + lane / 8 of this CTA's half, per 64 k.
        ptx::regs_down<kShares.load>();
        const uint32_t r8 = (uint32_t)(warp - kFirstLoad) * 4 + ((uint32_t)lane >> 3), piece = (uint32_t)lane & 7u;
        const uint32_t at = smem_base + off_act + r8 * 128u + ((piece ^ (r8 & 7u)) << 4);   // 16 rows on: the same place in the swizzle
        Ring r{0, 0};
        uint32_t issued = 0, parity = 0;
        bool ok = true;
        while (ok && next(x)) {
            const uint32_t act_rows = x.height / 2, slab_bytes = act_rows * 128u;   // act_rows: a multiple of 16
            constexpr int kTurns = LOW ? 2 : 8;
            // Low strips leave out what is behind the last row: the columns of D of those rows are never stored.  (High ones, whose last is not much lower, lose 2 to
            // 4 % to the test.)
            const uint32_t to_copy = !LOW ? act_rows : x.rows > rank * act_rows ? min(act_rows, x.rows - rank * act_rows) : 0u;
            uint32_t src[kTurns];
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {   // rows behind the last one, and those that A does not have: zeros
                const uint32_t r0 = 16u * i + r8, c = rank * act_rows + r0;
                src[i] = r0 < act_rows && c < x.rows ? source_row(p.x, x.row0 + c) : 0xffffffffu;
            }
            for (uint32_t l = 0; l < ns; ++l) {
                if (!warp_wait(step_empty(r.i), r.phase ^ 1u, abort_flag)) { give_up(62, x.expert, l); ok = false; break; }
                const uint32_t to = at + r.i * act_stride;
                const uint16_t* from = p.x.a + l * KS + piece * 8u;
#pragma unroll
                for (int i = 0; i < kTurns; ++i) {
                    if (16u * i >= to_copy) break;
                    const bool there = src[i] < p.x.a_rows;
                    const uint16_t* row = there ? from + (size_t)src[i] * p.x.lda : p.x.a;
#pragma unroll
                    for (int h = 0; h < KS / kSlab; ++h) cp_async16_or_zero(to + h * slab_bytes + i * 2048u, row + (there ? h * kSlab : 0), there ? 16u : 0u);
                }
                cp_async_arrive(step_full(r.i));
                issued |= 1u << r.i; parity = (parity & ~(1u << r.i)) | (r.phase << r.i);
                r.step(1, kSlots);
            }
        }
        cp_async_wait_all();   // never leave with a copy still writing this CTA's shared memory
        for (uint32_t s = 0; s < kSlots; ++s)   // not while a commit of rank 0 may still arrive here
            if (issued & (1u << s)) (void)warp_wait(step_empty(s), (parity >> s) & 1u, abort_flag);
    } else {
        // ======================= epilogue =======================
        ptx::regs_up<kShares.epi>();
        const uint32_t quarter = (uint32_t)warp & 3u, half = (uint32_t)(warp - kFirstEpi) >> 2, ch = quarter * 32 + lane;
        constexpr int kPacks = LOW ? 2 : 8;   // of 16 columns: this warp's half of a strip
        const bool odd = lane & 1, gated = p.x.gated != 0, act = p.x.silu != 0;
        const uint32_t stage = smem_base + kOffOut + (uint32_t)(warp - kFirstEpi) * 2 * kOutBytes;
        uint32_t acc_phase = 0;
        bool ok = true;
        auto drained = [&] {   // everything of the accumulator is in registers
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
#pragma unroll
                for (uint32_t h = 0; h < kIssuers; ++h) {
                    const uint32_t b = acc_empty(h);
                    if (rank == 0) ptx::mbar_arrive(b); else ptx::mbar_arrive_remote(b, 0);
                }
            }
        };
        auto pack2 = [](float lo, float hi) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
            return *reinterpret_cast<const uint32_t*>(&v);
        };
        auto put = [&](uint32_t at, uint32_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((uint16_t)v) : "memory"); };
        while (ok && next(x)) {
            const uint32_t cols = x.height / 2, nn = x.n0 + ch;
            const size_t chan = (size_t)x.expert * p.x.n + (nn < p.x.n ? nn : 0);
            // 16 finished sums of this lane's channel -> packed results.  Gated: the lanes of a pair hold gate (even) and up (odd) of one output
            // channel and exchange half of the 16 rows: the even lane finishes rows 0 to 7, the odd one 8 to 15.
            uint32_t o[kPacks][8];
            float factor[4] = {};   // group scales: what rows lane, lane + 32, ... have to be multiplied by
            auto row_scaled = [&](float v, uint32_t row) { return GROUPED ? v * __shfl_sync(0xffffffffu, factor[row / 32], row) : v; };
            auto finish = [&](uint32_t (&to)[8], const float (&v)[16], int at) {   // at: the first of the 16 rows
                if (gated) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        float f[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float lo = v[j + i], hi = v[j + i + 8], other = __shfl_xor_sync(0xffffffffu, odd ? lo : hi, 1);
                            // the two lanes of a pair have different rows: the factor is fetched from the lane that knows it
                            const float fr = GROUPED ? __shfl_sync(0xffffffffu, factor[at / 32], at % 32 + j + i + (odd ? 8 : 0)) : 1.f;
                            const float gate = (odd ? other : lo) * fr, up = (odd ? hi : other) * fr;
                            f[i] = (act ? silu(gate) : gate) * up;
                        }
                        to[j / 2] = pack2(f[0], f[1]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float lo = row_scaled(v[2 * j], at + 2 * j), hi = row_scaled(v[2 * j + 1], at + 2 * j + 1);
                        to[j] = pack2(act ? silu(lo) : lo, act ? silu(hi) : hi);
                    }
                }
            };
            const uint32_t column = tmem_base + ((quarter * 32u) << 16) + half * cols;
            // Per channel the sum of products times the scale; of group scales the powers of two that channel and row were given.
            const uint32_t first = half * cols, valid = x.rows > first ? min(cols, x.rows - first) : 0u;
            float scale = GROUPED ? 1.f / p.channel_mult[chan]
                                  : p.x.scale_dtype == AFB_SCALE_BF16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p.x.scale)[chan] << 16)
                                                                      : reinterpret_cast<const float*>(p.x.scale)[chan];
            // A sum, up to 2^53, meets the channel's power first: none of the warp's may be above 2^60, what is above goes to the rows' side.
            int above = 0;
            if (GROUPED) {
                above = max((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(scale)) >> 23) - 127 - 60, 0);
                scale *= power_of_two(-above);
            }
            const float unit = power_of_two(9 + above);   // 512: the weights' 2^-9
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t row = i * 32 + lane < valid ? p.x.row_pair ? source_row(p.x, x.row0 + first + i * 32 + lane) : x.row0 + first + i * 32 + lane : 0xffffffffu;
                factor[i] = GROUPED && row < p.x.a_rows ? fminf(p.row_factor[row] * unit, 0x1p127f) : 0.f;
            }
            if (!warp_wait(acc_full(0), acc_phase, abort_flag)) { give_up(68, x.expert, 0); break; }
            if (LOW && !warp_wait(acc_full(1), acc_phase, abort_flag)) { give_up(68, x.expert, 1); break; }
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int i = 0; i < kPacks; ++i) {
                if (16u * i >= cols) break;
                uint32_t a[16];
                float v[16];
                if (LOW) {   // the two issuers' sums
                    uint32_t b[16];
                    ptx::tmem_ld_32x16(column + 16 * i, a);
                    ptx::tmem_ld_32x16(column + acc_cols + 16 * i, b);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) + __uint_as_float(b[j]));
                } else {
                    ptx::tmem_ld_32x16(column + 16 * i, a);
                    ptx::tmem_ld_wait();
                }
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    v[j] = GROUPED ? __uint_as_float(a[j]) * scale : unscaled(__uint_as_float(a[j]), scale);
                finish(o[i], v, 16 * i);
            }
            drained();
            acc_phase ^= 1u;
            // Blocks of 16 rows turn round in shared memory and leave in 16-byte pieces, 64 (gated 32) contiguous bytes a row; two blocks take turns.
            const uint32_t c0 = x.n0 + quarter * 32u;   // first channel of this warp
            if (c0 >= p.x.n) continue;
            uint16_t* c = p.x.c + (size_t)(x.row0 + first) * p.x.ldc;
#pragma unroll
            for (int i = 0; i < kPacks; ++i) {
                if (16u * i >= valid) break;
                if (p.c_vec) {
                    const uint32_t out = stage + (i & 1) * kOutBytes;
                    if (gated) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t at = out + ((odd ? 8u : 0u) + 2 * j) * 32u + ((uint32_t)lane >> 1) * 2u;
                            put(at, o[i][j]); put(at + 32u, o[i][j] >> 16);
                        }
                        __syncwarp();
                        const uint32_t row = 16u * i + lane / 2, col = c0 / 2 + (lane & 1) * 8;
                        uint4 v;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(out + lane * 16u));
                        if (row < valid && col < p.x.n_out) *reinterpret_cast<uint4*>(c + (size_t)row * p.x.ldc + col) = v;   // n_out is a multiple of 8
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t at = out + (uint32_t)j * 128u + (uint32_t)lane * 2u;
                            put(at, o[i][j]); put(at + 64u, o[i][j] >> 16);
                        }
                        __syncwarp();
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const uint32_t piece = h * 32 + lane, row = 16u * i + piece / 4, col = c0 + piece % 4 * 8;
                            uint4 v;
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(out + piece * 16));
                            if (row < valid && col < p.x.n_out) *reinterpret_cast<uint4*>(c + (size_t)row * p.x.ldc + col) = v;
                        }
                    }
                } else if (gated) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t row = 16u * i + (odd ? 8u : 0u) + j;
                        if (row < valid && nn < p.x.n) c[(size_t)row * p.x.ldc + nn / 2] = (uint16_t)(o[i][j / 2] >> (j % 2 * 16));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (16u * i + j < valid && nn < p.x.n) c[(size_t)(16u * i + j) * p.x.ldc + nn] = (uint16_t)(o[i][j / 2] >> (j % 2 * 16));
                }
            }
            __syncwarp();   // the next tile's first block is written after this one's last has been read
        }
    }

    // ---- teardown: every thread gets here, also after an abort; neither CTA leaves while the other may read its shared memory or arrive there ----
    ptx::tc_fence_before_sync();
    __syncwarp();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    if (warp == 2) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

template <int BITS, bool GROUPED, int KS, bool LOW>
int launch_many(const CUtensorMap& tw, const ManyParams& p, uint32_t grid, uint32_t smem, DeviceCtx* ctx, cudaStream_t s) {
    auto kern = expert_many_kernel<BITS, GROUPED, KS, LOW>;
    static DeviceOnce attr_set;  // per template instance
    if (!attr_set.done(ctx->device)) {
        cudaFuncAttributes attr;
        cudaError_t e = cudaFuncGetAttributes(&attr, kern);
        if (e != cudaSuccess) return cuda_fail(e);
        if ((uint32_t)(attr.numRegs * kManyThreads) < regs_all(BITS == 4 && GROUPED)) return AFB_ERR_UNSUPPORTED;   // the shares come out of what the block is launched with
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (e != cudaSuccess) return cuda_fail(e);
        attr_set.mark(ctx->device);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kManyThreads); cfg.stream = s; cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // group scales: after expert_prepare_kernel
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = GROUPED ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw, p);
    count_launch();
    count_expert_many_launch();
    return e == cudaSuccess ? AFB_OK : cuda_fail(e);
}

template <int BITS, bool GROUPED, int KS>
int launch_cfg(const CUtensorMap& tw, const ManyParams& p, uint32_t grid, uint32_t smem, DeviceCtx* ctx, cudaStream_t s) {
    if constexpr (KS == 128)   // k an odd multiple of 64 leaves a raw block that is not whole: no low strips
        if (p.x.tile_rows <= 64) return launch_many<BITS, GROUPED, KS, true>(tw, p, grid, smem, ctx, s);
    return launch_many<BITS, GROUPED, KS, false>(tw, p, grid, smem, ctx, s);
}

}  // namespace

int launch_expert_many(const ExpertParams& q, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s, bool* done) {
    *done = false;
    ManyParams p{};
    p.x = q;
    const uint32_t ks = q.k % 128 == 0 ? 128 : 64, spb = (bits == 8 ? 128 : 256) / ks;
    p.x.set_blocks((q.n + 2 * kCh - 1) / (2 * kCh));
    p.steps = q.k / ks;
    const uint32_t per_block = p.steps % spb == 0 ? spb : 1;
    // Strips of up to 64 rows leave room for six slots and an accumulator for each of two issuers (whole raw blocks only, see below, and a step for each issuer).
    // By the mean of the rows per expert (us, strips up to 64 / up to 256): 64 experts of 2048 x 4096, int4 group-128: 16 rows 114 / 122, 32: 130 / 136, 40: 144 / 140;
    // int8: 16: 103 / 111, 40: 119 / 127, 48: 125 / 123;  39 of 8368 x 2176, int8: 32: 146 / 150, 40: 160 / 156.  (Strips up to 128 with two accumulators of one
    // issuer take more steps: 48 rows, int4: 142; 140: 222 where strips up to 256 take 206.)
    p.x.tile_rows = (uint64_t)q.m <= 36ull * q.experts && per_block == spb && p.steps > 1 ? 64 : 256;
    const bool low = p.x.tile_rows <= 64;
    const uint32_t kSlots = slots(ks, low);
    p.off_raw = (kOffTable + ExpertTable::bytes(q.experts) + 1023u) / 1024u * 1024u;
    const uint32_t act_bytes = kSlots * p.x.tile_rows * ks;
    p.raw_stages = (232448 - 1024 - p.off_raw - act_bytes) / kRawBytes;
    if (p.raw_stages > (uint32_t)kMaxRaw) p.raw_stages = kMaxRaw;
    // The parity waits of the converters: see stream.cu.  With two issuers a free slot tells about every second step only; so of the raw blocks either
    // every one has a step of each issuer, or the ring is of an even number of blocks with a step each, and the block that had its place in the
    // ring before had one of the same issuer's.
    if (low && spb == 1) p.raw_stages &= ~1u;
    p.slot_first = !low && p.raw_stages * per_block >= kConvGroups + kSlots + per_block - 1 ? 0u : 1u;
    if (p.raw_stages * per_block < kSlots + per_block - 1) return AFB_ERR_UNSUPPORTED;   // not with any size that this function takes
    p.c_vec = q.ldc % 8 == 0 && (uintptr_t)q.c % 16 == 0 && q.n_out % 8 == 0;
    p.status = ctx->status;
    const uint64_t tiles = expert_tiles(q.m, q.experts, p.x.tile_rows) * p.x.n_blocks;
    if (tiles >> 31) { *done = true; return AFB_ERR_TOO_LARGE; }
    const uint32_t pairs = (uint32_t)ctx->sm_count / 2, grid = 2 * (tiles < pairs ? (uint32_t)tiles : pairs);
    const uint32_t smem = 1024 + p.off_raw + p.raw_stages * kRawBytes + act_bytes;
    CUtensorMap tw;
    const int rc = tmap_2d(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, q.b, (uint64_t)q.k * bits / 8, (uint64_t)q.experts * q.n, q.ldb_bytes, 128, kCh, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) { *done = true; return rc; }
    if (!group) {
        *done = true;
        if (bits == 4) return launch_cfg<4, false, 128>(tw, p, grid, smem, ctx, s);   // k is a multiple of 128
        return ks == 128 ? launch_cfg<8, false, 128>(tw, p, grid, smem, ctx, s) : launch_cfg<8, false, 64>(tw, p, grid, smem, ctx, s);
    }
    // rows of A, their factors, the channels' multipliers, each from a multiple of 256 bytes on
    const uint64_t a_bytes = ((uint64_t)q.a_rows * q.k * 2 + 255) / 256 * 256, row_bytes = ((uint64_t)q.a_rows * 4 + 255) / 256 * 256;
    const uint64_t channels = (uint64_t)q.experts * q.n;
    const CallMemory memory(ctx, s, a_bytes + row_bytes + channels * 4);   // given back behind the second launch
    if (!memory.get()) return AFB_OK;
    *done = true;
    PrepareParams prep{};
    prep.x = q;
    prep.a = reinterpret_cast<uint16_t*>(memory.get());
    prep.row_factor = reinterpret_cast<float*>(reinterpret_cast<char*>(memory.get()) + a_bytes);
    prep.channel_mult = reinterpret_cast<float*>(reinterpret_cast<char*>(memory.get()) + a_bytes + row_bytes);
    prep.channel_blocks = (uint32_t)((channels + kPrepareThreads - 1) / kPrepareThreads);
    for (prep.row_threads = 32; prep.row_threads < (uint32_t)kPrepareThreads && prep.row_threads * kHeld * 8 < q.k;) prep.row_threads *= 2;
    const uint32_t rows = kPrepareThreads / prep.row_threads;
    expert_prepare_kernel<<<prep.channel_blocks + (q.a_rows + rows - 1) / rows, kPrepareThreads, 0, s>>>(prep);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e);
    p.x.a = prep.a; p.x.lda = q.k;
    p.row_factor = prep.row_factor; p.channel_mult = prep.channel_mult;
    if (bits == 4) return launch_cfg<4, true, 128>(tw, p, grid, smem, ctx, s);
    return ks == 128 ? launch_cfg<8, true, 128>(tw, p, grid, smem, ctx, s) : launch_cfg<8, true, 64>(tw, p, grid, smem, ctx, s);
}

}  // namespace afb

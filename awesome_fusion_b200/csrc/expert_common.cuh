// Shared by the two forms of the products grouped by expert (expert_few.cu, expert_many.cu): the parameter block and the table by which a CTA
// finds its tiles.  How many rows an expert has is known on the GPU only.
#pragma once
#include "afb_internal.h"

namespace afb {

struct ExpertParams {
    uint16_t* c;
    const uint16_t* a;
    const uint8_t* b;
    const void* scale;
    const uint8_t* zero;
    const int32_t* offsets;
    const int32_t* row_pair;   // nullptr: the rows of A as they lie
    uint32_t m, n, n_out, k, lda, ldc;
    size_t ldb_bytes;
    uint32_t experts, top_k, a_rows;
    uint32_t enc, scale_dtype, packed, group_shift;
    uint32_t gated, silu;
    uint32_t tile_rows;        // rows of a tile, at most
    uint32_t n_blocks;         // channel blocks
    uint32_t blocks_mul, blocks_shift;   // t / n_blocks = t * blocks_mul >> blocks_shift for t < 2^31
    // mul = 2^shift / n rounded up is too large by less than n <= 2^(shift - 31) of 2^shift, which t < 2^31 cannot carry over the next multiple of n.
    void set_blocks(uint32_t n) {
        n_blocks = n;
        for (blocks_shift = 31; n > 1u << (blocks_shift - 31); ++blocks_shift) {}
        blocks_mul = (uint32_t)(((1ull << blocks_shift) + n - 1) / n);
    }
};

// Tiles of at most `rows` rows that m rows of `experts` experts can make.
inline uint64_t expert_tiles(uint32_t m, uint32_t experts, uint32_t rows) {
    const uint32_t active = m < experts ? m : experts;   // each expert with a row adds at most one tile that is not full
    return active + (uint64_t)(m - active) / rows;
}

__device__ __forceinline__ uint32_t clamp_offset(int32_t o, uint32_t m) { return (uint32_t)min(max(o, 0), (int32_t)m); }

// One tile: rows [row0, row0 + rows) of an expert, at most `height` of them, x channel block `block`.
struct ExpertStrip { uint32_t expert, row0, rows, height, block; };

// Where each expert's rows and strips (its rows cut into as few as fit tile_rows, of equal height but for the last) begin, in shared memory.
struct ExpertTable {
    uint32_t *strips_before, *first_row, *row_count;   // [experts + 1], [experts], [experts]
    uint32_t experts;
    __host__ __device__ static uint32_t bytes(uint32_t experts) { return (3 * experts + 1) * (uint32_t)sizeof(uint32_t); }
    __device__ __forceinline__ ExpertTable(void* at, uint32_t n)
        : strips_before(reinterpret_cast<uint32_t*>(at)), first_row(strips_before + n + 1), row_count(first_row + n), experts(n) {}
    __device__ __forceinline__ uint32_t strips() const { return strips_before[experts]; }
    // By one warp, before a barrier of all.
    __device__ __forceinline__ void build(const ExpertParams& p, uint32_t lane) const {
        uint32_t before = 0;
        for (uint32_t e0 = 0; e0 < experts; e0 += 32) {
            const uint32_t e = e0 + lane;
            uint32_t lo = 0, hi = 0;
            if (e < experts) {
                lo = clamp_offset(__ldg(p.offsets + e), p.m);
                hi = max(lo, clamp_offset(__ldg(p.offsets + e + 1), p.m));
            }
            const uint32_t mine = (hi - lo + p.tile_rows - 1) / p.tile_rows;
            uint32_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += y;
            }
            if (e < experts) { strips_before[e] = before + upto - mine; first_row[e] = lo; row_count[e] = hi - lo; }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) strips_before[experts] = before;
    }
    // Tile t of strips() * n_blocks: inside an expert the channel blocks advance, strip fastest, so that its weights come from HBM once.
    // Heights are rounded up to a multiple of UNIT.  By a whole warp.  Every warp of a CTA asks for every tile: a binary search to the end and five divisions were 3 % of
    // the instructions of 1024 rows on 64 experts (form for few rows, 16384 rows: 1299 us, without them 1264).
    template <uint32_t UNIT>
    __device__ __forceinline__ void tile(const ExpertParams& p, uint32_t t, ExpertStrip& s) const {
        const uint32_t q = (uint32_t)((uint64_t)t * p.blocks_mul >> p.blocks_shift);
        uint32_t lo = 0, hi = experts;   // the expert with strips_before[e] <= q < strips_before[e + 1]
        while (hi - lo > 32) {
            const uint32_t mid = (lo + hi) / 2;
            if (strips_before[mid] <= q) lo = mid; else hi = mid;
        }
        const uint32_t e = lo + (threadIdx.x & 31u);
        lo += __popc(__ballot_sync(0xffffffffu, e < hi && strips_before[e] <= q)) - 1;   // they do not fall
        const uint32_t first = strips_before[lo], of = strips_before[lo + 1] - first, all = row_count[lo];
        s.expert = lo;
        s.block = t - first * p.n_blocks;
        s.height = all;
        uint32_t i = 0;
        if (of > 1) {
            const uint32_t r = s.block;
            s.block = r / of;
            i = r - s.block * of;
            s.height = (all + of - 1) / of;
        }
        s.height = (s.height + UNIT - 1) / UNIT * UNIT;
        s.row0 = first_row[lo] + i * s.height;
        s.rows = i * s.height < all ? min(s.height, all - i * s.height) : 0u;
    }
};

// `bytes` (0 or 16) from src, zeros behind them.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Of this thread, also those that no group was committed for.
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Arrives on `bar` when this thread's copies so far are complete.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Row of A behind row r of C; a value outside [0, a_rows): none, reads as zeros.
__device__ __forceinline__ uint32_t source_row(const ExpertParams& p, uint32_t r) {
    if (!p.row_pair) return r;
    const int32_t pair = __ldg(p.row_pair + r);
    return pair < 0 ? 0xffffffffu : (uint32_t)pair / p.top_k;
}

// v / (1 + exp(-v)) for a result that is rounded to bf16, as v * (2^-16 / (2^-16 + 2^(-v log2(e) - 16))): the factor keeps the sum below 2^126, from where on rcp
// returns 0, down to v = -98.4; the result is below half of the smallest bf16 there (without the factor it is lost from -87.3 on, -1e-36).  The argument is rounded
// once, so the exponential is off by 2^-17 at most (2^-20 for |v| < 11), a 200th of the rounding to come; below v = -87.3, where the quotient leaves the normal range,
// it loses bits towards 2^-149, as the result does towards 2^-133.  Infinite exponentials give -0, v = -infinity NaN, as the quotient would.
// (sigmoid() of pair.cu has more than twice the instructions: the drain of an accumulator of 256 gated columns waits for them.)
__device__ __forceinline__ float silu(float v) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(v, -1.44269504f, -16.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0x1p-16f + e));
    return v * (r * 0x1p-16f);
}

// `bits`, `group`: of the weights.  For group scales the form for many rows needs a workspace; *done = false: there is none to be had, and nothing has
// happened.
int launch_expert_many(const ExpertParams& p, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s, bool* done);
int launch_expert_few(const ExpertParams& p, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s);

}  // namespace afb

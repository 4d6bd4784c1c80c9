// Shared by the two forms of the products grouped by expert (expert_few.cu, expert_many.cu): the parameter block and the way a CTA finds its
// tile.  How many rows an expert has is known on the GPU only; the launch covers the most tiles there can be, the rest find nothing to do.
#pragma once
#include "activation.cuh"
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
};

// Tiles of at most `rows` rows that m rows of `experts` experts can make.
inline uint64_t expert_tiles(uint32_t m, uint32_t experts, uint32_t rows) {
    const uint32_t active = m < experts ? m : experts;   // each expert with a row adds at most one tile that is not full
    return active + (uint64_t)(m - active) / rows;
}

struct ExpertTile { uint32_t expert, row0, rows, tiles_before; };

__device__ __forceinline__ uint32_t clamp_offset(int32_t o, uint32_t m) { return (uint32_t)min(max(o, 0), (int32_t)m); }

// Tile number `slot` in the order of the experts, by a whole warp; false: there are fewer.  An expert's rows are cut into as few tiles as
// fit, of equal height but for the last; `unit` rounds the height up.
__device__ __forceinline__ bool find_tile(const ExpertParams& p, uint32_t slot, uint32_t unit, uint32_t lane, ExpertTile& x) {
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 32) {
        const uint32_t e = e0 + lane;
        uint32_t lo = 0, hi = 0;
        if (e < p.experts) {
            lo = clamp_offset(__ldg(p.offsets + e), p.m);
            hi = max(lo, clamp_offset(__ldg(p.offsets + e + 1), p.m));
        }
        const uint32_t rows = hi - lo, tiles = (rows + p.tile_rows - 1) / p.tile_rows;
        uint32_t upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += y;
        }
        const uint32_t found = __ballot_sync(0xffffffffu, slot < before + upto);
        if (found) {
            const int at = __ffs(found) - 1;
            const uint32_t nt = __shfl_sync(0xffffffffu, tiles, at), all = __shfl_sync(0xffffffffu, rows, at);
            const uint32_t first = before + __shfl_sync(0xffffffffu, upto, at) - nt, i = slot - first;
            const uint32_t height = ((all + nt - 1) / nt + unit - 1) / unit * unit;
            x.expert = e0 + at;
            x.row0 = __shfl_sync(0xffffffffu, lo, at) + i * height;
            x.rows = i * height < all ? min(height, all - i * height) : 0u;
            x.tiles_before = first;
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// Row of A behind row r of C; a value outside [0, a_rows): none, reads as zeros.
__device__ __forceinline__ uint32_t source_row(const ExpertParams& p, uint32_t r) {
    if (!p.row_pair) return r;
    const int32_t pair = __ldg(p.row_pair + r);
    return pair < 0 ? 0xffffffffu : (uint32_t)pair / p.top_k;
}

__device__ __forceinline__ float silu(float v) { return v * sigmoid(v); }

// `bits`, `group`: of the weights.  The form for many rows takes no empty A (a tensor map has at least one row).
int launch_expert_many(const ExpertParams& p, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s);
int launch_expert_few(const ExpertParams& p, uint32_t bits, uint32_t group, DeviceCtx* ctx, cudaStream_t s);

}  // namespace afb

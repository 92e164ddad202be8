// Where attn_tile and attn_own (attn_shared.hip) leave the parts of a row, for the merge that
// joins them: whole numbers only, so that it also runs, and is tested, on the host.
#pragma once
#include <hip/hip_runtime.h>

namespace sc {

// units of up to 64 columns of a sequence's n rows, and its blocks of 2^shift keys
__host__ __device__ __forceinline__ int own_coltiles(int n, int G) { return (n * G + 63) >> 6; }
__host__ __device__ __forceinline__ int own_keyblocks(int len, int shift = 6) {
    return (int)(((unsigned)len + (1u << shift) - 1) >> shift);
}
// blocks a workgroup takes of `total`
__host__ __device__ __forceinline__ int own_run(int total, int wgs) {
    return total > 0 ? (total - 1) / wgs + 1 : 1;
}

// Of part_rows rows' parts, attn_tile's of row `row`, the i-th of sequence r (-1: of none): the
// row's number, or, where they are kept by sequence (per_seq > 0 each), the sequence's i-th.
// part_rows: it has no part.
__host__ __device__ __forceinline__ int tile_part_row(int row, int r, int i, int per_seq, int part_rows) {
    if (per_seq == 0) return row;
    return r < 0 || i >= per_seq ? part_rows : r * per_seq + i;
}

struct OwnParts {
    int first, n, step, col;     // parts first, first + step, ..: n of them, and the column in each
};

// The parts of row `row`, q head gq of kv head hk, in a sequence of rows [first, first + n) and
// len keys whose first block is off and first unit is unit: of the workgroups that have
// blocks of the row's unit, the four waves' or (a wide unit) that of the wave whose column
// it is.  total: blocks of all sequences.  A row outside the sequence (row starts that begin
// above 0 or do not ascend) has none, nor has one whose parts would not all be there.
// shift: log2 of a block's keys; before: blocks that come before the sequence's own; rest:
// places in the line, after each unit's blocks, that hold no keys.
__host__ __device__ __forceinline__ OwnParts own_parts_of(int row, int first, int n, int len, int hk, int gq, int G,
                                                          int small_rows, int off, int unit, int total, int own_wgs,
                                                          int own_parts, int part_cols, int shift = 6,
                                                          int before = 0, int rest = 0) {
    OwnParts p = {0, 0, 1, 0};
    const int kt = before + (len > 0 ? own_keyblocks(len, shift) : 0);
    if (row < first || row >= first + n || n > small_rows || kt <= 0) return p;
    const int run = own_run(total, own_wgs), ct = own_coltiles(n, G);
    const int col = (row - first) * G + gq, u = hk * ct + (col >> 6);
    const int t0 = off + u * (kt + rest), w0 = t0 / run, wgs = (t0 + kt - 1) / run - w0 + 1;
    const bool wide = n * G > 16;
    p.first = 4 * (unit + u + w0) + (wide ? (col >> 4) & 3 : 0);
    p.step = wide ? 4 : 1;
    p.col = col & 15;
    p.n = wide ? wgs : 4 * wgs;
    if (p.first < 0 || p.first + p.step * (p.n - 1) >= own_parts || p.col >= part_cols) p.n = 0;
    return p;
}

}  // namespace sc

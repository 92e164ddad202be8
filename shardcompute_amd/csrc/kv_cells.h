// How a quantized key/value cache lies in memory: codes of 4 or 8 bits in groups of 64 dims,
// a scale and a bias (bf16) each, value = scale code + bias (the affine rule of the weights).
//
// A pool is [n_blocks, Hkv, bs / 16] cells; a cell is 16 consecutive positions of one kv
// head, keys and values, one run of bytes that a wave reads whole lines of:
//   keys' codes    lane (g, r) of 64 = 16 g + r: position r, dims 16 g .. 16 g + 15 of each group
//   values' codes  lane (g, l): positions 4 g .. 4 g + 3, dims l, 16 + l, 32 + l, ..
//   meta           [keys' groups, values' groups][16 positions]: scale | bias << 16
// A lane's codes are what it feeds as operand A of v_mfma_f32_16x16x32_bf16: keys as rows
// of S^T = K Q^T, whose result then lies as operand B of O^T += V^T P^T wants it, the 4 positions
// 4 g .. 4 g + 3 of a cell in lane row g.  A lane's bytes are one 16-byte load (8 with 4 bits
// and 64 dims; two planes of 1 KB with 8 bits and 128).
// Codes of 4 bits: of 8 dims of a key in a word, dim e is nibble (e >> 1) + 4 (e & 1), so that
// nib_pair(w, 4 i) is (e = 2 i, 2 i + 1).  Of a value's word byte i is position 4 g + i, its low
// nibble dim 32 m + l, its high one 32 m + 16 + l: positions of different rows are different
// bytes, written without reading what is there.
#pragma once
#include "sc_common.h"

namespace sc {

template <int D, int BITS>
struct Cell {
    static constexpr int GROUPS = D / 64;
    static constexpr int LANE = D * BITS / 32;              // bytes of codes a lane holds, keys' (and values')
    static constexpr int PLANE = LANE < 16 ? LANE : 16;     // bytes of one load
    static constexpr int PLANES = LANE / PLANE;
    static constexpr int CODES = 64 * LANE;
    static constexpr int ITEMS = 2 * GROUPS;                // meta words a position
    static constexpr int BYTES = 2 * CODES + 16 * ITEMS * 4;
    static constexpr int CHUNK = 8 * BITS / 8;              // bytes of 8 dims of a key

    // byte of the 8 dims 8 o .. 8 o + 7 of position t's key
    static __host__ __device__ constexpr int key_chunk(int t, int o) {
        const int grp = o >> 3, g = (o >> 1) & 3;
        return BITS == 4 ? (16 * g + t) * LANE + 8 * grp + 4 * (o & 1)
                         : 1024 * grp + (16 * g + t) * 16 + 8 * (o & 1);
    }
    // byte of dim d of position t's value (4 bits: its nibble d >> 4 & 1)
    static __host__ __device__ constexpr int value_byte(int t, int d) {
        const int lane = 16 * (t >> 2) + (d & 15), tile = d >> 4;
        return CODES + (BITS == 4 ? lane * LANE + 4 * (tile >> 1) : 1024 * (tile >> 2) + lane * 16 + 4 * (tile & 3)) + (t & 3);
    }
    // byte of a meta word: item grp of the keys, GROUPS + grp of the values
    static __host__ __device__ constexpr int meta(int t, int item) { return 2 * CODES + (item * 16 + t) * 4; }
};

// bytes of a cell, 0 for a head_dim or a number of bits that there is none for
inline long kv_cell_bytes(long D, int bits) {
    if (D == 128) return bits == 4 ? Cell<128, 4>::BYTES : bits == 8 ? Cell<128, 8>::BYTES : 0;
    if (D == 64) return bits == 4 ? Cell<64, 4>::BYTES : bits == 8 ? Cell<64, 8>::BYTES : 0;
    return 0;
}

}  // namespace sc

// What attention over a key/value cache in blocks does alike whether the cache is held in
// bf16 (attn_shared.hip) or in codes (attn_quant.hip): the column tiles (attn_tile, which takes
// key blocks from a ring in LDS however they came there), the merge of a row's parts, and
// where those lie in the workspace.
#pragma once
#include "sc_common.h"
#include "dma_util.h"
#include "attn_shared_parts.h"

#include <math.h>
#include <type_traits>

namespace sc {

int block_shift(long bs);       // blocks.hip

namespace {

using f4 = dma::f4;

constexpr int SA_KB = 64, SA_THREADS = 256;
constexpr int SA_AHEAD = 4;                              // operand reads in flight ahead of the MFMAs
constexpr int SA_MAX_SEQ = 2048;         // attn_own keeps two numbers of each in LDS, attn_line (attn_quant.hip) four
constexpr int SA_CU_LDS = 160 * 1024;    // of a CU

// What the kernels over a cache of either kind share; a kernel's own arguments are derived from
// it and say where keys and values lie.
struct SaArgs {
    const uint16_t *q;
    long q_stride;
    uint16_t *out;
    long out_stride;
    const int32_t *row_starts, *lengths, *tables, *prefix_table, *prefix_len;
    int N, R, H, Hkv, G, width, shift, n_blocks, prefix_width;
    int small_rows;          // a sequence of at most this many rows is attn_own's
    int any_big;             // some sequence may have more
    int nsplit;              // workgroups a column tile's keys are cut into
    int tile_wgs, own_wgs;   // their workgroups
    int part_rows, per_seq;  // attn_tile's parts: by row, or (per_seq > 0) by sequence, per_seq rows each
    int tiles, pair_half;    // attn_tile's column tiles; > 0: workgroups of a round, paired with the next round's
    float scale_log2;
    // parts: of attn_tile [nsplit][part_rows * H], of attn_own [own_parts][part_cols] columns
    float *tile_o;
    float2 *tile_ml;
    float *own_o;
    float2 *own_ml;
    int own_parts, part_cols;
    int own_shift, join;     // log2 of the keys of an own block; join: the prefix's come before a sequence's own
    int own_rest;            // own_unit[R] is the number of places after each unit's blocks that hold no keys, else there are none
    int32_t *own_off, *own_unit;         // [R + 1]: a sequence's first block (and all of them), its first unit
    int32_t *cut;            // null, or nsplit and own_wgs as the kernel has chosen them
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// rows of the batch that are there
__device__ __forceinline__ int live_rows(const SaArgs &a) { return clampi(a.row_starts[a.R], 0, a.N); }

struct Seq {
    int first, n, len;       // first row, rows, keys (its rows' own included)
};
__device__ __forceinline__ Seq seq_of(const SaArgs &a, int r, int rows) {
    Seq s;
    s.first = clampi(a.row_starts[r], 0, rows);
    s.n = max(clampi(a.row_starts[r + 1], 0, rows) - s.first, 0);
    s.len = clampi(a.lengths[r], 0, a.width << a.shift);
    return s;
}
__device__ __forceinline__ int prefix_keys(const SaArgs &a) {
    return a.prefix_width ? clampi(a.prefix_len[0], 0, a.prefix_width << a.shift) : 0;
}

// the sequence a row belongs to: the last r with row_starts[r] <= row, the 64 lanes
// looking at 64 candidates a step
__device__ __forceinline__ int find_seq(const SaArgs &a, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.R;
    while (n > 1) {
        const int step = (n + 63) >> 6, i = lo + lane * step;
        const bool le = lane * step < n && a.row_starts[i] <= row;
        const int c = max(__popcll(__ballot(le)), 1);
        const int cut = (c - 1) * step;
        lo += cut;
        n = min(step, n - cut);
    }
    return lo;
}

// ---------------------------------------------------------------- column tiles

template <int D>
struct SaGeo {
    static constexpr int KROW = D * 2;
    static constexpr int KTILE = SA_KB * KROW, VTILE = D * SA_KB * 2;
    static constexpr int STAGE = KTILE + VTILE;
    static constexpr int LDS = 2 * STAGE;
    static constexpr int KSTEPS = D / 16;
    static constexpr int DB = D / 32;
    static constexpr int DMA = KTILE / 1024 / 4;         // K (and Vt) copies of a wave, a key block
    // the growth of a column's maximum (log2) that moves it, as in the dense kernel
    static constexpr float LAZY = D == 64 ? 0.f : 8.f;
};

__device__ __forceinline__ int sa_swap23(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }
template <int D>
__device__ __forceinline__ uint32_t sa_kswz(int r, int c) {
    const int p = D == 128 ? c ^ (sa_swap23(r) & 15) : c ^ ((r >> 1) & 7);
    return (uint32_t)(r * (D * 2) + (p << 4));
}
__device__ __forceinline__ uint32_t sa_vswz(int d, int c) { return (uint32_t)(d * 128 + ((c ^ ((d >> 1) & 7)) << 4)); }

// bits 15 and 31 are set if the pair's low or high bf16 is inf or NaN (its exponent is all ones)
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t x) { return (x & 0x7F807F80u) + 0x00800080u; }
__device__ __forceinline__ uint32_t nonfinite_bits(uint4 v) {
    return nonfinite_bits(v.x) | nonfinite_bits(v.y) | nonfinite_bits(v.z) | nonfinite_bits(v.w);
}
// of the wave's lanes, some one's bits are set (a scalar)
__device__ __forceinline__ bool any_nonfinite(uint32_t bits) {
    return __builtin_amdgcn_readfirstlane((int)(__ballot((bits & 0x80008000u) != 0u) != 0ull)) != 0;
}

// word masks of 8 consecutive keys k0 .. k0 + 7, of which those below end are kept
__device__ __forceinline__ uint4 keep_below(int k0, int end) {
    uint4 m;
    m.x = (k0 + 0 < end ? 0xFFFFu : 0u) | (k0 + 1 < end ? 0xFFFF0000u : 0u);
    m.y = (k0 + 2 < end ? 0xFFFFu : 0u) | (k0 + 3 < end ? 0xFFFF0000u : 0u);
    m.z = (k0 + 4 < end ? 0xFFFFu : 0u) | (k0 + 5 < end ? 0xFFFF0000u : 0u);
    m.w = (k0 + 6 < end ? 0xFFFFu : 0u) | (k0 + 7 < end ? 0xFFFF0000u : 0u);
    return m;
}
// non-finite values replaced by 0
__device__ __forceinline__ uint32_t finite2(uint32_t x) {
    return ((x & 0x7F80u) == 0x7F80u ? 0u : x & 0xFFFFu) | ((x & 0x7F800000u) == 0x7F800000u ? 0u : x & 0xFFFF0000u);
}
__device__ __forceinline__ uint4 finite8(uint4 v) {
    return make_uint4(finite2(v.x), finite2(v.y), finite2(v.z), finite2(v.w));
}
__device__ __forceinline__ uint4 and4(uint4 v, uint4 m) { return make_uint4(v.x & m.x, v.y & m.y, v.z & m.z, v.w & m.w); }

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t cvt_pk_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{a, b}, half2_t));
}
__device__ __forceinline__ uint32_t word_of(bf16x8_t v, int e) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u4, v)[e];
}
__device__ __forceinline__ half8_t as_half8(bf16x8_t v) { return __builtin_bit_cast(half8_t, v); }
__device__ __forceinline__ f32x16_t mfma32x32x16_f16(bf16x8_t a, bf16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(as_half8(a), as_half8(b), c, 0, 0, 0);
}

// Where a stager has HALF, the values are rounded to 11 bits in place of 8: a key block comes as
// fp16, times 2^HALF_UP, where its range holds all of it (fits), 0 in the place of keys that are
// not there, else as bf16.  q then is kept as fp16: a column whose largest |q| is outside
// [2^-8, 2^15) is scaled by a power of two, so that what fp16 drops of q is 2^-17 of that at
// most.  P is 2^HALF_P times the probability, which may exceed 1 by 2^LAZY: at most 2^15, and
// a weight below 2^-32 of the largest is dropped.
constexpr int HALF_UP = 5, HALF_P = 7;
constexpr float pow2(int n) { return n >= 0 ? (float)(1 << n) : 1.f / (float)(1 << -n); }

// q as the bf16 blocks' scores take it, which are scaled by 2^-HALF_UP as the others
__device__ __forceinline__ bf16x8_t q_bf16(bf16x8_t v) {
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t w = word_of(v, e);
        asm volatile("" : "+v"(w));                      // opaque: not kept beside q over the loop
        const half2_t x = __builtin_bit_cast(half2_t, w);
        y[e] = cvt_pk_bf16((float)x[0] * pow2(HALF_UP), (float)x[1] * pow2(HALF_UP));
    }
    return as_bf16x8(y[0], y[1], y[2], y[3]);
}

// S: how the key blocks come into the ring (Args, COLS, HALF, Flow; open: the first, next: the one
// after blk, landed: what was begun is there.  HALF: looks_of and fits say whether the one in a
// stage fits, if not, again brings it as bf16).
template <int D, class S>
__device__ __forceinline__ void attn_tile(const typename S::Args &a, int id, uint8_t *smem) {
    using Gm = SaGeo<D>;
    constexpr int COLS = S::COLS;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    // later column tiles (of prompts: more keys) are dispatched first, the first two rounds,
    // resident together, in heavy and light pairs (an order only: results do not depend on it)
    if (a.pair_half > 0 && id < 2 * a.pair_half && id >= a.pair_half) id = 3 * a.pair_half - 1 - id;
    const int hk = id % a.Hkv;
    id /= a.Hkv;
    const int split = id % a.nsplit, tile = a.tiles - 1 - id / a.nsplit;
    const int rows = live_rows(a);
    const int col = tile * COLS + 32 * w + li;
    const int row = col / a.G, h = hk * a.G + col - row * a.G;
    const int row0 = tile * COLS / a.G, row1 = min((tile * COLS + COLS - 1) / a.G, rows - 1);
    if (row0 >= rows) return;
    const bool col_ok = row < rows;
    const int P = prefix_keys(a);

    // the column tile's keys: the prefix, then the own keys of its sequences with many
    // rows; this workgroup takes key blocks [t0, t1) of them
    auto own_blocks = [&](const Seq &s) {
        if (s.n <= a.small_rows) return 0;
        return (clampi(s.len - s.n + row1 - s.first + 1, 0, s.len) + SA_KB - 1) / SA_KB;
    };
    const int r0 = a.any_big ? find_seq(a, row0) : 0;
    int total = (P + SA_KB - 1) / SA_KB;
    bool big = false;                                   // this column's own keys are taken here
    int part_row = tile_part_row(row, -1, 0, a.per_seq, a.part_rows);      // where its part goes, if it has one
    if (a.any_big)
        for (int r = r0; r < a.R; ++r) {
            const Seq s = seq_of(a, r, rows);
            if (s.first > row1) break;
            if (row >= s.first && row < s.first + s.n) {
                big = s.n > a.small_rows;
                part_row = tile_part_row(row, r, row - s.first, a.per_seq, a.part_rows);
            }
            total += own_blocks(s);
        }
    const int t0 = (int)((long)total * split / a.nsplit), t1 = (int)((long)total * (split + 1) / a.nsplit);

    bf16x8_t qv[Gm::KSTEPS];
#pragma unroll
    for (int ks = 0; ks < Gm::KSTEPS; ++ks) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (col_ok) v = *reinterpret_cast<const uint4 *>(a.q + (size_t)row * a.q_stride + (size_t)h * D + 16 * ks + 8 * lh);
        qv[ks] = as_bf16x8(v);
    }
    float sc = a.scale_log2;
    if constexpr (S::HALF) {
        uint32_t top = 0;                                // the largest |q|
#pragma unroll
        for (int ks = 0; ks < Gm::KSTEPS; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = word_of(qv[ks], e);
                top = max(top, max(x << 16 & 0x7FFFFFFFu, x & 0x7FFF0000u));
            }
        top = max(top, (uint32_t)__shfl_xor((int)top, 32)) >> 23;
        // (its exponent, biased; a q that is no number keeps it)
        const bool keep = (top >= 127 - 8 && top < 127 + 15) || top == 255;
        const uint32_t up = keep ? 127u : 254u - clampi((int)top, 16, 240);
        const float by = __uint_as_float(up << 23);
#pragma unroll
        for (int ks = 0; ks < Gm::KSTEPS; ++ks) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = word_of(qv[ks], e);
                y[e] = cvt_pk_f16(__uint_as_float(x << 16) * by, __uint_as_float(x & 0xFFFF0000u) * by);
            }
            qv[ks] = as_bf16x8(y[0], y[1], y[2], y[3]);
        }
        sc = fmaxf(sc * __uint_as_float((254u - up) << 23) * pow2(-HALF_UP), 1e-37f);
    }
    f32x16_t o[Gm::DB];
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db) o[db] = f32x16_t{};
    float m = -INFINITY, lsum = 0.f;
    const int arow = sa_swap23(li);
    const uint32_t kat0 = sa_kswz<D>(arow, lh), vat0 = sa_vswz(li, lh);
    const S stager(a, smem, lane, w);

    // key blocks [b0, b1) of one table with `end` keys; the column sees keys <= limit
    auto segment = [&](const int32_t *table, int width, int end, int b0, int b1, int limit) {
        if (b0 >= b1) return;
        // of the wave's columns: the fewest and the most keys one of them sees
        int lo = limit, hi = limit;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            lo = min(lo, __shfl_xor(lo, x));
            hi = max(hi, __shfl_xor(hi, x));
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        typename S::Flow flow;
        // the stage is a compile-time constant in the copies without a mask, so that every
        // operand read is a loop-invariant lane offset plus an immediate
        auto block = [&](int blk, auto mask_tag, auto stage) {
            constexpr bool MASK = decltype(mask_tag)::value;
            constexpr bool F16 = S::HALF && !MASK;
            const int st = stage;
            const int kb = blk * SA_KB;
            const uint8_t *K = smem + (S::HALF ? 0 : st * Gm::STAGE);        // (of HALF in kplace and vplace)
            const uint8_t *V = K + Gm::KTILE;
            // operands' places: of HALF, whose registers are scarcer, from two offsets by one more
            // instruction each (opaque, else all are kept over the loop)
            uint32_t kat = kat0 + st * Gm::STAGE, vat = vat0 + st * Gm::STAGE;
            if constexpr (S::HALF) asm volatile("" : "+v"(kat), "+v"(vat));
            auto kplace = [&](int kh, int ks) {
                if constexpr (S::HALF) return (kat ^ (uint32_t)(ks << 5)) + 32 * kh * Gm::KROW;
                else return sa_kswz<D>(32 * kh + arow, 2 * ks + lh);
            };
            auto vplace = [&](int db, int s4) {
                if constexpr (S::HALF) return (vat ^ (uint32_t)(s4 << 5)) + 32 * 128 * db;
                else return sa_vswz(32 * db + li, 2 * s4 + lh);
            };
            if constexpr (!S::HALF)
                if (blk + 1 < b1) stager.next(flow, hk, table, width, blk, st);
            if ((!MASK && !F16) || kb <= hi) {           // else: nothing of it is seen by the wave
                f32x16_t sacc[2] = {f32x16_t{}, f32x16_t{}};
                // operand reads SA_AHEAD ahead of their MFMAs (the scheduler, left alone,
                // issues each read just before its MFMA)
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < Gm::KSTEPS; ++ks)
#pragma unroll
                    for (int kh = 0; kh < 2; ++kh) {
                        const bf16x8_t ka = as_bf16x8(*reinterpret_cast<const uint4 *>(K + kplace(kh, ks)));
                        if constexpr (F16) sacc[kh] = mfma32x32x16_f16(ka, qv[ks], sacc[kh]);
                        else sacc[kh] = mfma32x32x16(ka, S::HALF ? q_bf16(qv[ks]) : qv[ks], sacc[kh]);
                    }
                __builtin_amdgcn_sched_group_barrier(0x100, SA_AHEAD, 0);
#pragma unroll
                for (int i = 0; i < 2 * Gm::KSTEPS - SA_AHEAD; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, SA_AHEAD, 0);
                __builtin_amdgcn_sched_barrier(0);
                if (MASK || (F16 && kb + SA_KB - 1 > lo)) {
                    const int rel = limit - kb - 8 * lh;
#pragma unroll
                    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (32 * kh + 16 * (r >> 3) + (r & 7) > rel) sacc[kh][r] = -INFINITY;
                }
                float bm = -INFINITY;
#pragma unroll
                for (int kh = 0; kh < 2; ++kh)
#pragma unroll
                    for (int r = 0; r < 16; ++r) bm = fmaxf(bm, sacc[kh][r]);
                bm = fmaxf(bm, __shfl_xor(bm, 32));
                float alpha = 1.f;
                if ((bm - m) * sc > Gm::LAZY) {
                    alpha = __builtin_amdgcn_exp2f((m - bm) * sc);
                    m = bm;
                }
                // (a column that has seen no key yet has m = -inf: probabilities 0, not NaN)
                const float nms = (m == -INFINITY ? 0.f : -m * sc) + (S::HALF ? HALF_P : 0);
                float ps = 0.f;
#pragma unroll
                for (int kh = 0; kh < 2; ++kh)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(sacc[kh][r], sc, nms));
                        sacc[kh][r] = p;
                        ps += p;
                    }
                lsum = lsum * alpha + ps;
                if (__ballot(alpha != 1.f) != 0ull) {
#pragma unroll
                    for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
                }
                // keys at or past `end` may hold anything: their V is dropped.  Keys that only
                // some of the columns see (a later row's, another sequence's) meet zero
                // probabilities, which an inf or NaN among their values would turn into NaN
                // for every column: such values are dropped here and added afterwards to the
                // columns that see them
                bool bad = false;
                if (MASK) {
                    uint32_t bits = 0;
#pragma unroll 1                                         // (few registers: this block's P is live)
                    for (int s4 = 0; s4 < 4; ++s4) {
                        const uint4 mk = keep_below(kb + 16 * s4 + 8 * lh, end);
#pragma unroll
                        for (int db = 0; db < Gm::DB; ++db)
                            bits |= nonfinite_bits(and4(*reinterpret_cast<const uint4 *>(V + vplace(db, s4)), mk));
                    }
                    bad = any_nonfinite(bits);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s4 = 0; s4 < 4; ++s4) {
                    const int kh = s4 >> 1, q0 = 8 * (s4 & 1), c = 2 * s4 + lh;
                    auto pair = [&](int i) {
                        if constexpr (F16) return cvt_pk_f16(sacc[kh][q0 + i], sacc[kh][q0 + i + 1]);
                        else if constexpr (S::HALF) return cvt_pk_bf16(sacc[kh][q0 + i] * pow2(HALF_UP), sacc[kh][q0 + i + 1] * pow2(HALF_UP));
                        else return cvt_pk_bf16(sacc[kh][q0 + i], sacc[kh][q0 + i + 1]);
                    };
                    const bf16x8_t pb = as_bf16x8(pair(0), pair(2), pair(4), pair(6));
                    uint4 mk;
                    if (MASK) mk = keep_below(kb + 8 * c, end);
#pragma unroll
                    for (int db = 0; db < Gm::DB; ++db) {
                        uint4 v = *reinterpret_cast<const uint4 *>(V + vplace(db, s4));
                        if (MASK) {
                            v = and4(v, mk);
                            if (bad) v = finite8(v);
                        }
                        if constexpr (F16) o[db] = mfma32x32x16_f16(as_bf16x8(v), pb, o[db]);
                        else o[db] = mfma32x32x16(as_bf16x8(v), pb, o[db]);
                    }
                }
                if (!MASK) {
                    __builtin_amdgcn_sched_group_barrier(0x100, SA_AHEAD, 0);
#pragma unroll
                    for (int i = 0; i < 4 * Gm::DB - SA_AHEAD; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x008, SA_AHEAD, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (MASK && bad) {
                    // register r of o[db] is dim 32 db + 8 (r / 4) + 4 lh + r % 4; the weight
                    // of an inf is positive whatever it is
                    for (int j = 0; j < SA_KB && kb + j < end; ++j) {
                        const bool sees = kb + j <= limit;
                        int half = lh;                   // opaque: no addresses of this rare loop are kept
                        asm volatile("" : "+v"(half));
#pragma unroll
                        for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
                            for (int r = 0; r < 16; ++r) {
                                const int d = 32 * db + 8 * (r >> 2) + 4 * half + (r & 3);
                                const uint32_t x = *reinterpret_cast<const uint16_t *>(V + (S::HALF ? st * Gm::STAGE : 0) + sa_vswz(d, j >> 3) + 2 * (j & 7));
                                if (sees && (x & 0x7F80u) == 0x7F80u) o[db][r] += bf2f(x);
                            }
                    }
                }
            }
            // key block blk + 1 has landed, and this one is read, before the next is begun
            stager.landed();
            __syncthreads();
        };
        if constexpr (S::HALF) {
            stager.open(flow, hk, table, width, end, b0);
            __syncthreads();
            for (int blk = b0; blk < b1; ++blk) {
                bool half = true;
                for (; blk < b1; ++blk) {
                    const int st = (blk - b0) & 1;
                    const typename S::Looks looks = stager.looks_of(st);
                    if (blk + 1 < b1) stager.next(flow, hk, table, width, end, blk, st);
                    half = stager.fits(looks);
                    if (!half) break;
                    block(blk, std::false_type{}, st);
                }
                if (half) break;
                stager.again(hk, table, width, end, blk, (blk - b0) & 1);
                __syncthreads();
                block(blk, std::true_type{}, (blk - b0) & 1);
            }
        } else {
            stager.open(flow, hk, table, width, b0);
            stager.landed();
            __syncthreads();
            using S0 = std::integral_constant<int, 0>;
            using S1 = std::integral_constant<int, 1>;
            const int bf = min(b1, (lo + 1) / SA_KB);        // key blocks below it need no mask
            int blk = b0;
            for (; blk + 1 < bf; blk += 2) {
                block(blk, std::false_type{}, S0{});
                block(blk + 1, std::false_type{}, S1{});
            }
            if (blk < bf) block(blk++, std::false_type{}, S0{});
            for (; blk < b1; ++blk) block(blk, std::true_type{}, (blk - b0) & 1);
        }
    };

    // q's loads end here: a wait at their first use, in the loop, would also wait for the
    // copies in flight, which the compiler does not see
#pragma unroll
    for (int ks = 0; ks < Gm::KSTEPS; ++ks) asm volatile("" ::"v"(qv[ks]));
    // the prefix, then the sequences, in one loop (the body is compiled once)
    const int pb = (P + SA_KB - 1) / SA_KB;
    for (int r = r0 - 1, at = 0; r < a.R && at < t1; ++r) {
        const bool pre = r < r0;
        int nb = pb, end = P, limit = P - 1, width = a.prefix_width;
        const int32_t *table = a.prefix_table;
        if (!pre) {
            if (!a.any_big) break;
            const Seq s = seq_of(a, r, rows);
            if (s.first > row1) break;
            nb = own_blocks(s);
            end = s.len;
            limit = row >= s.first && row < s.first + s.n ? s.len - s.n + row - s.first : -1;
            table = a.tables + (size_t)r * a.width;
            width = a.width;
        }
        segment(table, width, end, clampi(t0 - at, 0, nb), clampi(t1 - at, 0, nb), limit);
        at += nb;
    }

    const float ltot = (lsum + __shfl_xor(lsum, 32)) * (S::HALF ? pow2(HALF_UP) : 1.f);      // (of P as o has it)
    if (!col_ok) return;
    if (big && a.nsplit == 1) {
        const float inv = ltot == 0.f ? 0.f : 1.f / ltot;      // (a row without a key: 0)
        uint16_t *orow = a.out + (size_t)row * a.out_stride + (size_t)h * D;
#pragma unroll
        for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *reinterpret_cast<uint2 *>(orow + 32 * db + 8 * r4 + 4 * lh) =
                    make_uint2(cvt_pk_bf16(o[db][4 * r4] * inv, o[db][4 * r4 + 1] * inv),
                               cvt_pk_bf16(o[db][4 * r4 + 2] * inv, o[db][4 * r4 + 3] * inv));
        return;
    }
    if (part_row >= a.part_rows) return;
    const size_t part = ((size_t)split * a.part_rows + part_row) * a.H + h;
    float *po = a.tile_o + part * D;
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
            *reinterpret_cast<float4 *>(po + 32 * db + 8 * r4 + 4 * lh) =
                make_float4(o[db][4 * r4], o[db][4 * r4 + 1], o[db][4 * r4 + 2], o[db][4 * r4 + 3]);
    if (lh == 0)     // (a sum that is no number: nor is the row)
        a.tile_ml[part] = make_float2(ltot == ltot ? m * sc - (S::HALF ? HALF_P + HALF_UP : 0) : INFINITY, ltot);
}

// ---------------------------------------------------------------- merge
//
// One wave a row and q head: the parts of attn_tile (nsplit), then those of attn_own.
// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i; parts of no key have m = -inf and
// weight 0, a row of no key at all is 0.  The waves go over every row, or, where only sequences of few rows have parts,
// over by_seq rows of every sequence, if that is less (prompts are then passed over).
//
// Bound by the latency of dependent loads, so there are two rounds of them: what says where
// the parts are, then the parts, lane i holding part i's place and (m, l), the values of
// AHEAD parts on their way together.
// 64 rows of 32 heads behind 8192 positions: 7.5 us.
// Few rows (up to four a CU): WPR = 4, a workgroup a row and q head, its waves taking the parts
// in turn: 8 rows of 32 heads, up to 300 own positions, behind 32768 33 us in all, 35 with one
// wave; but 64 rows, up to 1023 own, behind 2048 45 us, 40 with one.
template <int D, int WPR>
__global__ void __launch_bounds__(256) attn_merge_kernel(SaArgs a, int tile_parts, int by_seq) {
    constexpr int PER = D / 64;
    constexpr int AHEAD = WPR == 4 ? 16 : 8;
    __shared__ float2 sm_ml[WPR];
    __shared__ float sm_o[WPR][D];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long wid = WPR == 4 ? (long)blockIdx.x : (long)blockIdx.x * 4 + w;
    const int turn = WPR == 4 ? w : 0;
    const int rows = live_rows(a);
    if (a.cut) tile_parts = a.cut[0];
    int row = (int)(wid / a.H), r;
    const int h = (int)(wid - (long)row * a.H);
    Seq s;
    int part_row = row;
    if (by_seq) {
        r = row / by_seq;
        if (r >= a.R) return;
        s = seq_of(a, r, rows);
        const int i = row - r * by_seq;
        if (i >= s.n || s.n > a.small_rows) return;
        row = s.first + i;
        if (!a.per_seq) part_row = row;
    } else {
        if (row >= rows) return;
        r = find_seq(a, row);
        s = seq_of(a, r, rows);
        if (row < s.first || row >= s.first + s.n) return;     // no sequence's row
        if (s.n > a.small_rows && tile_parts <= 1) return;     // written by attn_tile
    }
    const int hk = h / a.G, gq = h - hk * a.G;
    const int own_wgs = a.cut ? a.cut[1] : a.own_wgs;
    const int joined = a.join ? own_keyblocks(prefix_keys(a), a.own_shift) : 0;
    const OwnParts own = own_parts_of(row, s.first, s.n, s.len, hk, gq, a.G, a.small_rows, a.own_off[r], a.own_unit[r],
                                      a.own_off[a.R], own_wgs, a.own_parts, a.part_cols, a.own_shift, joined,
                                      a.own_rest ? a.own_unit[a.R] : 0);
    const int parts = tile_parts + own.n;
    float M = -INFINITY, L = 0.f, acc[PER] = {};
    for (int i0 = 0; i0 * WPR + turn < parts; i0 += 64) {
        // this lane's part
        const int k = min(64, (parts - turn + WPR - 1) / WPR - i0);
        const int i = (i0 + min(lane, k - 1)) * WPR + turn;
        const bool t = i < tile_parts;
        long at = ((long)i * a.part_rows + part_row) * a.H + h;
        if (!t) at = (own.first + own.step * (i - tile_parts)) * (long)a.part_cols + own.col;
        float2 x = (t ? a.tile_ml : a.own_ml)[at];
        if (lane >= k) x = make_float2(-INFINITY, 0.f);
        const float *const po = (t ? a.tile_o : a.own_o) + at * D;
        const uint32_t plo = (uint32_t)(uintptr_t)po, phi = (uint32_t)((uintptr_t)po >> 32);
        float v[AHEAD][PER];
        auto fetch = [&](int i) {
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                const int y = min(i + e, k - 1);
                const uintptr_t p = (uintptr_t)(uint32_t)__builtin_amdgcn_readlane(plo, y);
                const float *o = reinterpret_cast<const float *>(p | (uintptr_t)(uint32_t)__builtin_amdgcn_readlane(phi, y) << 32);
#pragma unroll
                for (int z = 0; z < PER; ++z) v[e][z] = o[lane + 64 * z];
            }
        };
        fetch(0);
        float bm = x.x;
#pragma unroll
        for (int y = 32; y >= 1; y >>= 1) bm = fmaxf(bm, __shfl_xor(bm, y));
        if (bm == -INFINITY) continue;
        const float mn = fmaxf(M, bm), alpha = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mn);
        const float wi = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - mn);
        M = mn;
        L = L * alpha + wave_sum(wi * x.y);
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] *= alpha;
        for (int i = 0; i < k; i += AHEAD) {
            float u[AHEAD][PER];
#pragma unroll
            for (int e = 0; e < AHEAD; ++e)
#pragma unroll
                for (int z = 0; z < PER; ++z) u[e][z] = v[e][z];
            if (i + AHEAD < k) fetch(i + AHEAD);
#pragma unroll
            for (int e = 0; e < AHEAD; ++e) {
                const float wk = i + e < k ? __shfl(wi, min(i + e, 63)) : 0.f;
#pragma unroll
                for (int z = 0; z < PER; ++z) acc[z] += wk == 0.f ? 0.f : wk * u[e][z];
            }
        }
    }
    if (WPR == 4) {
        if (lane == 0) sm_ml[w] = make_float2(M, L);
#pragma unroll
        for (int e = 0; e < PER; ++e) sm_o[w][lane + 64 * e] = acc[e];
        __syncthreads();
        if (w != 0) return;
        float M4 = M;
#pragma unroll
        for (int q = 1; q < WPR; ++q) M4 = fmaxf(M4, sm_ml[q].x);
        L = 0.f;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
        for (int q = 0; q < WPR; ++q) {
            const float f = sm_ml[q].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm_ml[q].x - M4);
            L += f * sm_ml[q].y;
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] += f * sm_o[q][lane + 64 * e];
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint16_t *po = a.out + (size_t)row * a.out_stride + (size_t)h * D;
#pragma unroll
    for (int e = 0; e < PER; ++e) po[lane + 64 * e] = (uint16_t)f2bf(acc[e] * inv);
}

// ---------------------------------------------------------------- host side

struct SaPlan {
    int small_rows = 0, rows_max = 0, any_big = 0, nsplit = 1, own_wgs = 0, use_tile = 0, part_cols = 0;
    int own_shift = 6, own_rest = 0, join = 0, cut = 0;
    long tiles = 0, own_parts = 0, part_rows = 0;
    int by_seq = 0, per_seq = 0;     // the merge, and attn_tile's parts, by sequence: rows of each
    long tile_o = 0, tile_ml = 0, own_o = 0, own_ml = 0, own_idx = 0, bytes = 0;      // workspace offsets
};

// the merge's rows, and where the parts lie, of a plan whose splits and workgroups are set
void lay_out(SaPlan &p, long N, long R, long H, long D) {
    const long rows_max = p.rows_max;
    auto up = [](long v) { return (v + 255) / 256 * 256; };
    long at = 0;
    // With whole tiles only sequences of few rows have parts.  Where they can be few of the
    // batch's rows the parts are kept, and merged, by sequence
    const bool few = R * rows_max < N && p.any_big && p.nsplit == 1;
    p.by_seq = few || (!p.any_big && R * rows_max <= N) ? (int)rows_max : 0;
    p.per_seq = few ? (int)rows_max : 0;
    p.part_rows = few ? R * rows_max : N;
    const long tparts = p.use_tile ? p.nsplit * p.part_rows * H : 0;
    p.tile_o = at; at += up(tparts * D * 4);
    p.tile_ml = at; at += up(tparts * 8);
    p.own_o = at; at += up(p.own_parts * p.part_cols * D * 4);
    p.own_ml = at; at += up(p.own_parts * p.part_cols * 8);
    p.own_idx = at; at += up((R + 1) * 2 * 4 + 8);
    p.bytes = at;
}

template <int D>
int merge_parts(const SaArgs &a, const SaPlan &p, hipStream_t stream) {
    const long merge_rows = p.by_seq ? (long)a.R * p.by_seq : a.N;
    const long heads = merge_rows * a.H;
    const bool wide = heads <= 4L * device_info().num_cus;
    auto merge = wide ? attn_merge_kernel<D, 4> : attn_merge_kernel<D, 1>;
    hipLaunchKernelGGL(merge, dim3((unsigned)(wide ? heads : (heads + 3) / 4)), dim3(256), 0, stream, a,
                       p.use_tile ? p.nsplit : 0, p.by_seq);
    SC_HIP_CHECK(hipGetLastError());
    return SC_OK;
}

// the kernels' shared arguments, of a plan and its workspace
void fill_args(SaArgs &a, const SaPlan &p, void *workspace) {
    a.small_rows = p.small_rows; a.any_big = p.any_big; a.nsplit = p.nsplit;
    a.own_wgs = p.own_wgs;
    a.tile_wgs = p.use_tile ? (int)(p.tiles * p.nsplit * a.Hkv) : 0;
    a.tiles = (int)p.tiles;
    a.part_rows = (int)p.part_rows; a.per_seq = p.per_seq;
    char *ws = static_cast<char *>(workspace);
    a.tile_o = reinterpret_cast<float *>(ws + p.tile_o);
    a.tile_ml = reinterpret_cast<float2 *>(ws + p.tile_ml);
    a.own_o = reinterpret_cast<float *>(ws + p.own_o);
    a.own_ml = reinterpret_cast<float2 *>(ws + p.own_ml);
    a.own_parts = (int)p.own_parts; a.part_cols = p.part_cols;
    a.own_shift = p.own_shift; a.own_rest = p.own_rest; a.join = p.join;
    a.own_off = reinterpret_cast<int32_t *>(ws + p.own_idx);
    a.own_unit = a.own_off + a.R + 1;
    a.cut = p.cut ? a.own_unit + a.R + 1 : nullptr;
}

}  // namespace

}  // namespace sc

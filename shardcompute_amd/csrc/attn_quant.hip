// Attention over a quantized key/value cache in blocks (layout: kv_cells.h), for a ragged batch
// whose sequences share one prefix: row i of sequence r attends the prefix's P positions and its
// sequence's own positions up to its own,
//   out = softmax(scale q k^T) v   over prefix[0, P) + own_r[0, lengths[r] - new_r + i],
// where k and v are scale_j code + bias_j of their group j of 64 dims.
//
// The codes themselves are the operands of the matrix instructions, as bf16 whole numbers, and
// scales and biases act on sums over a group:
//   q k   = sum_j ks_j (q . code)_j + kb_j sum_j(q)
//   (p v)_d = sum_t (p_t vs_t) code_td + sum_t p_t vb_t           d in group j
// A code of 4 bits is 128 + code once or-ed into the mantissa of 128.0; the excess is taken off
// the sums: of q k with the bias; of p v, where codes are better centred first, by
//   sum_t P_t (code_td + EXCESS) - (EXCESS + MID) sum_t P_t + sum_t p_t (vb_t + MID vs_t)
// with P_t = bf16(p_t vs_t), the same P in both sums, and MID the middle code, so that the
// rounding of P meets code - MID, as it would meet v itself.
//
// As over the bf16 cache (attn_shared.hip), the keys of few columns are a stream of memory and
// those of many a product:
//   attn_line          the own keys of sequences with few rows (at most max(64 / (H / Hkv), 1),
//                      small_rows): the codes straight from memory into the operands' registers;
//                      the work cut evenly over the workgroups whatever the lengths are
//   attn_tile          (attn_shared_core.h) the prefix, then the own keys of sequences with many
//                      rows: the workgroup turns each key block into values in LDS once, in fp16
//                      where its range holds them, else in bf16
//   attn_merge_kernel  joins the parts of a row by their softmax maxima and sums
#include "attn_shared_core.h"
#include "kv_cells.h"

#include <algorithm>
#include <atomic>

namespace sc {

namespace {

struct QuantArgs : SaArgs {
    const uint8_t *pool;
    int cus;                 // of the device
    float part_us;           // of prompt_part_us
};

// the cell of position t (a multiple of 16) of a table, kv head hk
template <int BYTES>
__device__ __forceinline__ const uint8_t *cell_at(const QuantArgs &a, int hk, int block, int t) {
    const int per = a.shift - 4;
    return a.pool + ((((size_t)clampi(block, 0, a.n_blocks - 1) * a.Hkv + hk) << per) + ((t >> 4) & ((1 << per) - 1))) * BYTES;
}

// nib_pair, the mask from a scalar and the 128s from a vector register: one instruction
__device__ __forceinline__ bf16x8_t nibbles(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    uint32_t mask = 0x000F000Fu, one28 = 0x43004300u;
    asm("" : "+s"(mask));
    asm("" : "+v"(one28));
    return as_bf16x8(dma::and_or(a, mask, one28), dma::and_or(b, mask, one28), dma::and_or(c, mask, one28), dma::and_or(d, mask, one28));
}

// lane 16 (lane / 16) + n's value, n below 16 and known when the loop around is unrolled
__device__ __forceinline__ float row_lane(float v, int n) {
    const int x = __float_as_int(v);
#define SC_ROW_LANE(i) case i: return __int_as_float(__builtin_amdgcn_update_dpp(0, x, 0x150 + i, 0xF, 0xF, true));
    switch (n) {
        SC_ROW_LANE(0) SC_ROW_LANE(1) SC_ROW_LANE(2) SC_ROW_LANE(3) SC_ROW_LANE(4) SC_ROW_LANE(5) SC_ROW_LANE(6) SC_ROW_LANE(7)
        SC_ROW_LANE(8) SC_ROW_LANE(9) SC_ROW_LANE(10) SC_ROW_LANE(11) SC_ROW_LANE(12) SC_ROW_LANE(13) SC_ROW_LANE(14)
        default: SC_ROW_LANE(15)
    }
#undef SC_ROW_LANE
}

// What a wave reads of a cell's codes.
template <int D, int BITS>
struct CellRegs {
    using C = Cell<D, BITS>;
    static constexpr int WORDS = C::LANE / 4;
    uint32_t k[WORDS], v[WORDS];
    __device__ __forceinline__ void load(const uint8_t *cell, int lane) {
#pragma unroll
        for (int p = 0; p < C::PLANES; ++p) {
            const uint8_t *kp = cell + 1024 * p + lane * C::PLANE, *vp = kp + C::CODES;
            if (C::PLANE == 16) {
                const uint4 x = *reinterpret_cast<const uint4 *>(kp), y = *reinterpret_cast<const uint4 *>(vp);
                k[4 * p] = x.x; k[4 * p + 1] = x.y; k[4 * p + 2] = x.z; k[4 * p + 3] = x.w;
                v[4 * p] = y.x; v[4 * p + 1] = y.y; v[4 * p + 2] = y.z; v[4 * p + 3] = y.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2 *>(kp), y = *reinterpret_cast<const uint2 *>(vp);
                k[0] = x.x; k[1] = x.y; v[0] = y.x; v[1] = y.y;
            }
        }
    }
};

// Softmax over keys taken in, two cells at a time, for up to CW columns.
//
// Of a step's sums q . code there are 2 GROUPS kinds: one of each cell and group of dims, to be
// scaled apart.  With 16 columns each kind has a result of its own (the instruction's 16
// columns).  With CW = 8 or 4 the columns appear 16 / CW times, as blocks, each block with the
// q of one kind and zero in the place of the others', so that all kinds lie in one result (8
// columns of 128 dims: one a cell) and each lane scales what its block holds: the softmax,
// whose work is by the result, is done once for 4 keys of a lane in place of 16.
//   lane c = lane % 16:   128 dims  CW 4: column c % 4, cell c / 4 % 2, group c / 8
//                                   CW 8: column c % 8, group c / 8; a result a cell
//                          64 dims  CW 8: column c % 8, cell c / 8
// The weights P go back the same way: a block's columns of O take only the block's cell (its
// places of operand B, the other cell's are 0) with the weights of the block's group; what a
// block's group leaves in the other group's dims is not used, and the cells' are added at
// the end.
// One row of 131072 positions, 32 heads of 128 on 8 in 4 bits (4 columns): CW 4 36.7 us, 8 38.4, 16
// 46.9; 256 rows of the 70B shard's heads in 8 bits (8 columns) 40.8, with 16 53.2.
template <int D, int BITS, int CW>
struct Columns {
    using C = Cell<D, BITS>;
    static constexpr int DT = D / 16, GROUPS = C::GROUPS;
    static_assert(CW == 16 || CW == 8 || (CW == 4 && GROUPS == 2), "columns a lane row can hold");
    static constexpr bool BY_CELL = CW * GROUPS <= 8;           // a block has one cell
    static constexpr bool BY_GROUP = CW < 16 && GROUPS == 2;    // a block has one group
    static constexpr int NG = BY_GROUP ? 1 : GROUPS;            // groups a lane has
    static constexpr int NC = BY_CELL ? 1 : 2;                  // cells a lane has
    static constexpr int NQ = (BY_CELL ? 2 : 1) * 2 * GROUPS;   // operands with q
    static constexpr float EXCESS = BITS == 4 ? 128.f : 0.f, MID = BITS == 4 ? 8.f : 128.f;
    // the exponents' reference follows the maximum only when that is more than LAG (log2) above it
    static constexpr float LAG = 8.f;
    // Scales and biases of a lane's 4 keys a cell: in its own registers, or (16 columns, where
    // these would be 32) one word of each cell a lane, for its lane row: item l / 4, position 4 g + l % 4
    static constexpr bool ROWS = CW == 16;
    struct Own { uint4 k[NC][NG], v[NC][NG]; };
    struct Row { uint32_t w[2]; };
    using Meta = std::conditional_t<ROWS, Row, Own>;
    struct Affine { float scale, bias; };
    static __device__ __forceinline__ Affine affine(const Own &x, int j, int y, bool value, int i) {
        const uint32_t w = dma::wc(value ? x.v[j][y] : x.k[j][y], i);
        return {__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)};
    }
    static __device__ __forceinline__ Affine affine(const Row &x, int j, int y, bool value, int i) {
        const int n = 4 * ((value ? GROUPS : 0) + y) + i;
        return {row_lane(__uint_as_float(x.w[j] << 16), n), row_lane(__uint_as_float(x.w[j] & 0xFFFF0000u), n)};
    }

    bf16x8_t q[NQ];
    float qsum[NG];
    float m, ref, lsum, corr[NG];            // m: the maximum, of scores without the scale
    f4 o[DT], psum[NG];
    float sl, lag;                           // the scale, in log2 units; LAG without it
    int since;                               // steps since o was settled

    static __device__ __forceinline__ int cell_of(int c) { return BY_CELL ? (GROUPS == 2 ? (c >> 2) & 1 : c >> 3) : 0; }
    static __device__ __forceinline__ int group_of(int c) { return BY_GROUP ? c >> 3 : 0; }
    static __device__ __forceinline__ bf16x8_t ones() { return as_bf16x8(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u); }
    static __device__ __forceinline__ f4 mfma(bf16x8_t a, bf16x8_t b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    // 64 lanes' v, of lanes with the same column: the other block's (by cells)
    static __device__ __forceinline__ float other_cell(float v) { return GROUPS == 2 ? xor4_mov(v) : dpp_mov<DPP_ROR8>(v); }

    static __device__ __forceinline__ void load_meta(Own &x, const uint8_t *c0, const uint8_t *c1, int lane) {
        const int g = lane >> 4, c = lane & 15;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const uint8_t *cell = (BY_CELL ? cell_of(c) : j) ? c1 : c0;
#pragma unroll
            for (int y = 0; y < NG; ++y) {
                const int grp = BY_GROUP ? group_of(c) : y;
                x.k[j][y] = *reinterpret_cast<const uint4 *>(cell + C::meta(4 * g, grp));
                x.v[j][y] = *reinterpret_cast<const uint4 *>(cell + C::meta(4 * g, GROUPS + grp));
            }
        }
    }
    static __device__ __forceinline__ void load_meta(Row &x, const uint8_t *c0, const uint8_t *c1, int lane) {
        const int at = C::meta(4 * (lane >> 4) + (lane & 3), (lane >> 2) & (C::ITEMS - 1));
        x.w[0] = *reinterpret_cast<const uint32_t *>(c0 + at);
        x.w[1] = *reinterpret_cast<const uint32_t *>(c1 + at);
    }

    // this lane's share of its column's q row (null: none)
    struct Row4 { uint4 x[2 * GROUPS]; };
    static __device__ __forceinline__ void load_q(Row4 &r, const uint16_t *qp, int lane) {
#pragma unroll
        for (int s = 0; s < 2 * GROUPS; ++s) {
            r.x[s] = make_uint4(0u, 0u, 0u, 0u);
            if (qp) r.x[s] = *reinterpret_cast<const uint4 *>(qp + 64 * (s >> 1) + 16 * (lane >> 4) + 8 * (s & 1));
        }
    }
    __device__ __forceinline__ void open(const Row4 &r, int lane, float scale_log2) {
        const int c = lane & 15;
        sl = scale_log2;
        lag = LAG / scale_log2;
        f4 sum[NG];
#pragma unroll
        for (int y = 0; y < NG; ++y) sum[y] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NQ / (2 * GROUPS); ++j)
#pragma unroll
            for (int s = 0; s < 2 * GROUPS; ++s) {
                const uint32_t mine = (!BY_CELL || cell_of(c) == j) && (!BY_GROUP || group_of(c) == s >> 1) ? 0xFFFFFFFFu : 0u;
                q[2 * GROUPS * j + s] = as_bf16x8(r.x[s].x & mine, r.x[s].y & mine, r.x[s].z & mine, r.x[s].w & mine);
                const int y = BY_GROUP ? 0 : s >> 1;
                sum[y] = mfma(ones(), q[2 * GROUPS * j + s], sum[y]);
            }
#pragma unroll
        for (int y = 0; y < NG; ++y) {
            qsum[y] = sum[y][0];
            corr[y] = 0.f;
            psum[y] = f4{0.f, 0.f, 0.f, 0.f};
        }
        m = -INFINITY;
        ref = lsum = 0.f;
        since = 0;
#pragma unroll
        for (int y = 0; y < DT; ++y) o[y] = f4{0.f, 0.f, 0.f, 0.f};
    }

    // Of the cells' positions t0 .. t0 + 15 and t1 .. t1 + 15 the column sees those up to limit.
    // A lane whose meta words are its own hides a position by giving it none: values 0, and
    // -inf (pen) added to a score of 0, whatever the cell holds there.
    float pen[NC][4];
    __device__ __forceinline__ void hide(Own &x, int t0, int t1, int limit, int lane) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int t = ((BY_CELL ? cell_of(lane & 15) : j) ? t1 : t0) + 4 * (lane >> 4);
#pragma unroll
            for (int y = 0; y < NG; ++y) {
                uint4 &k = x.k[j][y], &v = x.v[j][y];
                k.x = t > limit ? 0u : k.x; k.y = t + 1 > limit ? 0u : k.y; k.z = t + 2 > limit ? 0u : k.z; k.w = t + 3 > limit ? 0u : k.w;
                v.x = t > limit ? 0u : v.x; v.y = t + 1 > limit ? 0u : v.y; v.z = t + 2 > limit ? 0u : v.z; v.w = t + 3 > limit ? 0u : v.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) pen[j][i] = t + i > limit ? -INFINITY : 0.f;
        }
    }
    __device__ __forceinline__ void show() {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) pen[j][i] = 0.f;
    }
    // The next 32 keys.  EDGE (with 16 columns): the column sees those up to limit; else all but
    // the hidden ones.
    template <bool EDGE>
    __device__ __forceinline__ void take(const CellRegs<D, BITS> (&c)[2], const Meta &x, int t0, int t1, int limit, int lane) {
        const int g = lane >> 4;
        f4 acc[NC][NG];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int y = 0; y < NG; ++y) {
                const float e = -EXCESS * qsum[y];
                acc[j][y] = f4{e, e, e, e};
            }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int s = 0; s < 2 * GROUPS; ++s) {
                bf16x8_t a;
                if (BITS == 4) {
                    const uint32_t w = c[j].k[s];
                    a = nibbles(w, w >> 4, w >> 8, w >> 12);
                } else {
                    const uint32_t w0 = c[j].k[2 * s], w1 = c[j].k[2 * s + 1];
                    a = as_bf16x8(byte_pair_lo(w0), byte_pair_hi(w0), byte_pair_lo(w1), byte_pair_hi(w1));
                }
                f4 &r = acc[BY_CELL ? 0 : j][BY_GROUP ? 0 : s >> 1];
                r = mfma(a, q[(BY_CELL ? 2 * GROUPS * j : 0) + s], r);
            }
        float p[NC][4];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float s = ROWS ? 0.f : pen[j][i];
#pragma unroll
                for (int y = 0; y < NG; ++y) {
                    const Affine k = affine(x, j, y, false, i);
                    s = fmaf(k.scale, acc[j][y][i], fmaf(k.bias, qsum[y], s));
                }
                if (BY_GROUP) s += dpp_mov<DPP_ROR8>(s);         // (both halves' -inf, or none)
                if (EDGE && ((BY_CELL ? cell_of(lane & 15) : j) ? t1 : t0) + 4 * g + i > limit) s = -INFINITY;
                p[j][i] = s;
            }
        float bm = -INFINITY;
#pragma unroll
        for (int j = 0; j < NC; ++j) bm = fmaxf(bm, fmaxf(fmaxf(p[j][0], p[j][1]), fmaxf(p[j][2], p[j][3])));
        if (since == SETTLE / 32 || __ballot(bm > m + lag)) {
            bm = fmaxf(bm, __shfl_xor(bm, 16));
            bm = fmaxf(bm, __shfl_xor(bm, 32));
            if (BY_CELL) bm = fmaxf(bm, other_cell(bm));
            const float mn = fmaxf(m, bm), to = mn == -INFINITY ? 0.f : mn * sl;
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - to);
            m = mn;
            ref = to;
            lsum *= alpha;
            settle(alpha);
        }
        ++since;
        // P of the lane's cells and groups; a position that the column does not see weighs 0
        // whatever its scale is
        uint32_t pw[2][NG][2];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            float pv[NG][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool sees = !EDGE || ((BY_CELL ? cell_of(lane & 15) : j) ? t1 : t0) + 4 * g + i <= limit;
                const float e = __builtin_amdgcn_exp2f(fmaf(p[j][i], sl, -ref));
                lsum += e;
#pragma unroll
                for (int y = 0; y < NG; ++y) {
                    const Affine v = affine(x, j, y, true, i);
                    pv[y][i] = sees ? e * v.scale : 0.f;
                    corr[y] = sees ? fmaf(e, fmaf(MID, v.scale, v.bias), corr[y]) : corr[y];
                }
            }
            constexpr int X = BITS == 4 ? 2 : 1, Y = BITS == 4 ? 1 : 2;      // order of a value's word
#pragma unroll
            for (int y = 0; y < NG; ++y) {
                pw[j][y][0] = cvt_pk_bf16(pv[y][0], pv[y][X]);
                pw[j][y][1] = cvt_pk_bf16(pv[y][Y], pv[y][3]);
            }
        }
        bf16x8_t pb[NG];
        if (BY_CELL) {
            const uint32_t m1 = cell_of(lane & 15) ? 0xFFFFFFFFu : 0u;
            pb[0] = as_bf16x8(pw[0][0][0] & ~m1, pw[0][0][1] & ~m1, pw[0][0][0] & m1, pw[0][0][1] & m1);
        } else {
#pragma unroll
            for (int y = 0; y < NG; ++y) pb[y] = as_bf16x8(pw[0][y][0], pw[0][y][1], pw[1][y][0], pw[1][y][1]);
        }
#pragma unroll
        for (int y = 0; y < NG; ++y) psum[y] = mfma(ones(), pb[y], psum[y]);
#pragma unroll
        for (int y = 0; y < DT; ++y) {
            bf16x8_t a;
            if (BITS == 4) {
                const uint32_t w0 = c[0].v[y >> 1], w1 = c[1].v[y >> 1];
                const int s = 4 * (y & 1);
                a = nibbles(w0 >> s, w0 >> (8 + s), w1 >> s, w1 >> (8 + s));
            } else {
                const uint32_t w0 = c[0].v[y], w1 = c[1].v[y];
                a = as_bf16x8(byte_pair_lo(w0), byte_pair_hi(w0), byte_pair_lo(w1), byte_pair_hi(w1));
            }
            o[y] = mfma(a, pb[NG == 1 ? 0 : y / 4], o[y]);
        }
    }

    // The excess of the codes and the biases' part go into o, which from then on is the sum of
    // p v, and is scaled.  Done every SETTLE keys at least: until then o holds up to EXCESS + MID
    // times a scale more than the sum itself, whose fp32 roundings would add up over a long walk
    // (512 keys: 16 sums of 32, at most 16 * 136 * 2^-24 = 2^-13 of a scale).
    static constexpr int SETTLE = 512;
    __device__ __forceinline__ void settle(float alpha) {
        since = 0;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float c = corr[j];
            c += __shfl_xor(c, 16);
            c += __shfl_xor(c, 32);
            c = fmaf(-(EXCESS + MID), psum[j][0], c) * alpha;
            corr[j] = 0.f;
            psum[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = NG == 1 ? 0 : 4 * j; y < (NG == 1 ? DT : 4 * j + 4); ++y)
#pragma unroll
                for (int z = 0; z < 4; ++z) o[y][z] = fmaf(o[y][z], alpha, c);
        }
    }
    // the column's sum of weights; o then is the column's sum of p v, in the tiles that the lane writes
    __device__ __forceinline__ float close() {
        settle(1.f);
        float l = lsum + __shfl_xor(lsum, 16);
        l += __shfl_xor(l, 32);
        if (BY_CELL) {
            l += other_cell(l);
#pragma unroll
            for (int y = 0; y < DT; ++y)
#pragma unroll
                for (int z = 0; z < 4; ++z) o[y][z] += other_cell(o[y][z]);
        }
        return l;
    }
    // whether this lane writes tile y of the column's dims
    static __device__ __forceinline__ bool writes(int y, int c) { return (BY_CELL ? cell_of(c) == 0 : true) && (!BY_GROUP || group_of(c) == y / 4); }
};

// ---------------------------------------------------------------- few columns
//
// A unit is up to 64 columns (row i, q head g: column i G + g) of one sequence and kv head; its
// keys are blocks of 128, the prefix's first where they are joined.  All units' blocks in a line
// (sequence, kv head, 64 columns, key block) are cut into equal runs, one a workgroup of 4
// waves.  Of a sequence with at most 16 columns wave w takes keys 32 w .. 32 w + 31 of every block;
// of one with more, all the keys for columns 16 w .. 16 w + 15.  A wave's share of a unit is one
// part, number 4 (unit + workgroup) + wave, as in attn_shared.hip.  The waves of a workgroup share
// nothing but their run, so there is no barrier; the next 32 keys' codes are on their way while
// these are computed.
//
// Bound by memory where the sequences are long: 131072 positions of one, 32 heads of 128 on 8 in
// 4 bits, 151 MB, 30.3 us, of which 26 from the first key on (5.8 TB/s); by the VALU of the
// codes, the affine sums and the softmax, about 300 instructions a wave and step of 32 keys, where
// codes come from a cache.
constexpr int LINE_SHIFT = 7, LINE_KB = 1 << LINE_SHIFT;
// Workgroups a CU, and waves a SIMD, where lines run alone: 64 dims leave room for three, of 4 bits
// and 64 sequences of 4000 positions 29.5 us in place of 30.8, 256 of up to 900 31.0 of 32.6.  Few
// units would be cut into more parts than their merge gains by: one sequence of 65536 positions
// 22.8 us with two, 26.9 with three.  128 dims with three spill: 131072 positions 38 us, with two 31.
constexpr int line_waves(int D) { return D == 64 ? 3 : 2; }
constexpr int FEW_UNITS = 32;

// sum of the lanes' values up to this one's: within rows of 16, then over the rows
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);          // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);          // lane 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);          // lane 31 into rows 2 and 3
    return v;
}

// the largest of the lanes' values, none below 0
__device__ __forceinline__ int wave_top(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

struct Line {
    int32_t *first_row, *keys, *off, *unit;      // of every sequence, in LDS: first row, keys, first block and unit in the line
    int rows, P, pb;                             // rows of the batch, joined keys of the prefix and their blocks
    int total, units;                            // places (blocks first, after places_of also the units' rests), units
    int rest;                                    // places after a unit's blocks that hold no keys
    __device__ __forceinline__ int start(int r) const { return off[r] + rest * unit[r]; }
};

// A unit's opening and end cost as much as a block's keys or nearly (64 rows on 32 heads of 128:
// workgroups with the short sequences' units took 39 us where the others took 26), so a unit is
// given a place more than it has blocks, unless that makes runs longer than it can save.
__device__ __forceinline__ bool with_rest(int total, int units, int wgs) {
    return 5 * own_run(total + units, wgs) < 8 * own_run(total, wgs);
}
__device__ __forceinline__ void places_of(const QuantArgs &a, Line &l) {
    l.rest = a.own_rest && with_rest(l.total, l.units, a.own_wgs) ? 1 : 0;
    l.total += l.rest * l.units;
}
constexpr int line_lds(int R) { return 4 * R * 4 + 64; }

__device__ __forceinline__ Line line_of(const QuantArgs &a, uint8_t *smem) {
    Line l;
    l.first_row = reinterpret_cast<int32_t *>(smem);
    l.keys = l.first_row + a.R;
    l.off = l.keys + a.R;
    l.unit = l.off + a.R;
    int32_t *wsum = l.unit + a.R;
    l.rows = __builtin_amdgcn_readfirstlane(live_rows(a));
    l.P = __builtin_amdgcn_readfirstlane(a.join ? prefix_keys(a) : 0);
    l.pb = own_keyblocks(l.P, LINE_SHIFT);
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    int t_before = 0, u_before = 0;
    for (int r0 = 0; r0 < a.R; r0 += threads) {
        const int r = r0 + tid;
        int t = 0, u = 0;
        if (r < a.R) {
            const Seq s = seq_of(a, r, l.rows);
            const int kt = l.pb + own_keyblocks(s.len, LINE_SHIFT);
            u = kt && s.n <= a.small_rows ? a.Hkv * own_coltiles(s.n, a.G) : 0;
            t = u * kt;
            l.first_row[r] = s.first;
            l.keys[r] = s.len;
        }
        const int ts = wave_scan(t), us = wave_scan(u);
        if (lane == 63) { wsum[wv] = ts; wsum[8 + wv] = us; }
        __syncthreads();
        int tb = t_before, ub = u_before;
        for (int i = 0; i < (min(threads, a.R - r0) + 63) >> 6; ++i) {       // the waves that have a sequence
            if (i < wv) { tb += wsum[i]; ub += wsum[8 + i]; }
            t_before += wsum[i];
            u_before += wsum[8 + i];
        }
        if (r < a.R) { l.off[r] = tb + ts - t; l.unit[r] = ub + us - u; }
        __syncthreads();
    }
    l.total = __builtin_amdgcn_readfirstlane(t_before);
    l.units = __builtin_amdgcn_readfirstlane(u_before);
    l.rest = 0;
    return l;
}

// for the merge
__device__ __forceinline__ void write_line(const QuantArgs &a, const Line &l, int i, int n) {
    for (int r = i; r < a.R; r += n) { a.own_off[r] = l.start(r); a.own_unit[r] = l.unit[r]; }
    if (i == 0) { a.own_off[a.R] = l.total; a.own_unit[a.R] = l.rest; }
}

template <int D, int BITS, int CW>
__device__ __forceinline__ void attn_line(const QuantArgs &a, const Line &l, int wg, int w) {
    using C = Cell<D, BITS>;
    using Cols = Columns<D, BITS, CW>;
    const int lane = threadIdx.x & 63, c = lane & (CW - 1), g = lane >> 4;
    const int rows = l.rows, P = l.P, pb = l.pb, total = l.total;
    int32_t *const first_row = l.first_row, *const keys = l.keys, *const unit = l.unit;
    if (wg == 0) write_line(a, l, lane + 64 * w, SA_THREADS);
    const int run = own_run(total, a.own_wgs);
    int t = (int)min((long)wg * run, (long)total);
    const int t_end = min(t + run, total);
    if (t >= t_end) return;
    // the sequence of block t: the last one that starts at or before it
    int r = 0;
    for (int n = a.R; n > 1;) {
        const int half = n >> 1;
        if (__builtin_amdgcn_readfirstlane(l.start(r + half)) <= t) { r += half; n -= half; }
        else n = half;
    }
    int in_seq = t - __builtin_amdgcn_readfirstlane(l.start(r));   // place t within sequence r

    struct Unit {                // the workgroup's run of one unit
        const int32_t *table;    // the sequence's
        int hk, part, first, n;
        int col0;                // this wave's first column
        bool wide;               // a wave takes 16 columns and every key, not all columns and 32 keys of a block
        int stop;                // the block its blocks end at
        int seen, all;           // own keys that some, that every column sees
        int rel;                 // its row i sees own keys up to rel + i
    };
    struct Step {                // 32 keys of it
        int kb;                  // the first of them in their table
        bool pre;                // the prefix's
        bool fresh, last;        // the unit's first, last step here
    };
    int blk = 0, sub = 0;        // the step's block in its unit; of a wide unit, which 32 keys of it
    auto place = [&](const Unit &u, Step &s) {
        s.pre = blk < pb;
        s.kb = (s.pre ? blk : blk - pb) * LINE_KB + 32 * (u.wide ? sub : w);
        s.last = blk + 1 >= u.stop && (!u.wide || sub == 3);
    };
    auto open = [&](Unit &u, Step &s) {      // the unit of block t; t moves to its end in the run
        int first, len, n, kt, ct, x, b0;
        for (;;) {
            if (t >= t_end) return false;
            first = __builtin_amdgcn_readfirstlane(first_row[r]);
            len = __builtin_amdgcn_readfirstlane(keys[r]);
            n = (r + 1 < a.R ? __builtin_amdgcn_readfirstlane(first_row[r + 1]) : rows) - first;
            if (n > a.small_rows) n = 0;
            kt = pb + own_keyblocks(len, LINE_SHIFT);
            ct = own_coltiles(n, a.G);
            const int places = kt + l.rest;
            if (kt == 0 || in_seq >= a.Hkv * ct * places) {
                if (++r == a.R) return false;
                in_seq = 0;
                continue;
            }
            x = in_seq / places;
            b0 = in_seq - x * places;
            if (b0 < kt) break;
            t += places - b0;
            in_seq += places - b0;
        }
        const int b1 = min(kt, b0 + t_end - t);
        t += b1 - b0;
        in_seq += b1 - b0;
        u.table = a.tables + (size_t)r * a.width;
        u.first = first;
        u.n = n;
        u.hk = x / ct;
        u.wide = n * a.G > 16;
        const int c0 = (x - u.hk * ct) * 64;
        u.col0 = u.wide ? c0 + 16 * w : 0;
        u.part = 4 * (__builtin_amdgcn_readfirstlane(unit[r]) + x + wg) + w;
        u.stop = b1;
        u.rel = len - n;
        const int last = min((c0 + 63) / a.G, n - 1);          // the unit's last row
        u.seen = clampi(u.rel + last + 1, 0, len);
        u.all = clampi(u.rel + c0 / a.G + 1, 0, len);
        blk = b0;
        sub = 0;
        s.fresh = true;
        place(u, s);
        return true;
    };
    auto advance = [&](Unit &u, Step &s) {
        s.fresh = false;
        if (u.wide && sub < 3) ++sub;
        else {
            sub = 0;
            if (++blk >= u.stop) return open(u, s);
        }
        place(u, s);
        return true;
    };
    // block numbers of a step's two cells
    struct Ids { int b0, b1; };
    auto ids_of = [&](const Unit &u, const Step &s) {
        const int32_t *table = s.pre ? a.prefix_table : u.table;
        const int last = (s.pre ? a.prefix_width : a.width) - 1;
        Ids x;
        x.b0 = table[min(s.kb >> a.shift, last)];
        x.b1 = table[min((s.kb + 16) >> a.shift, last)];
        return x;
    };
    auto end_of = [&](const Unit &u, const Step &s) { return s.pre ? P : u.seen; };      // keys that are seen
    struct Keys {                // what a step reads
        CellRegs<D, BITS> c[2];
        typename Cols::Meta meta;
    };
    auto load = [&](const Unit &u, const Step &s, const Ids &x, Keys &k) {
        const int end = end_of(u, s);
        if (s.kb >= end) return;             // nothing that is seen
        // (nor is a second cell read that no column sees: the first one again, its keys hidden)
        const int t1 = s.kb + 16 < end ? s.kb + 16 : s.kb;
        const int b0 = __builtin_amdgcn_readfirstlane(x.b0), b1 = __builtin_amdgcn_readfirstlane(t1 == s.kb ? x.b0 : x.b1);
        const uint8_t *c0 = cell_at<C::BYTES>(a, u.hk, b0, s.kb), *c1 = cell_at<C::BYTES>(a, u.hk, b1, t1);
        k.c[0].load(c0, lane);
        k.c[1].load(c1, lane);
        Cols::load_meta(k.meta, c0, c1, lane);
    };
    Cols col;
    typename Cols::Row4 qn;      // q of the unit whose keys are on their way
    auto load_q = [&](const Unit &u) {
        const int i = (u.col0 + c) / a.G, h = u.hk * a.G + u.col0 + c - i * a.G;
        Cols::load_q(qn, i < u.n ? a.q + (size_t)(u.first + i) * a.q_stride + (size_t)h * D : nullptr, lane);
    };
    auto end = [&](const Unit &u) {          // the part: the unit's columns that are there
        const float ltot = col.close();
        if ((u.col0 + c) / a.G >= u.n || u.part >= a.own_parts || c >= a.part_cols) return;
        const size_t at = (size_t)u.part * a.part_cols + c;
        if (lane < CW) a.own_ml[at] = make_float2(ltot == ltot ? col.m * a.scale_log2 : INFINITY, ltot);
        float *po = a.own_o + at * D + 4 * g;
#pragma unroll
        for (int y = 0; y < D / 16; ++y)
            if (Cols::writes(y, lane & 15)) *reinterpret_cast<f4 *>(po + 16 * y) = col.o[y];
    };

    Unit u, uf, un;              // of this step, the one whose keys are on their way, the one after it
    Step s, f, n;
    Keys k[2];
    if (!open(un, n)) return;
    uf = un;
    f = n;
    load(uf, f, ids_of(uf, f), k[0]);
    load_q(uf);
    bool more = advance(un, n);
    Ids ids = ids_of(un, n);
    int limit = -1;
    // Two waves on a SIMD: each goes first every other step (the older one always: it ended at 25 us
    // of 40, and the other went on alone; 64 decoded rows take 1 us less so)
    bool first = wg & 1;
    auto step = [&](Keys &cur, Keys &nxt) {              // false: the last one
        if (first) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        first = !first;
        if (f.fresh) {
            u = uf;
            col.open(qn, lane, a.scale_log2);
            const int i = (u.col0 + c) / a.G;
            limit = i >= u.n ? -1 : u.rel + i;
        }
        s = f;
        const bool go = more;
        if (go) {
            if (n.fresh) uf = un;
            f = n;
            load(uf, f, ids, nxt);
            if (f.fresh) load_q(uf);
            more = advance(un, n);
            ids = ids_of(un, n);
        }
        const bool edge = s.kb + 32 > (s.pre ? P : u.all);
        const int lim = s.pre ? P - 1 : limit;
        if constexpr (Cols::ROWS) {
            // (a wave of a wide unit may have no column)
            if (u.col0 < u.n * a.G && s.kb < end_of(u, s)) {
                if (!edge) col.template take<false>(cur.c, cur.meta, s.kb, s.kb + 16, lim, lane);
                else col.template take<true>(cur.c, cur.meta, s.kb, s.kb + 16, lim, lane);
            }
        } else {
            if (edge) col.hide(cur.meta, s.kb, s.kb + 16, lim, lane);
            else col.show();
            col.template take<false>(cur.c, cur.meta, s.kb, s.kb + 16, lim, lane);
        }
        if (s.last && u.col0 < u.n * a.G) end(u);
        return go;
    };
    if constexpr (Cols::ROWS) {
        do { k[1] = k[0]; } while (step(k[1], k[0]));
    } else {
        while (step(k[0], k[1]) && step(k[1], k[0])) {}
    }
}

// ---------------------------------------------------------------- many columns
//
// How attn_tile's key blocks come into its ring: K [64 keys x D] and Vt [D x 64 keys], placed as
// the bf16 cache's kernel copies them.  The waves load a key block's codes two blocks ahead and
// write their values one block ahead.  Of a block's 4 cells wave w has half of the words of cell
// w / 2, keys' and values' alike (8 waves and one path for all of them, so that nothing branches).
//
// The values are fp16, scale code + bias rounded once to 11 bits (pairs of 1024 + code, less 1024,
// one fused multiply-add): outputs are off by their own rounding, 0.0017 (relative, rms), where
// values rounded to bf16's 8 bits make it 0.0033.  A block that fp16 cannot hold (in_range) is
// read again and written in bf16 by its readers, who find it marked.
// A block of 256 columns is bound by the power of its products and the VALU of its softmax and
// values: 615 GFLOP of 16 prompts behind 4096 positions 737 us (835 TFLOP/s), with bf16 values 711:
// the same instructions on 11 in place of 8 bits lower the clock.
template <int D, int BITS>
struct Values {
    using Args = QuantArgs;
    using Gm = SaGeo<D>;
    using C = Cell<D, BITS>;
    static constexpr int COLS = 256;
    static constexpr bool HALF = true;
    static constexpr int WORDS = C::LANE / 8;        // words of a lane's half
    struct Flow {
        uint32_t k[WORDS], v[WORDS];
        uint32_t km, vm;         // scales and biases: of the lane's position's key; of position 4 g + l % 4's value
        int there;               // positions of the cell that are there, from the first
        int block;               // the next load's: its number in the pool, on its way
    };
    const QuantArgs &a;
    uint8_t *smem;
    int lane, half, cell;
    __device__ __forceinline__ Values(const QuantArgs &a_, uint8_t *smem_, int lane_, int w)
        : a(a_), smem(smem_), lane(lane_), half(w & 1), cell(w >> 1) {}

    static __device__ __forceinline__ void words(uint32_t (&x)[WORDS], const uint8_t *p) {
        if constexpr (WORDS == 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else if constexpr (WORDS == 2) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            x[0] = v.x; x[1] = v.y;
        } else {
            x[0] = *reinterpret_cast<const uint32_t *>(p);
        }
    }
    __device__ __forceinline__ int block_of(const int32_t *table, int width, int blk) const {
        return table[min((blk * SA_KB + 16 * cell) >> a.shift, width - 1)];
    }
    // the codes of key block blk, of keys below end, and the number of the one after it
    __device__ __forceinline__ void load(Flow &f, int hk, const int32_t *table, int width, int end, int blk) const {
        const int t = blk * SA_KB + 16 * cell, grp = C::GROUPS == 2 ? half : 0;
        const uint8_t *p = cell_at<C::BYTES>(a, hk, __builtin_amdgcn_readfirstlane(f.block), t);
        f.block = block_of(table, width, blk + 1);
        const int at = C::PLANES == 2 ? 1024 * half + lane * 16 : lane * C::LANE + 4 * WORDS * half;
        words(f.k, p + at);
        words(f.v, p + C::CODES + at);
        f.km = *reinterpret_cast<const uint32_t *>(p + C::meta(lane & 15, grp));
        f.vm = *reinterpret_cast<const uint32_t *>(p + C::meta(4 * (lane >> 4) + (lane & 3), C::GROUPS + grp));
        f.there = end - t;
    }
    // code e (0 .. 7) of a word of 4-bit codes, byte e (0 .. 3) of one of 8-bit codes
    static __device__ __forceinline__ float code(uint32_t w, int e) {
        return BITS == 4 ? (float)((w >> (4 * e)) & 15u) : ubyte_f32(w, e);
    }
    // fp16 holds these positions' values times 2^HALF_UP: none reaches its largest, and the scale
    // is whole, or what is dropped of it, 2^(-25 - HALF_UP) at most, is TOP times that in a value: below
    // 2^-22 in 8 bits (2^-26 in 4), 2^-11 (2^-15) of the group's largest.  (Rounded to bf16 in its place, such
    // keys move scores by 2^-8 of themselves: 0.0027 off in place of 0.0017 with scales of 2^-22.1.)
    static __device__ __forceinline__ bool in_range(uint32_t meta) {
        constexpr float TOP = BITS == 4 ? 15.f : 255.f;
        const float s = __uint_as_float(meta << 16), b = __uint_as_float(meta & 0xFFFF0000u), e = fmaf(s, TOP, b);
        const float most = fmaxf(fabsf(b), fabsf(e));
        return fabsf(b) < pow2(15 - HALF_UP) && fabsf(e) < pow2(15 - HALF_UP) &&
               (fabsf(s) >= pow2(-14 - HALF_UP) || most >= pow2(-11) || most == 0.f);
    }
    // Whether a stage's values were in range: a byte a wave, written with them.
    using Looks = uint2;
    __device__ __forceinline__ uint8_t *looks(int st) const { return smem + Gm::LDS + 8 * st; }
    __device__ __forceinline__ Looks looks_of(int st) const { return *reinterpret_cast<const uint2 *>(looks(st)); }
    static __device__ __forceinline__ bool fits(Looks x) { return __builtin_amdgcn_readfirstlane((int)(x.x | x.y)) == 0; }
    // the values of a position that is not there become 0, whatever its cell holds
    __device__ __forceinline__ void drop(Flow &f) const {
        f.km = (lane & 15) < f.there ? f.km : 0u;
        f.vm = 4 * (lane >> 4) + (lane & 3) < f.there ? f.vm : 0u;
    }
    // a pair of codes, whole numbers of 1024 + code in fp16, as values
    static __device__ __forceinline__ uint32_t pair(uint32_t codes, uint32_t s, uint32_t b) {
        const half2_t c = __builtin_bit_cast(half2_t, codes) - half2_t{(_Float16)1024.f, (_Float16)1024.f};
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, __builtin_bit_cast(half2_t, s), __builtin_bit_cast(half2_t, b)));
    }
    static __device__ __forceinline__ uint32_t up(uint32_t meta) {       // scale and bias
        return cvt_pk_f16(__uint_as_float(meta << 16) * pow2(HALF_UP), __uint_as_float(meta & 0xFFFF0000u) * pow2(HALF_UP));
    }
    __device__ __forceinline__ void store_half(Flow &f, int st) const {
        drop(f);
        // (by every lane, without a branch)
        looks(st)[2 * cell + half] = __ballot(!in_range(f.km) || !in_range(f.vm)) != 0ull;
        const int g = lane >> 4, r = lane & 15;
        uint8_t *K = smem + st * Gm::STAGE, *V = K + Gm::KTILE;
        uint32_t mask = 0x000F000Fu, one = 0x64006400u;
        asm("" : "+s"(mask));
        asm("" : "+v"(one));
        const uint32_t km = up(f.km);
        const uint32_t ks = __builtin_amdgcn_perm(km, km, 0x01000100u), kb = __builtin_amdgcn_perm(km, km, 0x03020302u);
#pragma unroll
        for (int h = 0; h < C::GROUPS; ++h) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (BITS == 4) o[e] = pair(dma::and_or(f.k[h] >> (4 * e), mask, one), ks, kb);
                else o[e] = pair(__builtin_amdgcn_perm(one, f.k[2 * h + (e >> 1)], e & 1 ? 0x07030702u : 0x05010500u), ks, kb);
            }
            const int chunk = C::GROUPS == 2 ? 8 * half + 2 * g + h : 2 * g + half;
            *reinterpret_cast<uint4 *>(K + sa_kswz<D>(16 * cell + r, chunk)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        const float vm = __uint_as_float(up(f.vm));
        uint32_t m[4], s[2], b[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = __float_as_uint(row_lane(vm, e));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            s[e] = __builtin_amdgcn_perm(m[2 * e + 1], m[2 * e], 0x05040100u);
            b[e] = __builtin_amdgcn_perm(m[2 * e + 1], m[2 * e], 0x07060302u);
        }
#pragma unroll
        for (int y = 0; y < 2 * C::GROUPS; ++y) {
            const uint32_t w = BITS == 4 ? (f.v[y >> 1] >> (4 * (y & 1))) & 0x0F0F0F0Fu : f.v[y];
            *reinterpret_cast<uint2 *>(V + sa_vswz(16 * (2 * C::GROUPS * half + y) + r, 2 * cell + (g >> 1)) + 8 * (g & 1)) =
                make_uint2(pair(__builtin_amdgcn_perm(one, w, 0x05010500u), s[0], b[0]),
                           pair(__builtin_amdgcn_perm(one, w, 0x07030702u), s[1], b[1]));
        }
    }
    __device__ __forceinline__ void store(const Flow &f, int st) const {
        int g = lane >> 4, r = lane & 15;
        asm volatile("" : "+v"(g), "+v"(r));             // opaque, as the bf16 blocks' addresses in attn_tile
        uint8_t *K = smem + st * Gm::STAGE, *V = K + Gm::KTILE;
        // keys: 8 dims a chunk, D / 64 of them
        const float ks = __uint_as_float(f.km << 16), kb = __uint_as_float(f.km & 0xFFFF0000u);
#pragma unroll
        for (int h = 0; h < C::GROUPS; ++h) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (BITS == 4) o[e] = cvt_pk_bf16(fmaf(ks, code(f.k[h], e), kb), fmaf(ks, code(f.k[h], 4 + e), kb));
                else {
                    const uint32_t wd = f.k[2 * h + (e >> 1)];
                    o[e] = cvt_pk_bf16(fmaf(ks, code(wd, 2 * (e & 1)), kb), fmaf(ks, code(wd, 2 * (e & 1) + 1), kb));
                }
            }
            const int chunk = C::GROUPS == 2 ? 8 * half + 2 * g + h : 2 * g + half;
            *reinterpret_cast<uint4 *>(K + sa_kswz<D>(16 * cell + r, chunk)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        // values: 4 positions of 2 D / 64 dims
        const float ms = __uint_as_float(f.vm << 16), mb = __uint_as_float(f.vm & 0xFFFF0000u);
        float s[4], b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) { s[e] = row_lane(ms, e); b[e] = row_lane(mb, e); }
#pragma unroll
        for (int y = 0; y < 2 * C::GROUPS; ++y) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = fmaf(s[e], BITS == 4 ? code(f.v[y >> 1], 2 * e + (y & 1)) : code(f.v[y], e), b[e]);
            *reinterpret_cast<uint2 *>(V + sa_vswz(16 * (2 * C::GROUPS * half + y) + r, 2 * cell + (g >> 1)) + 8 * (g & 1)) =
                make_uint2(cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]));
        }
    }
    __device__ __forceinline__ void open(Flow &f, int hk, const int32_t *table, int width, int end, int b0) const {
        f.block = block_of(table, width, b0);
        load(f, hk, table, width, end, b0);
        store_half(f, 0);
        load(f, hk, table, width, end, b0 + 1);
    }
    __device__ __forceinline__ void next(Flow &f, int hk, const int32_t *table, int width, int end, int blk, int st) const {
        store_half(f, st ^ 1);
        load(f, hk, table, width, end, blk + 2);
    }
    __device__ __forceinline__ void again(int hk, const int32_t *table, int width, int end, int blk, int st) const {
        Flow f;
        f.block = block_of(table, width, blk);
        load(f, hk, table, width, end, blk);
        drop(f);
        store(f, st);
    }
    __device__ __forceinline__ void landed() const {}
};

// ---------------------------------------------------------------- kernels

// Times in us that say how the CUs are shared out between tiles and lines, on a CU of its own: a
// tile's block (64 keys, 256 columns), what a tile takes beside its blocks, a place of a line's run
// (128 keys of a unit, two runs on a CU), and the bytes a us of parts, which the kernel's end has
// to bring from the caches to memory and the merge reads.  Stamped in the kernel at 64 decoded rows
// behind 8192 positions, 32 heads of 128 on 8: tiles end at 28 to 33 us, lines at 21 to 31.  Places
// taken for 1.8 us or parts for half as much change that case by less than 1 %; 24 rows of 5 on 32
// heads of 64 take 31.9 us in place of 29.2 with the parts at half.
constexpr float tile_block_us(int D) { return D == 128 ? 2.1f : 1.5f; }
constexpr float line_block_us(int D) { return D == 128 ? 2.3f : 1.4f; }
constexpr float TILE_OPEN_US = 5.f;
constexpr float PART_BYTES_US = 1.3e6f;

// Into how many workgroups each column tile's keys are cut: of 1 .. most the number with which the
// tiles' workgroups and the lines' on the CUs left are done first.  A lane a number.
__device__ __forceinline__ int best_cut(int wgs, int blocks, int most, int grid, const Line &l, float tile_us, float line_us, float part_us) {
    const int lane = threadIdx.x & 63, n = lane + 1;
    float us = INFINITY;
    if (n <= most) {                                       // (so that a CU is left)
        const float tile = (float)((blocks + n - 1) / n) * tile_us + TILE_OPEN_US;
        const int own = 2 * max(grid - wgs * n, 1);
        const float run = with_rest(l.total, l.units, own) ? (float)own_run(l.total + l.units, own) : 1.6f * (float)own_run(l.total, own);
        const float line = l.total == 0 ? 0.f : run * line_us;
        us = fmaxf(tile, line) + (float)n * part_us;
    }
    float least = us;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) least = fminf(least, __shfl_xor(least, x));
    return max(__ffsll((unsigned long long)__ballot(us == least)), 1);
}

// Where sequences of many rows are among them, column tiles of `wgs` workgroups, each with `blocks`
// key blocks that are cut into n: the walk at 2 us a block, `cus` workgroups at a time, and the
// parts, which are written and read at 2.5 TB/s (a tile that is not cut writes its rows' outputs
// itself).  (A prompt of 2048 rows in 33 column tiles on 8 kv heads stays whole: two cuts of each
// would write and read 140 MB of parts, 50 us, for half of a walk of 67.)  More blocks have their
// least time at the same n or a larger one, so that a cut planned for the tables' room is enough
// for whatever they hold.
template <class I>
__host__ __device__ __forceinline__ float cut_us(I wgs, I blocks, I n, I cus, float part_us) {
    const float walk = (float)blocks / (float)n * 2.f * (float)((wgs * n + cus - 1) / cus);
    return walk + (n == 1 ? 0.f : (float)n * part_us);
}
float prompt_part_us(long part_rows, long H, long D) { return (float)(part_rows * H * (8 * D + 16)) / 2.5e6f + 0.06f; }

// The cut by the keys that are held, those of the prefix and of the longest sequence with many rows,
// whatever the tables have room for: the n of the least time, less what leaves the longest walk as
// it is.  32 heads of 128 on 8 in 4 bits, tables with room for 131072 positions: a prompt of 2049 rows
// 82 us (75 where the tables end with it; cut for the room 258, in 12 pieces of which most hold no
// key), of 64 rows 15.2 (14.5; 22.2).  The lengths are read before the tile begins, 1 to 1.5 us where
// the cut for the room is as good: 24 rows behind 30000 held positions 39.4 us (38.6).
__device__ __forceinline__ int held_cut(const QuantArgs &a) {
    const int lane = threadIdx.x & 63, n = lane + 1, rows = live_rows(a), P = prefix_keys(a);
    int longest = 0;
    for (int r = lane; r < a.R; r += 64) {
        const Seq s = seq_of(a, r, rows);
        if (s.n > a.small_rows) longest = max(longest, s.len);
    }
    const int blocks = (P + wave_top(longest) + SA_KB - 1) / SA_KB;
    const float us = n == 1 || n <= min(a.nsplit, blocks) ? cut_us(a.tiles * a.Hkv, blocks, n, a.cus, a.part_us) : INFINITY;
    // (times are not negative: their bits are in their order)
    const int less = 0x7F800000 - __float_as_int(us);
    const int best = __ffsll((unsigned long long)__ballot(less == wave_top(less))), walk = max((blocks + best - 1) / best, 1);
    return max((blocks + walk - 1) / walk, 1);
}

// Column tiles and lines: workgroups of 8 waves, which take every register of a CU, of a tile of
// 256 columns or of two of the line's.
constexpr int QUANT_WAVES = 8;
template <int D, int BITS, int CW>
__global__ void __launch_bounds__(64 * QUANT_WAVES) __attribute__((amdgpu_waves_per_eu(2))) attn_quantized_kernel(QuantArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int id = (int)blockIdx.x, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Line l;
    // sequences with many rows are there only with 16 columns (small_rows of them make as many at least)
    const bool many = CW == 16 && a.any_big;
    if (a.cut && !many) {
        // tiles have the prefix alone, and everything else is in the line: cut by what there is
        l = line_of(a, smem);
        const int wgs = a.tiles * a.Hkv, blocks = (prefix_keys(a) + SA_KB - 1) / SA_KB;
        const float part_us = (float)a.part_rows * a.H * (8 * D + 16) / PART_BYTES_US;
        a.nsplit = __builtin_amdgcn_readfirstlane(best_cut(wgs, blocks, a.nsplit, (int)gridDim.x, l, tile_block_us(D), line_block_us(D), part_us));
        a.tile_wgs = wgs * a.nsplit;
        a.own_wgs = 2 * max((int)gridDim.x - a.tile_wgs, 1);
        if (id == 0 && threadIdx.x == 0) { a.cut[0] = a.nsplit; a.cut[1] = a.own_wgs; }
        places_of(a, l);
        if (id == 0) write_line(a, l, threadIdx.x, 64 * QUANT_WAVES);      // (the line may have no workgroup)
        if (id < a.tile_wgs) __syncthreads();                  // the ring takes the line's LDS
    }
    if (id < a.tile_wgs) {
        if (a.cut && many) {
            a.nsplit = held_cut(a);
            if (id >= a.tiles * a.Hkv * a.nsplit) return;
        }
        attn_tile<D, Values<D, BITS>>(a, id, smem);
        // (after the tile, which reads the lengths again)
        if (a.cut && many && id == 0 && threadIdx.x == 0) { a.cut[0] = a.nsplit; a.cut[1] = a.own_wgs; }
        return;
    }
    if (!a.cut || many) { l = line_of(a, smem); places_of(a, l); }
    attn_line<D, BITS, CW>(a, l, (id - a.tile_wgs) * (QUANT_WAVES / 4) + w / 4, w & 3);
}

// Lines alone.
template <int D, int BITS, int CW>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(line_waves(D)))) attn_line_kernel(QuantArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Line l = line_of(a, smem);
    places_of(a, l);
    attn_line<D, BITS, CW>(a, l, (int)blockIdx.x, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

// ---------------------------------------------------------------- host side

// The cut that is planned, for the keys that the tables have room for: what the workspace holds,
// and the most that held_cut takes.
int quant_splits(long wgs, long blocks, long cus, float part_us) {
    int best = 1;
    float least = INFINITY;
    for (int n = 1; n <= 64 && (n == 1 || n <= blocks); ++n) {
        const float us = cut_us(wgs, blocks, (long)n, cus, part_us);
        if (us < least) { least = us; best = n; }
    }
    return best;
}

// own_cap, prefix_cap: positions the tables have room for; max_new: at least the rows of
// the sequence with the most
SaPlan plan_quant(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new) {
    SaPlan p;
    const long G = H / Hkv, cols = N * G, cus = device_info().num_cus;
    if (max_new > N) max_new = N;
    p.own_shift = LINE_SHIFT;
    p.small_rows = (int)(64 / G > 1 ? 64 / G : 1);
    p.any_big = max_new > p.small_rows;
    p.own_rest = R > 1;                      // (a sequence's own units are alike)
    // one sequence: the prefix is keys of its own line (65536 positions, 32 heads of 128 on 8: 28 us, as
    // column tiles 79; 500 positions 15 either way)
    p.join = !p.any_big && prefix_cap > 0 && R == 1;
    p.use_tile = p.any_big || (prefix_cap > 0 && !p.join);
    p.tiles = (cols + 32 * QUANT_WAVES - 1) / (32 * QUANT_WAVES);
    const long wgs = p.tiles * Hkv;
    const long blocks = (prefix_cap + (p.any_big ? own_cap : 0) + SA_KB - 1) / SA_KB;
    // the kernel cuts them, into nsplit at most; where tiles have the prefix alone it shares the CUs out
    const bool shared = p.use_tile && !p.any_big && wgs < cus;
    if (shared) p.nsplit = (int)std::min({64L, blocks, (cus - 1) / wgs});
    else if (p.any_big) p.nsplit = quant_splits(wgs, blocks, cus, prompt_part_us(N, H, D));
    p.cut = shared || p.nsplit > 1;
    const long rows_max = max_new < p.small_rows ? max_new : p.small_rows;
    p.rows_max = (int)rows_max;
    long coltiles = R * ((rows_max * G + 63) / 64);
    if (coltiles > R + cols / 64) coltiles = R + cols / 64;
    const long keyblocks = coltiles * (own_keyblocks((int)own_cap, LINE_SHIFT) + (p.join ? own_keyblocks((int)prefix_cap, LINE_SHIFT) : 0) + p.own_rest);
    long ow = (p.use_tile || R * Hkv < FEW_UNITS ? 2 : line_waves((int)D)) * cus;
    if (!shared && ow > Hkv * keyblocks) ow = Hkv * keyblocks;
    p.own_wgs = (int)(ow < 1 ? 1 : ow);
    p.own_parts = 4 * (Hkv * coltiles + p.own_wgs);
    p.part_cols = (int)(rows_max * G < 16 ? (rows_max * G > 1 ? rows_max * G : 1) : 16);
    lay_out(p, N, R, H, D);
    return p;
}

template <int D, int BITS, int CW>
int run_quant(const QuantArgs &a, const SaPlan &p, hipStream_t stream) {
    const int line = line_lds(a.R);
    if (a.tile_wgs == 0) {
        hipLaunchKernelGGL((attn_line_kernel<D, BITS, CW>), dim3((unsigned)a.own_wgs), dim3(256), line, stream, a);
    } else {
        const int tile = SaGeo<D>::LDS + 16, lds = tile > line ? tile : line, per = QUANT_WAVES / 4;
        const int grid = a.cut && !a.any_big ? a.cus : a.tile_wgs + (a.own_wgs + per - 1) / per;
        if (lds > 65536) {
            // more than 64 KB of LDS has to be allowed, once a device
            static std::atomic<uint64_t> allowed;
            int dev = 0;
            SC_HIP_CHECK(hipGetDevice(&dev));
            const uint64_t bit = 1ull << (dev & 63);
            if (!(allowed.load() & bit)) {
                SC_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(&attn_quantized_kernel<D, BITS, CW>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, std::max(tile, line_lds(SA_MAX_SEQ))));
                allowed.fetch_or(bit);
            }
        }
        hipLaunchKernelGGL((attn_quantized_kernel<D, BITS, CW>), dim3((unsigned)grid), dim3(64 * QUANT_WAVES), lds, stream, a);
    }
    SC_HIP_CHECK(hipGetLastError());
    return merge_parts<D>(a, p, stream);
}

template <int D, int BITS>
int run_quant(const QuantArgs &a, const SaPlan &p, hipStream_t stream) {
    if (D == 128 && p.part_cols <= 4) return run_quant<D, BITS, D == 128 ? 4 : 8>(a, p, stream);
    if (p.part_cols <= 8) return run_quant<D, BITS, 8>(a, p, stream);
    return run_quant<D, BITS, 16>(a, p, stream);
}

bool bad_shape(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new, int bits) {
    return N < 0 || N >= (1L << 24) || R <= 0 || R > SA_MAX_SEQ || H <= 0 || Hkv <= 0 || H % Hkv || H > 4096 ||
           kv_cell_bytes(D, bits) == 0 || own_cap <= 0 || own_cap >= (1L << 30) || prefix_cap < 0 ||
           prefix_cap >= (1L << 30) || max_new < 0 ||
           // attn_line numbers its key blocks in 32 bits
           R * Hkv * ((H / Hkv + 63) / 64) * ((own_cap + prefix_cap) / LINE_KB + 3) >= (1L << 31);
}

}  // namespace

long attention_quantized_workspace_bytes(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap,
                                         long max_new, int bits) {
    if (bad_shape(N, R, H, Hkv, D, own_cap, prefix_cap, max_new, bits) || N == 0) return 0;
    return plan_quant(N, R, H, Hkv, D, own_cap, prefix_cap, max_new).bytes;
}

int launch_attention_quantized(const uint16_t *q, long q_stride, const uint8_t *pool, long n_blocks, long bs, int bits,
                               const int32_t *row_starts, const int32_t *lengths, const int32_t *tables, long width,
                               const int32_t *prefix_table, long prefix_width, const int32_t *prefix_len, uint16_t *out,
                               long out_stride, long N, long R, long H, long Hkv, long D, float scale, long max_new,
                               void *workspace, long workspace_bytes, hipStream_t stream) {
    if (N == 0) return SC_OK;
    if (!q || !pool || !row_starts || !lengths || !tables || !out || (prefix_width > 0 && (!prefix_table || !prefix_len)))
        return set_error(SC_EINVAL, "attention_quantized: null pointer");
    if (kv_cell_bytes(D, bits) == 0)
        return set_error(SC_EUNSUPPORTED, "attention_quantized: head_dim %ld in %d bits (64 or 128 in 4 or 8 supported)", D, bits);
    const int shift = block_shift(bs);
    if (shift < 0) return set_error(SC_EINVAL, "attention_quantized: block size %ld (16, 32, 64, 128 or 256)", bs);
    if (width <= 0 || width >= (1L << 26) || prefix_width < 0 || prefix_width >= (1L << 26) ||
        bad_shape(N, R, H, Hkv, D, width * bs, prefix_width * bs, max_new, bits))
        return set_error(SC_EINVAL, "attention_quantized: bad shape rows=%ld sequences=%ld (at most %d) H=%ld Hkv=%ld tables=%ld/%ld",
                         N, R, SA_MAX_SEQ, H, Hkv, width, prefix_width);
    if (n_blocks <= 0 || n_blocks * bs >= (1L << 31)) return set_error(SC_EINVAL, "attention_quantized: bad pool size");
    // the column tiles take the maximum of the unscaled scores
    if (!(scale >= 1e-30f && scale <= 1e30f)) return set_error(SC_EINVAL, "attention_quantized: scale must be positive (1e-30 to 1e30)");
    if (q_stride < H * D || out_stride < H * D || q_stride % 8 || out_stride % 4)
        return set_error(SC_EINVAL, "attention_quantized: bad row strides");
    if (((uintptr_t)q | (uintptr_t)pool) % 16 || (uintptr_t)out % 8)
        return set_error(SC_EINVAL, "attention_quantized: misaligned pointers");
    const SaPlan p = plan_quant(N, R, H, Hkv, D, width * bs, prefix_width * bs, max_new);
    if (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 16)
        return set_error(SC_EINVAL, "attention_quantized: a 16-byte aligned workspace of %ld bytes required", p.bytes);
    // 2^32 threads a launch
    if (p.tiles * p.nsplit * Hkv + p.own_wgs >= (1L << 23) || N * H >= (1L << 26))
        return set_error(SC_EINVAL, "attention_quantized: too many rows");
    QuantArgs a;
    a.q = q; a.q_stride = q_stride; a.pool = pool; a.out = out; a.out_stride = out_stride;
    a.row_starts = row_starts; a.lengths = lengths; a.tables = tables;
    a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.N = (int)N; a.R = (int)R; a.H = (int)H; a.Hkv = (int)Hkv; a.G = (int)(H / Hkv);
    a.width = (int)width; a.shift = shift; a.n_blocks = (int)n_blocks; a.prefix_width = (int)prefix_width;
    fill_args(a, p, workspace);
    a.pair_half = 0;
    a.cus = device_info().num_cus;
    a.part_us = prompt_part_us(p.part_rows, H, D);
    a.scale_log2 = scale * 1.4426950408889634f;
    if (D == 128) return bits == 4 ? run_quant<128, 4>(a, p, stream) : run_quant<128, 8>(a, p, stream);
    return bits == 4 ? run_quant<64, 4>(a, p, stream) : run_quant<64, 8>(a, p, stream);
}

}  // namespace sc

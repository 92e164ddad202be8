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
//                      rows: the workgroup turns each key block into bf16 values in LDS once
//   attn_merge_kernel  joins the parts of a row by their softmax maxima and sums
#include "attn_shared_core.h"
#include "kv_cells.h"

#include <atomic>

namespace sc {

namespace {

struct QuantArgs : SaArgs {
    const uint8_t *pool;
};

// the cell of position t (a multiple of 16) of a table, kv head hk
template <int BYTES>
__device__ __forceinline__ const uint8_t *cell_at(const QuantArgs &a, int hk, int block, int t) {
    const int per = a.shift - 4;
    return a.pool + ((((size_t)clampi(block, 0, a.n_blocks - 1) * a.Hkv + hk) << per) + ((t >> 4) & ((1 << per) - 1))) * BYTES;
}

// lane 16 (lane / 16) + SRC's value
template <int SRC>
__device__ __forceinline__ float row_lane(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + SRC, 0xF, 0xF, true));
}

// What a wave reads of a cell.
template <int D, int BITS>
struct CellRegs {
    using C = Cell<D, BITS>;
    static constexpr int WORDS = C::LANE / 4;
    uint32_t k[WORDS], v[WORDS], meta;
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
        // lane row g: positions 4 g .. 4 g + 3, item by item (64 dims: its lanes 8 .. 15 again)
        constexpr int PER = 4 * C::ITEMS;
        meta = *reinterpret_cast<const uint32_t *>(cell + 2 * C::CODES + ((lane >> 4) * PER + (lane & (PER - 1))) * 4);
    }
};

// Softmax over keys taken in, 32 at a time, for 16 columns (of which a lane has column lane & 15).
template <int D, int BITS>
struct Columns {
    using C = Cell<D, BITS>;
    static constexpr int DT = D / 16;
    static constexpr float EXCESS = BITS == 4 ? 128.f : 0.f, MID = BITS == 4 ? 8.f : 128.f;
    // the exponents' reference follows the maximum only when that is more than LAG (log2) above it
    static constexpr float LAG = 8.f;
    bf16x8_t q[2 * C::GROUPS];
    float qsum[C::GROUPS];
    float m, ref, lsum, corr[C::GROUPS];
    f4 o[DT], psum[C::GROUPS];

    static __device__ __forceinline__ bf16x8_t ones() { return as_bf16x8(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u); }

    // qp: this lane's column's q row (null: none)
    __device__ __forceinline__ void open(const uint16_t *qp, int g) {
#pragma unroll
        for (int s = 0; s < 2 * C::GROUPS; ++s) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (qp) x = *reinterpret_cast<const uint4 *>(qp + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
            q[s] = as_bf16x8(x);
        }
#pragma unroll
        for (int j = 0; j < C::GROUPS; ++j) {
            f4 s = {0.f, 0.f, 0.f, 0.f};
            s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones(), q[2 * j], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones(), q[2 * j + 1], s, 0, 0, 0);
            qsum[j] = s[0];
            corr[j] = 0.f;
            psum[j] = f4{0.f, 0.f, 0.f, 0.f};
        }
        m = -INFINITY;
        ref = lsum = 0.f;
#pragma unroll
        for (int y = 0; y < DT; ++y) o[y] = f4{0.f, 0.f, 0.f, 0.f};
    }

    // The cells' positions t0 .. t0 + 15 and t1 .. t1 + 15; the column sees those up to limit
    // (EDGE; else all).
    template <bool EDGE>
    __device__ __forceinline__ void take(const CellRegs<D, BITS> (&c)[2], int t0, int t1, int limit, float scale_log2, int lane) {
        const int g = lane >> 4;
        // this lane's item of meta: keys' scale and bias in log2 units, the excess taken off;
        // values' with the middle code
        float ma[2], mb[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float s = __uint_as_float(c[j].meta << 16), b = __uint_as_float(c[j].meta & 0xFFFF0000u);
            const bool key = (lane & C::GROUPS) == 0;
            const float f = key ? scale_log2 : 1.f;
            ma[j] = s * f;
            mb[j] = fmaf(key ? -EXCESS : MID, s, b) * f;
        }
        float p[2][4];
        f4 acc[2][C::GROUPS];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int y = 0; y < C::GROUPS; ++y) {
                f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bf16x8_t a;
                    if (BITS == 4) {
                        const uint32_t w = c[j].k[2 * y + h];
                        a = as_bf16x8(nib_pair(w, 0), nib_pair(w, 4), nib_pair(w, 8), nib_pair(w, 12));
                    } else {
                        const uint32_t w0 = c[j].k[4 * y + 2 * h], w1 = c[j].k[4 * y + 2 * h + 1];
                        a = as_bf16x8(byte_pair_lo(w0), byte_pair_hi(w0), byte_pair_lo(w1), byte_pair_hi(w1));
                    }
                    s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[2 * y + h], s, 0, 0, 0);
                }
                acc[j][y] = s;
            }
        constexpr int I = C::ITEMS;
        auto score = [&](int j, auto i_tag) {
            constexpr int i = decltype(i_tag)::value;
            float s = row_lane<I * i>(ma[j]) * acc[j][0][i];
            s = fmaf(row_lane<I * i>(mb[j]), qsum[0], s);
            if constexpr (C::GROUPS == 2) {
                s = fmaf(row_lane<I * i + 1>(ma[j]), acc[j][1][i], s);
                s = fmaf(row_lane<I * i + 1>(mb[j]), qsum[1], s);
            }
            if (EDGE && (j ? t1 : t0) + 4 * g + i > limit) s = -INFINITY;
            p[j][i] = s;
        };
        using I0 = std::integral_constant<int, 0>;
        using I1 = std::integral_constant<int, 1>;
        using I2 = std::integral_constant<int, 2>;
        using I3 = std::integral_constant<int, 3>;
#pragma unroll
        for (int j = 0; j < 2; ++j) { score(j, I0{}); score(j, I1{}); score(j, I2{}); score(j, I3{}); }
        float bm = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) bm = fmaxf(bm, fmaxf(fmaxf(p[j][0], p[j][1]), fmaxf(p[j][2], p[j][3])));
        if (__ballot(bm > m + LAG)) {
            bm = fmaxf(bm, __shfl_xor(bm, 16));
            bm = fmaxf(bm, __shfl_xor(bm, 32));
            const float mn = fmaxf(m, bm);
            ref = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - ref);
            m = mn;
            lsum *= alpha;
#pragma unroll
            for (int y = 0; y < C::GROUPS; ++y) {
                corr[y] *= alpha;
#pragma unroll
                for (int x = 0; x < 4; ++x) psum[y][x] *= alpha;
            }
#pragma unroll
            for (int y = 0; y < DT; ++y)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[y][x] *= alpha;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[j][i] = __builtin_amdgcn_exp2f(p[j][i] - ref);
                lsum += p[j][i];
            }
        // P of the groups; a position that the column does not see weighs 0 whatever its scale is
        bf16x8_t pb[C::GROUPS];
        float pv[2][C::GROUPS][4];
        auto weigh = [&](int j, auto i_tag) {
            constexpr int i = decltype(i_tag)::value;
            const bool sees = !EDGE || (j ? t1 : t0) + 4 * g + i <= limit;
            const float a0 = row_lane<I * i + C::GROUPS>(ma[j]), b0 = row_lane<I * i + C::GROUPS>(mb[j]);
            pv[j][0][i] = sees ? p[j][i] * a0 : 0.f;
            corr[0] = sees ? fmaf(p[j][i], b0, corr[0]) : corr[0];
            if constexpr (C::GROUPS == 2) {
                const float a1 = row_lane<I * i + 3>(ma[j]), b1 = row_lane<I * i + 3>(mb[j]);
                pv[j][1][i] = sees ? p[j][i] * a1 : 0.f;
                corr[1] = sees ? fmaf(p[j][i], b1, corr[1]) : corr[1];
            }
        };
#pragma unroll
        for (int j = 0; j < 2; ++j) { weigh(j, I0{}); weigh(j, I1{}); weigh(j, I2{}); weigh(j, I3{}); }
        constexpr int X = BITS == 4 ? 2 : 1, Y = BITS == 4 ? 1 : 2;      // order of a value's word
#pragma unroll
        for (int y = 0; y < C::GROUPS; ++y) {
            pb[y] = as_bf16x8(cvt_pk_bf16(pv[0][y][0], pv[0][y][X]), cvt_pk_bf16(pv[0][y][Y], pv[0][y][3]),
                              cvt_pk_bf16(pv[1][y][0], pv[1][y][X]), cvt_pk_bf16(pv[1][y][Y], pv[1][y][3]));
            psum[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones(), pb[y], psum[y], 0, 0, 0);
        }
#pragma unroll
        for (int y = 0; y < DT; ++y) {
            bf16x8_t a;
            if (BITS == 4) {
                const uint32_t w0 = c[0].v[y >> 1], w1 = c[1].v[y >> 1];
                const int s = 4 * (y & 1);
                a = as_bf16x8(nib_pair(w0, s), nib_pair(w0, 8 + s), nib_pair(w1, s), nib_pair(w1, 8 + s));
            } else {
                const uint32_t w0 = c[0].v[y], w1 = c[1].v[y];
                a = as_bf16x8(byte_pair_lo(w0), byte_pair_hi(w0), byte_pair_lo(w1), byte_pair_hi(w1));
            }
            o[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pb[y / 4], o[y], 0, 0, 0);
        }
    }

    // The excess of the codes and the biases' part go into o, which from then on is the sum of
    // p v.  Done every SETTLE keys: until then o holds up to EXCESS + MID times a scale more than
    // the sum itself, whose fp32 roundings would add up over a long walk (512 keys: 16 sums of 32,
    // at most 16 * 136 * 2^-24 = 2^-13 of a scale).
    static constexpr int SETTLE = 512;
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int j = 0; j < C::GROUPS; ++j) {
            float c = corr[j];
            c += __shfl_xor(c, 16);
            c += __shfl_xor(c, 32);
            c = fmaf(-(EXCESS + MID), psum[j][0], c);
            corr[j] = 0.f;
            psum[j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = 4 * j; y < 4 * j + 4; ++y)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[y][x] += c;
        }
    }
    // o and the sum of the column's weights
    __device__ __forceinline__ float close() {
        settle();
        const float l = lsum + __shfl_xor(lsum, 16);
        return l + __shfl_xor(l, 32);
    }
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
constexpr int LINE_SHIFT = 7, LINE_KB = 1 << LINE_SHIFT;

template <int D, int BITS>
__device__ __forceinline__ void attn_line(const QuantArgs &a, int wg, int w, uint8_t *smem) {
    using C = Cell<D, BITS>;
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    // of every sequence: its first row, its keys, its first block and unit in the line
    int32_t *first_row = reinterpret_cast<int32_t *>(smem), *keys = first_row + a.R, *off = keys + a.R, *unit = off + a.R;
    int32_t *wsum = unit + a.R;
    const int rows = live_rows(a);
    const int P = a.join ? prefix_keys(a) : 0, pb = own_keyblocks(P, LINE_SHIFT);

    int t_before = 0, u_before = 0;
    for (int r0 = 0; r0 < a.R; r0 += threads) {
        const int r = r0 + tid, wv = tid >> 6;
        int t = 0, u = 0;
        if (r < a.R) {
            const Seq s = seq_of(a, r, rows);
            const int kt = pb + own_keyblocks(s.len, LINE_SHIFT);
            u = kt && s.n <= a.small_rows ? a.Hkv * own_coltiles(s.n, a.G) : 0;
            t = u * kt;
            first_row[r] = s.first;
            keys[r] = s.len;
        }
        int ts = t, us = u;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const int t2 = __shfl_up(ts, x), u2 = __shfl_up(us, x);
            if (lane >= x) { ts += t2; us += u2; }
        }
        if (lane == 63) { wsum[wv] = ts; wsum[8 + wv] = us; }
        __syncthreads();
        int tb = t_before, ub = u_before;
        for (int i = 0; i < threads >> 6; ++i) {
            if (i < wv) { tb += wsum[i]; ub += wsum[8 + i]; }
            t_before += wsum[i];
            u_before += wsum[8 + i];
        }
        if (r < a.R) { off[r] = tb + ts - t; unit[r] = ub + us - u; }
        __syncthreads();
    }
    if (wg == 0) {
        for (int r = lane + 64 * w; r < a.R; r += SA_THREADS) { a.own_off[r] = off[r]; a.own_unit[r] = unit[r]; }
        if (lane + w == 0) a.own_off[a.R] = t_before;
    }
    const int total = t_before, run = own_run(total, a.own_wgs);
    int t = (int)min((long)wg * run, (long)total);
    const int t_end = min(t + run, total);
    if (t >= t_end) return;
    // the sequence of block t: the last one that starts at or before it
    int r = 0;
    for (int n = a.R; n > 1;) {
        const int half = n >> 1;
        if (off[r + half] <= t) { r += half; n -= half; }
        else n = half;
    }
    r = __builtin_amdgcn_readfirstlane(r);
    int u_next = __builtin_amdgcn_readfirstlane(unit[r]);      // unit number of the next unit opened
    int in_seq = t - __builtin_amdgcn_readfirstlane(off[r]);   // block t within sequence r

    struct Step {                // 32 keys of a wave's share of one unit
        const int32_t *table;
        int width;
        int hk, part, first, n;
        int col0;                // this wave's first column
        bool wide;               // a wave takes 16 columns and every key, not all columns and 32 keys of a block
        int blk, stop, sub;      // the unit's block, and the one its blocks end at; wide: which 32 keys of it
        int kb, end;             // the first of the 32 keys, and the keys some column sees, of the table
        int all;                 // keys that every column sees
        int rel;                 // the unit's row i sees keys up to rel + i (the prefix's: all)
        int seen_own, all_own;
        bool fresh, last;        // the unit's first, last step here
    };
    bool first_unit = true;
    auto place = [&](Step &s) {  // kb, table and bounds of the step
        const bool pre = s.blk < pb;
        s.kb = (pre ? s.blk : s.blk - pb) * LINE_KB + 32 * (s.wide ? s.sub : w);
        s.table = pre ? a.prefix_table : a.tables + (size_t)r * a.width;
        s.width = pre ? a.prefix_width : a.width;
        s.end = pre ? P : s.seen_own;
        s.all = pre ? P : s.all_own;
        s.last = s.blk + 1 >= s.stop && (!s.wide || s.sub == 3);
    };
    auto open = [&](Step &s) {   // the unit of block t; t moves to its end in the run
        if (t >= t_end) return false;
        int first, len, n, kt, ct;
        for (;; ++r, in_seq = 0) {
            first = __builtin_amdgcn_readfirstlane(first_row[r]);
            len = __builtin_amdgcn_readfirstlane(keys[r]);
            n = (r + 1 < a.R ? __builtin_amdgcn_readfirstlane(first_row[r + 1]) : rows) - first;
            if (n > a.small_rows) n = 0;
            kt = pb + own_keyblocks(len, LINE_SHIFT);
            ct = own_coltiles(n, a.G);
            if (in_seq < a.Hkv * ct * kt || r == a.R - 1) break;
        }
        const int u = in_seq / kt, b0 = in_seq - u * kt, b1 = min(kt, b0 + t_end - t);
        t += b1 - b0;
        in_seq += b1 - b0;
        if (first_unit) u_next += u;
        first_unit = false;
        s.fresh = true;
        s.first = first;
        s.n = n;
        s.hk = u / ct;
        s.wide = n * a.G > 16;
        const int c0 = (u - s.hk * ct) * 64;
        s.col0 = s.wide ? c0 + 16 * w : 0;
        s.part = 4 * (u_next + wg) + w;
        ++u_next;
        s.blk = b0;
        s.stop = b1;
        s.sub = 0;
        s.rel = len - n;
        const int last = min((c0 + 63) / a.G, n - 1);          // the unit's last row
        s.seen_own = clampi(s.rel + last + 1, 0, len);
        s.all_own = clampi(s.rel + c0 / a.G + 1, 0, len);
        place(s);
        return true;
    };
    auto advance = [&](Step &s) {
        if (s.wide && s.sub < 3) ++s.sub;
        else {
            s.sub = 0;
            if (++s.blk >= s.stop) return open(s);
        }
        s.fresh = false;
        place(s);
        return true;
    };
    // block numbers of a step's two cells
    struct Ids { int b0, b1; };
    auto ids_of = [&](const Step &s) {
        Ids x;
        x.b0 = s.table[min(s.kb >> a.shift, s.width - 1)];
        x.b1 = s.table[min((s.kb + 16) >> a.shift, s.width - 1)];
        return x;
    };
    auto load = [&](const Step &s, const Ids &x, CellRegs<D, BITS> (&regs)[2]) {
        if (s.kb >= s.end) return;           // nothing that is seen
        // (nor is a second cell read that no column sees: the first one again, its keys hidden)
        const int t1 = s.kb + 16 < s.end ? s.kb + 16 : s.kb;
        const int b0 = __builtin_amdgcn_readfirstlane(x.b0), b1 = __builtin_amdgcn_readfirstlane(t1 == s.kb ? x.b0 : x.b1);
        regs[0].load(cell_at<C::BYTES>(a, s.hk, b0, s.kb), lane);
        regs[1].load(cell_at<C::BYTES>(a, s.hk, b1, t1), lane);
    };
    Columns<D, BITS> col;
    auto column = [&](const Step &s) {       // this lane's column's q row
        const int i = (s.col0 + c) / a.G, h = s.hk * a.G + s.col0 + c - i * a.G;
        return i < s.n ? a.q + (size_t)(s.first + i) * a.q_stride + (size_t)h * D : nullptr;
    };
    auto end = [&](const Step &s) {          // the part: the unit's columns that are there
        const float ltot = col.close();
        if ((s.col0 + c) / a.G >= s.n || s.part >= a.own_parts || c >= a.part_cols) return;
        const size_t at = (size_t)s.part * a.part_cols + c;
        if (g == 0) a.own_ml[at] = make_float2(ltot == ltot ? col.m : INFINITY, ltot);
        float *po = a.own_o + at * D + 4 * g;
#pragma unroll
        for (int y = 0; y < D / 16; ++y) *reinterpret_cast<f4 *>(po + 16 * y) = col.o[y];
    };

    Step s, n;                   // this step, and the next
    CellRegs<D, BITS> cur[2], nxt[2];
    open(s);
    load(s, ids_of(s), nxt);
    n = s;
    bool more = advance(n);
    Ids ids = ids_of(n);
    int since = 0, limit = -1;
    for (;;) {
#pragma unroll
        for (int j = 0; j < 2; ++j) cur[j] = nxt[j];
        const Step f = n;
        const bool go = more;
        if (go) {
            load(f, ids, nxt);
            more = advance(n);
            ids = ids_of(n);
        }
        if (s.fresh) {
            col.open(column(s), g);
            since = 0;
            const int i = (s.col0 + c) / a.G;
            limit = i >= s.n ? -1 : s.rel + i;
        }
        if (s.col0 < s.n * a.G) {            // (a wave of a wide unit may have no column)
            if (s.kb < s.end) {
                if (since == Columns<D, BITS>::SETTLE / 32) { col.settle(); since = 0; }
                ++since;
                if (s.kb + 32 <= s.all) col.template take<false>(cur, s.kb, s.kb + 16, 0, a.scale_log2, lane);
                else col.template take<true>(cur, s.kb, s.kb + 16, s.blk < pb ? P - 1 : limit, a.scale_log2, lane);
            }
            if (s.last) end(s);
        }
        if (!go) break;
        s = f;
    }
}

// ---------------------------------------------------------------- many columns
//
// How attn_tile's key blocks come into its ring: K [64 keys x D] and Vt [D x 64 keys] in bf16, as
// the bf16 cache's kernel copies them.  The waves load a key block's codes two blocks ahead and
// write their values one block ahead; of 4 cells half of the waves have the keys, half the values.
template <int D, int BITS, int WAVES>
struct Values {
    using Args = QuantArgs;
    using Gm = SaGeo<D>;
    using C = Cell<D, BITS>;
    static constexpr int COLS = 32 * WAVES;
    static constexpr int CELLS = 8 / WAVES;          // cells' halves a wave has
    static constexpr int WORDS = C::LANE / 4;
    struct Flow {
        uint32_t x[CELLS][WORDS];
        uint32_t meta[CELLS];
    };
    const QuantArgs &a;
    uint8_t *smem;
    int lane, w;
    __device__ __forceinline__ Values(const QuantArgs &a_, uint8_t *smem_, int lane_, int w_) : a(a_), smem(smem_), lane(lane_), w(w_) {}

    __device__ __forceinline__ bool values_of(int i) const { return (w * CELLS + i) >= 4; }
    __device__ __forceinline__ int cell_of(int i) const { return (w * CELLS + i) & 3; }
    __device__ __forceinline__ void load(Flow &f, int hk, const int32_t *table, int width, int blk) const {
        constexpr int PER = 4 * C::ITEMS;
#pragma unroll
        for (int i = 0; i < CELLS; ++i) {
            const int t = blk * SA_KB + 16 * cell_of(i);
            const int b = __builtin_amdgcn_readfirstlane(table[min(t >> a.shift, width - 1)]);
            const uint8_t *cell = cell_at<C::BYTES>(a, hk, b, t);
            const uint8_t *p = cell + (values_of(i) ? C::CODES : 0) + lane * C::PLANE;
#pragma unroll
            for (int pl = 0; pl < C::PLANES; ++pl) {
                if (C::PLANE == 16) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(p + 1024 * pl);
                    f.x[i][4 * pl] = v.x; f.x[i][4 * pl + 1] = v.y; f.x[i][4 * pl + 2] = v.z; f.x[i][4 * pl + 3] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2 *>(p);
                    f.x[i][0] = v.x; f.x[i][1] = v.y;
                }
            }
            f.meta[i] = *reinterpret_cast<const uint32_t *>(cell + 2 * C::CODES + ((lane >> 4) * PER + (lane & (PER - 1))) * 4);
        }
    }
    // code e (0 .. 7) of a word of 4-bit codes, byte e (0 .. 3) of one of 8-bit codes
    static __device__ __forceinline__ float code(uint32_t w, int e) {
        return BITS == 4 ? (float)((w >> (4 * e)) & 15u) : ubyte_f32(w, e);
    }
    __device__ __forceinline__ void store(const Flow &f, int st) const {
        const int g = lane >> 4, r = lane & 15;
#pragma unroll
        for (int i = 0; i < CELLS; ++i) {
            uint8_t *K = smem + st * Gm::STAGE, *V = K + Gm::KTILE;
            const int ci = cell_of(i);
            if (!values_of(i)) {
                const int t = 16 * ci + r;
                // position r's scale and bias: lane row r / 4 of the meta words has them
#pragma unroll
                for (int j = 0; j < C::GROUPS; ++j) {
                    const uint32_t mw = (uint32_t)__shfl((int)f.meta[i], 16 * (r >> 2) + C::ITEMS * (r & 3) + j);
                    const float s = __uint_as_float(mw << 16), b = __uint_as_float(mw & 0xFFFF0000u);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t o[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (BITS == 4) {
                                const uint32_t wd = f.x[i][2 * j + h];
                                o[e] = cvt_pk_bf16(fmaf(s, code(wd, e), b), fmaf(s, code(wd, 4 + e), b));
                            } else {
                                const uint32_t wd = f.x[i][4 * j + 2 * h + (e >> 1)];
                                o[e] = cvt_pk_bf16(fmaf(s, code(wd, 2 * (e & 1)), b), fmaf(s, code(wd, 2 * (e & 1) + 1), b));
                            }
                        }
                        *reinterpret_cast<uint4 *>(K + sa_kswz<D>(t, 8 * j + 2 * g + h)) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            } else {
                const float ms = __uint_as_float(f.meta[i] << 16), mb = __uint_as_float(f.meta[i] & 0xFFFF0000u);
                auto group = [&](auto j_tag) {
                    constexpr int j = decltype(j_tag)::value, I = C::ITEMS, B = C::GROUPS + j;
                    const float s[4] = {row_lane<B>(ms), row_lane<I + B>(ms), row_lane<2 * I + B>(ms), row_lane<3 * I + B>(ms)};
                    const float b[4] = {row_lane<B>(mb), row_lane<I + B>(mb), row_lane<2 * I + B>(mb), row_lane<3 * I + B>(mb)};
#pragma unroll
                    for (int y = 4 * j; y < 4 * j + 4; ++y) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v[e] = fmaf(s[e], BITS == 4 ? code(f.x[i][y >> 1], 2 * e + (y & 1)) : code(f.x[i][y], e), b[e]);
                        *reinterpret_cast<uint2 *>(V + sa_vswz(16 * y + r, 2 * ci + (g >> 1)) + 8 * (g & 1)) =
                            make_uint2(cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3]));
                    }
                };
                group(std::integral_constant<int, 0>{});
                if constexpr (C::GROUPS == 2) group(std::integral_constant<int, 1>{});
            }
        }
    }
    __device__ __forceinline__ void open(Flow &f, int hk, const int32_t *table, int width, int b0) const {
        load(f, hk, table, width, b0);
        store(f, 0);
        load(f, hk, table, width, b0 + 1);
    }
    __device__ __forceinline__ void next(Flow &f, int hk, const int32_t *table, int width, int blk, int st) const {
        store(f, st ^ 1);
        load(f, hk, table, width, blk + 2);
    }
    __device__ __forceinline__ void landed() const {}
};

// ---------------------------------------------------------------- both

template <int D, int BITS, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(2))) attn_quantized_kernel(QuantArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    if ((int)blockIdx.x < a.tile_wgs) {
        attn_tile<D, Values<D, BITS, WAVES>>(a, (int)blockIdx.x, smem);
        return;
    }
    // a workgroup of the line is 4 waves
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    attn_line<D, BITS>(a, ((int)blockIdx.x - a.tile_wgs) * (WAVES / 4) + w / 4, w & 3, smem);
}

// ---------------------------------------------------------------- host side

constexpr int QUANT_WAVES_FEW = 4, QUANT_WAVES_MANY = 8;

// Into how many workgroups a column tile's key blocks are cut.
int quant_splits(long wgs, long blocks, double part_bytes, bool last_is_whole, long cus) {
    int best = 1;
    double least = 1e30;
    for (int n = 1; n <= 64 && (n == 1 || n <= blocks); ++n) {
        const long w = wgs * n;
        const double block = w <= cus ? 1.6 : 2.2 * ((w + 2 * cus - 1) / (2 * cus));
        const double walk = (double)((blocks + n - 1) / n) * block;
        const double parts = n == 1 && last_is_whole ? 0 : n * (part_bytes / (last_is_whole ? 2.5e6 : 1.3e6) + 0.06);
        if (walk + parts < least) { least = walk + parts; best = n; }
    }
    return best;
}

struct QuantPlan : SaPlan {
    int waves = QUANT_WAVES_FEW;
};

// own_cap, prefix_cap: positions the tables have room for; max_new: at least the rows of
// the sequence with the most
QuantPlan plan_quant(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new) {
    QuantPlan p;
    const long G = H / Hkv, cols = N * G, cus = device_info().num_cus;
    if (max_new > N) max_new = N;
    p.own_shift = LINE_SHIFT;
    p.small_rows = (int)(64 / G > 1 ? 64 / G : 1);
    p.any_big = max_new > p.small_rows;
    p.join = !p.any_big && prefix_cap > 0 && R == 1;
    p.use_tile = p.any_big || (prefix_cap > 0 && !p.join);
    p.waves = p.any_big ? QUANT_WAVES_MANY : QUANT_WAVES_FEW;
    p.tiles = (cols + 32 * p.waves - 1) / (32 * p.waves);
    const long wgs = p.tiles * Hkv;
    const long blocks = (prefix_cap + (p.any_big ? own_cap : 0) + SA_KB - 1) / SA_KB;
    p.nsplit = p.use_tile ? quant_splits(wgs, blocks, (double)N * H * (8 * D + 16), p.any_big, cus) : 1;
    const long rows_max = max_new < p.small_rows ? max_new : p.small_rows;
    p.rows_max = (int)rows_max;
    long coltiles = R * ((rows_max * G + 63) / 64);
    if (coltiles > R + cols / 64) coltiles = R + cols / 64;
    const long keyblocks = coltiles * (own_keyblocks((int)own_cap, LINE_SHIFT) + (p.join ? own_keyblocks((int)prefix_cap, LINE_SHIFT) : 0));
    long ow = p.use_tile && !p.any_big ? 2 * cus - wgs * p.nsplit : 2 * cus;
    if (ow < cus) ow = cus;
    if (ow > Hkv * keyblocks) ow = Hkv * keyblocks;
    p.own_wgs = (int)(ow < 1 ? 1 : ow);
    p.own_parts = 4 * (Hkv * coltiles + p.own_wgs);
    p.part_cols = (int)(rows_max * G < 16 ? (rows_max * G > 1 ? rows_max * G : 1) : 16);
    lay_out(p, N, R, H, D);
    return p;
}

template <int D, int BITS, int WAVES>
int run_quant(const QuantArgs &a, const QuantPlan &p, hipStream_t stream) {
    const int line_lds = 4 * a.R * 4 + 64;
    const int lds = a.tile_wgs && SaGeo<D>::LDS > line_lds ? SaGeo<D>::LDS : line_lds;
    auto kern = attn_quantized_kernel<D, BITS, WAVES>;
    const int per = WAVES / 4;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.tile_wgs + (a.own_wgs + per - 1) / per)), dim3(64 * WAVES), lds, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    return merge_parts<D>(a, p, stream);
}

template <int D, int BITS>
int run_quant(const QuantArgs &a, const QuantPlan &p, hipStream_t stream) {
    return p.waves == QUANT_WAVES_MANY ? run_quant<D, BITS, QUANT_WAVES_MANY>(a, p, stream)
                                       : run_quant<D, BITS, QUANT_WAVES_FEW>(a, p, stream);
}

bool bad_shape(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new, int bits) {
    return N < 0 || N >= (1L << 24) || R <= 0 || R > SA_MAX_SEQ || H <= 0 || Hkv <= 0 || H % Hkv || H > 4096 ||
           kv_cell_bytes(D, bits) == 0 || own_cap <= 0 || own_cap >= (1L << 30) || prefix_cap < 0 ||
           prefix_cap >= (1L << 30) || max_new < 0 ||
           // attn_line numbers its key blocks in 32 bits
           R * Hkv * ((H / Hkv + 63) / 64) * ((own_cap + prefix_cap) / LINE_KB + 2) >= (1L << 31);
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
    const QuantPlan p = plan_quant(N, R, H, Hkv, D, width * bs, prefix_width * bs, max_new);
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
    a.scale_log2 = scale * 1.4426950408889634f;
    if (D == 128) return bits == 4 ? run_quant<128, 4>(a, p, stream) : run_quant<128, 8>(a, p, stream);
    return bits == 4 ? run_quant<64, 4>(a, p, stream) : run_quant<64, 8>(a, p, stream);
}

}  // namespace sc

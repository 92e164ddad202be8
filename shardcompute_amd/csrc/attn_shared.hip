// Attention over a key/value cache in blocks, for a ragged batch whose sequences share
// one prefix: row i of sequence r attends the prefix's P positions and its sequence's own
// positions up to its own,
//   out = softmax(scale q k^T) v   over prefix[0, P) + own_r[0, lengths[r] - new_r + i].
//
// The prefix is one set of keys for every row, so its part is a product of all the
// batch's rows at once (128 "columns" = (row, q head of the kv head) a workgroup, matrix
// instructions, keys through LDS); read once for all instead of once per sequence.  A
// sequence's own keys serve its rows alone: few rows (a decoded token, a few guessed ones)
// make it a stream of memory, many rows (a prompt) a product again.  So:
//   attn_tile          128 columns: the prefix, then the own keys of sequences with many
//                      rows; over several workgroups where there are few
//   attn_own           units of up to 64 columns: the own keys of sequences with few rows
//                      (at most max(64 / (H / Hkv), 1), small_rows), the work cut evenly
//                      over the workgroups whatever the lengths are
//   attn_merge_kernel  joins the parts of a row by their softmax maxima and sums
// Parts are fp32 (O unnormalised, maximum in log2 units, sum).
// Scores, maxima, exponents and sums are fp32.  The probabilities are rounded to bf16 for the
// product with v, whose matrix instructions take 16-bit operands: half a step, 2^-8 of
// softmax |v| at most, beside the output's own 2^-8.  Against 64 bits 0.0019 to 0.0024 of the
// output's size (rms), where one rounding of the output alone gives 0.0017.
//
// Pool layout as in blocks.hip: K [n_blocks, Hkv, bs, D], Vt [n_blocks, Hkv, D, bs].
// Block numbers outside the pool are clamped into it; lengths to the tables' width and
// row starts to the rows, so nothing outside the buffers is touched whatever they hold.
#include "sc_common.h"
#include "dma_util.h"
#include "attn_shared_parts.h"

#include <math.h>
#include <atomic>
#include <type_traits>

namespace sc {

int block_shift(long bs);       // blocks.hip

namespace {

using f4 = dma::f4;

constexpr int SA_COLS = 128, SA_KB = 64, SA_THREADS = 256;
constexpr int SA_AHEAD = 4;                              // operand reads in flight ahead of the MFMAs
constexpr int SA_MAX_SEQ = 2048;         // attn_own keeps two numbers of each in LDS
constexpr int SA_CU_LDS = 160 * 1024;    // of a CU

struct SaArgs {
    const uint16_t *q;
    long q_stride;
    const uint16_t *kc, *vt;
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
    int32_t *own_off, *own_unit;         // [R + 1]: a sequence's first block (and all of them), its first unit
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

// ---------------------------------------------------------------- 128 columns
//
// As the dense prefill attention: 4 waves, wave w the columns [32 w, 32 w + 32), S^T[64 keys
// x 32] = K Q^T and O^T[D x 32] += Vt P^T on v_mfma_f32_32x32x16_bf16, keys swapped on their
// way into S^T (bits 2 and 3) so that the probabilities are operand B in registers, K and
// Vt by LDS-DMA one block of 64 keys ahead into a 2-stage ring, chunks XOR-swizzled by row.
// A key block takes its four 16-key groups from up to four cache blocks (block sizes below
// 64) or one.
//
// Bound by the matrix units: 16 ragged prompts behind 4096 positions 617 to 651 us with the
// card's clock, 945 to 1000 TFLOP/s.
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

// The copies of a key block (64 keys of one kv head) into a stage of the ring, by every wave
// of the workgroup.  ONE: a key block lies in one cache block (block sizes from 64 up).
template <int D, bool ONE>
struct Stager {
    using Gm = SaGeo<D>;
    // cache blocks of a key block: ONE, its block's number; else those of the wave's 16
    // keys of K and of the lane's two chunks of Vt
    struct Ids { int k, v0, v1; };
    const SaArgs &a;
    uint8_t *smem;
    int lane, w, sh, kr, vd, vc;
    size_t blk_bytes;

    // This lane's share.  Wave w issues K instructions of the keys 16 w .. 16 w + 15 and Vt
    // instructions of D / 4 dims; a lane's dim row and chunk of Vt instruction qq differ
    // between even and odd qq only in bit 2 of the chunk.
    __device__ __forceinline__ Stager(const SaArgs &a_, uint8_t *smem_, int lane_, int w_)
        : a(a_), smem(smem_), lane(lane_), w(w_), sh(a_.shift) {
        kr = D == 128 ? 16 * w + (lane >> 4) : 16 * w + (lane >> 3);    // key row at qq = 0
        vd = Gm::DMA * 8 * w + (lane >> 3);                             // dim at qq = 0
        vc = (lane & 7) ^ ((vd >> 1) & 7);                              // chunk at even qq; ^ 4 at odd
        blk_bytes = (size_t)a.Hkv * D * 2 << sh;
    }
    __device__ __forceinline__ Ids ids(const int32_t *table, int width, int kb) const {
        auto at = [&](int key) { return table[min(key >> sh, width - 1)]; };
        Ids x;
        x.k = at(ONE ? kb : kb + 16 * w);
        if (!ONE) { x.v0 = at(kb + 8 * vc); x.v1 = at(kb + 8 * (vc ^ 4)); }
        return x;
    }
    // CLAMP (with ONE): keys past kb + lim read that key's row (or chunk) again, so that no
    // memory is read for them
    template <bool CLAMP>
    __device__ __forceinline__ void copy(int hk, int kb, int lim, int st, const Ids &x) const {
        const int bs = 1 << sh;
        const char *kpool = reinterpret_cast<const char *>(a.kc) + ((size_t)hk * D * 2 << sh);
        const char *vpool = reinterpret_cast<const char *>(a.vt) + ((size_t)hk * D * 2 << sh);
        const uint32_t kl = (uint32_t)(uintptr_t)(smem + st * Gm::STAGE) + 1024 * Gm::DMA * w;
        const uint32_t vl = kl + Gm::KTILE;
        const int kid = clampi(__builtin_amdgcn_readfirstlane(x.k), 0, a.n_blocks - 1);
        const char *kp = kpool + kid * blk_bytes + (size_t)((ONE ? kb : kb + 16 * w) & (bs - 1)) * Gm::KROW;
#pragma unroll
        for (int qq = 0; qq < Gm::DMA; ++qq) {
            const int r = kr + (D == 128 ? 4 : 8) * qq;          // key row in the key block
            const int c = D == 128 ? (lane & 15) ^ (sa_swap23(r) & 15) : (lane & 7) ^ ((r >> 1) & 7);
            dma::dma16s(kp, (uint32_t)((ONE ? (CLAMP ? min(r, lim) : r) : r - 16 * w) * Gm::KROW + 16 * c), kl + 1024 * qq);
        }
        const char *vp = vpool + kid * blk_bytes + (ONE ? (size_t)(kb & (bs - 1)) * 2 : 0);
#pragma unroll
        for (int qq = 0; qq < Gm::DMA; ++qq) {
            const int c = (qq & 1) ? vc ^ 4 : vc;
            const uint32_t voff = ((uint32_t)(vd + 8 * qq) << sh) * 2;
            if (ONE) {
                dma::dma16s(vp, voff + 16 * (CLAMP ? min(c, lim >> 3) : c), vl + 1024 * qq);
            } else {
                const int vid = clampi((qq & 1) ? x.v1 : x.v0, 0, a.n_blocks - 1);
                dma::dma16(vpool + vid * blk_bytes + voff + ((kb + 8 * c) & (bs - 1)) * 2, vl + 1024 * qq);
            }
        }
    }
};

template <int D, bool ONE>
__device__ __forceinline__ void attn_tile(const SaArgs &a, int id, uint8_t *smem) {
    using Gm = SaGeo<D>;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    // later column tiles (of prompts: more keys) are dispatched first, the first two rounds,
    // resident together, in heavy and light pairs (an order only: results do not depend on it)
    if (a.pair_half > 0 && id < 2 * a.pair_half && id >= a.pair_half) id = 3 * a.pair_half - 1 - id;
    const int hk = id % a.Hkv;
    id /= a.Hkv;
    const int split = id % a.nsplit, tile = a.tiles - 1 - id / a.nsplit;
    const int rows = live_rows(a);
    const int col = tile * SA_COLS + 32 * w + li;
    const int row = col / a.G, h = hk * a.G + col - row * a.G;
    const int row0 = tile * SA_COLS / a.G, row1 = min((tile * SA_COLS + SA_COLS - 1) / a.G, rows - 1);
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
    f32x16_t o[Gm::DB];
#pragma unroll
    for (int db = 0; db < Gm::DB; ++db) o[db] = f32x16_t{};
    float m = -INFINITY, lsum = 0.f;
    const float sc = a.scale_log2;
    const int arow = sa_swap23(li);
    const Stager<D, ONE> stager(a, smem, lane, w);

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
        // cache block numbers, one key block ahead of its copies
        typename Stager<D, ONE>::Ids ids;
        // the stage is a compile-time constant in the copies without a mask, so that every
        // operand read is a loop-invariant lane offset plus an immediate
        auto block = [&](int blk, auto mask_tag, auto stage) {
            constexpr bool MASK = decltype(mask_tag)::value;
            const int st = stage;
            const int kb = blk * SA_KB;
            const uint8_t *K = smem + st * Gm::STAGE;
            const uint8_t *V = K + Gm::KTILE;
            if (blk + 1 < b1) {
                stager.template copy<false>(hk, kb + SA_KB, 0, st ^ 1, ids);
                ids = stager.ids(table, width, kb + 2 * SA_KB);
            }
            if (!MASK || kb <= hi) {                     // else: nothing of it is seen by the wave
                f32x16_t sacc[2] = {f32x16_t{}, f32x16_t{}};
                // operand reads SA_AHEAD ahead of their MFMAs (the scheduler, left alone,
                // issues each read just before its MFMA)
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < Gm::KSTEPS; ++ks)
#pragma unroll
                    for (int kh = 0; kh < 2; ++kh) {
                        const bf16x8_t ka = as_bf16x8(*reinterpret_cast<const uint4 *>(K + sa_kswz<D>(32 * kh + arow, 2 * ks + lh)));
                        sacc[kh] = mfma32x32x16(ka, qv[ks], sacc[kh]);
                    }
                __builtin_amdgcn_sched_group_barrier(0x100, SA_AHEAD, 0);
#pragma unroll
                for (int i = 0; i < 2 * Gm::KSTEPS - SA_AHEAD; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, SA_AHEAD, 0);
                __builtin_amdgcn_sched_barrier(0);
                if (MASK) {
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
                const float nms = m == -INFINITY ? 0.f : -m * sc;
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
                            bits |= nonfinite_bits(and4(*reinterpret_cast<const uint4 *>(V + sa_vswz(32 * db + li, 2 * s4 + lh)), mk));
                    }
                    bad = any_nonfinite(bits);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s4 = 0; s4 < 4; ++s4) {
                    const int kh = s4 >> 1, q0 = 8 * (s4 & 1), c = 2 * s4 + lh;
                    const bf16x8_t pb = as_bf16x8(cvt_pk_bf16(sacc[kh][q0], sacc[kh][q0 + 1]),
                                                  cvt_pk_bf16(sacc[kh][q0 + 2], sacc[kh][q0 + 3]),
                                                  cvt_pk_bf16(sacc[kh][q0 + 4], sacc[kh][q0 + 5]),
                                                  cvt_pk_bf16(sacc[kh][q0 + 6], sacc[kh][q0 + 7]));
                    uint4 mk;
                    if (MASK) mk = keep_below(kb + 8 * c, end);
#pragma unroll
                    for (int db = 0; db < Gm::DB; ++db) {
                        uint4 v = *reinterpret_cast<const uint4 *>(V + sa_vswz(32 * db + li, c));
                        if (MASK) {
                            v = and4(v, mk);
                            if (bad) v = finite8(v);
                        }
                        o[db] = mfma32x32x16(as_bf16x8(v), pb, o[db]);
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
                                const uint32_t x = *reinterpret_cast<const uint16_t *>(V + sa_vswz(d, j >> 3) + 2 * (j & 7));
                                if (sees && (x & 0x7F80u) == 0x7F80u) o[db][r] += bf2f(x);
                            }
                    }
                }
            }
            // key block blk + 1 has landed, and this one is read, before the next is begun
            dma::wait_vm<0>();
            __syncthreads();
        };
        ids = stager.ids(table, width, b0 * SA_KB);
        stager.template copy<false>(hk, b0 * SA_KB, 0, 0, ids);
        ids = stager.ids(table, width, b0 * SA_KB + SA_KB);
        dma::wait_vm<0>();
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

    const float ltot = lsum + __shfl_xor(lsum, 32);
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
        a.tile_ml[part] = make_float2(ltot == ltot ? m * sc : INFINITY, ltot);
}

// ---------------------------------------------------------------- few columns
//
// A unit is up to 64 columns (row i, q head g: column i G + g) of one sequence and kv head;
// its keys are blocks of 64.  All units' blocks in a line (sequence, kv head, 64 columns, key
// block) are cut into equal runs, one a workgroup, whatever the lengths are.  A block is
// staged as attn_tile stages it, one ahead, also from one unit into the next.  A wave takes
// 16 keys x 16 columns at a time: S^T[16 x 16] = K Q^T on v_mfma_f32_16x16x32_bf16, whose result
// is operand B of O^T[D x 16] += Vt P^T on v_mfma_f32_16x16x16_bf16 as it lies in the registers.
// Of a sequence with at most 16 columns wave w takes keys 16 w .. 16 w + 15 of every block,
// with a maximum, a sum and an O of its own; of one with more, all the keys for columns 16 w ..
// 16 w + 15, so that the keys are read once for them all.  A wave's share of a unit is one
// part, number 4 (unit + workgroup) + wave (two consecutive runs meet in one unit at most, so
// the numbers differ).
//
// Bound by memory.  The copies read whole cache lines, 256 bytes a K row and 128 a Vt row:
// 5.6 TB/s (64 sequences of 4096 positions, no prefix, 191 us; operands loaded straight into
// the registers in the MFMA's order, 64 bytes of 16 rows an instruction, 250 us).
static_assert(SA_KB == 64, "own_keyblocks counts blocks of 64 keys");

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_t;

template <int D, bool ONE>
__device__ __forceinline__ void attn_own(const SaArgs &a, int wg, uint8_t *smem) {
    constexpr int U = D / 32, DT = D / 16;
    using Gm = SaGeo<D>;
    // behind the ring, of every sequence: its first row, and its keys; in the ring, before it
    // is used: the sequences' first blocks and units
    int32_t *first_row = reinterpret_cast<int32_t *>(smem + Gm::LDS), *keys = first_row + a.R;
    int32_t *off = reinterpret_cast<int32_t *>(smem), *unit = off + a.R, *wsum = unit + a.R;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int rows = live_rows(a);

    // a short burst between two waits, beside a column tile's waves that always have work: it
    // goes first (64 rows of up to 1023 own positions behind 8192 61.0 -> 58.8 us, host-timed;
    // 24 x 5 rows 24.4 -> 23.0)
    if (!a.any_big) __builtin_amdgcn_s_setprio(2);

    int t_before = 0, u_before = 0;
    for (int r0 = 0; r0 < a.R; r0 += SA_THREADS) {
        const int r = r0 + tid;
        int t = 0, u = 0;
        if (r < a.R) {
            const Seq s = seq_of(a, r, rows);
            const int kt = own_keyblocks(s.len);
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
        if (lane == 63) { wsum[w] = ts; wsum[4 + w] = us; }
        __syncthreads();
        int tb = t_before, ub = u_before;
        for (int i = 0; i < 4; ++i) {
            if (i < w) { tb += wsum[i]; ub += wsum[4 + i]; }
            t_before += wsum[i];
            u_before += wsum[4 + i];
        }
        if (r < a.R) { off[r] = tb + ts - t; unit[r] = ub + us - u; }
        __syncthreads();
    }
    if (wg == 0) {
        for (int r = tid; r < a.R; r += SA_THREADS) { a.own_off[r] = off[r]; a.own_unit[r] = unit[r]; }
        if (tid == 0) a.own_off[a.R] = t_before;
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
    __syncthreads();                                           // off and unit have been read: the ring is free

    struct Run {                 // the workgroup's share of one unit
        const int32_t *table;
        int hk, part, first, n;
        int col0;                // this wave's first column
        bool wide;               // a wave takes 16 columns and every key, not all columns and 16 keys
        int kb, stop;            // the key block, and the key its blocks end at
        int all, seen;           // keys that every, that some column sees
        int rel;                 // the unit's row i sees keys up to rel + i
        bool fresh;              // the unit's first block here
    };
    bool first_unit = true;
    auto open = [&](Run &s) {    // the unit of block t; t moves to its end in the run
        if (t >= t_end) return false;
        int first, len, n, kt, ct;
        for (;; ++r, in_seq = 0) {
            first = __builtin_amdgcn_readfirstlane(first_row[r]);
            len = __builtin_amdgcn_readfirstlane(keys[r]);
            n = (r + 1 < a.R ? __builtin_amdgcn_readfirstlane(first_row[r + 1]) : rows) - first;
            if (n > a.small_rows) n = 0;
            kt = own_keyblocks(len);
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
        s.col0 = s.wide ? (u - s.hk * ct) * 64 + 16 * w : 0;
        s.table = a.tables + (size_t)r * a.width;
        s.part = 4 * (u_next + wg) + w;
        ++u_next;
        s.kb = b0 * SA_KB;
        s.stop = b1 * SA_KB;
        s.rel = len - n;
        const int c0 = (u - s.hk * ct) * 64, last = min((c0 + 63) / a.G, n - 1);     // the unit's last row
        s.seen = clampi(s.rel + last + 1, 0, len);
        s.all = clampi(s.rel + c0 / a.G + 1, 0, len);
        return true;
    };
    auto advance = [&](Run &s) {
        s.kb += SA_KB;
        s.fresh = false;
        return s.kb < s.stop || open(s);
    };
    const Stager<D, ONE> stager(a, smem, lane, w);
    auto stage = [&](const Run &s, int st, const typename Stager<D, ONE>::Ids &ids) {
        const int lim = max(s.seen - 1 - s.kb, 0);
        if (ONE && lim < SA_KB - 1) stager.template copy<true>(s.hk, s.kb, lim, st, ids);
        else stager.template copy<false>(s.hk, s.kb, 0, st, ids);
    };
    auto load_q = [&](const Run &s, uint4 (&q)[U]) {
        const int i = (s.col0 + c) / a.G, h = s.hk * a.G + s.col0 + c - i * a.G;
#pragma unroll
        for (int x = 0; x < U; ++x) {
            q[x] = make_uint4(0u, 0u, 0u, 0u);
            if (i < s.n) q[x] = *reinterpret_cast<const uint4 *>(a.q + (size_t)(s.first + i) * a.q_stride + (size_t)h * D + 32 * x + 8 * g);
        }
    };
    bf16x8_t qv[U];
    // Of this lane's column: the exponents' reference (m = -inf: no key seen yet, 0 taken).  It
    // follows the maximum only when that is more than LAG above, so that most blocks spare
    // the two exchanges and the scaling of O: 64 rows of up to 1023 own positions behind 8192
    // 61.8 -> 60.0 us, host-timed, 24 x 5 rows 24.7 -> 24.1
    constexpr float LAG = 8.f;
    float m = -INFINITY, ref = 0.f, lsum = 0.f;
    f4 o[DT];
    int limit = -1;              // the last key this lane's column sees
    // keys 16 sub .. 16 sub + 15 of the block
    auto compute = [&](const Run &s, int st, int sub) {
        const uint8_t *K = smem + st * Gm::STAGE, *V = K + Gm::KTILE;
        const int k0 = s.kb + 16 * sub + 4 * g;            // this lane's keys: k0 .. k0 + 3
        f4 sv = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < U; ++y)
            sv = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                as_bf16x8(*reinterpret_cast<const uint4 *>(K + sa_kswz<D>(16 * sub + c, 4 * y + g))), qv[y], sv, 0, 0, 0);
        // Vt of the 16 keys: dim 16 y + c, keys 4 g .. 4 g + 3
        uint2 v[DT];
#pragma unroll
        for (int y = 0; y < DT; ++y)
            v[y] = *reinterpret_cast<const uint2 *>(V + sa_vswz(16 * y + c, 2 * sub + (g >> 1)) + 8 * (g & 1));
        float p[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) p[x] = sv[x] * a.scale_log2;
        const bool edge = s.kb + SA_KB > s.all;          // some column does not see all of the keys
        if (edge)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (k0 + x > limit) p[x] = -INFINITY;
        float bm = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
        if (__ballot(bm > m + LAG)) {
            bm = fmaxf(bm, __shfl_xor(bm, 16));
            bm = fmaxf(bm, __shfl_xor(bm, 32));
            const float mn = fmaxf(m, bm);
            ref = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - ref);
            m = mn;
            lsum *= alpha;
#pragma unroll
            for (int y = 0; y < DT; ++y)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[y][x] *= alpha;
        }
        float ps = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            p[x] = __builtin_amdgcn_exp2f(p[x] - ref);
            ps += p[x];
        }
        lsum += ps;
        const s16x4_t pb = __builtin_bit_cast(s16x4_t, make_uint2(cvt_pk_bf16(p[0], p[1]), cvt_pk_bf16(p[2], p[3])));
        // V of keys nobody sees is dropped, and values that are not finite where some
        // column does not see their key are added to those that do (as in attn_tile)
        if (edge) {
            const uint32_t m0 = (k0 + 0 < s.seen ? 0xFFFFu : 0u) | (k0 + 1 < s.seen ? 0xFFFF0000u : 0u);
            const uint32_t m1 = (k0 + 2 < s.seen ? 0xFFFFu : 0u) | (k0 + 3 < s.seen ? 0xFFFF0000u : 0u);
            uint32_t bits = 0;
#pragma unroll
            for (int y = 0; y < DT; ++y) {
                v[y].x &= m0;
                v[y].y &= m1;
                bits |= nonfinite_bits(v[y].x) | nonfinite_bits(v[y].y);
            }
            if (any_nonfinite(bits)) {
#pragma unroll 1
                for (int j = 0; j < 16; ++j) {
                    const int key = s.kb + 16 * sub + j;
                    const bool sees = key <= limit;
                    int quad = g;                        // opaque: no addresses of this rare loop are kept
                    asm volatile("" : "+v"(quad));
#pragma unroll
                    for (int y = 0; y < DT; ++y)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int d = 16 * y + 4 * quad + x;
                            const uint32_t z = *reinterpret_cast<const uint16_t *>(V + sa_vswz(d, 2 * sub + (j >> 3)) + 2 * (j & 7));
                            if (sees && (z & 0x7F80u) == 0x7F80u) o[y][x] += bf2f(z);
                        }
                }
#pragma unroll
                for (int y = 0; y < DT; ++y) v[y] = make_uint2(finite2(v[y].x), finite2(v[y].y));
            }
        }
#pragma unroll
        for (int y = 0; y < DT; ++y)
            o[y] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, v[y]), pb, o[y], 0, 0, 0);
    };
    auto end = [&](const Run &s) {           // the part: the unit's columns that are there
        float ltot = lsum + __shfl_xor(lsum, 16);
        ltot += __shfl_xor(ltot, 32);
        if ((s.col0 + c) / a.G >= s.n || s.part >= a.own_parts || c >= a.part_cols) return;
        const size_t at = (size_t)s.part * a.part_cols + c;
        float *po = a.own_o + at * D + 4 * g;
#pragma unroll
        for (int y = 0; y < DT; ++y) *reinterpret_cast<f4 *>(po + 16 * y) = o[y];
        if (g == 0) a.own_ml[at] = make_float2(ltot == ltot ? m : INFINITY, ltot);
    };

    Run f, n;                    // the block staged last, and the one after it
    uint4 qn[U];                 // q of the unit of block f, where f is its first
    open(f);
    stage(f, 0, stager.ids(f.table, a.width, f.kb));
    load_q(f, qn);
    n = f;
    bool more = advance(n);
    typename Stager<D, ONE>::Ids ids = stager.ids(n.table, a.width, n.kb);
    for (int st = 0;; st ^= 1) {
        // block f has landed, and the other stage has been read
        dma::wait_vm<0>();
        __syncthreads();
        const Run s = f;
        if (s.fresh) {
            const int i = (s.col0 + c) / a.G;
            limit = i >= s.n ? -1 : s.rel + i;
#pragma unroll
            for (int x = 0; x < U; ++x) qv[x] = as_bf16x8(qn[x]);
            m = -INFINITY;
            ref = lsum = 0.f;
#pragma unroll
            for (int y = 0; y < DT; ++y) o[y] = f4{0.f, 0.f, 0.f, 0.f};
        }
        const bool go = more;
        if (go) {
            f = n;
            stage(f, st ^ 1, ids);
            if (f.fresh) load_q(f, qn);
            more = advance(n);
            ids = stager.ids(n.table, a.width, n.kb);
        }
        if (s.col0 < s.n * a.G) {                        // (a wave of a wide unit may have no column)
            const int sub1 = s.wide ? 4 : w + 1;
            for (int sub = s.wide ? 0 : w; sub < sub1; ++sub) compute(s, st, sub);
            if (s.kb + SA_KB >= s.stop) end(s);
        }
        if (!go) break;
    }
}

// ---------------------------------------------------------------- both
//
// One launch: the own workgroups, which wait for memory, run beside tile workgroups, which
// keep the matrix units busy.
template <int D, bool ONE>
__global__ void __launch_bounds__(SA_THREADS) __attribute__((amdgpu_waves_per_eu(2))) attn_shared_kernel(SaArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    if ((int)blockIdx.x < a.tile_wgs) attn_tile<D, ONE>(a, (int)blockIdx.x, smem);
    else attn_own<D, ONE>(a, (int)blockIdx.x - a.tile_wgs, smem);
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
        if (s.n > a.small_rows && a.nsplit == 1) return;       // written by attn_tile
    }
    const int hk = h / a.G, gq = h - hk * a.G;
    const OwnParts own = own_parts_of(row, s.first, s.n, s.len, hk, gq, a.G, a.small_rows, a.own_off[r], a.own_unit[r],
                                      a.own_off[a.R], a.own_wgs, a.own_parts, a.part_cols);
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

// Into how many workgroups a column tile's key blocks are cut (wgs: workgroups without a cut).
// A key block takes a workgroup alone on its CU 1.5 us, 2.1 us where two share it, further
// ones wait (head_dim 128, measured: 300 rows behind 30000 positions 199 to 222 us in 3 pieces
// of 80 workgroups, 16 prompts 633 us in 2117 workgroups of 72 blocks; head_dim 64 ~0.8 of it,
// the softmax is the same), and the keys come at 5.3 TB/s at most; a row's part is written and
// read at about 2.5 TB/s and lengthens the merge by 0.06 us; at 1.3 TB/s where no tile takes own
// keys (last_is_whole false), which then come by themselves beside it.  Measured, 32 heads of
// 128 on 8: 200 rows of up to 500 own positions behind 1000 60 us, at 2.5 69; 64 of up to 1023
// behind 2048 40.3 and 41.5; but 300 rows of a prompt behind 8000 77 us at 1.3, 64 at 2.5.  The
// sum is least at the count returned: 16 rows of up to 300 own positions behind 65536 58 us (in
// 31), 65 in 24, 64 in 64; a prompt's 768 rows behind 2048 60 us (whole), 62 in 2.  64 pieces are
// what the merge's lanes take in one round; more have not been measured.
int tile_splits(long wgs, long blocks, long Hkv, long D, double part_bytes, bool last_is_whole, long cus) {
    const double stream = (double)Hkv * blocks * SA_KB * D * 4 / 5.3e6;
    int best = 1;
    double least = 1e30;
    for (int n = 1; n <= 64 && (n == 1 || n <= blocks); ++n) {
        const long w = wgs * n;
        const double block = (D == 64 ? 0.8 : 1.0) * (w <= cus ? 1.5 : 2.1 * ((w + 2 * cus - 1) / (2 * cus)));
        const double walk = (double)((blocks + n - 1) / n) * block;
        const double parts = n == 1 && last_is_whole ? 0 : n * (part_bytes / (last_is_whole ? 2.5e6 : 1.3e6) + 0.06);
        const double us = (walk > stream ? walk : stream) + parts;
        if (us < least) { least = us; best = n; }
    }
    return best;
}

struct SaPlan {
    int small_rows, rows_max, any_big, nsplit, own_wgs, use_tile, part_cols;
    long tiles, own_parts, part_rows;
    int by_seq, per_seq;     // the merge, and attn_tile's parts, by sequence: rows of each
    long tile_o, tile_ml, own_o, own_ml, own_idx, bytes;       // workspace offsets
};

// own_cap, prefix_cap: positions the tables have room for; max_new: at least the rows of
// the sequence with the most
SaPlan plan_shared(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new) {
    SaPlan p = {};
    const long G = H / Hkv, cols = N * G, cus = device_info().num_cus;
    if (max_new > N) max_new = N;
    p.small_rows = (int)(64 / G > 1 ? 64 / G : 1);
    p.any_big = max_new > p.small_rows;
    p.use_tile = p.any_big || prefix_cap > 0;
    p.tiles = (cols + SA_COLS - 1) / SA_COLS;
    const long wgs = p.tiles * Hkv;
    const long blocks = (prefix_cap + (p.any_big ? own_cap : 0) + SA_KB - 1) / SA_KB;
    p.nsplit = p.use_tile ? tile_splits(wgs, blocks, Hkv, D, (double)N * H * (8 * D + 16), p.any_big, cus) : 1;
    // attn_own: at most R coltiles of the most rows a sequence has here, and no more
    // than the rows make
    const long rows_max = max_new < p.small_rows ? max_new : p.small_rows;
    p.rows_max = (int)rows_max;
    long coltiles = R * ((rows_max * G + 63) / 64);
    if (coltiles > R + cols / 64) coltiles = R + cols / 64;
    const long keyblocks = coltiles * ((own_cap + SA_KB - 1) / SA_KB);
    // Equal runs of key blocks over what the column tiles leave of two workgroups a CU, so that
    // one round holds all (64 rows of up to 1023 own positions behind 2048, 64 tile workgroups:
    // 40 us with 448 here, 47 with 256 or 512), but at least one a CU (128 such rows behind 8192,
    // 256 tile workgroups: 87 us, 95 with two a CU).  Where tiles take own keys as well they end
    // at different times, and two a CU fill in (the mixed batch 70 us, 72 with one)
    long ow = p.use_tile && !p.any_big ? 2 * cus - wgs * p.nsplit : 2 * cus;
    if (ow < cus) ow = cus;
    if (ow > Hkv * keyblocks) ow = Hkv * keyblocks;
    p.own_wgs = (int)(ow < 1 ? 1 : ow);
    p.own_parts = 4 * (Hkv * coltiles + p.own_wgs);
    p.part_cols = (int)(rows_max * G < 16 ? (rows_max * G > 1 ? rows_max * G : 1) : 16);
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
    p.own_idx = at; at += up((R + 1) * 2 * 4);
    p.bytes = at;
    return p;
}

template <int D>
int run_shared(const SaArgs &a, const SaPlan &p, hipStream_t stream) {
    const int lds = SaGeo<D>::LDS + 2 * a.R * 4;
    // plan_shared counts on two workgroups a CU, whatever the sequences are: 2048 of up to 200
    // positions behind 4096, 32 heads of 128 on 8, 433 us, with one a CU 480
    static_assert(2 * (SaGeo<D>::LDS + 2 * SA_MAX_SEQ * 4) <= SA_CU_LDS, "two workgroups on a CU");
    auto kern = a.shift >= 6 ? attn_shared_kernel<D, true> : attn_shared_kernel<D, false>;
    // more than 64 KB of LDS has to be allowed, once a device
    static std::atomic<uint64_t> allowed[2];
    int dev = 0;
    SC_HIP_CHECK(hipGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(allowed[a.shift >= 6].load() & bit)) {
        SC_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                         SaGeo<D>::LDS + 2 * SA_MAX_SEQ * 4));
        allowed[a.shift >= 6].fetch_or(bit);
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.own_wgs + a.tile_wgs)), dim3(SA_THREADS), lds, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    const long merge_rows = p.by_seq ? (long)a.R * p.by_seq : a.N;
    const long heads = merge_rows * a.H;
    const bool wide = heads <= 4L * device_info().num_cus;
    auto merge = wide ? attn_merge_kernel<D, 4> : attn_merge_kernel<D, 1>;
    hipLaunchKernelGGL(merge, dim3((unsigned)(wide ? heads : (heads + 3) / 4)), dim3(256), 0, stream, a,
                       p.use_tile ? p.nsplit : 0, p.by_seq);
    SC_HIP_CHECK(hipGetLastError());
    return SC_OK;
}

bool bad_shape(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new) {
    return N < 0 || N >= (1L << 24) || R <= 0 || R > SA_MAX_SEQ || H <= 0 || Hkv <= 0 || H % Hkv || H > 4096 ||
           (D != 64 && D != 128) || own_cap <= 0 || own_cap >= (1L << 30) || prefix_cap < 0 || prefix_cap >= (1L << 30) ||
           max_new < 0 ||
           // attn_own numbers its key blocks in 32 bits
           R * Hkv * ((H / Hkv + 63) / 64) * ((own_cap + SA_KB - 1) / SA_KB) >= (1L << 31);
}

}  // namespace

long attention_shared_workspace_bytes(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap,
                                      long max_new) {
    if (bad_shape(N, R, H, Hkv, D, own_cap, prefix_cap, max_new) || N == 0) return 0;
    return plan_shared(N, R, H, Hkv, D, own_cap, prefix_cap, max_new).bytes;
}

int launch_attention_shared(const uint16_t *q, long q_stride, const uint16_t *kc, const uint16_t *vt, long n_blocks,
                            long bs, const int32_t *row_starts, const int32_t *lengths, const int32_t *tables,
                            long width, const int32_t *prefix_table, long prefix_width, const int32_t *prefix_len,
                            uint16_t *out, long out_stride, long N, long R, long H, long Hkv, long D, float scale,
                            long max_new, void *workspace, long workspace_bytes, hipStream_t stream) {
    if (N == 0) return SC_OK;
    if (!q || !kc || !vt || !row_starts || !lengths || !tables || !out || (prefix_width > 0 && (!prefix_table || !prefix_len)))
        return set_error(SC_EINVAL, "attention_shared: null pointer");
    if (D != 64 && D != 128) return set_error(SC_EUNSUPPORTED, "attention_shared: head_dim %ld (64 or 128 supported)", D);
    const int shift = block_shift(bs);
    if (shift < 0) return set_error(SC_EINVAL, "attention_shared: block size %ld (16, 32, 64, 128 or 256)", bs);
    if (width <= 0 || width >= (1L << 26) || prefix_width < 0 || prefix_width >= (1L << 26) ||
        bad_shape(N, R, H, Hkv, D, width * bs, prefix_width * bs, max_new))
        return set_error(SC_EINVAL, "attention_shared: bad shape rows=%ld sequences=%ld (at most %d) H=%ld Hkv=%ld tables=%ld/%ld",
                         N, R, SA_MAX_SEQ, H, Hkv, width, prefix_width);
    if (n_blocks <= 0 || n_blocks * bs >= (1L << 31)) return set_error(SC_EINVAL, "attention_shared: bad pool size");
    // the maximum is taken of the unscaled scores
    if (!(scale >= 1e-30f && scale <= 1e30f)) return set_error(SC_EINVAL, "attention_shared: scale must be positive (1e-30 to 1e30)");
    if (q_stride < H * D || out_stride < H * D || q_stride % 8 || out_stride % 4)
        return set_error(SC_EINVAL, "attention_shared: bad row strides");
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vt) % 16 || (uintptr_t)out % 8)
        return set_error(SC_EINVAL, "attention_shared: misaligned pointers");
    const SaPlan p = plan_shared(N, R, H, Hkv, D, width * bs, prefix_width * bs, max_new);
    if (!workspace || workspace_bytes < p.bytes || (uintptr_t)workspace % 16)
        return set_error(SC_EINVAL, "attention_shared: a 16-byte aligned workspace of %ld bytes required", p.bytes);
    if (p.tiles * p.nsplit * Hkv >= (1L << 30) || N * H >= (1L << 31))
        return set_error(SC_EINVAL, "attention_shared: too many rows");
    SaArgs a;
    a.q = q; a.q_stride = q_stride; a.kc = kc; a.vt = vt; a.out = out; a.out_stride = out_stride;
    a.row_starts = row_starts; a.lengths = lengths; a.tables = tables;
    a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.N = (int)N; a.R = (int)R; a.H = (int)H; a.Hkv = (int)Hkv; a.G = (int)(H / Hkv);
    a.width = (int)width; a.shift = shift; a.n_blocks = (int)n_blocks; a.prefix_width = (int)prefix_width;
    a.small_rows = p.small_rows; a.any_big = p.any_big; a.nsplit = p.nsplit;
    a.own_wgs = p.own_wgs;
    a.tile_wgs = p.use_tile ? (int)(p.tiles * p.nsplit * Hkv) : 0;
    a.tiles = (int)p.tiles;
    a.part_rows = (int)p.part_rows; a.per_seq = p.per_seq;
    a.pair_half = p.any_big && a.tile_wgs >= 2 * device_info().num_cus ? device_info().num_cus : 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    char *ws = static_cast<char *>(workspace);
    a.tile_o = reinterpret_cast<float *>(ws + p.tile_o);
    a.tile_ml = reinterpret_cast<float2 *>(ws + p.tile_ml);
    a.own_o = reinterpret_cast<float *>(ws + p.own_o);
    a.own_ml = reinterpret_cast<float2 *>(ws + p.own_ml);
    a.own_parts = (int)p.own_parts; a.part_cols = p.part_cols;
    a.own_off = reinterpret_cast<int32_t *>(ws + p.own_idx);
    a.own_unit = a.own_off + R + 1;
    return D == 128 ? run_shared<128>(a, p, stream) : run_shared<64>(a, p, stream);
}

}  // namespace sc

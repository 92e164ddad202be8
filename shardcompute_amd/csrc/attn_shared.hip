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
#include "attn_shared_core.h"

#include <atomic>

namespace sc {

namespace {

constexpr int SA_COLS = 128;

struct SharedArgs : SaArgs {
    const uint16_t *kc, *vt;
};

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
// The copies of a key block (64 keys of one kv head) into a stage of the ring, by every wave
// of the workgroup.  ONE: a key block lies in one cache block (block sizes from 64 up).
template <int D, bool ONE>
struct Stager {
    using Gm = SaGeo<D>;
    using Args = SharedArgs;
    static constexpr int COLS = SA_COLS;
    static constexpr bool HALF = false;
    // cache blocks of a key block: ONE, its block's number; else those of the wave's 16
    // keys of K and of the lane's two chunks of Vt
    struct Ids { int k, v0, v1; };
    using Flow = Ids;            // attn_tile's: one key block ahead of its copies
    const SharedArgs &a;
    uint8_t *smem;
    int lane, w, sh, kr, vd, vc;
    size_t blk_bytes;

    // This lane's share.  Wave w issues K instructions of the keys 16 w .. 16 w + 15 and Vt
    // instructions of D / 4 dims; a lane's dim row and chunk of Vt instruction qq differ
    // between even and odd qq only in bit 2 of the chunk.
    __device__ __forceinline__ Stager(const SharedArgs &a_, uint8_t *smem_, int lane_, int w_)
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
    __device__ __forceinline__ void open(Flow &f, int hk, const int32_t *table, int width, int b0) const {
        f = ids(table, width, b0 * SA_KB);
        copy<false>(hk, b0 * SA_KB, 0, 0, f);
        f = ids(table, width, b0 * SA_KB + SA_KB);
    }
    __device__ __forceinline__ void next(Flow &f, int hk, const int32_t *table, int width, int blk, int st) const {
        copy<false>(hk, blk * SA_KB + SA_KB, 0, st ^ 1, f);
        f = ids(table, width, blk * SA_KB + 2 * SA_KB);
    }
    __device__ __forceinline__ void landed() const { dma::wait_vm<0>(); }
};

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
__device__ __forceinline__ void attn_own(const SharedArgs &a, int wg, uint8_t *smem) {
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
__global__ void __launch_bounds__(SA_THREADS) __attribute__((amdgpu_waves_per_eu(2))) attn_shared_kernel(SharedArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    if ((int)blockIdx.x < a.tile_wgs) attn_tile<D, Stager<D, ONE>>(a, (int)blockIdx.x, smem);
    else attn_own<D, ONE>(a, (int)blockIdx.x - a.tile_wgs, smem);
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

// own_cap, prefix_cap: positions the tables have room for; max_new: at least the rows of
// the sequence with the most
SaPlan plan_shared(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new) {
    SaPlan p;
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
    lay_out(p, N, R, H, D);
    return p;
}

template <int D>
int run_shared(const SharedArgs &a, const SaPlan &p, hipStream_t stream) {
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
    return merge_parts<D>(a, p, stream);
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
    SharedArgs a;
    a.q = q; a.q_stride = q_stride; a.kc = kc; a.vt = vt; a.out = out; a.out_stride = out_stride;
    a.row_starts = row_starts; a.lengths = lengths; a.tables = tables;
    a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.N = (int)N; a.R = (int)R; a.H = (int)H; a.Hkv = (int)Hkv; a.G = (int)(H / Hkv);
    a.width = (int)width; a.shift = shift; a.n_blocks = (int)n_blocks; a.prefix_width = (int)prefix_width;
    fill_args(a, p, workspace);
    a.pair_half = p.any_big && a.tile_wgs >= 2 * device_info().num_cus ? device_info().num_cus : 0;
    a.scale_log2 = scale * 1.4426950408889634f;
    return D == 128 ? run_shared<128>(a, p, stream) : run_shared<64>(a, p, stream);
}

}  // namespace sc

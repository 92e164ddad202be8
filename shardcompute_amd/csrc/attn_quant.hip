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
#include "sc_common.h"
#include "kv_cells.h"
#include "dma_util.h"

#include <math.h>
#include <type_traits>

namespace sc {

int block_shift(long bs);       // blocks.hip

namespace {

using f4 = dma::f4;

struct QaArgs {
    const uint16_t *q;
    long q_stride;
    const uint8_t *pool;
    uint16_t *out;
    long out_stride;
    const int32_t *row_starts, *lengths, *tables, *prefix_table, *prefix_len;
    int N, R, H, Hkv, G, width, shift, n_blocks, prefix_width;
    float scale_log2;
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

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

// One wave 16 columns (q heads of one kv head) of one row.
template <int D, int BITS>
__global__ void __launch_bounds__(256) attn_quantized_kernel(QaArgs a) {
    using C = Cell<D, BITS>;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int tiles = (a.G + 15) / 16;
    const long wid = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = (int)(wid / (a.Hkv * tiles)), rest = (int)(wid - (long)row * (a.Hkv * tiles));
    const int hk = rest / tiles, tile = rest - hk * tiles;
    const int rows = clampi(a.row_starts[a.R], 0, a.N);
    if (row >= rows || row < a.row_starts[0]) return;
    int lo = 0, hi = a.R;                                      // the last sequence that starts at or before the row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.row_starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    const int r = lo, first = clampi(a.row_starts[r], 0, rows), next = clampi(a.row_starts[r + 1], 0, rows);
    if (row < first || row >= next) return;
    const int len = clampi(a.lengths[r], 0, a.width << a.shift);
    const int own = clampi(len - (next - first) + (row - first) + 1, 0, len);
    const int P = a.prefix_width ? clampi(a.prefix_len[0], 0, a.prefix_width << a.shift) : 0;

    const int head = tile * 16 + c, h = hk * a.G + head;
    Columns<D, BITS> col;
    col.open(head < a.G ? a.q + (size_t)row * a.q_stride + (size_t)h * D : nullptr, g);
    const int cells_log2 = a.shift - 4;
    auto walk = [&](const int32_t *table, int width, int end) {
        for (int kb = 0; kb < end; kb += 32) {
            if (kb && kb % Columns<D, BITS>::SETTLE == 0) col.settle();
            CellRegs<D, BITS> x[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int t = min(kb + 16 * j, (width << a.shift) - 16);
                const int blk = clampi(__builtin_amdgcn_readfirstlane(table[t >> a.shift]), 0, a.n_blocks - 1);
                x[j].load(a.pool + ((((size_t)blk * a.Hkv + hk) << cells_log2) + ((t >> 4) & ((1 << cells_log2) - 1))) * C::BYTES, lane);
            }
            if (kb + 32 <= end) col.template take<false>(x, kb, kb + 16, 0, a.scale_log2, lane);
            else col.template take<true>(x, kb, kb + 16, end - 1, a.scale_log2, lane);
        }
    };
    walk(a.prefix_table, a.prefix_width, P);
    walk(a.tables + (size_t)r * a.width, a.width, own);
    const float l = col.close(), inv = l == 0.f ? 0.f : 1.f / l;
    if (head >= a.G) return;
    uint16_t *po = a.out + (size_t)row * a.out_stride + (size_t)h * D + 4 * g;
#pragma unroll
    for (int y = 0; y < D / 16; ++y)
        *reinterpret_cast<uint2 *>(po + 16 * y) = make_uint2(cvt_pk_bf16(col.o[y][0] * inv, col.o[y][1] * inv),
                                                             cvt_pk_bf16(col.o[y][2] * inv, col.o[y][3] * inv));
}

bool bad_shape(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap, long max_new, int bits) {
    return N < 0 || N >= (1L << 24) || R <= 0 || R > 2048 || H <= 0 || Hkv <= 0 || H % Hkv || H > 4096 ||
           kv_cell_bytes(D, bits) == 0 || own_cap <= 0 || own_cap >= (1L << 30) || prefix_cap < 0 ||
           prefix_cap >= (1L << 30) || max_new < 0;
}

}  // namespace

long attention_quantized_workspace_bytes(long N, long R, long H, long Hkv, long D, long own_cap, long prefix_cap,
                                         long max_new, int bits) {
    (void)N; (void)R; (void)H; (void)Hkv; (void)D; (void)own_cap; (void)prefix_cap; (void)max_new; (void)bits;
    return 0;
}

int launch_attention_quantized(const uint16_t *q, long q_stride, const uint8_t *pool, long n_blocks, long bs, int bits,
                               const int32_t *row_starts, const int32_t *lengths, const int32_t *tables, long width,
                               const int32_t *prefix_table, long prefix_width, const int32_t *prefix_len, uint16_t *out,
                               long out_stride, long N, long R, long H, long Hkv, long D, float scale, long max_new,
                               void *workspace, long workspace_bytes, hipStream_t stream) {
    (void)workspace; (void)workspace_bytes;
    if (N == 0) return SC_OK;
    if (!q || !pool || !row_starts || !lengths || !tables || !out || (prefix_width > 0 && (!prefix_table || !prefix_len)))
        return set_error(SC_EINVAL, "attention_quantized: null pointer");
    if (kv_cell_bytes(D, bits) == 0)
        return set_error(SC_EUNSUPPORTED, "attention_quantized: head_dim %ld in %d bits (64 or 128 in 4 or 8 supported)", D, bits);
    const int shift = block_shift(bs);
    if (shift < 0) return set_error(SC_EINVAL, "attention_quantized: block size %ld (16, 32, 64, 128 or 256)", bs);
    if (width <= 0 || width >= (1L << 26) || prefix_width < 0 || prefix_width >= (1L << 26) ||
        bad_shape(N, R, H, Hkv, D, width * bs, prefix_width * bs, max_new, bits))
        return set_error(SC_EINVAL, "attention_quantized: bad shape rows=%ld sequences=%ld (at most 2048) H=%ld Hkv=%ld tables=%ld/%ld",
                         N, R, H, Hkv, width, prefix_width);
    if (n_blocks <= 0 || n_blocks * bs >= (1L << 31)) return set_error(SC_EINVAL, "attention_quantized: bad pool size");
    // maxima are taken of the scores in log2 units
    if (!(scale >= 1e-30f && scale <= 1e30f)) return set_error(SC_EINVAL, "attention_quantized: scale must be positive (1e-30 to 1e30)");
    if (q_stride < H * D || out_stride < H * D || q_stride % 8 || out_stride % 4)
        return set_error(SC_EINVAL, "attention_quantized: bad row strides");
    if (((uintptr_t)q | (uintptr_t)pool) % 16 || (uintptr_t)out % 8)
        return set_error(SC_EINVAL, "attention_quantized: misaligned pointers");
    if (N * H >= (1L << 31)) return set_error(SC_EINVAL, "attention_quantized: too many rows");
    QaArgs a;
    a.q = q; a.q_stride = q_stride; a.pool = pool; a.out = out; a.out_stride = out_stride;
    a.row_starts = row_starts; a.lengths = lengths; a.tables = tables;
    a.prefix_table = prefix_table; a.prefix_len = prefix_len;
    a.N = (int)N; a.R = (int)R; a.H = (int)H; a.Hkv = (int)Hkv; a.G = (int)(H / Hkv);
    a.width = (int)width; a.shift = shift; a.n_blocks = (int)n_blocks; a.prefix_width = (int)prefix_width;
    a.scale_log2 = scale * 1.4426950408889634f;
    const long waves = N * Hkv * ((a.G + 15) / 16);
    if (waves >= (1L << 26)) return set_error(SC_EINVAL, "attention_quantized: too many rows");
    auto kern = D == 128 ? (bits == 4 ? attn_quantized_kernel<128, 4> : attn_quantized_kernel<128, 8>)
                         : (bits == 4 ? attn_quantized_kernel<64, 4> : attn_quantized_kernel<64, 8>);
    hipLaunchKernelGGL(kern, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    return SC_OK;
}

}  // namespace sc

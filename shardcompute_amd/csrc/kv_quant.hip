// A key/value cache in blocks of 4- or 8-bit codes: the append of a step's keys and values
// (rope_append_quantized) and reading positions back (read_quantized).  Layout: kv_cells.h.
#include "sc_common.h"
#include "kv_cells.h"

namespace sc {

int block_shift(long bs);       // blocks.hip

namespace {

// ---------------------------------------------------------------- rotation, quantization, append
//
// Row t of qkv goes to slot slots[t], rotated for positions[t] as rope_append_blocks rotates it
// (the same fp32 products and sums, rounded to bf16); k and v are then quantized as `quantize`
// quantizes a weight row, bit for bit, 64 dims a group:
//     scale = max((max - min) / n, 1e-7), n = 2^bits - 1; edge = |min| > |max| ? min : max
//     (scale negated where edge = max); q0 = rint(edge / scale); where q0 != 0: scale = edge / q0
//     and bias = edge, else bias = 0; code = clamp(rint((x - bias) / scale), 0, n)
// in fp32; scale and bias are kept as bf16, as NaN where a value of the group is not finite.  Rows whose slot or position lies outside the pool
// or the tables are left alone.
struct QuantAppendArgs {
    const uint16_t *qkv;
    long qkv_stride;
    uint16_t *q;
    long q_stride;
    uint8_t *pool;
    const float *cos_t, *sin_t;
    const int32_t *slots, *positions;
    int N, H, Hkv, shift, table_len;
    long n_slots;
    int kv_wgs, kv_rows;     // workgroups that have keys and values, rows of one
    int heads_per_wave;      // of q, the others'
};

struct Affine { float scale, bias; };

template <int BITS>
__device__ __forceinline__ Affine affine_of(float lo, float hi) {
    constexpr float n_bins = (float)((1 << BITS) - 1);
    Affine a;
    a.scale = fmaxf((hi - lo) / n_bins, 1e-7f);
    const bool use_min = fabsf(lo) > fabsf(hi);
    a.scale = use_min ? a.scale : -a.scale;
    const float edge = use_min ? lo : hi;
    const float q0 = rintf(edge / a.scale);
    a.bias = 0.f;
    if (q0 != 0.f) {
        a.scale = edge / q0;
        a.bias = edge;
    }
    return a;
}
template <int BITS>
__device__ __forceinline__ uint32_t code_of(float x, const Affine &a) {
    constexpr float n_bins = (float)((1 << BITS) - 1);
    return (uint32_t)fminf(fmaxf(rintf((x - a.bias) / a.scale), 0.f), n_bins);
}

__device__ __forceinline__ uint4 pack8(const float *x) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// D / 16 lanes of a row's head: a lane has the dims i0 .. i0 + 7 and D / 2 above them, so that a
// pair that is rotated together is in one lane.
template <int D>
struct Lane {
    uint4 a1, a2;
    float c[8], sn[8];
    __device__ __forceinline__ void values(const uint16_t *p) {
        a1 = *reinterpret_cast<const uint4 *>(p);
        a2 = *reinterpret_cast<const uint4 *>(p + D / 2);
    }
    __device__ __forceinline__ void angles(const QuantAppendArgs &a, int pos, int i0) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const float4 cv = *reinterpret_cast<const float4 *>(a.cos_t + (size_t)pos * (D / 2) + i0 + 4 * q);
            const float4 sv = *reinterpret_cast<const float4 *>(a.sin_t + (size_t)pos * (D / 2) + i0 + 4 * q);
            c[4 * q] = cv.x; c[4 * q + 1] = cv.y; c[4 * q + 2] = cv.z; c[4 * q + 3] = cv.w;
            sn[4 * q] = sv.x; sn[4 * q + 1] = sv.y; sn[4 * q + 2] = sv.z; sn[4 * q + 3] = sv.w;
        }
    }
    __device__ __forceinline__ void rotate(uint4 &o1, uint4 &o2) const {
        float x[2][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x1 = bfe(a1, e), x2 = bfe(a2, e);
            x[0][e] = add_rn(mul_rn(x1, c[e]), mul_rn(-x2, sn[e]));
            x[1][e] = add_rn(mul_rn(x2, c[e]), mul_rn(x1, sn[e]));
        }
        o1 = pack8(x[0]);
        o2 = pack8(x[1]);
    }
};

// maxima over the D / 16 lanes of a head (every lane has it)
template <int D>
__device__ __forceinline__ float head_max(float v) {
    v = fmaxf(v, dpp_mov<DPP_XOR1>(v));
    v = fmaxf(v, dpp_mov<DPP_XOR2>(v));
    return D == 128 ? fmaxf(v, dpp_mov<DPP_HALF_MIRROR>(v)) : v;
}

// Workgroups with keys and values have kv_rows rows of one kv head, the others q heads of a row a
// wave.  Codes go to LDS first, as the rows lie in a cell, and leave from there: a key in
// pieces of 16 bytes (8 of 4 bits and 64 dims), 4 values of consecutive slots that begin at a
// multiple of 4 in pieces of 16 too (a lane of the cell: PLANE), other values byte by byte.
//
// Prompts: 22000 rows of 8 + 1 heads of 128 in 8 bits, 113 MB, 28.1 us: 4.0 TB/s, 63 % of what a large
// copy moves; what holds it there has not been found.  Single rows are bound by the chain slot, row,
// scale, codes, store (64 rows of 32 + 8 heads in 4 bits: 5.7 us).  A wave with the keys of one row
// and no LDS, its values stored byte by byte: 48.8 and 9.7 us.
constexpr int QA_ROWS = 32, QA_FEW_ROWS = 16;
constexpr long QA_FEW = 512;          // rows up to which the groups are the smaller

template <int D, int BITS>
__global__ void __launch_bounds__(256) rope_append_quantized_kernel(QuantAppendArgs a) {
    using C = Cell<D, BITS>;
    constexpr int LPH = D / 16, HALF = D / 2;
    constexpr int KROW = D * BITS / 8, KPAD = KROW + 16, VPAD = QA_ROWS + 8;
    __shared__ __align__(16) uint8_t kcode[QA_ROWS * KPAD];      // [row][plane, g][PLANE]
    __shared__ __align__(16) uint8_t vcode[D * VPAD];            // [dim][row]
    __shared__ int slot_of[QA_ROWS + 4];
    const int tid = threadIdx.x, lane = tid & 63;
    if ((int)blockIdx.x >= a.kv_wgs) {
        constexpr int HPW = 64 / LPH;
        const int parts = (a.H + a.heads_per_wave - 1) / a.heads_per_wave;
        const long wid = (long)((int)blockIdx.x - a.kv_wgs) * 4 + (tid >> 6);
        const int tok = (int)(wid / parts), part = (int)(wid - (long)tok * parts);
        if (tok >= a.N) return;
        const int i0 = 8 * (lane % LPH), h0 = part * a.heads_per_wave + lane / LPH;
        const int slot = a.slots[tok], pos = a.positions[tok];
        const uint16_t *row = a.qkv + (size_t)tok * a.qkv_stride + i0;
        Lane<D> x;
        x.values(row + (size_t)min(h0, a.H - 1) * D);            // on its way while the slot and the angles are read
        if (slot < 0 || slot >= a.n_slots || pos < 0 || pos >= a.table_len) return;
        x.angles(a, pos, i0);
        const int h1 = min(a.H, (part + 1) * a.heads_per_wave);
#pragma unroll 4
        for (int h = h0; h < h1; h += HPW) {
            if (h != h0) x.values(row + (size_t)h * D);
            uint4 o1, o2;
            x.rotate(o1, o2);
            uint16_t *dst = a.q + (size_t)tok * a.q_stride + (size_t)h * D + i0;
            *reinterpret_cast<uint4 *>(dst) = o1;
            *reinterpret_cast<uint4 *>(dst + HALF) = o2;
        }
        return;
    }
    const int hk = (int)blockIdx.x % a.Hkv, t0 = (int)blockIdx.x / a.Hkv * a.kv_rows, rows = min(a.kv_rows, a.N - t0);
    const int shift = a.shift, cells = 1 << (shift - 4);
    auto cell_of = [&](int slot) {
        return a.pool + (((size_t)(slot >> shift) * a.Hkv + hk) * cells + ((slot & ((1 << shift) - 1)) >> 4)) * C::BYTES;
    };
    // Threads 0 .. 127 have keys, the others values.
    constexpr int STEP = 128 / LPH;                              // rows at a time
    const bool value = tid >= 128;
    const int hl = lane % LPH, i0 = 8 * hl;
    constexpr int TIMES = QA_ROWS / STEP;
    Lane<D> xs[TIMES];
    int slots[TIMES], poss[TIMES] = {};
#pragma unroll
    for (int u = 0; u < TIMES; ++u) {                            // all loads before the first use
        const int r = u * STEP + (tid & 127) / LPH, tok = t0 + r;
        slots[u] = -1;
        if (r < rows) {
            slots[u] = a.slots[tok];
            poss[u] = a.positions[tok];
            xs[u].values(a.qkv + (size_t)tok * a.qkv_stride + (size_t)(a.H + (value ? a.Hkv : 0) + hk) * D + i0);
        }
    }
#pragma unroll
    for (int u = 0; u < TIMES; ++u) {
        const int r = u * STEP + (tid & 127) / LPH, pos = poss[u];
        int slot = slots[u];
        Lane<D> &x = xs[u];
        if (slot >= a.n_slots || pos < 0 || pos >= a.table_len) slot = -1;
        if (value && hl == 0) slot_of[r] = slot;
        if (slot < 0) continue;                                  // (all of a head's lanes)
        if (!value) {
            x.angles(a, pos, i0);
            x.rotate(x.a1, x.a2);
        }
        float v[2][8], lo[2], hi[2], zero[2];                    // zero: 0, or no number if a value is not finite
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[y][e] = bfe(y ? x.a2 : x.a1, e);
            lo[y] = hi[y] = v[y][0];
            zero[y] = v[y][0] * 0.f;
#pragma unroll
            for (int e = 1; e < 8; ++e) {
                lo[y] = fminf(lo[y], v[y][e]);
                hi[y] = fmaxf(hi[y], v[y][e]);
                zero[y] = fmaf(v[y][e], 0.f, zero[y]);
            }
        }
        // 128 dims: a group in each half; 64: both halves one group
        if (C::GROUPS == 1) {
            lo[0] = fminf(lo[0], lo[1]);
            hi[0] = fmaxf(hi[0], hi[1]);
            zero[0] += zero[1];
        }
        Affine af[2];
#pragma unroll
        for (int y = 0; y < C::GROUPS; ++y) {
            lo[y] = -head_max<D>(-lo[y]);
            hi[y] = head_max<D>(hi[y]);
            af[y] = affine_of<BITS>(lo[y], hi[y]);
            // minima and maxima pass a NaN over: the group's scale keeps it
            if (head_max<D>(zero[y] == 0.f ? 0.f : 1.f) != 0.f) af[y].scale = af[y].bias = __builtin_nanf("");
        }
        if (C::GROUPS == 1) af[1] = af[0];
        if (hl < C::GROUPS)
            *reinterpret_cast<uint32_t *>(cell_of(slot) + C::meta(slot & 15, (value ? C::GROUPS : 0) + hl)) =
                f2bf(hl ? af[1].scale : af[0].scale) | f2bf(hl ? af[1].bias : af[0].bias) << 16;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            uint32_t code[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) code[e] = code_of<BITS>(v[y][e], af[y]);
            const int o = hl + y * LPH;                          // of the row's chunks of 8 dims
            if (value) {
#pragma unroll
                for (int e = 0; e < 8; ++e) vcode[(8 * o + e) * VPAD + r] = (uint8_t)code[e];
            } else {
                const int grp = o >> 3, g = (o >> 1) & 3;
                if (BITS == 4) {
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < 8; ++e) w |= code[e] << (4 * ((e >> 1) + 4 * (e & 1)));
                    *reinterpret_cast<uint32_t *>(kcode + r * KPAD + g * C::PLANE + 8 * grp + 4 * (o & 1)) = w;
                } else {
                    uint32_t w[2] = {0u, 0u};
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e >> 2] |= code[e] << (8 * (e & 3));
                    *reinterpret_cast<uint2 *>(kcode + r * KPAD + (4 * grp + g) * 16 + 8 * (o & 1)) = make_uint2(w[0], w[1]);
                }
            }
        }
    }
    __syncthreads();
    // keys: a piece is PLANE bytes of a row
    constexpr int PIECES = 4 * C::PLANES;
    for (int i = tid; i < rows * PIECES; i += 256) {
        const int r = i / PIECES, pc = i % PIECES, slot = slot_of[r];
        if (slot < 0) continue;
        uint8_t *dst = cell_of(slot) + 1024 * (pc >> 2) + (16 * (pc & 3) + (slot & 15)) * C::PLANE;
        const uint8_t *src = kcode + r * KPAD + pc * C::PLANE;
        if (C::PLANE == 16) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
        else *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(src);
    }
    // values: rows r .. r + 3 are a quad if their slots are 4 q .. 4 q + 3
    auto leads = [&](int r) {
        const int s = slot_of[r];
        return r + 3 < rows && s >= 0 && (s & 3) == 0 && slot_of[r + 1] == s + 1 && slot_of[r + 2] == s + 2 && slot_of[r + 3] == s + 3;
    };
    constexpr int WORDS = C::PLANE / 4, PER_ROW = 16 * C::PLANES;
    for (int i = tid; i < rows * PER_ROW; i += 256) {
        const int r = i / PER_ROW, l = i % 16, pl = i / 16 % C::PLANES;
        if (!leads(r)) continue;
        const int slot = slot_of[r];
        // 4 codes of dim d, rows r .. r + 3: bytes r .. r + 3 of two aligned words
        auto four = [&](int d) {
            const uint32_t *p = reinterpret_cast<const uint32_t *>(vcode + d * VPAD + (r & ~3));
            return __builtin_amdgcn_alignbyte(p[1], p[0], r & 3);
        };
        uint32_t w[WORDS];
#pragma unroll
        for (int m = 0; m < WORDS; ++m)
            w[m] = BITS == 4 ? four(32 * m + l) | four(32 * m + 16 + l) << 4 : four(16 * (4 * pl + m) + l);
        uint8_t *dst = cell_of(slot) + C::CODES + 1024 * pl + (16 * ((slot & 15) >> 2) + l) * C::PLANE;
        if constexpr (WORDS == 4) *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    }
    constexpr int BYTES = D * BITS / 8;
    for (int i = tid; i < rows * BYTES; i += 256) {
        const int r = i / BYTES, b = i % BYTES, slot = slot_of[r];
        if (slot < 0) continue;
        const int first = r - (slot & 3);
        if (first >= 0 && leads(first) && slot_of[first] == slot - (slot & 3)) continue;
        // byte b: of 4 bits, dims 32 m + l and 16 above it
        const int l = b & 15, m = b >> 4, d = BITS == 4 ? 32 * m + l : 16 * m + l;
        const uint32_t lo = vcode[d * VPAD + r], up = BITS == 4 ? vcode[(d + 16) * VPAD + r] : 0u;
        cell_of(slot)[C::value_byte(slot & 15, d)] = (uint8_t)(lo | up << 4);
    }
}

// ---------------------------------------------------------------- reading back
//
// k, v [n, Hkv, D] bf16 of the positions at slots[n]: bf16(scale code + bias), the sum rounded
// once (as dequantize); 0 for a slot outside the pool.  D / 8 lanes of a row of one kv head: a lane
// has 8 dims of the key, and of the value the dims l, 16 + l, .. of its place in the cell (two
// places with 64 dims), which go through LDS into the row's order.
//
// Bound by memory: 40000 positions of 8 kv heads of 128 in 4 bits (164 MB of outputs, a pool of 46):
// 35 us into outputs that the caches hold with two pools in turn, 48 with four, 53 into outputs that
// were not written lately.  With stores past the caches it takes 34 to 36 in each case, but with
// whoever uses the outputs next (one pass over them) 103 us in place of 95: ordinary stores.
struct QuantReadArgs {
    const uint8_t *pool;
    const int32_t *slots;
    uint16_t *k, *v;
    long n, n_slots;
    int Hkv, shift;
};

template <int D, int BITS>
__global__ void __launch_bounds__(256) read_quantized_kernel(QuantReadArgs a) {
    using C = Cell<D, BITS>;
    constexpr int OCT = D / 8, ROWS = 256 / OCT, PAD = D + 8;
    __shared__ __align__(16) uint16_t tile[ROWS * PAD];
    const int hk = (int)(blockIdx.x % (unsigned)a.Hkv), r = threadIdx.x / OCT, o = threadIdx.x % OCT;
    const long row = (long)(blockIdx.x / (unsigned)a.Hkv) * ROWS + r;
    const int slot = row < a.n ? a.slots[row] : -1;
    uint4 key = make_uint4(0u, 0u, 0u, 0u), val = key;
    const bool there = slot >= 0 && slot < a.n_slots;
    if (there) {
        const int t = slot & 15;
        const uint8_t *cell = a.pool + (((size_t)(slot >> a.shift) * a.Hkv + hk) * (1u << (a.shift - 4)) + ((slot & ((1 << a.shift) - 1)) >> 4)) * C::BYTES;
        // the place's codes: byte t & 3 of each word is this position's
        constexpr int PLACES = 16 / OCT, WORDS = C::LANE / 4;
        uint32_t w[PLACES][WORDS], kw[2], m[C::ITEMS];
#pragma unroll
        for (int q = 0; q < PLACES; ++q) {
            const int l = o + q * OCT;
#pragma unroll
            for (int pl = 0; pl < C::PLANES; ++pl) {
                const uint8_t *p = cell + C::CODES + 1024 * pl + (16 * (t >> 2) + l) * C::PLANE;
                if constexpr (C::PLANE == 16) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(p);
                    w[q][4 * pl] = x.x; w[q][4 * pl + 1] = x.y; w[q][4 * pl + 2] = x.z; w[q][4 * pl + 3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2 *>(p);
                    w[q][0] = x.x; w[q][1] = x.y;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < BITS / 4; ++e) kw[e] = *reinterpret_cast<const uint32_t *>(cell + C::key_chunk(t, o) + 4 * e);
#pragma unroll
        for (int i = 0; i < C::ITEMS; ++i) m[i] = *reinterpret_cast<const uint32_t *>(cell + C::meta(t, i));
        float x[8];
        const uint32_t mk = C::GROUPS == 2 && o >= 8 ? m[1] : m[0];
        const float ks = bf2f(mk & 0xFFFFu), kb = bf2f(mk >> 16);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[e] = fmaf(ks, BITS == 4 ? (float)((kw[0] >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) : ubyte_f32(kw[e >> 2], e & 3), kb);
        key = pack8(x);
#pragma unroll
        for (int q = 0; q < PLACES; ++q)
#pragma unroll
            for (int y = 0; y < D / 16; ++y) {
                const uint32_t mv = m[C::GROUPS + y / 4];
                uint32_t c = (w[q][BITS == 4 ? y >> 1 : y] >> (8 * (t & 3))) & 0xFFu;
                if (BITS == 4) c = (y & 1) ? c >> 4 : c & 15u;
                tile[r * PAD + 16 * y + o + q * OCT] = (uint16_t)f2bf(fmaf(bf2f(mv & 0xFFFFu), (float)c, bf2f(mv >> 16)));
            }
    }
    __syncthreads();
    if (row >= a.n) return;
    if (there) val = *reinterpret_cast<const uint4 *>(tile + r * PAD + 8 * o);
    const long at = (row * a.Hkv + hk) * D + 8 * o;
    *reinterpret_cast<uint4 *>(a.k + at) = key;
    *reinterpret_cast<uint4 *>(a.v + at) = val;
}

}  // namespace

int launch_rope_append_quantized(const uint16_t *qkv, long qkv_stride, uint16_t *q, long q_stride, long N, long H,
                                 long Hkv, long D, const float *cos_t, const float *sin_t, long table_len,
                                 uint8_t *pool, long n_blocks, long bs, int bits, const int32_t *slots,
                                 const int32_t *positions, hipStream_t stream) {
    if (N == 0) return SC_OK;
    if (!qkv || !q || !cos_t || !sin_t || !pool || !slots || !positions)
        return set_error(SC_EINVAL, "rope_append_quantized: null pointer");
    if (kv_cell_bytes(D, bits) == 0)
        return set_error(SC_EUNSUPPORTED, "rope_append_quantized: head_dim %ld in %d bits (64 or 128 in 4 or 8 supported)", D, bits);
    const int shift = block_shift(bs);
    if (shift < 0) return set_error(SC_EINVAL, "rope_append_quantized: block size %ld (16, 32, 64, 128 or 256)", bs);
    if (N < 0 || N >= (1L << 30) || H <= 0 || Hkv <= 0 || H % Hkv || H > 65536)
        return set_error(SC_EINVAL, "rope_append_quantized: bad shape N=%ld H=%ld Hkv=%ld", N, H, Hkv);
    if (n_blocks <= 0 || n_blocks * bs >= (1L << 31) || table_len <= 0 || table_len >= (1L << 31))
        return set_error(SC_EINVAL, "rope_append_quantized: bad pool or table size");
    if (qkv_stride < (H + 2 * Hkv) * D || q_stride < H * D || qkv_stride % 8 || q_stride % 8)
        return set_error(SC_EINVAL, "rope_append_quantized: bad row strides");
    if (((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)pool | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16)
        return set_error(SC_EINVAL, "rope_append_quantized: pointers must be 16-byte aligned");
    QuantAppendArgs a;
    a.qkv = qkv; a.qkv_stride = qkv_stride; a.q = q; a.q_stride = q_stride; a.pool = pool;
    a.cos_t = cos_t; a.sin_t = sin_t; a.slots = slots; a.positions = positions;
    a.N = (int)N; a.H = (int)H; a.Hkv = (int)Hkv; a.shift = shift; a.table_len = (int)table_len;
    a.n_slots = n_blocks * bs;
    // few rows in smaller groups, so that more of the GPU has work: 64 rows of 32 + 8 heads of 128
    // 5.7 us, in groups of 32 rows 8.9; 22000 rows of 8 + 1 heads 28.4 us, in groups of 64 31.5
    a.kv_rows = N <= QA_FEW ? QA_FEW_ROWS : QA_ROWS;
    const long kv_wgs = (N + a.kv_rows - 1) / a.kv_rows * Hkv;
    // A token's q heads over several waves while tokens alone leave CUs idle; from 4 tokens a CU on a
    // wave each.  (8600 rows of 32 heads of 64: 19.9 us, all in their own waves 20.8.)
    const long hpw = 64 / (D / 16), cus = device_info().num_cus;
    long per = N >= 4 * cus ? H : N >= cus ? 2 * hpw : hpw;
    if (per > H) per = H;
    a.heads_per_wave = (int)per;
    const long blocks = kv_wgs + (N * ((H + per - 1) / per) + 3) / 4;
    if (blocks >= (1L << 24)) return set_error(SC_EINVAL, "rope_append_quantized: too many rows");     // 2^32 threads
    a.kv_wgs = (int)kv_wgs;
    auto kern = D == 128 ? (bits == 4 ? rope_append_quantized_kernel<128, 4> : rope_append_quantized_kernel<128, 8>)
                         : (bits == 4 ? rope_append_quantized_kernel<64, 4> : rope_append_quantized_kernel<64, 8>);
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    return SC_OK;
}

int launch_read_quantized(const uint8_t *pool, long n_blocks, long bs, int bits, long Hkv, long D,
                          const int32_t *slots, long n, uint16_t *k, uint16_t *v, hipStream_t stream) {
    if (n == 0) return SC_OK;
    if (!pool || !slots || !k || !v) return set_error(SC_EINVAL, "read_quantized: null pointer");
    if (kv_cell_bytes(D, bits) == 0)
        return set_error(SC_EUNSUPPORTED, "read_quantized: head_dim %ld in %d bits (64 or 128 in 4 or 8 supported)", D, bits);
    const int shift = block_shift(bs);
    if (shift < 0) return set_error(SC_EINVAL, "read_quantized: block size %ld (16, 32, 64, 128 or 256)", bs);
    if (n < 0 || n >= (1L << 30) || Hkv <= 0 || Hkv > 65536) return set_error(SC_EINVAL, "read_quantized: bad shape n=%ld Hkv=%ld", n, Hkv);
    if (n_blocks <= 0 || n_blocks * bs >= (1L << 31)) return set_error(SC_EINVAL, "read_quantized: bad pool size");
    if (((uintptr_t)pool | (uintptr_t)k | (uintptr_t)v) % 16)
        return set_error(SC_EINVAL, "read_quantized: pointers must be 16-byte aligned");
    QuantReadArgs a;
    a.pool = pool; a.slots = slots; a.k = k; a.v = v; a.n = n; a.n_slots = n_blocks * bs; a.Hkv = (int)Hkv; a.shift = shift;
    const long rows = 256 / (D / 8), blocks = (n + rows - 1) / rows * Hkv;
    if (blocks >= (1L << 24)) return set_error(SC_EINVAL, "read_quantized: too many rows");            // 2^32 threads
    auto kern = D == 128 ? (bits == 4 ? read_quantized_kernel<128, 4> : read_quantized_kernel<128, 8>)
                         : (bits == 4 ? read_quantized_kernel<64, 4> : read_quantized_kernel<64, 8>);
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    return SC_OK;
}

}  // namespace sc

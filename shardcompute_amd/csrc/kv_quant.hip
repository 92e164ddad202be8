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

// A wave takes the heads of one row, D / 16 lanes a head: a lane has the dims i0 .. i0 + 7 and
// D / 2 above them, so that a pair that is rotated together is in one lane.
template <int D, int BITS>
__global__ void __launch_bounds__(256) rope_append_quantized_kernel(QuantAppendArgs a) {
    using C = Cell<D, BITS>;
    constexpr int LPH = D / 16, HPW = 64 / LPH, HALF = D / 2;
    const int heads = a.H + 2 * a.Hkv, parts = (heads + HPW - 1) / HPW;
    const long wid = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, hl = lane % LPH;
    const int tok = (int)(wid / parts), h = (int)(wid - (long)tok * parts) * HPW + lane / LPH;
    if (tok >= a.N || h >= heads) return;
    const int slot = a.slots[tok], pos = a.positions[tok];
    if (slot < 0 || slot >= a.n_slots || pos < 0 || pos >= a.table_len) return;
    const int i0 = 8 * hl;
    const uint16_t *row = a.qkv + (size_t)tok * a.qkv_stride + (size_t)h * D + i0;
    const uint4 a1 = *reinterpret_cast<const uint4 *>(row), a2 = *reinterpret_cast<const uint4 *>(row + HALF);
    float x[2][8];
    if (h < a.H + a.Hkv) {
        const float *ct = a.cos_t + (size_t)pos * HALF + i0, *st = a.sin_t + (size_t)pos * HALF + i0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x1 = bfe(a1, e), x2 = bfe(a2, e), c = ct[e], s = st[e];
            x[0][e] = add_rn(mul_rn(x1, c), mul_rn(-x2, s));
            x[1][e] = add_rn(mul_rn(x2, c), mul_rn(x1, s));
        }
        const uint4 o1 = pack8(x[0]), o2 = pack8(x[1]);
        if (h < a.H) {
            uint16_t *dst = a.q + (size_t)tok * a.q_stride + (size_t)h * D + i0;
            *reinterpret_cast<uint4 *>(dst) = o1;
            *reinterpret_cast<uint4 *>(dst + HALF) = o2;
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[0][e] = bfe(o1, e); x[1][e] = bfe(o2, e); }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) { x[0][e] = bfe(a1, e); x[1][e] = bfe(a2, e); }
    }
    const bool value = h >= a.H + a.Hkv;
    const int hk = value ? h - a.H - a.Hkv : h - a.H;
    // the groups' bounds: 128 dims, a group in each half; 64, both halves one group
    float lo[2], hi[2], zero[2];                // zero: 0, or no number if a value is not finite
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        lo[y] = hi[y] = x[y][0];
        zero[y] = x[y][0] * 0.f;
#pragma unroll
        for (int e = 1; e < 8; ++e) {
            lo[y] = fminf(lo[y], x[y][e]);
            hi[y] = fmaxf(hi[y], x[y][e]);
            zero[y] = fmaf(x[y][e], 0.f, zero[y]);
        }
    }
    if (C::GROUPS == 1) {
        lo[0] = fminf(lo[0], lo[1]);
        hi[0] = fmaxf(hi[0], hi[1]);
        zero[0] += zero[1];
    }
    Affine af[2];
#pragma unroll
    for (int y = 0; y < C::GROUPS; ++y) {
#pragma unroll
        for (int m = 1; m < LPH; m <<= 1) {
            lo[y] = fminf(lo[y], __shfl_xor(lo[y], m));
            hi[y] = fmaxf(hi[y], __shfl_xor(hi[y], m));
            zero[y] += __shfl_xor(zero[y], m);
        }
        af[y] = affine_of<BITS>(lo[y], hi[y]);
        // minima and maxima pass a NaN over: the group's scale keeps it
        if (zero[y] != 0.f) af[y].scale = af[y].bias = __builtin_nanf("");
    }
    if (C::GROUPS == 1) af[1] = af[0];
    const int t = slot & 15;
    uint8_t *cell = a.pool + (((size_t)(slot >> a.shift) * a.Hkv + hk) * (1u << (a.shift - 4)) + ((slot & ((1 << a.shift) - 1)) >> 4)) * C::BYTES;
    if (hl < C::GROUPS)
        *reinterpret_cast<uint32_t *>(cell + C::meta(t, (value ? C::GROUPS : 0) + hl)) =
            f2bf(af[hl].scale) | f2bf(af[hl].bias) << 16;
    uint32_t code[2][8];
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int e = 0; e < 8; ++e) code[y][e] = code_of<BITS>(x[y][e], af[y]);
    if (!value) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            uint8_t *dst = cell + C::key_chunk(t, hl + y * LPH);
            if (BITS == 4) {
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) w |= code[y][e] << (4 * ((e >> 1) + 4 * (e & 1)));
                *reinterpret_cast<uint32_t *>(dst) = w;
            } else {
                uint32_t w[2] = {0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e >> 2] |= code[y][e] << (8 * (e & 3));
                *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
            }
        }
        return;
    }
    if (BITS == 8) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int e = 0; e < 8; ++e) cell[C::value_byte(t, i0 + y * HALF + e)] = (uint8_t)code[y][e];
        return;
    }
    // 4 bits: dims d and d + 16 share a byte, lane ^ 2 has the other; of a pair of lanes one
    // writes the lower half's bytes and one the upper half's
    const int y = (hl >> 1) & 1, d0 = (i0 & ~16) + y * HALF;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t give = y ? code[0][e] : code[1][e], keep = y ? code[1][e] : code[0][e];
        const uint32_t got = (uint32_t)__shfl_xor((int)give, 2);
        cell[C::value_byte(t, d0 + e)] = (uint8_t)(y ? got | keep << 4 : keep | got << 4);
    }
}

// ---------------------------------------------------------------- reading back
//
// k, v [n, Hkv, D] bf16 of the positions at slots[n]: bf16(scale code + bias), the sum rounded
// once (as dequantize); 0 for a slot outside the pool.  A thread 8 dims of a key and of a value.
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
    constexpr int OCT = D / 8;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = i / (a.Hkv * OCT);
    if (row >= a.n) return;
    const int rest = (int)(i - row * (a.Hkv * OCT)), hk = rest / OCT, o = rest % OCT;
    const int slot = a.slots[row];
    uint16_t *k = a.k + (row * a.Hkv + hk) * D + 8 * o, *v = a.v + (row * a.Hkv + hk) * D + 8 * o;
    if (slot < 0 || slot >= a.n_slots) {
        *reinterpret_cast<uint4 *>(k) = *reinterpret_cast<uint4 *>(v) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    const int t = slot & 15, grp = o >> 3;
    const uint8_t *cell = a.pool + (((size_t)(slot >> a.shift) * a.Hkv + hk) * (1u << (a.shift - 4)) + ((slot & ((1 << a.shift) - 1)) >> 4)) * C::BYTES;
    const uint32_t mk = *reinterpret_cast<const uint32_t *>(cell + C::meta(t, grp));
    const uint32_t mv = *reinterpret_cast<const uint32_t *>(cell + C::meta(t, C::GROUPS + grp));
    const float ks = bf2f(mk & 0xFFFFu), kb = bf2f(mk >> 16), vs = bf2f(mv & 0xFFFFu), vb = bf2f(mv >> 16);
    float x[8];
    if (BITS == 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(cell + C::key_chunk(t, o));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(ks, (float)((w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u), kb);
    } else {
        const uint2 w = *reinterpret_cast<const uint2 *>(cell + C::key_chunk(t, o));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(ks, ubyte_f32(e < 4 ? w.x : w.y, e & 3), kb);
    }
    *reinterpret_cast<uint4 *>(k) = pack8(x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint32_t c = cell[C::value_byte(t, 8 * o + e)];
        if (BITS == 4) c = (c >> (4 * ((o >> 1) & 1))) & 15u;
        x[e] = fmaf(vs, (float)c, vb);
    }
    *reinterpret_cast<uint4 *>(v) = pack8(x);
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
    const long hpw = 64 / (D / 16), blocks = (N * ((H + 2 * Hkv + hpw - 1) / hpw) + 3) / 4;
    if (blocks >= (1L << 24)) return set_error(SC_EINVAL, "rope_append_quantized: too many rows");     // 2^32 threads
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
    const long blocks = (n * Hkv * (D / 8) + 255) / 256;
    if (blocks >= (1L << 24)) return set_error(SC_EINVAL, "read_quantized: too many rows");            // 2^32 threads
    auto kern = D == 128 ? (bits == 4 ? read_quantized_kernel<128, 4> : read_quantized_kernel<128, 8>)
                         : (bits == 4 ? read_quantized_kernel<64, 4> : read_quantized_kernel<64, 8>);
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    return SC_OK;
}

}  // namespace sc

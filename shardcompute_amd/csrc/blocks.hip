// A key/value cache in blocks: the tables of one model step (block_tables) and the
// append of its keys and values (rope_append_blocks).
//
// A pool holds blocks of bs positions (a power of two, 16 to 256):
//   K  [n_blocks, Hkv, bs, D]   keys in rows
//   Vt [n_blocks, Hkv, D, bs]   values transposed, as the dense cache holds them
// Sequence r's own position p lies in block tables[r, p / bs] at offset p % bs: slot
// tables[r, p / bs] bs + p % bs.  Blocks nobody holds are a stack, free[0, n_free).
#include "sc_common.h"

namespace sc {

namespace {

// ---------------------------------------------------------------- tables of a step
//
// Of sequence r: old = release ? 0 : lengths[r], total = old + new[r], it holds
// ceil(old / bs) blocks and takes need = ceil(total / bs) - ceil(old / bs) more.  Blocks
// given back go onto the stack in the order (sequence, place), then block i of
// sequence r's new ones is stack[top - 1 - E_r - i] with E the exclusive sum of need.
// row_starts is the exclusive sum of new; row row_starts[r] + i is position old + i.
//
// Integer work of a few bytes per sequence and row, so what counts is the chain of
// dependent loads and launches.  One workgroup sums, checks and fills the tables; where
// rows are few it writes them too (STEP_ROWS), else a second launch does, whose
// workgroups read the finished tables.  Up to STEP_THREADS sequences, a thread each, take
// one pass (block_step_kernel: every sum in one exchange between the waves, a decoded
// token's slot from registers); more go through in chunks, three times (block_step_many_kernel).
// One decoded sequence 2.3 us, 256 with 32 of them starting anew 5.0; 512 prompts of up to
// 700 positions, 180 thousand rows, 4.3 + 6.1.  With the host's call 1024 decoded sequences
// 9.7 us, 2048 15.
constexpr int STEP_THREADS = 1024;
constexpr int STEP_ROWS = 4096;

enum StepStatus { STEP_NO_BLOCKS = 1, STEP_NO_TABLE = 2, STEP_NO_ROWS = 4, STEP_NO_STACK = 8 };

struct StepArgs {
    const int32_t *lengths, *fresh;
    const uint8_t *release;
    int32_t *tables, *free_blocks;
    const int32_t *n_free, *prefix_len;
    int32_t *lengths_out, *n_free_out, *row_starts, *slots, *positions, *status;
    int R, width, shift, cap, rows;
    int rows_here;           // the rows are written by block_step_kernel
};

// inclusive sum over the workgroup's threads; total: of all of them
__device__ __forceinline__ int block_scan(int v, int *wsum, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();                       // wsum of the previous call has been read
    if (lane == 63) wsum[w] = v;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < nw; ++i) {
        const int s = wsum[i];
        before += i < w ? s : 0;
        all += s;
    }
    total = all;
    return v + before;
}

// the largest i in [0, n) with start[i] <= x, start ascending and start[0] <= x
__device__ __forceinline__ int last_at_most(const int32_t *start, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One thread a sequence.  Sums saturate at STEP_MOST, above every limit they are compared
// with, so none wraps.
constexpr int STEP_MOST = (1 << 30) - 1;

__global__ void __launch_bounds__(STEP_THREADS) block_step_kernel(StepArgs a) {
    struct Sums { int back, need, fresh; };
    __shared__ Sums wave_sum_[STEP_THREADS / 64];
    __shared__ int wave_flags[STEP_THREADS / 64];
    __shared__ int first_back[STEP_THREADS], first_need[STEP_THREADS], first_row[STEP_THREADS], held[STEP_THREADS];
    const int r = threadIdx.x, lane = r & 63, w = r >> 6, n = blockDim.x, nw = n >> 6, R = a.R;
    const int bs = 1 << a.shift;
    const long most = (long)a.width << a.shift;                // positions a table has room for
    const int32_t *table = a.tables + (long)r * a.width;

    int len = 0, fresh = 0, gone = 0;
    if (r < R) {
        len = a.lengths[r];
        fresh = a.fresh[r];
        gone = a.release ? a.release[r] : 0;
    }
    const int n_free = a.n_free[0], prefix = a.prefix_len ? a.prefix_len[0] : 0;
    len = (int)min((long)max(len, 0), most);
    fresh = max(fresh, 0);
    const int old = gone ? 0 : len;
    int last = 0;                                              // the block an unfilled last one goes on in
    if (old & (bs - 1)) last = table[old >> a.shift];
    enum { FLAG_TABLE = STEP_NO_TABLE, FLAG_MANY = 256 };
    int flags = 0;
    if ((long)old + fresh > most) flags |= FLAG_TABLE;
    if (fresh > 1) flags |= FLAG_MANY;
    if (flags & FLAG_TABLE) fresh = 0;                         // (the step is refused; in 32 bits from here)
    const int have = (old + bs - 1) >> a.shift, need = ((old + fresh + bs - 1) >> a.shift) - have;
    Sums x = {gone ? (len + bs - 1) >> a.shift : 0, need, fresh};
    const Sums mine = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int b = __shfl_up(x.back, o), d = __shfl_up(x.need, o), f = __shfl_up(x.fresh, o);
        if (lane >= o) {
            x.back = min(x.back + b, STEP_MOST);
            x.need = min(x.need + d, STEP_MOST);
            x.fresh = min(x.fresh + f, STEP_MOST);
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) flags |= __shfl_xor(flags, o);
    if (lane == 63) {
        wave_sum_[w] = x;
        wave_flags[w] = flags;
    }
    __syncthreads();
    Sums before = {0, 0, 0}, all = {0, 0, 0};
    for (int i = 0; i < nw; ++i) {
        const Sums y = wave_sum_[i];
        if (i == w) before = all;
        all.back = min(all.back + y.back, STEP_MOST);
        all.need = min(all.need + y.need, STEP_MOST);
        all.fresh = min(all.fresh + y.fresh, STEP_MOST);
        flags |= wave_flags[i];
    }
    const int stack = min(max(n_free, 0), a.cap);
    const long top = (long)stack + all.back;
    int bad = flags & FLAG_TABLE;
    if (all.fresh > a.rows) bad |= STEP_NO_ROWS;
    if (all.need > top) bad |= STEP_NO_BLOCKS;
    if (top > a.cap) bad |= STEP_NO_STACK;
    if (bad) {
        if (r == 0) {
            a.status[0] |= bad;
            a.n_free_out[0] = n_free;
        }
        if (r < R) a.lengths_out[r] = a.lengths[r];
        for (int i = r; i <= R; i += n) a.row_starts[i] = 0;
        if (a.rows_here)
            for (int i = r; i < a.rows; i += n) a.slots[i] = a.positions[i] = -1;
        return;
    }
    // exclusive sums of the sequences before this one
    const int e_back = before.back + x.back - mine.back, e_need = before.need + x.need - need;
    const int row = before.fresh + x.fresh - fresh;
    if (r < R) {
        a.lengths_out[r] = old + fresh;
        a.row_starts[r] = row;
    }
    if (r == 0) {
        a.row_starts[R] = all.fresh;
        a.n_free_out[0] = (int)top - all.need;
    }
    const bool many = flags & FLAG_MANY;
    if (many || all.back) {
        first_back[r] = e_back;
        first_need[r] = e_need;
        first_row[r] = row;
        held[r] = old;
        __syncthreads();
    }
    // blocks given back
    if (all.back) {
        for (int e = r; e < all.back; e += n) {
            const int i = last_at_most(first_back, R, e);
            a.free_blocks[stack + e] = a.tables[(long)i * a.width + e - first_back[i]];
        }
        __syncthreads();                                       // before blocks are popped and tables written
    }
    if (!many) {
        // decode: at most one new position, and one new block, a sequence
        if (need) {
            last = a.free_blocks[top - 1 - e_need];
            a.tables[(long)r * a.width + have] = last;
        }
        if (fresh && a.rows_here) {
            a.slots[row] = (last << a.shift) + (old & (bs - 1));
            a.positions[row] = prefix + old;
        }
    } else if (a.rows_here) {                                  // (else block_rows_kernel's)
        for (int e = r; e < all.need; e += n) {
            const int i = last_at_most(first_need, R, e);
            a.tables[(long)i * a.width + ((held[i] + bs - 1) >> a.shift) + e - first_need[i]] = a.free_blocks[top - 1 - e];
        }
        for (int e = r; e < all.fresh; e += n) {
            // a position of the blocks held is in the table, of the new ones on the stack
            const int i = last_at_most(first_row, R, e), p = held[i] + e - first_row[i];
            const int j = (p >> a.shift) - ((held[i] + bs - 1) >> a.shift);
            const int block = j < 0 ? a.tables[(long)i * a.width + (p >> a.shift)] : a.free_blocks[top - 1 - first_need[i] - j];
            a.slots[e] = (block << a.shift) + (p & (bs - 1));
            a.positions[e] = prefix + p;
        }
    }
    if (a.rows_here)
        for (int i = all.fresh + r; i < a.rows; i += n) a.slots[i] = a.positions[i] = -1;
}

// More sequences than threads.
__global__ void __launch_bounds__(STEP_THREADS) block_step_many_kernel(StepArgs a) {
    __shared__ int wsum[STEP_THREADS / 64];
    __shared__ int start[STEP_THREADS], base[STEP_THREADS];     // of this chunk: exclusive sums, and held blocks
    __shared__ int row0[STEP_THREADS], held[STEP_THREADS];
    __shared__ unsigned long long sums[3];
    __shared__ int bad;
    const int tid = threadIdx.x, n = blockDim.x, R = a.R;
    const int bs = 1 << a.shift;
    const long most = (long)a.width << a.shift;                // positions a table has room for
    if (tid < 3) sums[tid] = 0;
    if (tid == 0) bad = 0;
    __syncthreads();

    int old = 0, w = 0, back = 0;
    auto load = [&](int r) {
        old = w = back = 0;
        if (r >= R) return;
        const int len = min((long)max(a.lengths[r], 0), most);
        w = max(a.fresh[r], 0);
        const bool gone = a.release && a.release[r];
        back = gone ? (len + bs - 1) >> a.shift : 0;
        old = gone ? 0 : len;
    };
    auto need = [&]() { return ((old + w + bs - 1) >> a.shift) - ((old + bs - 1) >> a.shift); };

    // what the step asks for, before anything is changed
    unsigned long long s_new = 0, s_need = 0, s_back = 0;
    for (int r0 = 0; r0 < R; r0 += n) {
        load(r0 + tid);
        if ((long)old + w > most) {                            // (need() may not be asked: 32-bit)
            atomicOr(&bad, STEP_NO_TABLE);
        } else {
            s_new += w;
            s_need += need();
        }
        s_back += back;
    }
    if (s_new) atomicAdd(&sums[0], s_new);
    if (s_need) atomicAdd(&sums[1], s_need);
    if (s_back) atomicAdd(&sums[2], s_back);
    const int stack = min(max(a.n_free[0], 0), a.cap);
    __syncthreads();
    const long top = (long)stack + (long)sums[2];
    if (tid == 0) {
        int b = bad;
        if ((long)sums[0] > a.rows) b |= STEP_NO_ROWS;
        if ((long)sums[1] > top) b |= STEP_NO_BLOCKS;
        if (top > a.cap) b |= STEP_NO_STACK;
        bad = b;
        if (b) a.status[0] |= b;
    }
    __syncthreads();
    const bool refused = bad != 0;
    if (refused) {
        for (int r = tid; r <= R; r += n) a.row_starts[r] = 0;
        for (int r = tid; r < R; r += n) a.lengths_out[r] = a.lengths[r];
        if (tid == 0) a.n_free_out[0] = a.n_free[0];
        if (a.rows_here)
            for (int i = tid; i < a.rows; i += n) a.slots[i] = a.positions[i] = -1;
        return;
    }

    // blocks given back
    if (sums[2]) {
        int before = 0;
        for (int r0 = 0; r0 < R; r0 += n) {
            load(r0 + tid);
            int all;
            start[tid] = block_scan(back, wsum, all) - back;
            __syncthreads();
            for (int e = tid; e < all; e += n) {
                const int i = last_at_most(start, min(n, R - r0), e);
                a.free_blocks[stack + before + e] = a.tables[(long)(r0 + i) * a.width + e - start[i]];
            }
            before += all;
            __syncthreads();
        }
    }

    // blocks taken, lengths, row starts and rows, a chunk of sequences at a time
    const int prefix = a.prefix_len ? a.prefix_len[0] : 0;
    int taken = 0, rows = 0;
    for (int r0 = 0; r0 < R; r0 += n) {
        const int r = r0 + tid, chunk = min(n, R - r0);
        load(r);
        const int nd = need();
        int all, rall;
        start[tid] = block_scan(nd, wsum, all) - nd;
        row0[tid] = block_scan(w, wsum, rall) - w;
        base[tid] = (old + bs - 1) >> a.shift;
        held[tid] = old;
        if (r < R) {
            a.lengths_out[r] = old + w;
            a.row_starts[r] = rows + row0[tid];
        }
        __syncthreads();
        for (int e = tid; e < all; e += n) {
            const int i = last_at_most(start, chunk, e);
            a.tables[(long)(r0 + i) * a.width + base[i] + e - start[i]] = a.free_blocks[top - 1 - taken - e];
        }
        if (a.rows_here) {
            __syncthreads();                                   // the tables of this chunk are whole
            for (int e = tid; e < rall; e += n) {
                const int i = last_at_most(row0, chunk, e), p = held[i] + e - row0[i];
                a.slots[rows + e] = (a.tables[(long)(r0 + i) * a.width + (p >> a.shift)] << a.shift) + (p & (bs - 1));
                a.positions[rows + e] = prefix + p;
            }
        }
        taken += all;
        rows += rall;
        __syncthreads();
    }
    if (tid == 0) {
        a.row_starts[R] = rows;
        a.n_free_out[0] = (int)top - taken;
    }
    if (a.rows_here)
        for (int i = rows + tid; i < a.rows; i += n) a.slots[i] = a.positions[i] = -1;
}

// Slots and positions of many rows, four rows a thread (one search, 16-byte stores where the
// buffers are aligned).  FILL (up to STEP_THREADS sequences): block_step_kernel has left the
// tables to this launch; a new position's block is popped here, by every row of it, and the
// row that begins it writes the table's entry.  Otherwise the tables are whole.
template <bool FILL>
__global__ void __launch_bounds__(256) block_rows_kernel(StepArgs a) {
    __shared__ int first_need[FILL ? STEP_THREADS + 1 : 1], wsum[4];
    const int bs = 1 << a.shift;
    if (FILL) {
        // the exclusive sums of the blocks the sequences take, four sequences a thread
        int need[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 4 * (int)threadIdx.x + i;
            need[i] = 0;
            if (r < a.R) {
                const int len = a.lengths_out[r], fresh = a.row_starts[r + 1] - a.row_starts[r];
                need[i] = ((len + bs - 1) >> a.shift) - ((len - fresh + bs - 1) >> a.shift);
            }
            sum += need[i];
        }
        int all, at = block_scan(sum, wsum, all) - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            first_need[4 * threadIdx.x + i] = at;
            at += need[i];
        }
        if (threadIdx.x == 0) first_need[STEP_THREADS] = all;
        __syncthreads();
    }
    const int row = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
    if (row >= a.rows) return;
    const int total = a.row_starts[a.R], prefix = a.prefix_len ? a.prefix_len[0] : 0;
    const int top = FILL ? a.n_free_out[0] + first_need[STEP_THREADS] : 0;
    int r = row < total ? last_at_most(a.row_starts, a.R, row) : 0;
    int begin = a.row_starts[r], end = a.row_starts[r + 1], first = a.lengths_out[r] - end;   // position of row j: first + j
    int sl[4], po[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = row + i;
        sl[i] = po[i] = -1;
        if (j >= total) continue;
        while (j >= end) {
            ++r;
            begin = end;
            end = a.row_starts[r + 1];
            first = a.lengths_out[r] - end;
        }
        const int p = first + j, b = p >> a.shift;
        int32_t *entry = a.tables + (long)r * a.width + b;
        int block;
        const int have = (first + begin + bs - 1) >> a.shift;          // blocks held before the step
        if (FILL && b >= have) {
            block = a.free_blocks[top - 1 - first_need[r] - (b - have)];
            if ((p & (bs - 1)) == 0) *entry = block;
        } else {
            block = *entry;
        }
        sl[i] = (block << a.shift) + (p & (bs - 1));
        po[i] = prefix + p;
    }
    if (row + 4 <= a.rows && (((uintptr_t)a.slots | (uintptr_t)a.positions) & 15) == 0) {
        *reinterpret_cast<int4 *>(a.slots + row) = make_int4(sl[0], sl[1], sl[2], sl[3]);
        *reinterpret_cast<int4 *>(a.positions + row) = make_int4(po[0], po[1], po[2], po[3]);
    } else {
        for (int i = 0; i < 4 && row + i < a.rows; ++i) {
            a.slots[row + i] = sl[i];
            a.positions[row + i] = po[i];
        }
    }
}

// ---------------------------------------------------------------- rotation and append
//
// Row t of qkv goes to slot slots[t], rotated for positions[t] (rotate-half, fp32
// tables, rope_append_kernel's arithmetic element by element; attention.py:130-151):
// q to its own buffer, k and v to the pool.  Rows whose slot or position lies outside
// the pool or the tables are left alone.
//
// Bound by memory: every row is read and written once.  Rotation: a wave a token and
// head range, 16-byte accesses.  V: the pool holds it transposed, so 64 rows of one kv
// head go through LDS and leave in 16-byte pieces of 8 consecutive slots (rows of one
// sequence are consecutive slots within a block); rows that no whole piece covers,
// single decoded tokens among them, in 2-byte stores.  24 prompts, 8.6 thousand rows of 32 + 4 + 4
// heads of 64: 18 us, 4.9 TB/s.  Single rows are bound by their values' cache lines, D of
// them a row and kv head: 2048 rows of 8 kv heads of 128 111 us where no cache holds those lines
// (blocks of 64), 38 where one does.
struct RopeBlocksArgs {
    const uint16_t *qkv;
    long qkv_stride;
    uint16_t *q;
    long q_stride;
    uint16_t *kc, *vt;
    const float *cos_t, *sin_t;
    const int32_t *slots, *positions;
    int N, H, Hkv, shift, table_len;
    long n_slots;
    int v_blocks, heads_per_wave;
    int v_heads;             // Hkv: the waves write v too (no v blocks)
};

constexpr int RB_ROWS = 64, RB_HALO = 8;
constexpr long RB_FEW = 512;

template <int D>
__global__ void __launch_bounds__(256) rope_append_blocks_kernel(RopeBlocksArgs a) {
    constexpr int W = D / 2 + 1;                             // LDS words a row (odd: conflict-free columns)
    __shared__ uint32_t tile[(RB_ROWS + RB_HALO) * W];
    __shared__ int slot_of[RB_HALO + RB_ROWS + RB_HALO];
    const int bs = 1 << a.shift;
    if ((int)blockIdx.x < a.v_blocks) {
        const int hk = (int)blockIdx.x % a.Hkv, t0 = (int)blockIdx.x / a.Hkv * RB_ROWS;
        constexpr int CPT = D / 8;
        for (int i = threadIdx.x; i < RB_HALO + RB_ROWS + RB_HALO; i += 256) {
            const int t = t0 - RB_HALO + i;
            int s = -1;
            if (t >= 0 && t < a.N) {
                s = a.slots[t];
                const int p = a.positions[t];
                if (s < 0 || s >= a.n_slots || p < 0 || p >= a.table_len) s = -1;
            }
            slot_of[i] = s;
        }
        for (int i = threadIdx.x; i < (RB_ROWS + RB_HALO) * CPT; i += 256) {
            const int t = i / CPT, c = i - t * CPT;
            if (t0 + t < a.N) {
                const uint4 v = *reinterpret_cast<const uint4 *>(a.qkv + (size_t)(t0 + t) * a.qkv_stride +
                                                                 (size_t)(a.H + a.Hkv + hk) * D + 8 * c);
                uint32_t *row = tile + t * W + 4 * c;
                row[0] = v.x; row[1] = v.y; row[2] = v.z; row[3] = v.w;
            }
        }
        __syncthreads();
        // row t leads a piece if its slot is a multiple of 8 and the next 7 rows follow it;
        // it is covered if the row that would lead its piece does (that row may belong to
        // the workgroup before).  Each wave finds this for the 64 rows, a row a lane
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        auto leads = [&](int i) {                            // i: index into slot_of
            const int s = slot_of[i];
            bool ok = s >= 0 && (s & 7) == 0;
            for (int j = 1; j < 8; ++j) ok = ok && slot_of[i + j] == s + j;
            return ok;
        };
        const int s = slot_of[RB_HALO + lane], off = s & 7;
        const bool lead = leads(RB_HALO + lane);
        const bool covered = s >= 0 && slot_of[RB_HALO + lane - off] == s - off && leads(RB_HALO + lane - off);
        unsigned long long lm = __ballot(lead), sm = __ballot(s >= 0 && !covered);
        const size_t head = (size_t)hk * D << a.shift, blk = (size_t)a.Hkv * D << a.shift;
        // pieces: lanes take (pair of dims, leader), leaders fastest so that stores of one
        // dim are neighbours
        const int nl = __popcll(lm);
        if (nl) {
            for (int i = (int)threadIdx.x; i < nl * (D / 2); i += 256) {
                const int dp = i / nl;
                int k = i - dp * nl;
                // the k-th leader's row
                unsigned long long m = lm;
                while (k--) m &= m - 1;
                const int t = __ffsll((unsigned long long)m) - 1;
                const int st = slot_of[RB_HALO + t];
                uint32_t x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = tile[(t + j) * W + dp];
                uint4 lo, hi;
                lo.x = __builtin_amdgcn_perm(x[1], x[0], 0x05040100u); hi.x = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
                lo.y = __builtin_amdgcn_perm(x[3], x[2], 0x05040100u); hi.y = __builtin_amdgcn_perm(x[3], x[2], 0x07060302u);
                lo.z = __builtin_amdgcn_perm(x[5], x[4], 0x05040100u); hi.z = __builtin_amdgcn_perm(x[5], x[4], 0x07060302u);
                lo.w = __builtin_amdgcn_perm(x[7], x[6], 0x05040100u); hi.w = __builtin_amdgcn_perm(x[7], x[6], 0x07060302u);
                uint16_t *dst = a.vt + (size_t)(st >> a.shift) * blk + head + ((size_t)(2 * dp) << a.shift) + (st & (bs - 1));
                *reinterpret_cast<uint4 *>(dst) = lo;
                *reinterpret_cast<uint4 *>(dst + bs) = hi;
            }
        }
        // single rows: a wave a row, lanes over the dims
        int turn = 0;
        while (sm) {
            const int t = __ffsll((unsigned long long)sm) - 1;
            sm &= sm - 1;
            if ((turn++ & 3) != w) continue;
            const int st = slot_of[RB_HALO + t];
            uint16_t *dst = a.vt + (size_t)(st >> a.shift) * blk + head + (st & (bs - 1));
            for (int d = lane; d < D / 2; d += 64) {
                const uint32_t x = tile[t * W + d];
                dst[(size_t)(2 * d) << a.shift] = (uint16_t)x;
                dst[(size_t)(2 * d + 1) << a.shift] = (uint16_t)(x >> 16);
            }
        }
        return;
    }
    constexpr int LPH = D / 16, HPW = 64 / LPH, HALF = D / 2;   // lanes a head, heads a wave at a time
    const int heads = a.H + a.Hkv + a.v_heads, parts = (heads + a.heads_per_wave - 1) / a.heads_per_wave;
    const int wid = ((int)blockIdx.x - a.v_blocks) * 4 + ((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int tok = wid / parts, part = wid - tok * parts;
    if (tok >= a.N) return;
    const int slot = a.slots[tok], pos = a.positions[tok];
    const int i0 = 8 * (lane % LPH), h0 = part * a.heads_per_wave + lane / LPH;
    const uint16_t *row = a.qkv + (size_t)tok * a.qkv_stride + i0;
    // the first head's values are on their way while the slot and the angles are read
    uint4 a1, a2;
    {
        const uint16_t *hp = row + (size_t)min(h0, heads - 1) * D;
        a1 = *reinterpret_cast<const uint4 *>(hp);
        a2 = *reinterpret_cast<const uint4 *>(hp + HALF);
    }
    if (slot < 0 || slot >= a.n_slots || pos < 0 || pos >= a.table_len) return;
    float c[8], sn[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const float4 cv = *reinterpret_cast<const float4 *>(a.cos_t + (size_t)pos * HALF + i0 + 4 * q);
        const float4 sv = *reinterpret_cast<const float4 *>(a.sin_t + (size_t)pos * HALF + i0 + 4 * q);
        c[4 * q] = cv.x; c[4 * q + 1] = cv.y; c[4 * q + 2] = cv.z; c[4 * q + 3] = cv.w;
        sn[4 * q] = sv.x; sn[4 * q + 1] = sv.y; sn[4 * q + 2] = sv.z; sn[4 * q + 3] = sv.w;
    }
    const int h1 = min(heads, (part + 1) * a.heads_per_wave);
#pragma unroll 4
    for (int h = h0; h < h1; h += HPW) {
        if (h != h0) {
            const uint16_t *hp = row + (size_t)h * D;
            a1 = *reinterpret_cast<const uint4 *>(hp);
            a2 = *reinterpret_cast<const uint4 *>(hp + HALF);
        }
        if (h >= a.H + a.Hkv) {                              // a v head: a slot's values lie bs apart
            uint16_t *dst = a.vt + ((((size_t)(slot >> a.shift) * a.Hkv + (h - a.H - a.Hkv)) * D + i0) << a.shift) + (slot & (bs - 1));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t w1 = e < 2 ? a1.x : e < 4 ? a1.y : e < 6 ? a1.z : a1.w;
                const uint32_t w2 = e < 2 ? a2.x : e < 4 ? a2.y : e < 6 ? a2.z : a2.w;
                dst[(size_t)e << a.shift] = (uint16_t)((e & 1) ? w1 >> 16 : w1);
                dst[(size_t)(e + HALF) << a.shift] = (uint16_t)((e & 1) ? w2 >> 16 : w2);
            }
            continue;
        }
        uint32_t o1[4], o2[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float r1[2], r2[2];
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const float x1 = bfe(a1, e + f), x2 = bfe(a2, e + f);
                r1[f] = add_rn(mul_rn(x1, c[e + f]), mul_rn(-x2, sn[e + f]));
                r2[f] = add_rn(mul_rn(x2, c[e + f]), mul_rn(x1, sn[e + f]));
            }
            o1[e / 2] = pack_bf16x2(r1[0], r1[1]);
            o2[e / 2] = pack_bf16x2(r2[0], r2[1]);
        }
        uint16_t *dst = h < a.H ? a.q + (size_t)tok * a.q_stride + (size_t)h * D + i0
                                : a.kc + ((((size_t)(slot >> a.shift) * a.Hkv + (h - a.H)) << a.shift) + (slot & (bs - 1))) * D + i0;
        *reinterpret_cast<uint4 *>(dst) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
        *reinterpret_cast<uint4 *>(dst + HALF) = make_uint4(o2[0], o2[1], o2[2], o2[3]);
    }
}

}  // namespace

// log2 of a block size the kernels take, or -1
int block_shift(long bs) {
    for (int s = 4; s <= 8; ++s)
        if (bs == (1L << s)) return s;
    return -1;
}

int launch_block_tables(const int32_t *lengths, const int32_t *fresh, const uint8_t *release, int32_t *tables,
                        int32_t *free_blocks, const int32_t *n_free, const int32_t *prefix_len, long R, long width,
                        long bs, long cap, long rows, int32_t *lengths_out, int32_t *n_free_out, int32_t *row_starts,
                        int32_t *slots, int32_t *positions, int32_t *status, hipStream_t stream) {
    if (!lengths || !fresh || !tables || !free_blocks || !n_free || !lengths_out || !n_free_out || !row_starts ||
        !status || (rows > 0 && (!slots || !positions)))
        return set_error(SC_EINVAL, "block_tables: null pointer");
    const int shift = block_shift(bs);
    if (shift < 0) return set_error(SC_EINVAL, "block_tables: block size %ld (16, 32, 64, 128 or 256)", bs);
    if (R <= 0 || R > 65536) return set_error(SC_EINVAL, "block_tables: %ld sequences (1 to 65536)", R);
    if (width <= 0 || width * bs >= (1L << 30)) return set_error(SC_EINVAL, "block_tables: bad table width %ld", width);
    if (cap <= 0 || cap * bs >= (1L << 31)) return set_error(SC_EINVAL, "block_tables: bad stack size %ld", cap);
    if (rows < 0 || rows >= STEP_MOST) return set_error(SC_EINVAL, "block_tables: bad row count %ld", rows);
    StepArgs a;
    a.lengths = lengths; a.fresh = fresh; a.release = release; a.tables = tables; a.free_blocks = free_blocks;
    a.n_free = n_free; a.prefix_len = prefix_len; a.lengths_out = lengths_out; a.n_free_out = n_free_out;
    a.row_starts = row_starts; a.slots = slots; a.positions = positions; a.status = status;
    a.R = (int)R; a.width = (int)width; a.shift = shift; a.cap = (int)cap; a.rows = (int)rows;
    a.rows_here = rows <= STEP_ROWS;
    const long want = R > rows / 4 ? R : rows / 4;
    const int threads = (int)(want >= STEP_THREADS || !a.rows_here ? STEP_THREADS : (want + 63) / 64 * 64);
    if (R <= threads) hipLaunchKernelGGL(block_step_kernel, dim3(1), dim3(threads), 0, stream, a);
    else hipLaunchKernelGGL(block_step_many_kernel, dim3(1), dim3(threads), 0, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    if (!a.rows_here) {
        auto kern = R <= threads ? block_rows_kernel<true> : block_rows_kernel<false>;
        hipLaunchKernelGGL(kern, dim3((unsigned)((rows + 1023) / 1024)), dim3(256), 0, stream, a);
        SC_HIP_CHECK(hipGetLastError());
    }
    return SC_OK;
}

int launch_rope_append_blocks(const uint16_t *qkv, long qkv_stride, uint16_t *q, long q_stride, long N, long H,
                              long Hkv, long D, const float *cos_t, const float *sin_t, long table_len, uint16_t *kc,
                              uint16_t *vt, long n_blocks, long bs, const int32_t *slots, const int32_t *positions,
                              hipStream_t stream) {
    if (N == 0) return SC_OK;
    if (!qkv || !q || !cos_t || !sin_t || !kc || !vt || !slots || !positions)
        return set_error(SC_EINVAL, "rope_append_blocks: null pointer");
    if (D != 64 && D != 128) return set_error(SC_EUNSUPPORTED, "rope_append_blocks: head_dim %ld (64 or 128 supported)", D);
    const int shift = block_shift(bs);
    if (shift < 0) return set_error(SC_EINVAL, "rope_append_blocks: block size %ld (16, 32, 64, 128 or 256)", bs);
    if (N < 0 || N >= (1L << 30) || H <= 0 || Hkv <= 0 || H % Hkv || H > 65536)
        return set_error(SC_EINVAL, "rope_append_blocks: bad shape N=%ld H=%ld Hkv=%ld", N, H, Hkv);
    if (n_blocks <= 0 || n_blocks * bs >= (1L << 31) || table_len <= 0 || table_len >= (1L << 31))
        return set_error(SC_EINVAL, "rope_append_blocks: bad pool or table size");
    if (qkv_stride < (H + 2 * Hkv) * D || q_stride < H * D || qkv_stride % 8 || q_stride % 8)
        return set_error(SC_EINVAL, "rope_append_blocks: bad row strides");
    if (((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)kc | (uintptr_t)vt | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16)
        return set_error(SC_EINVAL, "rope_append_blocks: pointers must be 16-byte aligned");
    RopeBlocksArgs a;
    a.qkv = qkv; a.qkv_stride = qkv_stride; a.q = q; a.q_stride = q_stride; a.kc = kc; a.vt = vt;
    a.cos_t = cos_t; a.sin_t = sin_t; a.slots = slots; a.positions = positions;
    a.N = (int)N; a.H = (int)H; a.Hkv = (int)Hkv; a.shift = shift; a.table_len = (int)table_len;
    a.n_slots = n_blocks * bs;
    // few rows: v in 2-byte stores by the rotation's waves, which spares the way through LDS
    // (64 single rows of 32 + 8 heads of 128: 8.1 -> 4.0 us; at 1024 rows of a
    // prompt 10.0 -> 15.5)
    const bool few = N <= RB_FEW;
    a.v_heads = few ? (int)Hkv : 0;
    const long v_blocks = few ? 0 : (N + RB_ROWS - 1) / RB_ROWS * Hkv, heads = H + Hkv + a.v_heads;
    // a token's heads over several waves while tokens alone leave CUs idle
    const int hpw = (int)(64 / (D / 16));
    long per = N >= 4L * device_info().num_cus ? heads : N >= device_info().num_cus ? 2 * hpw : hpw;
    if (per > heads) per = heads;
    a.heads_per_wave = (int)per;
    const long waves = N * ((heads + per - 1) / per);
    const long blocks = v_blocks + (waves + 3) / 4;
    if (blocks >= (1L << 31)) return set_error(SC_EINVAL, "rope_append_blocks: too many rows");
    a.v_blocks = (int)v_blocks;
    auto kern = D == 128 ? rope_append_blocks_kernel<128> : rope_append_blocks_kernel<64>;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    SC_HIP_CHECK(hipGetLastError());
    return SC_OK;
}

}  // namespace sc

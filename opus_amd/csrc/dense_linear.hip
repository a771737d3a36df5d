// linear:  z = x W^T + bias,  y = residual + D(act(z)), and its gradients dx = dz W, dW = dz^T x, dbias = sum dz.
//
// All three are one product C[i, j] = sum_r A(i, r) B(j, r); an operand lies in memory either with r running fastest
// ("RC": x and W in the forward, dz in dx) or with i (j) running fastest (W in dx, both operands in dW).
//
// A workgroup makes a BM x BN tile of C.  128 bytes of r at a time (64 bf16 / fp16 or 32 fp32 values), both operands'
// tiles go to LDS by 16-byte transfers straight from memory (global_load_lds), double-buffered: the next tile is on
// its way while the matrix cores work on this one.  Where a base or a row is not 16-byte aligned, or r ends inside a
// tile, the tile goes through registers instead, zeros filled in.
//
// In LDS a 16-byte piece of an RC tile's row `row` stands at position piece ^ ((row >> 1) & 7): 16 rows read at the
// same piece hit all 64 banks.  The other kind of tile keeps memory's order of r rows; a wave reads its operands with
// ds_read_b64_tr_b16, which hands a lane four values of r at one i (fp32: plain 4-byte reads), and pieces are moved
// so that the rows of one read lie in different banks.
//
// Matrix instructions: 32 x 32 x 16 (16-bit types) and 32 x 32 x 2 (fp32), sums in fp32.  fp32 operands stay fp32.
//
// The epilogue turns a wave's 32-row strip of C round through LDS, so that a lane holds eight consecutive columns of
// one row: 16-byte accesses to bias, residual, z and y, and one generator call of the dropout for the eight.  Few
// tiles and a long r: r is cut up over workgroups, each stores its fp32 share, and a second kernel adds the shares in
// order and runs the epilogue.  No atomics: the result does not depend on the order of the workgroups.
//
// Measured on one MI355X (the library's plain products in brackets, same card and run; dW with the bias' gradient):
// 8192 x 4096 x 4096 bf16 forward 218 us = 1263 TFLOP/s (187), dx 218 (210), dW 224 (235); 4096^3 fp32 962 us = 143 TFLOP/s
// (916); 4800 x 256 -> 18432 bf16 forward 86 (88), both gradients 130 (200); 4800 x 8192 -> 256 fp32 forward 189 (224), both
// gradients 335 (355).  With silu and a residual the wide tile's matrix cores are busy 63 % of its cycles, LDS 26 %: without
// the transfers, or without the reads of LDS, it would be 15 % faster each, so both have to run beside the matrix
// instructions, which are interleaved with them.  With few steps of r (256) start and epilogue weigh as much as the product.
#include "dense_common.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------------------------------------
// epilogue
// ------------------------------------------------------------------------------------------------
struct Epilogue {
    const void *bias, *residual;
    void *y, *z;
    int act;
    DnDrop drop;
};

// v: eight values of C at (row, col ..), element `at` of y, `n` of them inside its `cols` columns (all of them, where !EDGE); col is a
// multiple of 8.  bias: those columns' (zeros without one).
template <class T, bool EDGE>
__device__ __forceinline__ void finish(const Epilogue &e, dn_floats<8> v, const dn_floats<8> &bias, uint64_t at, uint64_t row,
                                       uint32_t col, int n, int cols, uint64_t seed)
{
    if (!EDGE)
        n = 8;
    v += bias;
    if (e.z) {
        dn_floats<8> z = v;
        // What the rounding to 16 bits must not do: make a tiny z 0, which relu's gradient would take for a negative one, or a
        // large finite one inf, whose slope under gelu or silu would be inf x 0.
        if constexpr (sizeof(T) == 2) {
            constexpr float MOST = __is_same(T, dn_f16) ? 65504.f : 0x1.FEp127f;
            if (e.act == OPUS_DENSE_ACT_RELU) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if ((float)(T)z[j] == 0.f && z[j] > 0.f)
                        z[j] = 6e-8f;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    z[j] = __builtin_isinf(z[j]) || z[j] != z[j] ? z[j] : __builtin_amdgcn_fmed3f(z[j], -MOST, MOST);
            }
        }
        dn_store_n<8>(static_cast<T *>(e.z) + at, z, n);
    }
    dn_act<8, T>(v, e.act);
    if (e.drop.threshold)
        dn_drop<8>(v, row, col, seed, e.drop);
    if (e.residual)
        v += dn_load_n<8>(static_cast<const T *>(e.residual) + at, n, cols);
    dn_store_n<8>(static_cast<T *>(e.y) + at, v, n);
}

// ------------------------------------------------------------------------------------------------
// tiles
// ------------------------------------------------------------------------------------------------
struct GemmArgs {
    const void *a, *b;           // A(i, r), B(j, r)
    long long I, J, R;
    int tiles_i, tiles_j, splits, steps, steps_per_split;       // steps: tiles of 128 bytes along r
    float *partial;              // [splits][I][pitch], where splits > 1
    long long pitch;
    float *colsum;               // [splits * sharers][I]: shares of the sums over r of A(i, r) ..
    void *colsum_out;            // .. which belong here (at once, where there is one share); NULL: not wanted
    int sharers;                 // tiles of a row of tiles that share the sums' work (0: `colsum` holds sums made before)
    int sum_parts;               // rows of `colsum`
    Epilogue e;
};

template <class T> struct Elem;
template <> struct Elem<float> { static constexpr int PIECE = 4, STEP = 32; };
template <> struct Elem<dn_bf16> { static constexpr int PIECE = 8, STEP = 64; };
template <> struct Elem<dn_f16> { static constexpr int PIECE = 8, STEP = 64; };

// position of 16-byte piece `c` in row `row` of an LDS tile
__device__ __forceinline__ int place_rc(int row, int c) { return c ^ ((row >> 1) & 7); }
template <class T, int W> __device__ __forceinline__ int place_ic(int r, int c)
{
    if constexpr (sizeof(T) == 2 && W >= 128)
        return c ^ ((r & 3) << 2);              // four r rows of a transposing read: 64 bytes apart
    else if constexpr (sizeof(T) == 2)
        return c ^ ((r & 2) << 1);              // (a row of 128 bytes: its neighbour is in the other banks already)
    else
        return c ^ ((r & 4) << 1);              // rows r and r + 4 of a read: the two halves of the banks
}

// One operand's tile: W rows of C (i or j) x 128 bytes of r.
template <class T, bool RC, int W>
struct Tile {
    static constexpr int PIECE = Elem<T>::PIECE, STEP = Elem<T>::STEP;
    static constexpr int PIECES = W * 8;                             // 16-byte pieces
    static constexpr int ROW = RC ? 8 : W / PIECE;                   // pieces a row of the LDS tile
    static constexpr int BYTES = PIECES * 16;

    // piece p of the tile -> its coordinates: `w` (first i or the i), `r`
    static __device__ __forceinline__ void coords(int p, int &w, int &r)
    {
        const int row = p / ROW, pos = p % ROW;
        if constexpr (RC) {
            w = row;
            r = place_rc(row, pos) * PIECE;
        } else {
            r = row;
            w = place_ic<T, W>(row, pos) * PIECE;
        }
    }

    // Straight to LDS: a thread's pieces of the first tile, in bytes from the tile's base; the following tiles are a
    // uniform distance further.  Rows beyond `I` (columns, where !RC) fetch the last valid one: what they make of C is
    // never stored.
    template <int THREADS>
    static __device__ __forceinline__ void offsets(uint32_t (&off)[PIECES / THREADS], long long w0, long long I, long long R, int tid)
    {
        static_assert(PIECES % THREADS == 0, "whole turns");
#pragma unroll
        for (int t = 0; t < PIECES / THREADS; ++t) {
            int w, r;
            coords(t * THREADS + tid, w, r);
            if constexpr (RC)
                off[t] = (uint32_t)(min((long long)w, I - 1 - w0) * R + r) * sizeof(T);
            else
                off[t] = (uint32_t)(r * I + min((long long)w, I - PIECE - w0)) * sizeof(T);
        }
    }
    // the tile's base, and how far the next one is
    static __device__ __forceinline__ const char *origin(const T *base, long long w0, long long r0, long long I, long long R)
    {
        return reinterpret_cast<const char *>(RC ? base + w0 * R + r0 : base + r0 * I + w0);
    }
    static __device__ __forceinline__ long long advance(long long I) { return RC ? STEP * sizeof(T) : STEP * I * sizeof(T); }

    template <int THREADS>
    static __device__ __forceinline__ void fetch(const char *from, const uint32_t (&off)[PIECES / THREADS], char *lds, int wave)
    {
#pragma unroll
        for (int t = 0; t < PIECES / THREADS; ++t)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + off[t]),
                                             (__attribute__((address_space(3))) void *)(lds + (t * THREADS + wave * 64) * 16),
                                             16, 0, 0);
    }

    // Through registers: any alignment, zeros outside.
    template <int THREADS> using Pieces = typename DnVec<T, PIECE>::type[PIECES / THREADS];

    template <int THREADS>
    static __device__ __forceinline__ void read(Pieces<THREADS> &v, const T *base, long long w0, long long r0, long long I,
                                                long long R, int tid)
    {
#pragma unroll
        for (int t = 0; t < PIECES / THREADS; ++t) {
            int w, r;
            coords(t * THREADS + tid, w, r);
            const long long i = w0 + w, rr = r0 + r;
            const T *src = RC ? base + i * R + rr : base + rr * I + i;
            const long long inside = RC ? (i < I ? R - rr : 0) : (rr < R ? I - i : 0);
            v[t] = dn_load_raw<PIECE>(src, (int)max(-1ll, min(inside, (long long)PIECE)), (int)min((long long)PIECE, RC ? R : I));
        }
    }
    template <int THREADS> static __device__ __forceinline__ void write(const Pieces<THREADS> &v, char *lds, int tid)
    {
#pragma unroll
        for (int t = 0; t < PIECES / THREADS; ++t)
            *reinterpret_cast<typename DnVec<T, PIECE>::type *>(lds + (t * THREADS + tid) * 16) = v[t];
    }

    // A lane's operands of rows w .. w+31 (lane % 32) for k-group `ks` (of 4): RC order of r: pieces 2 ks + lane / 32.
    static __device__ __forceinline__ typename DnVec<T, PIECE>::type frag(const char *lds, int w, int ks, int lane)
    {
        if constexpr (RC) {
            const int row = w + (lane & 31);
            return *reinterpret_cast<const typename DnVec<T, PIECE>::type *>(
                lds + (row * 8 + place_rc(row, ks * 2 + (lane >> 5))) * 16);
        } else if constexpr (sizeof(T) == 2) {
            // 16 lanes transpose 4 r rows x 16 columns: lane q of the 16 points at row q / 4, columns 4 (q % 4) ..,
            // and receives the four rows of column q
            const int q = lane & 15;
            const int r = ks * 16 + (lane >> 5) * 8 + (q >> 2);
            const int col = w + ((lane >> 4) & 1) * 16 + (q & 3) * 4;
            const int at = (place_ic<T, W>(r, col >> 3) * 8 + (col & 7)) * 2;       // (r + 4 has the same r & 3)
            typedef __attribute__((address_space(3))) s16x4 *lp;
            const char *p = lds + r * (W * 2) + at;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * W * 2));
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(typename DnVec<T, 8>::type, v);
        } else {
            f32x4 v;
            const int col = w + (lane & 31);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int r = ks * 8 + (lane >> 5) * 4 + t;
                v[t] = *reinterpret_cast<const float *>(lds + r * (W * 4) + place_ic<T, W>(r, col >> 2) * 16 + (col & 3) * 4);
            }
            return v;
        }
    }
};

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c)
{
    // a lane's four values are four r of the eight of the group: any order serves, as long as A and B have the same
#pragma unroll
    for (int t = 0; t < 4; ++t)
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
    return c;
}

// s + the lane's values of an operand (two at a time: products with one)
__device__ __forceinline__ float add_up(bf16x8 v, float s)
{
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int t = 0; t < 8; t += 2)
        s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[t], v[t + 1]}, one, s, false);
    return s;
}
__device__ __forceinline__ float add_up(f16x8 v, float s)
{
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
    for (int t = 0; t < 8; t += 2)
        s = __builtin_amdgcn_fdot2(f16x2{v[t], v[t + 1]}, one, s, false);
    return s;
}
__device__ __forceinline__ float add_up(f32x4 v, float s) { return s + ((v[0] + v[1]) + (v[2] + v[3])); }

constexpr int STRIP = 72;       // floats a row of a wave's strip in LDS: rows four apart then start 32 banks apart

// LDS of a workgroup: two stages of both operands' tiles, and in their place the epilogue's strips
template <class T, int WI, int WJ, int MI, int MJ>
constexpr int gemm_lds = (2 * (WI * MI + WJ * MJ) * 32 * 128 > WI * WJ * 32 * STRIP * 4) ? 2 * (WI * MI + WJ * MJ) * 32 * 128
                                                                                        : WI * WJ * 32 * STRIP * 4;

// Workgroup `id` of a product: WI x WJ waves, each MI x MJ blocks of 32 x 32.  DIRECT: bases and rows are 16-byte aligned.
template <class T, bool ARC, bool BRC, int WI, int WJ, int MI, int MJ, bool DIRECT>
__device__ __forceinline__ void gemm_tile(const GemmArgs &g, int id, char *lds)
{
    constexpr int THREADS = WI * WJ * 64, BM = WI * MI * 32, BN = WJ * MJ * 32, STEP = Elem<T>::STEP;
    using TA = Tile<T, ARC, BM>;
    using TB = Tile<T, BRC, BN>;
    constexpr int STAGE = TA::BYTES + TB::BYTES;
    static_assert(2 * STAGE <= gemm_lds<T, WI, WJ, MI, MJ>, "two stages");

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi = wave / WJ, wj = wave % WJ;

    // Workgroups go to the eight XCDs in turn: give each XCD a contiguous run of tiles, so that the tiles sharing an
    // operand share an L2.
    const int total = g.tiles_i * g.tiles_j * g.splits, per = total >> 3, rest = total & 7, xcd = id & 7;
    id = xcd * per + min(xcd, rest) + (id >> 3);
    const int split = id / (g.tiles_i * g.tiles_j);
    id -= split * g.tiles_i * g.tiles_j;
    // tiles in bands of eight tile rows, down each band's columns
    const int band = id / (8 * g.tiles_j), high = min(8, g.tiles_i - band * 8);
    const int in = id - band * 8 * g.tiles_j;
    const int tj = in / high, ti = band * 8 + in % high;
    const long long i0 = (long long)ti * BM, j0 = (long long)tj * BN;
    const int s0 = split * g.steps_per_split, s1 = min(s0 + g.steps_per_split, g.steps);

    const T *pa = static_cast<const T *>(g.a), *pb = static_cast<const T *>(g.b);
    typename TA::template Pieces<THREADS> va;
    typename TB::template Pieces<THREADS> vb;
    const auto read = [&](int s) __attribute__((always_inline)) {
        TA::template read<THREADS>(va, pa, i0, (long long)s * STEP, g.I, g.R, tid);
        TB::template read<THREADS>(vb, pb, j0, (long long)s * STEP, g.J, g.R, tid);
    };
    const auto write = [&](char *to) __attribute__((always_inline)) {
        TA::template write<THREADS>(va, to, tid);
        TB::template write<THREADS>(vb, to + TA::BYTES, tid);
    };
    // whole tiles, which may go straight to LDS; the last one of all may not be
    const int whole = DIRECT ? min(s1, (int)(g.R / STEP)) : s0;
    uint32_t oa[TA::PIECES / THREADS], ob[TB::PIECES / THREADS];
    const char *fa0 = TA::origin(pa, i0, (long long)s0 * STEP, g.I, g.R), *fb0 = TB::origin(pb, j0, (long long)s0 * STEP, g.J, g.R);
    const long long na = TA::advance(g.I), nb = TB::advance(g.J);
    if constexpr (DIRECT) {
        TA::template offsets<THREADS>(oa, i0, g.I, g.R, tid);
        TB::template offsets<THREADS>(ob, j0, g.J, g.R, tid);
    }
    const auto fetch = [&](char *to) __attribute__((always_inline)) {
        TA::template fetch<THREADS>(fa0, oa, to, wave);
        TB::template fetch<THREADS>(fb0, ob, to + TA::BYTES, wave);
        fa0 += na;
        fb0 += nb;
    };

    f32x16 acc[MI][MJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j)
            acc[i][j] = 0.f;
    float sum[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
        sum[i] = 0.f;
    // The sums of A's rows: of a row of tiles the first `sharers` take turns at the steps of r, and of the waves that hold
    // the same rows each takes its k-groups of a step.
    const bool summing = !ARC && g.colsum_out && tj < g.sharers;

    typename DnVec<T, Elem<T>::PIECE>::type fa[2][MI], fb[2][MJ];
    constexpr bool F32 = sizeof(T) == 4;
    const auto load = [&](const char *from, int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
            fa[ks & 1][i] = TA::frag(from, (wi * MI + i) * 32, ks, lane);
#pragma unroll
        for (int j = 0; j < MJ; ++j)
            fb[ks & 1][j] = TB::frag(from + TA::BYTES, (wj * MJ + j) * 32, ks, lane);
    };
    bool turn_to_sum = false;
    const auto multiply = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < MJ; ++j)
                acc[i][j] = mma(fa[ks & 1][i], fb[ks & 1][j], acc[i][j]);
        if (!ARC && turn_to_sum && ks % WJ == wj)
#pragma unroll
            for (int i = 0; i < MI; ++i)
                sum[i] = add_up(fa[ks & 1][i], sum[i]);
    };
    // One barrier a tile, before its last k-group is multiplied: by then every wave holds that group in registers, so
    // the tile's buffer is free for the transfers of the tile after next, and the next tile, under way for a whole
    // tile's time, is complete; its first group is read while the last of this one is multiplied.
    const auto arrived = [] {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if (s0 < s1) {
        char *cur = lds, *next = lds + STAGE;
        if (DIRECT && s0 < whole) {
            fetch(cur);
        } else {
            read(s0);
            write(cur);
        }
        arrived();
        if (DIRECT && s0 + 1 < whole)
            fetch(next);
        load(cur, 0);
        int s = s0;
        if constexpr (DIRECT)
            for (; s + 2 < whole; ++s) {
                turn_to_sum = summing && s % g.sharers == tj;
                // matrix instructions between the operands' reads, and between the transfers, which the memory pipeline
                // takes in slowly (8192 x 4096 x 4096 bf16: 246 -> 225 us)
                constexpr int READS = (ARC ? MI : MI * (F32 ? 4 : 2)) + (BRC ? MJ : MJ * (F32 ? 4 : 2));
                constexpr int TRANSFERS = TA::PIECES / THREADS + TB::PIECES / THREADS;
                constexpr int PRODUCTS = MI * MJ, PAIR = (READS + PRODUCTS - 1) / PRODUCTS;
#pragma unroll
                for (int ks = 0; ks < 3; ++ks) {
                    load(cur, ks + 1);
                    multiply(ks);
                    if constexpr (!F32)          // (a group of fp32's is long enough: measured, no gain)
#pragma unroll
                        for (int k = 0; k < PRODUCTS; ++k) {
                            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x100, PAIR, 0);
                        }
                }
                arrived();
                load(next, 0);
                fetch(cur);
                multiply(3);
                __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
                for (int k = 0; k < TRANSFERS; ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
                }
                char *t = cur;
                cur = next;
                next = t;
            }
        for (; s < s1; ++s) {
            turn_to_sum = summing && s % g.sharers == tj;
            const bool more = s + 1 < s1, by_hand = more && s + 1 >= whole;
            if (!DIRECT && by_hand)             // under way while this tile is multiplied
                read(s + 1);
            load(cur, 1);
            multiply(0);
            load(cur, 2);
            multiply(1);
            load(cur, 3);
            multiply(2);
            if (more) {
                if (by_hand) {
                    if (DIRECT)                 // one tile of a product: not worth the registers it would hold
                        read(s + 1);
                    write(next);
                }
                arrived();
                if (DIRECT && s + 2 < whole)
                    fetch(cur);
                load(next, 0);
            }
            multiply(3);
            char *t = cur;
            cur = next;
            next = t;
        }
    }

    if constexpr (!ARC)
        if (summing) {                            // (uniform over the workgroup)
            __syncthreads();
            float *rows = reinterpret_cast<float *>(lds);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const float t = sum[i] + __shfl_xor(sum[i], 32);
                if (lane < 32)
                    rows[wj * BM + (wi * MI + i) * 32 + lane] = t;
            }
            __syncthreads();
            for (int r = tid; r < BM; r += THREADS)
                if (i0 + r < g.I) {
                    float t = rows[r];
#pragma unroll
                    for (int k = 1; k < WJ; ++k)
                        t += rows[k * BM + r];
                    if (g.colsum)
                        g.colsum[((long long)split * g.sharers + tj) * g.I + i0 + r] = t;
                    else
                        static_cast<T *>(g.colsum_out)[i0 + r] = (T)t;
                }
        }

    // ---- epilogue: a wave turns 32 rows x (32 MJ, at most 64) columns at a time through its own strip
    constexpr int SJ = MJ < 2 ? MJ : 2, CPR = SJ * 4, RPT = 64 / CPR;
    const uint64_t seed = dn_seed(g.e.drop);
    float *strip = reinterpret_cast<float *>(lds) + wave * 32 * STRIP;
    __syncthreads();
    const bool inside = i0 + BM <= g.I && j0 + BN <= g.J;
    // one turn of the loop a strip: the code behind it exists once, whatever the number of blocks
#pragma unroll 1
    for (int turn = 0; turn < MI * MJ / SJ; ++turn) {
        const int i = turn / (MJ / SJ), jj = turn % (MJ / SJ) * SJ;
#pragma unroll
        for (int k = 0; k < MI * MJ / SJ; ++k)
            if (turn == k)
#pragma unroll
                for (int j = 0; j < SJ; ++j)
#pragma unroll
                    for (int t = 0; t < 16; ++t)
                        strip[((t >> 2) * 8 + (lane >> 5) * 4 + (t & 3)) * STRIP + j * 32 + (lane & 31)] =
                            acc[k / (MJ / SJ)][k % (MJ / SJ) * SJ + j][t];
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int col = (lane % CPR) * 8;
        const float *from = strip + lane / CPR * STRIP + col;
        const long long ci = i0 + (wi * MI + i) * 32 + lane / CPR, cj = j0 + (wj * MJ + jj) * 32 + col;
        const auto value = [&](int q) __attribute__((always_inline)) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(from + q * RPT * STRIP);
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(from + q * RPT * STRIP + 4);
            return (dn_floats<8>)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        if (g.partial) {
            float *to = g.partial + (split * g.I + ci) * g.pitch + cj;
#pragma unroll
            for (int q = 0; q < 32 / RPT; ++q)
                if (ci + q * RPT < g.I && cj < g.J)
                    *reinterpret_cast<dn_floats<8> *>(to + q * RPT * g.pitch) = value(q);
        } else {
            const int n = (int)min(8ll, g.J - cj);
            dn_floats<8> bias = 0.f;
            if (g.e.bias)
                bias = dn_load_n<8>(static_cast<const T *>(g.e.bias) + cj, n, (int)g.J);
            uint64_t at = (uint64_t)ci * g.J + cj;
            if (inside) {
#pragma unroll
                for (int q = 0; q < 32 / RPT; ++q, at += RPT * g.J)
                    finish<T, false>(g.e, value(q), bias, at, ci + q * RPT, (uint32_t)cj, 8, (int)g.J, seed);
            } else {
#pragma unroll 1
                for (int q = 0; q < 32 / RPT; ++q, at += RPT * g.J)
                    if (ci + q * RPT < g.I && n > 0)
                        finish<T, true>(g.e, value(q), bias, at, ci + q * RPT, (uint32_t)cj, n, (int)g.J, seed);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    }
}

template <class T, bool ARC, bool BRC, int WI, int WJ, int MI, int MJ, bool DIRECT>
__global__ void __launch_bounds__(WI * WJ * 64) dense_gemm_kernel(GemmArgs g)
{
    __shared__ __align__(128) char lds[gemm_lds<T, WI, WJ, MI, MJ>];
    gemm_tile<T, ARC, BRC, WI, WJ, MI, MJ, DIRECT>(g, blockIdx.x, lds);
}

// Both products of the backward in one launch: first the one whose workgroups take longer (more steps of r each), then
// the other's, which fill up the CUs as those run out.
template <class T, int WI, int WJ, int MI, int MJ, bool DIRECT>
__global__ void __launch_bounds__(WI * WJ * 64) dense_gemm_pair_kernel(GemmArgs dx, GemmArgs dw, int dx0, int dw0)
{
    __shared__ __align__(128) char lds[gemm_lds<T, WI, WJ, MI, MJ>];
    // (one of dx0, dw0, the products' first workgroups, is 0)
    if ((int)blockIdx.x >= dx0 && (dx0 || (int)blockIdx.x < dw0))
        gemm_tile<T, true, false, WI, WJ, MI, MJ, DIRECT>(dx, blockIdx.x - dx0, lds);
    else
        gemm_tile<T, false, false, WI, WJ, MI, MJ, DIRECT>(dw, blockIdx.x - dw0, lds);
}

// The column sums' shares added up, by 256 threads: 16 columns, 16 lanes a column.
template <class T>
__device__ __forceinline__ void join_sums(const float *part, int parts, long long n, T *out, long long block)
{
    __shared__ float lds[16][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const long long i = block * 16 + x;
    float s = 0.f;
    if (i < n) {
#pragma unroll 4
        for (int k = y; k < parts; k += 16)
            s += part[k * n + i];
    }
    lds[y][x] = s;
    __syncthreads();
    if (y == 0 && i < n) {
#pragma unroll
        for (int k = 1; k < 16; ++k)
            s += lds[k][x];
        out[i] = (T)s;
    }
}

// Adds the shares of r in order and runs the epilogue, for one product or two; a thread takes eight columns of a row.
// The workgroups behind those, if any, add the second (or only) one's column sums' shares.
struct JoinArgs {
    GemmArgs g[2];
    unsigned blocks[2], sum_blocks;
};

template <class T>
__global__ void __launch_bounds__(256) dense_gemm_join_kernel(JoinArgs a)
{
    unsigned block = blockIdx.x;
    const int which = block >= a.blocks[0];
    if (which)
        block -= a.blocks[0];
    const GemmArgs &g = a.g[which];
    if (which && block >= a.blocks[1]) {
        join_sums<T>(g.colsum, g.sum_parts, g.I, static_cast<T *>(g.colsum_out), block - a.blocks[1]);
        return;
    }
    const uint64_t seed = dn_seed(g.e.drop);
    const uint32_t units = (uint32_t)(g.pitch / 8);
    const uint64_t u = (uint64_t)block * 256 + threadIdx.x;
    const uint64_t row = u / units;
    const uint32_t col = (uint32_t)(u - row * units) * 8;
    if (row >= (uint64_t)g.I)
        return;
    dn_floats<8> v = 0.f;
    const float *p = g.partial + row * g.pitch + col;
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s)
        v += *reinterpret_cast<const dn_floats<8> *>(p + s * g.I * g.pitch);
    const int n = (int)min(8ll, g.J - (long long)col);
    dn_floats<8> bias = 0.f;
    if (g.e.bias)
        bias = dn_load_n<8>(static_cast<const T *>(g.e.bias) + col, n, (int)g.J);
    finish<T, true>(g.e, v, bias, row * g.J + col, row, col, n, (int)g.J, seed);
}

// The product for up to 16 rows of x (single tokens), bound by reading W once: 16 columns of y a workgroup, r dealt to
// its waves.  W's rows are the matrix instruction's A operand and x's its B, both straight from memory in 16-byte
// pieces, eight steps of r at a time; the waves' shares meet in LDS, then the epilogue.  One launch, where tiles would
// need a second one to add the shares of r.
__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(f32x4 a, f32x4 b, f32x4 c)
{
#pragma unroll
    for (int t = 0; t < 4; ++t)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0);
    return c;
}

constexpr int FEW_ROWS = 16;

template <class T, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) dense_few_rows_kernel(const T *x, const T *w, int M, long long N, long long K, Epilogue e)
{
    constexpr int PIECE = Elem<T>::PIECE, STEP = 4 * PIECE, AHEAD = 8;
    __shared__ __align__(16) float lds[WAVES][16][20];               // [wave][row of x][column], padded
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long n0 = (long long)blockIdx.x * 16;
    const int r = lane & 15;
    const T *pw = w + min(n0 + r, N - 1) * K + (lane >> 4) * PIECE;  // (columns beyond N are never stored)
    const T *px = x + (long long)min(r, M - 1) * K + (lane >> 4) * PIECE;
    const long long each = (K + STEP * WAVES - 1) / (STEP * WAVES) * STEP;
    const long long k0 = wave * each, k1 = min(k0 + each, K);
    f32x4 acc = 0.f;
    long long k = k0;
    typename DnVec<T, PIECE>::type a[AHEAD], b[AHEAD];
    for (; k + AHEAD * STEP <= k1; k += AHEAD * STEP) {
#pragma unroll
        for (int t = 0; t < AHEAD; ++t) {
            a[t] = dn_load<PIECE>(pw + k + t * STEP);
            b[t] = dn_load<PIECE>(px + k + t * STEP);
        }
#pragma unroll
        for (int t = 0; t < AHEAD; ++t)
            acc = mma16(a[t], b[t], acc);
    }
    for (; k < k1; k += STEP) {
        const int left = (int)min(k1 - k - (lane >> 4) * PIECE, (long long)PIECE), row = (int)min(K, (long long)PIECE);
        acc = mma16(dn_load_raw<PIECE>(pw + k, left, row), dn_load_raw<PIECE>(px + k, left, row), acc);
    }
    // lane: row of x lane % 16, columns 4 (lane / 16) ..
    *reinterpret_cast<f32x4 *>(&lds[wave][r][(lane >> 4) * 4]) = acc;
    __syncthreads();
    const int m = threadIdx.x >> 1, c = (threadIdx.x & 1) * 8;
    const long long col = n0 + c;
    const int n = (int)min(8ll, N - col);
    if (m < M && n > 0) {
        dn_floats<8> v = 0.f;
#pragma unroll 4
        for (int s = 0; s < WAVES; ++s) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(&lds[s][m][c]), hi = *reinterpret_cast<const f32x4 *>(&lds[s][m][c + 4]);
            v += (dn_floats<8>)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        dn_floats<8> bias = 0.f;
        if (e.bias)
            bias = dn_load_n<8>(static_cast<const T *>(e.bias) + col, n, (int)N);
        finish<T, true>(e, v, bias, (uint64_t)m * N + col, m, (uint32_t)col, n, (int)N, dn_seed(e.drop));
    }
}

template <class T>
__global__ void __launch_bounds__(256) dense_colsum_join_kernel(const float *part, int parts, long long n, T *out)
{
    join_sums<T>(part, parts, n, out, blockIdx.x);
}

// Column sums of dz [M, N] by themselves (where dW is not wanted, or has no elements): 32 columns a workgroup
// and a run of rows, which the kernel above adds.
template <class T>
__global__ void __launch_bounds__(256) dense_colsum_kernel(const T *dz, long long M, long long N, long long rows_per, float *part)
{
    __shared__ float lds[8][33];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * 32 + x, first = blockIdx.y * rows_per, last = min(first + rows_per, M);
    float s = 0.f;
    if (col < N)
        for (long long m = first + y; m < last; m += 8)
            s += (float)dz[m * N + col];
    lds[y][x] = s;
    __syncthreads();
    if (y == 0 && col < N) {
#pragma unroll
        for (int k = 1; k < 8; ++k)
            s += lds[k][x];
        part[blockIdx.y * N + col] = s;
    }
}

// dz = D(dy) act'(z), and its column sums before it is rounded to 16 bits (after that the sums would be off by 1.4 times
// what their own rounding costs, 2 times where the kept elements' scale is half a step from a 16-bit number).  1 << lx
// threads a row, eight columns each; 256 >> lx rows at a time, whose sums meet in LDS; a run of rows a workgroup, which
// the kernels above add.  8192 x 4096 bf16 with silu and dropout: 46 us (201 MB, 4.4 TB/s, beside the generator and the slope);
// loading the next row ahead gains nothing.
//
// dz itself is rounded to 16 bits, and so was z before it: a 16-bit matrix instruction takes 16-bit operands, and dz in two parts
// would double both products of the backward.  Of fp16 gradients of 1237 x 333 -> 777 with gelu and dropout, relative to 64
// bits: 3.0e-4; z alone rounded 2.2e-4, dz alone 2.9e-4, only the results 2.1e-4.
struct DzArgs {
    const void *dy, *z;
    void *dz;
    long long M, N, rows_per;
    int lx, act;
    DnDrop drop;
    float *part;                 // [runs][N]
};

template <class T>
__global__ void __launch_bounds__(256) dense_dz_kernel(DzArgs a)
{
    __shared__ dn_floats<8> lds[256];
    const int tid = threadIdx.x, x = tid & ((1 << a.lx) - 1), y = tid >> a.lx, lanes = 256 >> a.lx;
    const long long col = (((long long)blockIdx.x << a.lx) + x) * 8, first = blockIdx.y * a.rows_per, last = min(first + a.rows_per, a.M);
    const int n = (int)max(0ll, min(8ll, a.N - col));
    const uint64_t seed = dn_seed(a.drop);
    dn_floats<8> s = 0.f;
    if (n > 0)
        for (long long row = first + y; row < last; row += lanes) {
            const long long at = row * a.N + col;
            dn_floats<8> v = dn_load_n<8>(static_cast<const T *>(a.dy) + at, n, (int)a.N);
            if (a.drop.threshold)
                dn_drop<8>(v, row, (uint32_t)col, seed, a.drop);
            if (a.z)
                dn_act_slope<8, T>(v, dn_load_n<8>(static_cast<const T *>(a.z) + at, n, (int)a.N), a.act);
            s += v;
            dn_store_n<8>(static_cast<T *>(a.dz) + at, v, n);
        }
    lds[tid] = s;
    for (int half = lanes >> 1; half; half >>= 1) {
        __syncthreads();
        if (y < half)
            lds[tid] = s += lds[tid + (half << a.lx)];
    }
    if (y == 0)
        dn_store_n<8>(a.part + blockIdx.y * a.N + col, s, n);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
constexpr int CUS = 256;

struct Plan {
    int tile;                    // index into TILES
    int tiles_i, tiles_j, splits, steps, steps_per_split;
    long long pitch;
    size_t bytes;                // of the fp32 shares
    int sharers;                 // of the column sums
    double cost;                 // the estimate
};

// The tiles a workgroup can make, rows x columns of C, the workgroups of a kind that fit a CU together (by LDS), and what
// a step of r costs one of them, in cycles, where the CU is full (16-bit types, fp32).
struct TileKind {
    int i, j, per_cu, cost16, cost32;
};
constexpr TileKind TILES[] = {{64, 64, 4, 330, 1350}, {128, 128, 2, 800, 4700}, {256, 256, 1, 2560, 18200}};

// Which tile, and into how many shares r is cut: the cheapest by this estimate.  A CU works through its workgroups in
// turns of as many as fit it; a step of r costs them together the cost above, and never less than the time a transfer
// takes to arrive; a workgroup's start and end cost about as much as a few steps; shares are written, read and added by
// a further kernel.  Against the best of a sweep over tiles and cuts it comes within 5 % for 30 of 33 products, within 12 %
// for two and 25 % for one (the odd 1237 x 333 -> 777's dx in 16 bits, which goes through registers: 17.2 us and 13.8).
constexpr double ARRIVE = 1400, START_END = 8000, JOIN = 14000, JOIN_BYTES = 2000;

// `only`: that kind of tile.
Plan plan(int type, long long I, long long J, long long R, int only = -1)
{
    Plan p = {};
    p.splits = 1;
    if (I < 1 || J < 1)
        return p;
    p.steps = (int)dn_ceil(R, type == OPUS_DENSE_F32 ? 32 : 64);
    p.pitch = dn_ceil(J, 8) * 8;
    const int most = p.steps / 2 < 64 ? p.steps / 2 : 64;
    const bool fp32 = type == OPUS_DENSE_F32;
    double &best = p.cost;
    for (int k = 0; k < 3; ++k) {
        if (only >= 0 && k != only)
            continue;
        const TileKind &t = TILES[k];
        const long long tiles = dn_ceil(I, t.i) * dn_ceil(J, t.j);
        // no cut, and the cuts that give every CU 1, 2, ... workgroups, up to two turns
        for (int m = 0; m <= 2 * t.per_cu; ++m) {
            const long long cut = m * CUS / tiles;
            const int n = m == 0 ? 1 : (int)(cut < most ? cut : most);
            if (m > 0 && n < 2)
                continue;
            const int each = (p.steps + n - 1) / n;
            const double a_cu = (double)((tiles * n + CUS - 1) / CUS);
            const double together = a_cu < t.per_cu ? a_cu : t.per_cu, turns = __builtin_ceil(a_cu / together);
            const double step = together * (fp32 ? t.cost32 : t.cost16);
            double cost = turns * (each * (step > ARRIVE ? step : ARRIVE) + START_END);
            if (n > 1)
                cost += JOIN + 8.0 * n * I * p.pitch / JOIN_BYTES;
            if (best == 0 || cost < best) {
                best = cost;
                p.tile = k;
                p.splits = n;
            }
            if (n == most)
                break;
        }
    }
    const TileKind &t = TILES[p.tile];
    p.tiles_i = (int)dn_ceil(I, t.i);
    p.tiles_j = (int)dn_ceil(J, t.j);
    p.steps_per_split = (int)dn_ceil(p.steps > 0 ? p.steps : 1, p.splits);
    p.splits = p.steps > 0 ? (int)dn_ceil(p.steps, p.steps_per_split) : 1;
    // the column sums are shared where there is much of r to a tile, else one tile's work costs less than another launch
    const int share = p.splits == 1 && p.steps >= 48 ? 8 : 1;
    p.sharers = p.tiles_j < share ? p.tiles_j : share;
    p.bytes = p.splits > 1 ? (size_t)p.splits * I * p.pitch * sizeof(float) : 0;
    return p;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class T, bool ARC, bool BRC, bool DIRECT>
void launch_tiles(const Plan &p, const GemmArgs &g, hipStream_t s)
{
    const dim3 grid((unsigned)(p.tiles_i * p.tiles_j * p.splits));
    if (p.tile == 2)
        hipLaunchKernelGGL((dense_gemm_kernel<T, ARC, BRC, 2, 4, 4, 2, DIRECT>), grid, dim3(512), 0, s, g);
    else if (p.tile == 1)
        hipLaunchKernelGGL((dense_gemm_kernel<T, ARC, BRC, 2, 2, 2, 2, DIRECT>), grid, dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((dense_gemm_kernel<T, ARC, BRC, 2, 2, 1, 1, DIRECT>), grid, dim3(256), 0, s, g);
}

// C = A B^T with an epilogue, planned as `p`.  shares: p.bytes of workspace.  sums_out [I]: the sums over r of A(i, r), or
// NULL; sums: [p.splits * p.sharers][I] of workspace for them.
struct Product {
    GemmArgs g;
    bool direct;
    long long blocks;
};

template <class T, bool ARC, bool BRC>
Product product(const Plan &p, const void *a, const void *b, long long I, long long J, long long R, const Epilogue &e,
                float *shares, float *sums, void *sums_out)
{
    const int piece = Elem<T>::PIECE;
    // (a tile's pieces are addressed in 32 bits from its corner)
    const auto near = [](bool rc, long long i, long long r) { return (rc ? 256 * r : 64 * i) * sizeof(T) < (1ll << 31); };
    return {{a, b, I, J, R, p.tiles_i, p.tiles_j, p.splits, p.steps, p.steps_per_split, p.splits > 1 ? shares : nullptr, p.pitch,
             p.splits * p.sharers > 1 ? sums : nullptr, sums_out, p.sharers, p.splits * p.sharers, e},
            aligned16(a) && aligned16(b) && (ARC ? R : I) % piece == 0 && (BRC ? R : J) % piece == 0 && near(ARC, I, R) && near(BRC, J, R),
            (long long)p.tiles_i * p.tiles_j * p.splits};
}

// What is left to do behind one product or two (NULL): shares to add, and the second one's column sums.
template <class T>
hipError_t join(const GemmArgs *one, const GemmArgs &two, hipStream_t s)
{
    JoinArgs a = {};
    long long blocks[2] = {0, 0};
    if (one && one->splits > 1) {
        a.g[0] = *one;
        blocks[0] = dn_ceil(one->I * (one->pitch / 8), 256);
    }
    a.g[1] = two;
    if (two.splits > 1)
        blocks[1] = dn_ceil(two.I * (two.pitch / 8), 256);
    const long long sums = two.colsum_out && two.colsum ? dn_ceil(two.I, 16) : 0, all = blocks[0] + blocks[1] + sums;
    if (all * 256 > 0xFFFFFFFFll)
        return hipErrorInvalidValue;
    a.blocks[0] = (unsigned)blocks[0];
    a.blocks[1] = (unsigned)blocks[1];
    a.sum_blocks = (unsigned)sums;
    if (all)
        hipLaunchKernelGGL(dense_gemm_join_kernel<T>, dim3((unsigned)all), dim3(256), 0, s, a);
    return hipSuccess;
}

template <class T, bool ARC, bool BRC>
hipError_t gemm(const Plan &p, const Product &q, hipStream_t s)
{
    if (q.blocks * (p.tile == 2 ? 512 : 256) > 0xFFFFFFFFll)
        return hipErrorInvalidValue;
    if (q.direct)
        launch_tiles<T, ARC, BRC, true>(p, q.g, s);
    else
        launch_tiles<T, ARC, BRC, false>(p, q.g, s);
    return join<T>(nullptr, q.g, s);
}

// runs of rows of dense_colsum_kernel
long long colsum_runs(long long M, long long N)
{
    const long long want = dn_ceil(4 * CUS, dn_ceil(N, 32)), most = dn_ceil(M, 64);
    const long long runs = want < most ? want : most;
    return runs < 1 ? 1 : runs > 65535 ? 65535 : runs;
}

// dense_dz_kernel's threads a row (their logarithm), and its runs of rows: eight workgroups a CU, of a row a thread or more
// (1237 x 777 fp16: 7.5 us, of two rows 10.9)
int dz_lanes(long long N)
{
    int lx = 0;
    while (lx < 5 && (8ll << lx) < N)
        ++lx;
    return lx;
}
long long dz_runs(long long M, long long N)
{
    const int lx = dz_lanes(N);
    const long long want = dn_ceil(8 * CUS, dn_ceil(N, 8 << lx)), most = dn_ceil(M, 256 >> lx);
    const long long runs = want < most ? want : most;
    return runs < 1 ? 1 : runs;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// The backward's two products, as they are planned where both are wanted: side by side in one launch if their tiles
// are of one of the kinds of four waves (then of the kind that is cheaper for both).
struct PlanPair {
    Plan dx, dw;
    bool together;
};

PlanPair plan_pair(int type, long long M, long long N, long long K)
{
    PlanPair p = {plan(type, M, K, N), plan(type, N, K, M), false};
    if (M > 0 && N > 0 && K > 0 && p.dx.tile < 2 && p.dw.tile < 2) {
        if (p.dx.tile != p.dw.tile) {
            const PlanPair a = {plan(type, M, K, N, 0), plan(type, N, K, M, 0), false};
            const PlanPair b = {plan(type, M, K, N, 1), plan(type, N, K, M, 1), false};
            p = a.dx.cost + a.dw.cost < b.dx.cost + b.dw.cost ? a : b;
        }
        p.together = true;
    }
    return p;
}

size_t sums_bytes(const Plan &p, long long N) { return (size_t)p.splits * p.sharers * N * sizeof(float); }

// made: dz's column sums, [dz_runs][N], where they were made along with dz (else NULL)
template <class T>
hipError_t backward(int type, const void *dz, const void *x, const void *w, long long M, long long N, long long K,
                    void *dx, void *dw, void *db, float *ws, const float *made, hipStream_t s)
{
    const auto take = [&](Product q) {
        if (made) {
            q.g.colsum = const_cast<float *>(made);
            q.g.sharers = 0;
            q.g.sum_parts = (int)dz_runs(M, N);
        }
        return q;
    };
    const bool want_dx = dx && M && K, want_dw = dw && N && K;
    const Epilogue ex = {nullptr, nullptr, dx, nullptr, OPUS_DENSE_ACT_NONE, {}}, ew = {nullptr, nullptr, dw, nullptr, OPUS_DENSE_ACT_NONE, {}};
    if (want_dx && want_dw) {
        const PlanPair p = plan_pair(type, M, N, K);
        if (p.together) {
            float *const shares = ws + align256(p.dx.bytes) / sizeof(float), *const sums = shares + align256(p.dw.bytes) / sizeof(float);
            const Product qx = product<T, true, false>(p.dx, dz, w, M, K, N, ex, ws, nullptr, nullptr);
            const Product qw = take(product<T, false, false>(p.dw, dz, x, N, K, M, ew, shares, sums, db));
            const long long blocks = qx.blocks + qw.blocks;
            if (blocks * 256 > 0xFFFFFFFFll)
                return hipErrorInvalidValue;
            const dim3 grid((unsigned)blocks);
            const bool dw_first = p.dw.steps_per_split > p.dx.steps_per_split;
            const int dx0 = dw_first ? (int)qw.blocks : 0, dw0 = dw_first ? 0 : (int)qx.blocks;
            const bool direct = qx.direct && qw.direct;
            if (p.dx.tile == 1 && direct)
                hipLaunchKernelGGL((dense_gemm_pair_kernel<T, 2, 2, 2, 2, true>), grid, dim3(256), 0, s, qx.g, qw.g, dx0, dw0);
            else if (p.dx.tile == 1)
                hipLaunchKernelGGL((dense_gemm_pair_kernel<T, 2, 2, 2, 2, false>), grid, dim3(256), 0, s, qx.g, qw.g, dx0, dw0);
            else if (direct)
                hipLaunchKernelGGL((dense_gemm_pair_kernel<T, 2, 2, 1, 1, true>), grid, dim3(256), 0, s, qx.g, qw.g, dx0, dw0);
            else
                hipLaunchKernelGGL((dense_gemm_pair_kernel<T, 2, 2, 1, 1, false>), grid, dim3(256), 0, s, qx.g, qw.g, dx0, dw0);
            return join<T>(&qx.g, qw.g, s);
        }
    }
    hipError_t e = hipSuccess;
    if (want_dx) {
        const Plan p = plan(type, M, K, N);
        e = gemm<T, true, false>(p, product<T, true, false>(p, dz, w, M, K, N, ex, ws, nullptr, nullptr), s);
    }
    if (e != hipSuccess)
        return e;
    if (want_dw) {
        const Plan p = plan(type, N, K, M);
        float *const sums = ws + align256(p.bytes) / sizeof(float);
        e = gemm<T, false, false>(p, take(product<T, false, false>(p, dz, x, N, K, M, ew, ws, sums, db)), s);
    } else if (db && N && made) {
        hipLaunchKernelGGL(dense_colsum_join_kernel<T>, dim3((unsigned)dn_ceil(N, 16)), dim3(256), 0, s, made,
                           (int)dz_runs(M, N), N, static_cast<T *>(db));
    } else if (db && N) {
        const long long runs = colsum_runs(M, N), per = dn_ceil(M > 0 ? M : 1, runs);
        hipLaunchKernelGGL(dense_colsum_kernel<T>, dim3((unsigned)dn_ceil(N, 32), (unsigned)runs), dim3(256), 0, s,
                           static_cast<const T *>(dz), M, N, per, ws);
        hipLaunchKernelGGL(dense_colsum_join_kernel<T>, dim3((unsigned)dn_ceil(N, 16)), dim3(256), 0, s, ws,
                           (int)runs, N, static_cast<T *>(db));
    }
    return e;
}

}  // namespace

// Few rows take their own kernel rather than tiles (1 row, 1024 -> 4096 bf16: 3.5 us and 7.3; 16 rows, 4096 -> 4096: 10.3
// and 12.8; 1 row, 8192 -> 8192 fp32: 44 and 78), but for two shapes: few columns over long rows of W, which leave most of
// the chip idle (1 row, 8192 -> 256 fp32: 20.0 and 16.0), and many 16-bit rows over a large W, where reading x again for
// every 16 columns shows (16 rows, 8192 -> 8192 bf16: 32 and 25).  Of 252 products measured around the limits the rule takes
// the slower kernel for 30, by 26 % at most (8 rows, 16384 -> 2048 bf16: 25.7 and 20.4).
static bool few_rows(int type, long long M, long long N, long long K)
{
    if (M > FEW_ROWS)
        return false;
    if (N <= 1024 && K * (long long)dn_type_bytes(type) >= 32768)
        return false;
    return type == OPUS_DENSE_F32 || M <= 8 || N * K < (1ll << 25);
}

size_t dn_linear_forward_workspace(int type, long long M, long long N, long long K)
{
    return M > 0 && N > 0 && !few_rows(type, M, N, K) ? plan(type, M, N, K).bytes : 0;
}

template <class T>
static hipError_t forward(int type, const void *x, const void *w, long long M, long long N, long long K, const Epilogue &e,
                          float *workspace, hipStream_t s)
{
    if (!few_rows(type, M, N, K)) {
        const Plan p = plan(type, M, N, K);
        return gemm<T, true, true>(p, product<T, true, true>(p, x, w, M, N, K, e, workspace, nullptr, nullptr), s);
    }
    if (dn_ceil(N, 16) * 256 > 0xFFFFFFFFll)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)dn_ceil(N, 16));
    const T *tx = static_cast<const T *>(x), *tw = static_cast<const T *>(w);
    // sixteen waves where four would leave each a long run of r, and there are too few columns to fill the chip
    if (N <= 16 * 2 * CUS && K >= 64 * Elem<T>::STEP)
        hipLaunchKernelGGL((dense_few_rows_kernel<T, 16>), grid, dim3(1024), 0, s, tx, tw, (int)M, N, K, e);
    else
        hipLaunchKernelGGL((dense_few_rows_kernel<T, 4>), grid, dim3(256), 0, s, tx, tw, (int)M, N, K, e);
    return hipSuccess;
}

hipError_t dn_launch_linear_forward(int type, const void *x, const void *w, const void *bias, const void *residual,
                                    long long M, long long N, long long K, int act, const DnDrop &drop, void *y,
                                    void *z, float *workspace, hipStream_t s)
{
    if (M == 0 || N == 0)
        return hipSuccess;
    const Epilogue e = {bias, residual, y, z, act, drop};
    const hipError_t stale = hipPeekAtLastError();
    const hipError_t r = type == OPUS_DENSE_F32 ? forward<float>(type, x, w, M, N, K, e, workspace, s)
                       : type == OPUS_DENSE_BF16 ? forward<dn_bf16>(type, x, w, M, N, K, e, workspace, s)
                                                 : forward<dn_f16>(type, x, w, M, N, K, e, workspace, s);
    return r != hipSuccess ? r : msmv_launch_status(stale);
}

// the products' part of the backward's workspace; behind it, for 16-bit types, the column sums made along with dz
static size_t products_workspace(int type, long long M, long long N, long long K)
{
    if (N <= 0)
        return 0;
    const Plan px = plan(type, M, K, N), pw = plan(type, N, K, M);
    const PlanPair both = plan_pair(type, M, N, K);
    size_t most = px.bytes;
    const auto at_least = [&](size_t n) { most = most > n ? most : n; };
    at_least(align256(pw.bytes) + sums_bytes(pw, N));
    at_least((size_t)colsum_runs(M, N) * N * sizeof(float));
    if (both.together)
        at_least(align256(both.dx.bytes) + align256(both.dw.bytes) + sums_bytes(both.dw, N));
    return align256(most);
}

size_t dn_linear_backward_workspace(int type, long long M, long long N, long long K)
{
    if (N <= 0)
        return 0;
    const size_t products = products_workspace(type, M, N, K);
    return type == OPUS_DENSE_F32 ? products : products + (size_t)dz_runs(M, N) * N * sizeof(float);
}

// The column sums are made along with dz only for 16-bit types: an fp32 dz is not rounded, and the products' workgroups
// add it up at less cost.
hipError_t dn_launch_linear_backward(int type, const void *dy, const void *x, const void *w, const void *z, long long M,
                                     long long N, long long K, int act, const DnDrop &drop, void *dz_buffer, void *dx,
                                     void *dw, void *db, float *workspace, hipStream_t s)
{
    const bool prepare = (act != OPUS_DENSE_ACT_NONE || drop.threshold) && M > 0 && N > 0;
    float *made = nullptr;
    hipError_t r = hipSuccess;
    const hipError_t stale = hipPeekAtLastError();
    if (prepare && db && type != OPUS_DENSE_F32) {
        made = workspace + products_workspace(type, M, N, K) / sizeof(float);
        const long long runs = dz_runs(M, N);
        const DzArgs a = {dy, act != OPUS_DENSE_ACT_NONE ? z : nullptr, dz_buffer, M, N, dn_ceil(M, runs), dz_lanes(N), act, drop, made};
        const dim3 grid((unsigned)dn_ceil(N, 8 << a.lx), (unsigned)runs);
        if (type == OPUS_DENSE_BF16)
            hipLaunchKernelGGL(dense_dz_kernel<dn_bf16>, grid, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL(dense_dz_kernel<dn_f16>, grid, dim3(256), 0, s, a);
    } else if (prepare) {
        r = dn_launch_elementwise(type, dy, nullptr, act != OPUS_DENSE_ACT_NONE ? z : nullptr, act, M, N, drop, dz_buffer, s);
    }
    if (r != hipSuccess)
        return r;
    const void *dz = prepare ? dz_buffer : dy;
    r = type == OPUS_DENSE_F32 ? backward<float>(type, dz, x, w, M, N, K, dx, dw, db, workspace, made, s)
      : type == OPUS_DENSE_BF16 ? backward<dn_bf16>(type, dz, x, w, M, N, K, dx, dw, db, workspace, made, s)
                                : backward<dn_f16>(type, dz, x, w, M, N, K, dx, dw, db, workspace, made, s);
    return r != hipSuccess ? r : msmv_launch_status(stale);
}

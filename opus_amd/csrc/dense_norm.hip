// residual_norm:  r = scale * x + gate * D(post(block)),  y = norm(r), forward and backward.
//
// Bound by memory: forward two reads and up to two writes an element, backward four reads and two writes.  A row is
// read once and stays in registers: TPR threads share it, each holding CH runs of VEC consecutive elements, so the
// mean, the sum of squared deviations from it (two passes over registers, not over memory: no cancellation) and the
// results cost no second read.  A wave takes a row of up to 512 elements by itself (sums by lane exchange alone);
// wider rows take 2 to 16 waves and one LDS exchange a sum.
//
// Backward: r, and with a post-norm the block's normed rows, are computed again from x and block with the forward's
// statistics.  Sums over rows (dweight, dbias, dpost_*, dgate) stay with the thread while its workgroup
// walks a run of rows, are stored once a workgroup as fp32 rows, and a second small kernel adds those up: no atomics,
// the same order every time.  All sums are in fp32.
//
// Where that is more than a thread has registers for, the compiler keeps the rest in scratch memory: in the backward above
// 8192 elements (320 to 1312 bytes a lane), of odd widths above 4096 (36 to 652), and of whole ones there with post-norm and
// biases (52 to 60); in the forward above 8192 in fp32 and of odd widths (44 to 244).
//
// Measured on one MI355X: 38400 x 256 fp32 LayerNorm with dropout 28 us forward (157 MB, 5.6 TB/s), 40 backward (236 MB,
// 5.9 TB/s) and 6 for the sums over rows; 8192 x 8192 bf16 RMS with post-norm and a gate a sample 110 forward (537 MB,
// 4.9 TB/s), 215 backward (805 MB, 3.7 TB/s: a row of 8192 and its sums fill a thread's registers, so only one row is worked
// on and one under way) and 10.  Whole steps' backwards of 8192 bf16 rows with post-norm: 8192 wide RMS 202 us, LayerNorm 262;
// 5003 RMS 273; 10001 RMS 1879; 16384 RMS 1433, LayerNorm 1914, against 340 for that one's bytes at a copy's rate: above 8192
// it is bound by the scratch memory.
#include "dense_common.h"

namespace {

struct NormArgs {
    const void *x, *block, *weight, *bias, *post_weight, *post_bias, *gate;
    void *y, *stream_out;
    float *stats;
    const void *dy, *dstream;
    void *dx, *dblock, *dgate;                               // dgate: in T, where a workgroup owns whole gate rows
    float *part_w, *part_b, *part_pw, *part_pb, *part_gate;  // [workgroups, width], NULL: not wanted
    long long rows, gate_rows, rows_per_gate, rows_per_group;
    int chunks;                                              // workgroups a gate row (1: a workgroup takes rows_per_group whole ones)
    int gate_per_row;                                        // backward: a gate row for every row (dgate then needs no sum)
    int width, rms;
    float eps, scale, inv_width;
    DnDrop drop;
};

// Sums N values over the TPR threads of a row; every thread gets the totals.  `lds` holds N * 16 floats and is free
// again at the next call's first barrier: calls alternate between two halves.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float *lds, int &phase)
{
#pragma unroll
    for (int m = 32; m; m >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] += __shfl_xor(v[i], m);
    if constexpr (TPR > 64) {
        constexpr int WAVES = TPR / 64;
        float *half = lds + phase * 32;
        phase ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i)
                half[i * 16 + (threadIdx.x >> 6)] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
                t += half[i * 16 + w];
            v[i] = t;
        }
    }
}

template <int CH, int VEC> using Row = dn_floats<VEC>[CH];
template <class T, int CH, int VEC> using Raw = typename DnVec<T, VEC>::type[CH];       // a row as it lies in memory

template <class T, int TPR, int VEC, int CH, bool WHOLE>
__device__ __forceinline__ void load_row(Raw<T, CH, VEC> &r, const T *p, int lane, int width)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + lane) * VEC;
        r[c] = dn_load_raw<VEC, WHOLE>(p + col, width - col, width);
    }
}

template <class T, int TPR, int VEC, int CH, bool WHOLE>
__device__ __forceinline__ void store_row(T *p, const Row<CH, VEC> &r, int lane, int width)
{
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + lane) * VEC;
        dn_store_n<VEC, WHOLE>(p + col, r[c], width - col);
    }
}

// A vector of `width` that every row uses: held in registers where a thread's part is small (KEEP), else loaded again
// (from the caches) for every row.
template <class T, int TPR, int VEC, int CH, bool WHOLE, bool KEEP>
struct Param {
    Raw<T, KEEP ? CH : 1, VEC> held;
    const T *p;
    __device__ __forceinline__ Param(const void *from, int lane, int width) : p(static_cast<const T *>(from))
    {
        if constexpr (KEEP)
            if (p)
                load_row<T, TPR, VEC, CH, WHOLE>(held, p, lane, width);
    }
    __device__ __forceinline__ explicit operator bool() const { return p; }
    __device__ __forceinline__ dn_floats<VEC> at(int c, int lane, int width) const
    {
        if constexpr (KEEP) {
            return __builtin_convertvector(held[c], dn_floats<VEC>);
        } else {
            const int col = (c * TPR + lane) * VEC;
            return dn_load_n<VEC, WHOLE>(p + col, width - col, width);
        }
    }
};

// mean (0 for RMS) and 1 / sigma of a row in registers (zeros beyond `width`)
template <int TPR, int VEC, int CH>
__device__ __forceinline__ void row_stats(const Row<CH, VEC> &r, int lane, const NormArgs &a, float *lds, int &phase,
                                          float &mean, float &rstd)
{
    float s[1] = {0.f};
    mean = 0.f;
    if (!a.rms) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                s[0] += r[c][j];
        row_sum<TPR, 1>(s, lds, phase);
        mean = s[0] * a.inv_width;
        s[0] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int n = a.width - (c * TPR + lane) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float d = j < n ? r[c][j] - mean : 0.f;
            s[0] += d * d;
        }
    }
    row_sum<TPR, 1>(s, lds, phase);
    rstd = 1.f / sqrtf(s[0] * a.inv_width + a.eps);
}

constexpr int group_threads(int TPR) { return TPR < 128 ? 256 : TPR; }

// The next row's values are on their way while a row is worked on.
template <class T, int TPR, int VEC, int CH, bool WHOLE>
__global__ void __launch_bounds__(group_threads(TPR)) dense_norm_forward_kernel(NormArgs a)
{
    constexpr int ROWS = group_threads(TPR) / TPR;
    constexpr bool KEEP = sizeof(T) * VEC * CH <= 16;
    __shared__ float lds[64];
    int phase = 0;
    const int lane = threadIdx.x % TPR, sub = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
    // every thread of a workgroup makes the same number of turns (the sums have barriers where TPR > 64, and then
    // ROWS is 1)
    const long long first = (long long)blockIdx.x * ROWS + sub, stride = (long long)gridDim.x * ROWS;
    if (first >= a.rows)
        return;
    const uint64_t seed = dn_seed(a.drop);
    const T *x = static_cast<const T *>(a.x), *block = static_cast<const T *>(a.block);
    Raw<T, CH, VEC> next_h, next_x;
    load_row<T, TPR, VEC, CH, WHOLE>(next_h, block + first * a.width, lane, a.width);
    load_row<T, TPR, VEC, CH, WHOLE>(next_x, x + first * a.width, lane, a.width);
    using P = Param<T, TPR, VEC, CH, WHOLE, KEEP>;
    const P weight(a.weight, lane, a.width), bias(a.bias, lane, a.width);
    const P pw(a.post_weight, lane, a.width), pb(a.post_bias, lane, a.width);
    for (long long row = first; row < a.rows; row += stride) {
        const long long at = row * a.width;
        Row<CH, VEC> h, r;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            h[c] = __builtin_convertvector(next_h[c], dn_floats<VEC>);
            r[c] = __builtin_convertvector(next_x[c], dn_floats<VEC>);
        }
        if (row + stride < a.rows) {
            load_row<T, TPR, VEC, CH, WHOLE>(next_h, block + at + stride * a.width, lane, a.width);
            load_row<T, TPR, VEC, CH, WHOLE>(next_x, x + at + stride * a.width, lane, a.width);
        }
        float mean2 = 0.f, rstd2 = 1.f, mean, rstd;
        const T *gate = a.gate ? static_cast<const T *>(a.gate) + row / a.rows_per_gate * a.width : nullptr;
        if (pw)
            row_stats<TPR, VEC, CH>(h, lane, a, lds, phase, mean2, rstd2);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + lane) * VEC, n = a.width - col;
            dn_floats<VEC> u = h[c];
            if (pw) {
                u = (u - mean2) * rstd2 * pw.at(c, lane, a.width);
                if (pb)
                    u += pb.at(c, lane, a.width);
            }
            if (a.drop.threshold)
                dn_drop<VEC>(u, row, col, seed, a.drop);
            if (gate)
                u *= dn_load_n<VEC, WHOLE>(gate + col, n, a.width);
            r[c] = r[c] * a.scale + u;
            if (!WHOLE && n < VEC)                 // what lies beyond the row stays out of its sums
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    r[c][j] = j < n ? r[c][j] : 0.f;
        }
        if (a.stream_out)
            store_row<T, TPR, VEC, CH, WHOLE>(static_cast<T *>(a.stream_out) + at, r, lane, a.width);
        row_stats<TPR, VEC, CH>(r, lane, a, lds, phase, mean, rstd);
        if (a.stats && lane == 0)
            *reinterpret_cast<float4 *>(a.stats + row * 4) = make_float4(mean2, rstd2, mean, rstd);
        if (a.y) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                r[c] = (r[c] - mean) * rstd;
                if (weight)
                    r[c] *= weight.at(c, lane, a.width);
                if (bias)
                    r[c] += bias.at(c, lane, a.width);
            }
            store_row<T, TPR, VEC, CH, WHOLE>(static_cast<T *>(a.y) + at, r, lane, a.width);
        }
    }
}

// Adds `acc` of the workgroup's ROWS row lanes and stores it as one row of `width` floats (or of T).
template <class O, int TPR, int VEC, int CH, bool WHOLE>
__device__ __forceinline__ void flush(O *out, Row<CH, VEC> &acc, float *cols, int lane, int sub, int width)
{
    constexpr int ROWS = group_threads(TPR) / TPR;
    if constexpr (ROWS == 1) {
        store_row<O, TPR, VEC, CH, WHOLE>(out, acc, lane, width);
    } else {
        static_assert(CH == 1, "the first row's threads add a whole row");
        __syncthreads();
        *reinterpret_cast<dn_floats<VEC> *>(cols + (sub * TPR + lane) * VEC) = acc[0];
        __syncthreads();
        if (sub == 0) {
            dn_floats<VEC> t = acc[0];
#pragma unroll
            for (int w = 1; w < ROWS; ++w)
                t += *reinterpret_cast<const dn_floats<VEC> *>(cols + (w * TPR + lane) * VEC);
            dn_store_n<VEC, WHOLE>(out + lane * VEC, t, width - lane * VEC);
        }
    }
}

// POST: with a post-norm.  BIAS: a bias' gradient may be wanted.  A workgroup works on rows_per_group consecutive rows of one gate row where chunks > 1,
// otherwise on rows_per_group whole gate rows.  AHEAD: the next row's
// values are on their way while a row is worked on.
template <class T, int TPR, int VEC, int CH, bool WHOLE, bool POST, bool BIAS>
__global__ void __launch_bounds__(group_threads(TPR)) dense_norm_backward_kernel(NormArgs a)
{
    constexpr int ROWS = group_threads(TPR) / TPR;
    constexpr bool KEEP = sizeof(T) * VEC * CH <= 16;
    // Not where the next row's registers would spill, or spill more: 8192 x 8192 bf16 with a post-norm 337 us ahead, 376 not, but
    // with biases as well 454 and 421; 5003 wide, whose last vectors are partial, 293 and 279 (RMS).  (Eight elements a thread
    // of 1024 threads instead of 16 of 512: 397 and up.)
    constexpr bool AHEAD = CH == 1 || (WHOLE && TPR < 1024 && sizeof(T) == 2 && !(POST && BIAS));
    __shared__ float lds[64];
    __shared__ __align__(16) float cols[ROWS > 1 ? ROWS * TPR * VEC : 4];
    int phase = 0;
    const int lane = threadIdx.x % TPR, sub = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR), width = a.width;
    const uint64_t seed = dn_seed(a.drop);
    const T *x = static_cast<const T *>(a.x), *block = static_cast<const T *>(a.block);
    const T *dy_in = static_cast<const T *>(a.dy), *ds_in = static_cast<const T *>(a.dstream);

    Row<CH, VEC> dw, db, dpw, dpb, dg;
#pragma unroll
    for (int c = 0; c < CH; ++c)
        dw[c] = db[c] = dpw[c] = dpb[c] = dg[c] = 0.f;

    // rows first .. last of gate rows g0 .. g1
    long long g0, g1, first, last;
    if (a.chunks > 1) {
        g0 = blockIdx.x / a.chunks;
        g1 = g0 + 1;
        first = g0 * a.rows_per_gate + (blockIdx.x - g0 * a.chunks) * a.rows_per_group;
        last = min(first + a.rows_per_group, g1 * a.rows_per_gate);
    } else {
        g0 = blockIdx.x * a.rows_per_group;
        g1 = min(g0 + a.rows_per_group, a.gate_rows);
        first = g0 * a.rows_per_gate;
        last = g1 * a.rows_per_gate;
    }
    Raw<T, CH, VEC> raw_h, raw_x, raw_dy, raw_ds;
    float4 raw_st = make_float4(0.f, 1.f, 0.f, 1.f);
    const auto load = [&](long long row) __attribute__((always_inline)) {
        const long long at = row * width;
        load_row<T, TPR, VEC, CH, WHOLE>(raw_h, block + at, lane, width);
        load_row<T, TPR, VEC, CH, WHOLE>(raw_x, x + at, lane, width);
        if (dy_in)
            load_row<T, TPR, VEC, CH, WHOLE>(raw_dy, dy_in + at, lane, width);
        if (ds_in)
            load_row<T, TPR, VEC, CH, WHOLE>(raw_ds, ds_in + at, lane, width);
        raw_st = *reinterpret_cast<const float4 *>(a.stats + row * 4);
    };
#pragma unroll
    for (int c = 0; c < CH; ++c)
        raw_dy[c] = raw_ds[c] = (T)0.f;
    if (AHEAD && first + sub < last)
        load(first + sub);
    using P = Param<T, TPR, VEC, CH, WHOLE, KEEP>;
    const P weight(a.weight, lane, width), pw(POST ? a.post_weight : nullptr, lane, width), pb(POST ? a.post_bias : nullptr, lane, width);

    long long row = first + sub;
    for (long long g = g0; g < g1; ++g) {
        const long long end = min((g + 1) * a.rows_per_gate, last);
        const T *gate = a.gate ? static_cast<const T *>(a.gate) + g * width : nullptr;
        for (; row < end; row += ROWS) {
            const long long at = row * width;
            if (a.gate_per_row)
                gate = static_cast<const T *>(a.gate) + at;
            if (!AHEAD)
                load(row);
            Row<CH, VEC> h, r, dy;
            Raw<T, CH, VEC> ds;
            const float4 st = raw_st;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                h[c] = __builtin_convertvector(raw_h[c], dn_floats<VEC>);
                r[c] = __builtin_convertvector(raw_x[c], dn_floats<VEC>);
                dy[c] = __builtin_convertvector(raw_dy[c], dn_floats<VEC>);
                ds[c] = raw_ds[c];
            }
            if (AHEAD && row + ROWS < last)
                load(row + ROWS);
            // xhat in r, D(post(block)) in u
            float s[2] = {0.f, 0.f};
            Row<CH, VEC> u;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * TPR + lane) * VEC, n = width - col;
                if constexpr (POST) {
                    h[c] = (h[c] - st.x) * st.y;                        // hhat
                    u[c] = h[c] * pw.at(c, lane, width);
                    if (pb)
                        u[c] += pb.at(c, lane, width);
                } else {
                    u[c] = h[c];
                }
                if (a.drop.threshold)
                    dn_drop<VEC>(u[c], row, col, seed, a.drop);
                r[c] = r[c] * a.scale + (gate ? u[c] * dn_load_n<VEC, WHOLE>(gate + col, n, width) : u[c]);
                r[c] = (r[c] - st.z) * st.w;
                dw[c] += dy[c] * r[c];
                if constexpr (BIAS)
                    db[c] += dy[c];
                if (weight)
                    dy[c] *= weight.at(c, lane, width);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {                         // (dy is zero beyond the row)
                    s[0] += dy[c][j];
                    s[1] += dy[c][j] * r[c][j];
                }
            }
            row_sum<TPR, 2>(s, lds, phase);
            const float m0 = a.rms ? 0.f : s[0] * a.inv_width, m1 = s[1] * a.inv_width;
            float t[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * TPR + lane) * VEC, n = width - col;
                dn_floats<VEC> dr = st.w * (dy[c] - m0 - r[c] * m1) + __builtin_convertvector(ds[c], dn_floats<VEC>);
                if (a.dx)
                    dn_store_n<VEC, WHOLE>(static_cast<T *>(a.dx) + at + col, dr * a.scale, n);
                if (gate) {
                    const dn_floats<VEC> dgate = dr * u[c];
                    dg[c] += dgate;
                    if (a.dgate && a.gate_per_row)
                        dn_store_n<VEC, WHOLE>(static_cast<T *>(a.dgate) + at + col, dgate, n);
                    dr *= dn_load_n<VEC, WHOLE>(gate + col, n, width);
                }
                if (a.drop.threshold)
                    dn_drop<VEC>(dr, row, col, seed, a.drop);
                if constexpr (POST) {
                    dpw[c] += dr * h[c];
                    if constexpr (BIAS)
                        dpb[c] += dr;
                    u[c] = dr * pw.at(c, lane, width);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        t[0] += u[c][j];
                        t[1] += u[c][j] * h[c][j];
                    }
                } else if (a.dblock) {
                    dn_store_n<VEC, WHOLE>(static_cast<T *>(a.dblock) + at + col, dr, n);
                }
            }
            if constexpr (POST) {
                row_sum<TPR, 2>(t, lds, phase);
                const float n0 = a.rms ? 0.f : t[0] * a.inv_width, n1 = t[1] * a.inv_width;
                if (a.dblock) {
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        u[c] = st.y * (u[c] - n0 - h[c] * n1);
                    store_row<T, TPR, VEC, CH, WHOLE>(static_cast<T *>(a.dblock) + at, u, lane, width);
                }
            }
        }
        if (gate && !a.gate_per_row) {
            if (a.part_gate)
                flush<float, TPR, VEC, CH, WHOLE>(a.part_gate + (long long)blockIdx.x * width, dg, cols, lane, sub, width);
            else if (a.dgate)
                flush<T, TPR, VEC, CH, WHOLE>(static_cast<T *>(a.dgate) + g * width, dg, cols, lane, sub, width);
#pragma unroll
            for (int c = 0; c < CH; ++c)
                dg[c] = 0.f;
        }
    }
    const long long mine = (long long)blockIdx.x * width;
    if (a.part_w)
        flush<float, TPR, VEC, CH, WHOLE>(a.part_w + mine, dw, cols, lane, sub, width);
    if (BIAS && a.part_b)
        flush<float, TPR, VEC, CH, WHOLE>(a.part_b + mine, db, cols, lane, sub, width);
    if constexpr (POST) {
        if (a.part_pw)
            flush<float, TPR, VEC, CH, WHOLE>(a.part_pw + mine, dpw, cols, lane, sub, width);
        if (BIAS && a.part_pb)
            flush<float, TPR, VEC, CH, WHOLE>(a.part_pb + mine, dpb, cols, lane, sub, width);
    }
}

// out[g, col] = sum of part[g * count .. +count][col], for up to five tensors (blockIdx.z) of one row and the gate's
// of gate_rows.  16 columns a workgroup, 16 row lanes that are added in LDS.
struct ReduceArgs {
    const float *part[5];
    void *out[5];
    long long groups[5];
    long long count[5];
    int width;
};

template <class T>
__global__ void __launch_bounds__(256) dense_reduce_rows_kernel(ReduceArgs a)
{
    __shared__ float lds[16][17];
    const int z = blockIdx.z, x = threadIdx.x & 15, y = threadIdx.x >> 4, col = blockIdx.x * 16 + x;
    for (long long g = blockIdx.y; g < a.groups[z]; g += gridDim.y) {
        const long long first = g * a.count[z], last = first + a.count[z];
        float s = 0.f;
        if (col < a.width) {
#pragma unroll 8
            for (long long i = first + y; i < last; i += 16)
                s += a.part[z][i * a.width + col];
        }
        lds[y][x] = s;
        __syncthreads();
        if (y == 0 && col < a.width) {
#pragma unroll
            for (int i = 1; i < 16; ++i)
                s += lds[i][x];
            static_cast<T *>(a.out[z])[g * a.width + col] = (T)s;
        }
        __syncthreads();
    }
}

// How the backward's rows are dealt to workgroups.
struct NormPlan {
    long long groups_rows, rows_per_gate, rows_per_group, workgroups;
    int chunks;
};

int threads_per_row(long long width)
{
    return width <= 512 ? 64 : width <= 1024 ? 128 : width <= 2048 ? 256 : width <= 8192 ? 512 : 1024;
}

NormPlan plan_backward(long long rows, long long width, long long gate_rows)
{
    const int tpr = threads_per_row(width), lanes = group_threads(tpr) / tpr;
    // 16 waves a CU hide each other's latency (8 of the widest kinds fill its registers); more workgroups, or ones of
    // fewer than four rows a wave, would only lengthen the second kernel's sums
    const long long full = width > 4096 ? 256 : 256 * (1024 / group_threads(tpr)), worth = dn_ceil(rows, 4 * lanes);
    const long long target = full < worth ? full : worth;
    NormPlan p;
    if (rows < 1) {                      // nothing to add: every sum is empty
        p = {gate_rows > 0 ? gate_rows : 1, 0, 0, 0, 1};
        return p;
    }
    p.groups_rows = gate_rows <= 0 || gate_rows == rows ? 1 : gate_rows;     // a gate row of its own for every row needs no sums
    p.rows_per_gate = rows / p.groups_rows;
    if (p.groups_rows >= target) {
        p.chunks = 1;
        p.rows_per_group = dn_ceil(p.groups_rows, target);
        p.workgroups = dn_ceil(p.groups_rows, p.rows_per_group);
    } else {
        const long long want = dn_ceil(target, p.groups_rows);
        p.rows_per_group = dn_ceil(dn_ceil(p.rows_per_gate, want), lanes) * lanes;
        p.chunks = (int)dn_ceil(p.rows_per_gate, p.rows_per_group);
        if (p.chunks <= 1) {
            p.chunks = 1;
            p.rows_per_group = 1;
        }
        p.workgroups = p.groups_rows * p.chunks;
    }
    return p;
}

template <class T, int TPR, int VEC, int CH, bool WHOLE>
void launch_forward(const NormArgs &a, hipStream_t s)
{
    constexpr int ROWS = group_threads(TPR) / TPR;
    const long long blocks = dn_ceil(a.rows, ROWS);
    const unsigned grid = (unsigned)(blocks < 2048 ? blocks : 2048);
    hipLaunchKernelGGL((dense_norm_forward_kernel<T, TPR, VEC, CH, WHOLE>), dim3(grid), dim3(group_threads(TPR)), 0, s, a);
}

template <class T, int TPR, int VEC, int CH, bool WHOLE, bool POST>
void launch_backward(const NormArgs &a, unsigned grid, hipStream_t s)
{
    // sums nobody wants are left out where registers are short
    const bool bias = a.part_b || a.part_pb;
    if (CH > 1 && !bias)
        hipLaunchKernelGGL((dense_norm_backward_kernel<T, TPR, VEC, CH, WHOLE, POST, CH == 1>), dim3(grid), dim3(group_threads(TPR)), 0, s, a);
    else
        hipLaunchKernelGGL((dense_norm_backward_kernel<T, TPR, VEC, CH, WHOLE, POST, true>), dim3(grid), dim3(group_threads(TPR)), 0, s, a);
}
template <class T, int TPR, int VEC, int CH, bool WHOLE>
void launch_backward(const NormArgs &a, unsigned grid, hipStream_t s)
{
    if (a.post_weight)
        launch_backward<T, TPR, VEC, CH, WHOLE, true>(a, grid, s);
    else
        launch_backward<T, TPR, VEC, CH, WHOLE, false>(a, grid, s);
}

// The narrowest variant that holds the row: 4 or 8 elements a thread (16 in the last two).  WHOLE: no thread's elements cross
// the row's end.
#define NORM_DISPATCH(CALL)                              \
    if (a.width <= 256) { CALL(64, 4, 1); }              \
    else if (a.width <= 512) { CALL(64, 8, 1); }         \
    else if (a.width <= 1024) { CALL(128, 8, 1); }       \
    else if (a.width <= 2048) { CALL(256, 8, 1); }       \
    else if (a.width <= 4096) { CALL(512, 8, 1); }       \
    else if (a.width <= 8192) { CALL(512, 8, 2); }       \
    else { CALL(1024, 8, 2); }

template <class T>
void dispatch_forward(const NormArgs &a, hipStream_t s)
{
#define CALL(TPR, VEC, CH) a.width % VEC ? launch_forward<T, TPR, VEC, CH, false>(a, s) : launch_forward<T, TPR, VEC, CH, true>(a, s)
    NORM_DISPATCH(CALL)
#undef CALL
}

template <class T>
void dispatch_backward(const NormArgs &a, unsigned grid, hipStream_t s)
{
#define CALL(TPR, VEC, CH) a.width % VEC ? launch_backward<T, TPR, VEC, CH, false>(a, grid, s) : launch_backward<T, TPR, VEC, CH, true>(a, grid, s)
    NORM_DISPATCH(CALL)
#undef CALL
}

NormArgs common_args(const opus_dense_norm_t &in, const DnDrop &drop)
{
    NormArgs a = {};
    a.x = in.x; a.block = in.block; a.weight = in.weight; a.bias = in.bias;
    a.post_weight = in.post_weight; a.post_bias = in.post_weight ? in.post_bias : nullptr; a.gate = in.gate;
    a.rows = in.rows;
    a.gate_rows = in.gate && in.gate_rows > 0 ? in.gate_rows : 1;
    a.rows_per_gate = in.rows / a.gate_rows;
    a.width = (int)in.width;
    a.rms = in.kind == OPUS_DENSE_NORM_RMS;
    a.eps = in.eps; a.scale = in.scale; a.inv_width = 1.f / (float)in.width;
    a.drop = drop;
    return a;
}

}  // namespace

hipError_t dn_launch_norm_forward(const opus_dense_norm_t &in, const DnDrop &drop, void *y, void *stream_out,
                                  float *stats, hipStream_t s)
{
    NormArgs a = common_args(in, drop);
    a.y = y; a.stream_out = stream_out; a.stats = stats;
    const hipError_t stale = hipPeekAtLastError();
    if (in.type == OPUS_DENSE_F32) dispatch_forward<float>(a, s);
    else if (in.type == OPUS_DENSE_BF16) dispatch_forward<dn_bf16>(a, s);
    else dispatch_forward<dn_f16>(a, s);
    return msmv_launch_status(stale);
}

size_t dn_norm_backward_workspace(long long rows, long long width, long long gate_rows)
{
    if (rows < 1 || width < 1)
        return 0;
    const NormPlan p = plan_backward(rows, width, gate_rows);
    return (size_t)p.workgroups * 5 * width * sizeof(float);
}

hipError_t dn_launch_norm_backward(const opus_dense_norm_t &in, const DnDrop &drop, const void *dy,
                                   const void *dstream, const float *stats, const opus_dense_norm_grads_t &out,
                                   float *workspace, hipStream_t s)
{
    NormArgs a = common_args(in, drop);
    const NormPlan p = plan_backward(in.rows, in.width, in.gate ? in.gate_rows : 0);
    a.stats = const_cast<float *>(stats);
    a.dy = dy; a.dstream = dstream;
    a.dx = out.dx; a.dblock = out.dblock;
    a.chunks = p.chunks;
    a.gate_rows = p.groups_rows;
    a.rows_per_gate = p.rows_per_gate;
    a.rows_per_group = p.rows_per_group;
    a.gate_per_row = in.gate && in.gate_rows == in.rows;
    const long long plane = p.workgroups * in.width;
    float *const w = workspace;
    a.part_w = out.dweight ? w : nullptr;
    a.part_b = out.dbias ? w + plane : nullptr;
    if (in.post_weight) {
        a.part_pw = out.dpost_weight ? w + 2 * plane : nullptr;
        a.part_pb = out.dpost_bias ? w + 3 * plane : nullptr;
    }
    if (in.gate && out.dgate) {
        if (a.gate_per_row || p.chunks == 1)
            a.dgate = out.dgate;
        else
            a.part_gate = w + 4 * plane;
    }
    ReduceArgs r = {};
    int n = 0;
    const auto add = [&](const float *part, void *o, long long groups, long long count) {
        if (o) {
            r.part[n] = part; r.out[n] = o; r.groups[n] = groups; r.count[n] = count;
            ++n;
        }
    };
    add(a.part_w, out.dweight, 1, p.workgroups);
    add(a.part_b, out.dbias, 1, p.workgroups);
    add(a.part_pw, out.dpost_weight, 1, p.workgroups);
    add(a.part_pb, out.dpost_bias, 1, p.workgroups);
    if (a.part_gate || (in.rows == 0 && in.gate_rows > 0))
        add(a.part_gate, out.dgate, p.groups_rows, in.rows ? p.chunks : 0);
    r.width = (int)in.width;
    long long groups = 1;
    for (int i = 0; i < n; ++i)
        groups = r.groups[i] > groups ? r.groups[i] : groups;
    groups = groups < 65535 ? groups : 65535;

    const unsigned grid = (unsigned)p.workgroups;
    const dim3 rgrid((unsigned)dn_ceil(in.width, 16), (unsigned)groups, (unsigned)n);
    const hipError_t stale = hipPeekAtLastError();
    if (in.type == OPUS_DENSE_F32) {
        if (grid) dispatch_backward<float>(a, grid, s);
        if (n) hipLaunchKernelGGL(dense_reduce_rows_kernel<float>, rgrid, dim3(256), 0, s, r);
    } else if (in.type == OPUS_DENSE_BF16) {
        if (grid) dispatch_backward<dn_bf16>(a, grid, s);
        if (n) hipLaunchKernelGGL(dense_reduce_rows_kernel<dn_bf16>, rgrid, dim3(256), 0, s, r);
    } else {
        if (grid) dispatch_backward<dn_f16>(a, grid, s);
        if (n) hipLaunchKernelGGL(dense_reduce_rows_kernel<dn_f16>, rgrid, dim3(256), 0, s, r);
    }
    return msmv_launch_status(stale);
}

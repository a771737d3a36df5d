// Shared by the dense operators (include/opus_dense.h): element types and vector access, the dropout generator,
// activations, and the host-side launchers.
#pragma once
#include "../../include/opus_dense.h"
#include "msmv_launch.h"

#include <stdint.h>

typedef __bf16 dn_bf16;
typedef _Float16 dn_f16;

// N elements of T in registers.  `at` is the same vector with T's own alignment: gfx950 takes global vector accesses
// at any element address, so rows of odd length are loaded and stored in vectors too (an aligned address costs
// nothing extra, an odd one a second cache line at times).
template <class T, int N> struct DnVec {
    typedef T type __attribute__((ext_vector_type(N)));
    typedef T at __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <int N> using dn_floats = typename DnVec<float, N>::type;

template <int N, class T> __device__ __forceinline__ typename DnVec<T, N>::type dn_load(const T *p)
{
    return *reinterpret_cast<const typename DnVec<T, N>::at *>(p);
}
template <int N, class T> __device__ __forceinline__ void dn_store(T *p, typename DnVec<T, N>::type v)
{
    *reinterpret_cast<typename DnVec<T, N>::at *>(p) = v;
}

// The n elements at p, 0 < n < N, and zeros: the vector that ends with them, shifted down.  N - n elements before p
// have to be readable (the row has N elements or more).
template <int N, class T> __device__ __forceinline__ typename DnVec<T, N>::type dn_load_tail(const T *p, int n)
{
    constexpr int W = N * sizeof(T) / 4;
    typedef uint32_t words __attribute__((ext_vector_type(W)));
    const int skip = N - n;
    words a = __builtin_bit_cast(words, dn_load<N>(p - skip));
    const int whole = sizeof(T) == 4 ? skip : skip >> 1;
#pragma unroll
    for (int b = W / 2; b; b /= 2)
#pragma unroll
        for (int i = 0; i < W; ++i)
            a[i] = whole & b ? (i + b < W ? a[i + b] : 0u) : a[i];
    if (sizeof(T) == 2)
#pragma unroll
        for (int i = 0; i < W; ++i)
            a[i] = skip & 1 ? (uint32_t)(((i + 1 < W ? (uint64_t)a[i + 1] << 32 : 0) | a[i]) >> 16) : a[i];
    return __builtin_bit_cast(typename DnVec<T, N>::type, a);
}

// Up to N elements: all N where `n` >= N, zeros beyond `n` otherwise.  `row`: how many the whole row has.  WHOLE: n is
// no less than N if it is positive at all.
template <int N, bool WHOLE = false, class T>
__device__ __forceinline__ typename DnVec<T, N>::type dn_load_raw(const T *p, int n, int row)
{
    typename DnVec<T, N>::type r = (T)0.f;
    if (WHOLE) {
        if (n > 0)
            r = dn_load<N>(p);
    } else if (n >= N) {
        r = dn_load<N>(p);
    } else if (n > 0) {
        if (row >= N) {
            r = dn_load_tail<N>(p, n);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j < n)
                    r[j] = p[j];
        }
    }
    return r;
}
template <int N, bool WHOLE = false, class T>
__device__ __forceinline__ dn_floats<N> dn_load_n(const T *p, int n, int row)
{
    return __builtin_convertvector(dn_load_raw<N, WHOLE>(p, n, row), dn_floats<N>);
}

// The first `n` of N floats, each rounded to T once, to nearest even.
template <int N, bool WHOLE = false, class T> __device__ __forceinline__ void dn_store_n(T *p, dn_floats<N> v, int n)
{
    typename DnVec<T, N>::type r = __builtin_convertvector(v, typename DnVec<T, N>::type);
    if (WHOLE) {
        if (n > 0)
            dn_store<N>(p, r);
    } else if (n >= N) {
        dn_store<N>(p, r);
    } else if (n > 0) {
        // halves, quarters, ... of the vector, the stored part shifted out each time
#pragma unroll
        for (int b = N / 2; b; b /= 2)
            if (n & b) {
                if (b == 4)
                    dn_store<4>(p, __builtin_shufflevector(r, r, 0, 1, 2, 3));
                else if (b == 2)
                    dn_store<2>(p, __builtin_shufflevector(r, r, 0, 1));
                else
                    p[0] = r[0];
                p += b;
#pragma unroll
                for (int j = 0; j + b < N; ++j)
                    r[j] = r[j + b];
            }
    }
}

// ------------------------------------------------------------------------------------------------
// dropout
// ------------------------------------------------------------------------------------------------
struct DnDrop {
    uint32_t threshold;          // 0: no dropout
    uint32_t offset;
    float scale;                 // 65536 / (65536 - threshold); 0 where everything is dropped
    uint64_t seed;
    const uint64_t *seed_ptr;
};

__device__ __forceinline__ uint64_t dn_seed(const DnDrop &d)
{
    return d.threshold && d.seed_ptr ? *d.seed_ptr : d.seed;
}

// Philox 4x32-10 (Salmon, Moraes, Dror, Shaw, SC'11): ten rounds of two 32 x 32 -> 64-bit products.  The round keys
// depend on the seed alone and stay in scalar registers.
__device__ __forceinline__ void dn_philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint64_t seed,
                                          uint32_t (&out)[4])
{
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

// D on N (4 or 8) consecutive elements of a row, the first at column `col`, a multiple of N.  16 bits an element:
// one generator call serves eight, which keeps a 16-bit tensor's dropout bound by memory (with 32 bits an element
// the ten rounds, about 480 cycles of a SIMD for 64 calls, would take longer than the bytes).  A dropped element is
// selected away, not multiplied by zero: inf and NaN vanish with it.
template <int N>
__device__ __forceinline__ void dn_drop(dn_floats<N> &v, uint64_t row, uint32_t col, uint64_t seed, const DnDrop &d)
{
    uint32_t w[4];
    dn_philox(col >> 3, (uint32_t)row, (uint32_t)(row >> 32), d.offset, seed, w);
    if (N == 4 && (col & 4)) {
        w[0] = w[2];
        w[1] = w[3];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t bits = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
        v[j] = bits >= d.threshold ? v[j] * d.scale : 0.f;
    }
}

// ------------------------------------------------------------------------------------------------
// activations (in fp32)
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float dn_relu(float z) { return z > 0.f ? z : (z != z ? z : 0.f); }
// 0.5 z (1 + tanh u) = z / (1 + exp(-2u)), u = sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float dn_gelu_tanh(float z)
{
    return z / (1.f + expf(-1.59576912f * (z + 0.044715f * z * z * z)));
}
__device__ __forceinline__ float dn_silu(float z) { return z / (1.f + expf(-z)); }

// 1 / (1 + exp(-a)), for results that are rounded to 16 bits with the hardware's exponential and reciprocal: the error is
// within 2^-21 (1 + |a|) of the value against a half step of 2^-11 (fp16) or 2^-8 (bf16), and 0 instead of the 1e-38 that is
// left below a = -87.  8192 x 4096 x 4096 bf16 with silu: 225 us, 242 with expf and a division; with gelu_tanh 228 and 244
// (221 without either); 4800 x 256 -> 18432 bf16 with silu 109 and 160 (96 without).  dz of 8192 x 4096 bf16 with silu and
// dropout 46 and 58.
template <class T> __device__ __forceinline__ float dn_sigmoid(float a)
{
    if constexpr (sizeof(T) == 4)
        return 1.f / (1.f + expf(-a));
    else
        return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * a));
}

// Phi(z), the normal distribution, and exp(-z^2 / 2).  1 + erf would cancel for negative z, where Phi is what is left: gelu(-5)
// would be off by 2 %, gelu(-5.5) be 0.  For 16-bit types Phi(-|z|) = exp(-z^2 / 2) times a polynomial in 1 / (1 + 0.26 |z|),
// fitted to erfcx(|z| / sqrt 2) / 2 over 0 .. 15 by least squares, reweighted until the largest relative error was smallest
// (2^-24.9; with its roundings and the hardware's exponential and reciprocal within 2^-20 (1 + z^2)).  8192 x 4096 x 4096
// bf16 with gelu: 237 us (erff 246, erfcf 256; 221 without activation); 4800 x 256 -> 18432 bf16: 146 (173, 208; 96).  fp32,
// 4800 x 256 -> 1024: erfcf 48 us, erff 45.5.
template <class T> __device__ __forceinline__ float dn_normal(float z, float &bell)
{
    if constexpr (sizeof(T) == 4) {
        bell = expf(-0.5f * z * z);
        return 0.5f * erfcf(-0.70710678f * z);
    } else {
        constexpr float C[] = {1.03755139e-01f, 1.03083022e-01f, 1.02560110e-01f,
                               5.28595224e-02f, 1.56652570e-01f, -1.44729093e-01f,
                               2.46046543e-01f, -1.50188193e-01f, 2.99603622e-02f};
        const float t = __builtin_amdgcn_rcpf(1.f + 0.26f * __builtin_fabsf(z));
        float p = C[8];
#pragma unroll
        for (int i = 7; i >= 0; --i)
            p = p * t + C[i];
        bell = __builtin_amdgcn_exp2f(-0.72134752f * z * z);
        const float tail = p * t * bell;
        return z < 0.f ? tail : 1.f - tail;
    }
}
template <class T> __device__ __forceinline__ float dn_gelu(float z)
{
    float bell;
    return z * dn_normal<T>(z, bell);
}
template <class T> __device__ __forceinline__ float dn_gelu_slope(float z)
{
    float bell;
    const float cdf = dn_normal<T>(z, bell);
    return cdf + z * 0.39894228f * bell;
}

// s = (1 + tanh u) / 2;  s + 2 z s (1 - s) u'.  Beyond |z| = 16 s is 0 or 1, and z^2 may not become inf beside that zero.
template <class T> __device__ __forceinline__ float dn_gelu_tanh_slope(float z)
{
    z = z > 16.f ? 16.f : z < -16.f ? -16.f : z;                 // NaN stays
    const float z2 = z * z, s = dn_sigmoid<T>(1.59576912f * (z + 0.044715f * z * z2));
    return s + 2.f * z * s * (1.f - s) * 0.79788456f * (1.f + 0.134145f * z2);
}
template <class T> __device__ __forceinline__ float dn_silu_slope(float z)
{
    const float s = dn_sigmoid<T>(z);
    return s * (1.f + z * (1.f - s));
}

// v[j] = act(v[j]), rounded to T next; the choice is uniform and outside the loops
template <int N, class T> __device__ __forceinline__ void dn_act(dn_floats<N> &v, int act)
{
#define DN_EACH(expr) _Pragma("unroll") for (int j = 0; j < N; ++j) v[j] = expr
    switch (act) {
    case OPUS_DENSE_ACT_RELU: DN_EACH(dn_relu(v[j])); break;
    case OPUS_DENSE_ACT_GELU: DN_EACH(dn_gelu<T>(v[j])); break;
    case OPUS_DENSE_ACT_GELU_TANH:
        if constexpr (sizeof(T) == 4)
            DN_EACH(dn_gelu_tanh(v[j]));
        else
            DN_EACH(v[j] * dn_sigmoid<T>(1.59576912f * (v[j] + 0.044715f * v[j] * v[j] * v[j])));
        break;
    case OPUS_DENSE_ACT_SILU:
        if constexpr (sizeof(T) == 4)
            DN_EACH(dn_silu(v[j]));
        else
            DN_EACH(v[j] * dn_sigmoid<T>(v[j]));
        break;
    default: break;
    }
}

// v[j] *= act'(z[j])
template <int N, class T> __device__ __forceinline__ void dn_act_slope(dn_floats<N> &v, const dn_floats<N> &z, int act)
{
    switch (act) {
    case OPUS_DENSE_ACT_RELU: DN_EACH(z[j] > 0.f ? v[j] : 0.f); break;
    case OPUS_DENSE_ACT_GELU: DN_EACH(v[j] * dn_gelu_slope<T>(z[j])); break;
    case OPUS_DENSE_ACT_GELU_TANH: DN_EACH(v[j] * dn_gelu_tanh_slope<T>(z[j])); break;
    case OPUS_DENSE_ACT_SILU: DN_EACH(v[j] * dn_silu_slope<T>(z[j])); break;
    default: break;
    }
#undef DN_EACH
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
inline size_t dn_type_bytes(int type) { return type == OPUS_DENSE_F32 ? 4 : 2; }
inline long long dn_ceil(long long a, long long b) { return (a + b - 1) / b; }

// y = residual + D(x) (slope == NULL), or D(x) * act'(slope) (slope = z, residual NULL).
hipError_t dn_launch_elementwise(int type, const void *x, const void *residual, const void *slope, int act,
                                 long long rows, long long cols, const DnDrop &drop, void *y, hipStream_t s);

hipError_t dn_launch_norm_forward(const opus_dense_norm_t &in, const DnDrop &drop, void *y, void *stream_out,
                                  float *stats, hipStream_t s);
size_t dn_norm_backward_workspace(long long rows, long long width, long long gate_rows);
hipError_t dn_launch_norm_backward(const opus_dense_norm_t &in, const DnDrop &drop, const void *dy,
                                   const void *dstream, const float *stats, const opus_dense_norm_grads_t &out,
                                   float *workspace, hipStream_t s);

size_t dn_linear_forward_workspace(int type, long long M, long long N, long long K);
hipError_t dn_launch_linear_forward(int type, const void *x, const void *w, const void *bias, const void *residual,
                                    long long M, long long N, long long K, int act, const DnDrop &drop, void *y,
                                    void *z, float *workspace, hipStream_t s);
size_t dn_linear_backward_workspace(int type, long long M, long long N, long long K);
hipError_t dn_launch_linear_backward(int type, const void *dy, const void *x, const void *w, const void *z, long long M,
                                     long long N, long long K, int act, const DnDrop &drop, void *dz_buffer, void *dx,
                                     void *dw, void *db, float *workspace, hipStream_t s);

// Dropout as an operator of its own, and dz = D(dy) act'(z) of linear's backward: element by element, bound by memory.
//
// A thread takes eight consecutive elements of a row, the unit one call of the generator serves; a row starts a new
// unit, so rows of any length can be cut up.  Consecutive threads take consecutive units: 16 (32) bytes a lane.
//
// Measured on one MI355X: 65536 x 2048 bf16 87 us (537 MB, 6.2 TB/s; torch's copy of it 99), 38400 x 256 fp32 with a
// residual 18.5 us (118 MB, 6.4 TB/s).  The generator's ten rounds stay hidden behind the bytes because one call serves
// eight elements: with nothing to drop the same kernel takes 90 and 18 us.
#include "dense_common.h"

namespace {

constexpr int EW_THREADS = 256;

struct EwArgs {
    const void *x, *residual, *slope;
    void *y;
    long long rows;
    uint32_t cols, units;        // elements and units of eight a row
    MsmvDiv div_units;
    int act;
    DnDrop drop;
};

template <class T, bool SLOPE>
__global__ void __launch_bounds__(EW_THREADS) dense_elementwise_kernel(EwArgs a)
{
    const uint64_t seed = dn_seed(a.drop);
    // the block's first unit, split into row and unit once; a thread's own unit is then a 31-bit division away
    const uint64_t first = (uint64_t)blockIdx.x * EW_THREADS;
    const uint64_t row0 = first / a.units;
    const uint32_t unit0 = (uint32_t)(first - row0 * a.units) + threadIdx.x;
    const uint32_t down = msmv_div(unit0, a.div_units);
    const uint64_t row = row0 + down;
    const uint32_t col = (unit0 - down * a.units) * 8;
    if (row >= (uint64_t)a.rows)
        return;
    const uint64_t at = row * a.cols + col;
    const int n = (int)min(8u, a.cols - col);
    dn_floats<8> v = dn_load_n<8>(static_cast<const T *>(a.x) + at, n, (int)a.cols);
    if (a.drop.threshold)
        dn_drop<8>(v, row, col, seed, a.drop);
    if constexpr (SLOPE) {
        dn_act_slope<8, T>(v, dn_load_n<8>(static_cast<const T *>(a.slope) + at, n, (int)a.cols), a.act);
    } else if (a.residual) {
        v += dn_load_n<8>(static_cast<const T *>(a.residual) + at, n, (int)a.cols);
    }
    dn_store_n<8>(static_cast<T *>(a.y) + at, v, n);
}

template <class T>
hipError_t launch(const EwArgs &a, hipStream_t s)
{
    const long long blocks = dn_ceil(a.rows * (long long)a.units, EW_THREADS);
    if (blocks * EW_THREADS > 0xFFFFFFFFll)          // a grid's threads are counted in 32 bits
        return hipErrorInvalidValue;
    if (a.slope)
        hipLaunchKernelGGL((dense_elementwise_kernel<T, true>), dim3((unsigned)blocks), dim3(EW_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((dense_elementwise_kernel<T, false>), dim3((unsigned)blocks), dim3(EW_THREADS), 0, s, a);
    return hipSuccess;
}

}  // namespace

hipError_t dn_launch_elementwise(int type, const void *x, const void *residual, const void *slope, int act,
                                 long long rows, long long cols, const DnDrop &drop, void *y, hipStream_t s)
{
    if (rows == 0 || cols == 0)
        return hipSuccess;
    EwArgs a = {x, residual, slope, y, rows, (uint32_t)cols, (uint32_t)dn_ceil(cols, 8), {}, act, drop};
    a.div_units = msmv_make_div((int)a.units);
    const hipError_t stale = hipPeekAtLastError();
    const hipError_t e = type == OPUS_DENSE_F32 ? launch<float>(a, s)
                       : type == OPUS_DENSE_BF16 ? launch<dn_bf16>(a, s) : launch<dn_f16>(a, s);
    return e != hipSuccess ? e : msmv_launch_status(stale);
}

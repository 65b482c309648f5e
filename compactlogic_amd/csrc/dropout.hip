// Dropout whose mask is a function of (seed, offset, row, column) and is never stored: the
// backward makes it again.
//
// The generator is Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC'11): key = seed, counter = (column / 8, row, offset low,
// offset high).  Its four words are eight 16-bit halves, low half first; half number column % 8
// decides the element: dropped where half < t, t = round(65536 p).  Sixteen bits an element
// keep p to 2^-16 and halve the generator's work, which bounds the 16-bit types.
#include "storage.h"

#include <algorithm>

namespace cl {
namespace {

constexpr int kDropThreads = 256;
constexpr int kDropBlock = 8;  // elements of one generator block

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                        uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = uint64_t(0xD2511F53u) * c0, b = uint64_t(0xCD9E8D57u) * c2;
        c0 = uint32_t(b >> 32) ^ c1 ^ k0;
        c1 = uint32_t(b);
        c2 = uint32_t(a >> 32) ^ c3 ^ k1;
        c3 = uint32_t(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words{{c0, c1, c2, c3}};
}

__device__ __forceinline__ bool kept(const Words& w, int e, uint32_t t) {
    return ((w.w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu) >= t;
}

template <typename T>
struct DropArgs {
    const T* x;
    T* y;
    int64_t xs, ys;  // strides of the outer dimension (the inner one is contiguous)
    int64_t rows, cols;
    uint32_t t;
    wide_t<T> scale;
    T fill;
    uint64_t seed, offset;
    const int64_t* rng;  // (seed, offset) on the device, or null
};

template <typename T>
__device__ __forceinline__ void drop_state(const DropArgs<T>& a, uint64_t& seed, uint64_t& off) {
    seed = a.rng ? uint64_t(a.rng[0]) : a.seed;
    off = a.rng ? uint64_t(a.rng[1]) : a.offset;
}

template <typename T>
__device__ __forceinline__ T dropped(T x, bool keep, const DropArgs<T>& a) {
    return keep ? T(wide_t<T>(x) * a.scale) : a.fill;
}

// Columns contiguous: one thread per generator block of eight columns.
template <typename T>
__global__ __launch_bounds__(kDropThreads) void k_dropout_rows(DropArgs<T> a, int64_t blocks) {
    const int64_t item = int64_t(blockIdx.x) * kDropThreads + threadIdx.x;
    if (item >= a.rows * blocks) return;
    const int64_t row = item / blocks, blk = item % blocks;
    uint64_t seed, off;
    drop_state(a, seed, off);
    const Words w = philox(uint32_t(blk), uint32_t(row), uint32_t(off), uint32_t(off >> 32),
                           uint32_t(seed), uint32_t(seed >> 32));
    const int64_t c0 = blk * kDropBlock;
    const T* x = a.x + row * a.xs + c0;
    T* y = a.y + row * a.ys + c0;
    const int n = int(std::min<int64_t>(kDropBlock, a.cols - c0));
    for (int e = 0; e < n; ++e) y[e] = dropped(x[e], kept(w, e, a.t), a);
}

// Rows contiguous (the view a LogicLayer returns): one thread per row and eight columns, so
// that a wave reads runs of 64 elements.
template <typename T>
__global__ __launch_bounds__(kDropThreads) void k_dropout_cols(DropArgs<T> a, int64_t blocks) {
    const int64_t item = int64_t(blockIdx.x) * kDropThreads + threadIdx.x;
    if (item >= a.rows * blocks) return;
    const int64_t row = item % a.rows, blk = item / a.rows;
    uint64_t seed, off;
    drop_state(a, seed, off);
    const Words w = philox(uint32_t(blk), uint32_t(row), uint32_t(off), uint32_t(off >> 32),
                           uint32_t(seed), uint32_t(seed >> 32));
    const int64_t c0 = blk * kDropBlock;
    const T* x = a.x + c0 * a.xs + row;
    T* y = a.y + c0 * a.ys + row;
    const int n = int(std::min<int64_t>(kDropBlock, a.cols - c0));
    for (int e = 0; e < n; ++e) y[e * a.ys] = dropped(x[e * a.xs], kept(w, e, a.t), a);
}

__global__ void k_dropout_next(int64_t* __restrict__ rng, int64_t* __restrict__ used) {
    const int64_t seed = rng[0], off = rng[1];
    used[0] = seed;
    used[1] = off;
    rng[1] = int64_t(uint64_t(off) + 1);
}

}  // namespace
}  // namespace cl

using namespace cl;

extern "C" int cl_dropout(int dtype, const void* x, int64_t x_stride_row, int64_t x_stride_col,
                          void* y, int64_t y_stride_row, int64_t y_stride_col, int64_t rows,
                          int64_t cols, int64_t threshold, int rescale, double fill,
                          uint64_t seed, uint64_t offset, const int64_t* rng, void* stream) {
    clear_error();
    CL_ARG(rows >= 0 && cols >= 0, "negative shape");
    CL_ARG(rows <= int64_t(UINT32_MAX) && cols <= int64_t(UINT32_MAX),
           "rows and columns of a dropped tensor are counted in 32 bits");
    CL_ARG(threshold >= 0 && threshold <= 65536, "threshold must be in [0, 65536], got %lld",
           (long long)threshold);
    if (rows == 0 || cols == 0) return CL_OK;
    CL_ARG(x && y, "null pointer argument");
    const bool by_rows = (x_stride_col == 1 && y_stride_col == 1) || cols == 1;
    const bool by_cols = (x_stride_row == 1 && y_stride_row == 1) || rows == 1;
    CL_ARG(by_rows || by_cols, "x and y must be contiguous along the same dimension");
    const int64_t xs = by_rows ? x_stride_row : x_stride_col;
    const int64_t ys = by_rows ? y_stride_row : y_stride_col;
    CL_ARG(xs >= 0 && ys >= 0, "negative strides are not supported");
    CL_ARG(ys >= (by_rows ? cols : rows) || (by_rows ? rows : cols) == 1,
           "the rows of y overlap");
    const int64_t blocks = ceil_div(cols, kDropBlock);
    const int64_t grid = ceil_div(rows * blocks, kDropThreads);
    CL_ARG(grid < (int64_t(1) << 31), "too many elements for one call");
    hipStream_t s = as_stream(stream);
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        DropArgs<T> a;
        a.x = static_cast<const T*>(x);
        a.y = static_cast<T*>(y);
        a.xs = xs;
        a.ys = ys;
        a.rows = rows;
        a.cols = cols;
        a.t = uint32_t(threshold);
        a.scale = wide_t<T>(rescale && threshold < 65536 ? 65536.0 / double(65536 - threshold) : 1.0);
        a.fill = T(wide_t<T>(fill));
        a.seed = seed;
        a.offset = offset;
        a.rng = rng;
        if (by_rows)
            k_dropout_rows<T><<<unsigned(grid), kDropThreads, 0, s>>>(a, blocks);
        else
            k_dropout_cols<T><<<unsigned(grid), kDropThreads, 0, s>>>(a, blocks);
    });
    return check_launch("cl_dropout");
}

extern "C" int cl_dropout_next(int64_t* rng, int64_t* used, void* stream) {
    clear_error();
    CL_ARG(rng && used, "null pointer argument");
    k_dropout_next<<<1, 1, 0, as_stream(stream)>>>(rng, used);
    return check_launch("cl_dropout_next");
}

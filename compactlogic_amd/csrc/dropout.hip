// Dropout whose mask is a function of (seed, offset, row, column) and is never stored: the
// backward makes it again.
//
// The generator is Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC'11): key = seed, counter = (column / 8, row, offset low,
// offset high).  Its four words are eight 16-bit halves, low half first; half number column % 8
// decides the element: dropped where half < t, t = round(65536 p).  Sixteen bits an element
// keep p to 2^-16; 32 would double the generator's work, some 110 vector instructions a block,
// which would then take longer than the memory accesses of 16-bit types.
#include "storage.h"

#include <algorithm>

namespace cl {
namespace {

constexpr int kDropThreads = 256;
constexpr int kDropBlock = 8;  // elements of one generator block

struct Words {
    uint32_t w[4];
};

// One instruction: the truth table of a ^ b ^ c over the three inputs' patterns.
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_amdgcn_bitop3_b32(a, b, c, 0xF0 ^ 0xCC ^ 0xAA);
}

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                        uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = uint64_t(0xD2511F53u) * c0, b = uint64_t(0xCD9E8D57u) * c2;
        c0 = xor3(uint32_t(b >> 32), c1, k0);
        c1 = uint32_t(b);
        c2 = xor3(uint32_t(a >> 32), c3, k1);
        c3 = uint32_t(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words{{c0, c1, c2, c3}};
}

template <typename T>
struct DropArgs {
    const T* x;
    T* y;
    int64_t xs, ys;  // strides of the outer dimension (the inner one is contiguous)
    int64_t rows, cols;
    uint32_t last;   // t * 2^16 - 1: a word whose upper half is below t is at most this
    wide_t<T> scale;
    wide_t<T> fill;  // as T holds it
    uint64_t seed, offset;
    const int64_t* rng;  // (seed, offset) on the device, or null
};

// The generator of a row: element e of block blk is dropped where bit e of mask(blk) is set.
template <typename T>
struct Generator {
    uint32_t k0, k1, o0, o1, last;
    __device__ __forceinline__ explicit Generator(const DropArgs<T>& a) : last(a.last) {
        const uint64_t seed = a.rng ? uint64_t(a.rng[0]) : a.seed;
        const uint64_t off = a.rng ? uint64_t(a.rng[1]) : a.offset;
        k0 = uint32_t(seed);
        k1 = uint32_t(seed >> 32);
        o0 = uint32_t(off);
        o1 = uint32_t(off >> 32);
    }
    __device__ __forceinline__ Words words(uint32_t row, uint32_t blk) const {
        return philox(blk, row, o0, o1, k0, k1);
    }
    // compared as whole words: the upper half as it lies, the lower one moved up
    __device__ __forceinline__ bool drops(const Words& w, int e) const {
        return (e & 1 ? w.w[e >> 1] : w.w[e >> 1] << 16) <= last;
    }
};

// chosen in the wide type, so that two 16-bit results are rounded by one instruction
template <typename T>
__device__ __forceinline__ T after(T x, bool drop, const DropArgs<T>& a) {
    const wide_t<T> kept = wide_t<T>(x) * a.scale;
    return T(drop ? a.fill : kept);
}

// item / d and item % d, by a multiplication where there are fewer than 2^31 items.
template <bool WIDE>
struct Split;
template <>
struct Split<false> {
    FastDiv d;
    __device__ __forceinline__ void operator()(int64_t item, int64_t& q, int64_t& r) const {
        const uint32_t i = uint32_t(item), k = fast_div(i, d);
        q = k;
        r = i - k * d.d;
    }
};
template <>
struct Split<true> {
    int64_t d;
    __device__ __forceinline__ void operator()(int64_t item, int64_t& q, int64_t& r) const {
        q = item / d;
        r = item - q * d;
    }
};

// Columns contiguous: one thread per generator block of eight columns, which are one 16-byte
// access each way for 16-bit types and two for fp32.  Bound by memory: 16384 x 11999 bf16 (786 MB)
// 130 us = 6.0 TB/s; element by element it took 428 us.
template <typename T, bool WIDE>
__global__ __launch_bounds__(kDropThreads) void k_dropout_rows(DropArgs<T> a, int64_t items,
                                                               Split<WIDE> split) {
    const int64_t item = group_index() * kDropThreads + threadIdx.x;
    if (item >= items) return;
    int64_t row, blk;
    split(item, row, blk);
    const Generator<T> gen(a);
    const int64_t c0 = blk * kDropBlock;
    const T* x = a.x + row * a.xs + c0;
    T* y = a.y + row * a.ys + c0;
    if (c0 + kDropBlock <= a.cols) {
        Pack<T, kDropBlock> v = pload<T, kDropBlock>(x);
        const Words w = gen.words(uint32_t(row), uint32_t(blk));
#pragma unroll
        for (int e = 0; e < kDropBlock; ++e) v.v[e] = after(v.v[e], gen.drops(w, e), a);
        pstore<T, kDropBlock>(y, v);
    } else {
        const Words w = gen.words(uint32_t(row), uint32_t(blk));
        const int n = int(a.cols - c0);
#pragma unroll
        for (int e = 0; e < kDropBlock - 1; ++e)
            if (e < n) y[e] = after(x[e], gen.drops(w, e), a);
    }
}

// Rows contiguous (the view a LogicLayer returns): one thread per eight columns and as many rows
// as 16 bytes hold, so that every access is of 16 bytes and no generator block is made twice.
// 1024 x 12000 fp32 (98 MB, in the cache) 15.1 us = 6.5 TB/s; a thread per row 28.9 us.
template <typename T, bool WIDE>
__global__ __launch_bounds__(kDropThreads) void k_dropout_cols(DropArgs<T> a, int64_t items,
                                                               Split<WIDE> split) {
    constexpr int R = wide_vec<T>();
    const int64_t item = group_index() * kDropThreads + threadIdx.x;
    if (item >= items) return;
    int64_t blk, rb;
    split(item, blk, rb);
    const Generator<T> gen(a);
    const int64_t row = rb * R, c0 = blk * kDropBlock;
    const T* x = a.x + c0 * a.xs + row;
    T* y = a.y + c0 * a.ys + row;
    const int n = int(std::min<int64_t>(kDropBlock, a.cols - c0));
    uint32_t mask[R];  // bit e: column c0 + e of the row is dropped
    if (row + R <= a.rows) {
        Pack<T, R> v[kDropBlock];
#pragma unroll
        for (int e = 0; e < kDropBlock; ++e)
            if (e < n) v[e] = pload<T, R>(x + e * a.xs);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const Words w = gen.words(uint32_t(row) + i, uint32_t(blk));
            mask[i] = 0;
#pragma unroll
            for (int e = 0; e < kDropBlock; ++e) mask[i] |= gen.drops(w, e) ? 1u << e : 0u;
        }
#pragma unroll
        for (int e = 0; e < kDropBlock; ++e)
            if (e < n) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                    v[e].v[i] = after(v[e].v[i], (mask[i] >> e & 1) != 0, a);
                pstore<T, R>(y + e * a.ys, v[e]);
            }
    } else {
        const int rows = int(a.rows - row);
        for (int i = 0; i < rows; ++i) {
            const Words w = gen.words(uint32_t(row) + i, uint32_t(blk));
#pragma unroll
            for (int e = 0; e < kDropBlock; ++e)
                if (e < n) y[e * a.ys + i] = after(x[e * a.xs + i], gen.drops(w, e), a);
        }
    }
}

template <typename T>
int launch_dropout(const DropArgs<T>& a, bool by_rows, hipStream_t s) {
    const int64_t blocks = ceil_div(a.cols, kDropBlock);
    const int64_t bands = ceil_div(a.rows, wide_vec<T>());
    const int64_t items = by_rows ? a.rows * blocks : bands * blocks;
    const int64_t grid = ceil_div(items, kDropThreads);
    CL_ARG(grid < (int64_t(1) << 31), "too many elements for one call");
    const int64_t d = by_rows ? blocks : bands;
    if (items < (int64_t(1) << 31)) {
        const Split<false> split{make_fastdiv(uint32_t(d))};
        if (by_rows)
            k_dropout_rows<T, false><<<wide_grid(grid), kDropThreads, 0, s>>>(a, items, split);
        else
            k_dropout_cols<T, false><<<wide_grid(grid), kDropThreads, 0, s>>>(a, items, split);
    } else {
        const Split<true> split{d};
        if (by_rows)
            k_dropout_rows<T, true><<<wide_grid(grid), kDropThreads, 0, s>>>(a, items, split);
        else
            k_dropout_cols<T, true><<<wide_grid(grid), kDropThreads, 0, s>>>(a, items, split);
    }
    return check_launch("cl_dropout");
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
    CL_ARG(threshold >= 1 && threshold <= 65536, "threshold must be in [1, 65536], got %lld",
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
        a.last = uint32_t((uint64_t(threshold) << 16) - 1);
        const double keep = double(65536 - threshold);
        a.scale = wide_t<T>(rescale && keep > 0 ? 65536.0 / keep : 1.0);
        a.fill = wide_t<T>(T(wide_t<T>(fill)));
        a.seed = seed;
        a.offset = offset;
        a.rng = rng;
        return launch_dropout(a, by_rows, s);
    });
}

extern "C" int cl_dropout_next(int64_t* rng, int64_t* used, void* stream) {
    clear_error();
    CL_ARG(rng && used, "null pointer argument");
    k_dropout_next<<<1, 1, 0, as_stream(stream)>>>(rng, used);
    return check_launch("cl_dropout_next");
}

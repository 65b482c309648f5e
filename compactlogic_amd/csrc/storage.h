// Element types of the operators that also take 16-bit tensors: storage only, arithmetic in
// wide_t (fp32; fp64 for fp64), each result rounded once on store.
#pragma once

#include "common.h"

#include <type_traits>

namespace cl {

using half_t = _Float16;
using bf16_t = __bf16;

template <typename T>
struct WideType {
    using type = float;
};
template <>
struct WideType<double> {
    using type = double;
};
template <typename T>
using wide_t = typename WideType<T>::type;

// Runs the statement block with scalar_t bound to the storage type of `dtype`.
#define CL_STORAGE_SWITCH(dtype, ...)                                                    \
    do {                                                                                 \
        if ((dtype) == CL_DTYPE_F32) {                                                   \
            using scalar_t = float;                                                      \
            __VA_ARGS__                                                                  \
        } else if ((dtype) == CL_DTYPE_F64) {                                            \
            using scalar_t = double;                                                     \
            __VA_ARGS__                                                                  \
        } else if ((dtype) == CL_DTYPE_F16) {                                            \
            using scalar_t = ::cl::half_t;                                               \
            __VA_ARGS__                                                                  \
        } else if ((dtype) == CL_DTYPE_BF16) {                                           \
            using scalar_t = ::cl::bf16_t;                                               \
            __VA_ARGS__                                                                  \
        } else {                                                                         \
            ::cl::set_error("unsupported dtype code %d (expected F32, F64, F16 or BF16)", \
                            int(dtype));                                                 \
            return CL_ERR_INVALID_ARGUMENT;                                              \
        }                                                                                \
    } while (0)

// Any number of workgroups below 2^31: a launch counts the threads of a grid dimension in 32 bits,
// so what lies past 2^21 workgroups goes to the second one.  The last row of a grid may be partly
// past the end.
constexpr int64_t kGridRow = int64_t(1) << 21;

inline dim3 wide_grid(int64_t groups) {
    return dim3(unsigned(groups < kGridRow ? groups : kGridRow),
                unsigned((groups + kGridRow - 1) / kGridRow));
}
__device__ __forceinline__ int64_t group_index() { return blockIdx.y * kGridRow + blockIdx.x; }

// N elements moved in 16-byte accesses, at any address that is a multiple of the element size:
// the hardware takes them off 16 bytes, so rows need no alignment of their own.
template <typename T, int N>
struct Pack {
    static_assert(N * sizeof(T) % 16 == 0, "whole 16-byte accesses");
    T v[N];
};

typedef uint32_t quad2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t quad4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t quad8 __attribute__((ext_vector_type(4), aligned(8)));

template <typename T>
using quad_of = std::conditional_t<sizeof(T) == 2, quad2,
                                   std::conditional_t<sizeof(T) == 4, quad4, quad8>>;

// THROUGH: past the caches (non-temporal), for what is read or written once and does not fit them.
template <typename T, int N, bool THROUGH = false>
__device__ __forceinline__ Pack<T, N> pload(const T* p) {
    using Q = quad_of<T>;
    struct Words {
        Q q[N * sizeof(T) / 16];
    } w;
#pragma unroll
    for (int i = 0; i < int(N * sizeof(T) / 16); ++i) {
        if constexpr (THROUGH)
            w.q[i] = __builtin_nontemporal_load(reinterpret_cast<const Q*>(p) + i);
        else
            w.q[i] = reinterpret_cast<const Q*>(p)[i];
    }
    return __builtin_bit_cast(Pack<T, N>, w);
}

template <typename T, int N, bool THROUGH = false>
__device__ __forceinline__ void pstore(T* p, const Pack<T, N>& r) {
    using Q = quad_of<T>;
    struct Words {
        Q q[N * sizeof(T) / 16];
    };
    const Words w = __builtin_bit_cast(Words, r);
#pragma unroll
    for (int i = 0; i < int(N * sizeof(T) / 16); ++i) {
        if constexpr (THROUGH)
            __builtin_nontemporal_store(w.q[i], reinterpret_cast<Q*>(p) + i);
        else
            reinterpret_cast<Q*>(p)[i] = w.q[i];
    }
}

}  // namespace cl

// Element types of the operators that also take 16-bit tensors: storage only, arithmetic in
// wide_t (fp32; fp64 for fp64), each result rounded once on store.
#pragma once

#include "common.h"

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

// N elements moved as one access, at any address that is a multiple of the element size: the
// hardware takes 16-byte global accesses off 16 bytes, so rows need no alignment of their own.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pload(const T* p) {
    Pack<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}

template <typename T, int N>
__device__ __forceinline__ void pstore(T* p, const Pack<T, N>& r) {
    __builtin_memcpy(p, &r, sizeof(r));
}

}  // namespace cl

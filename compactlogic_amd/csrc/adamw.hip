// One AdamW step over many tensors, with moments in 32 bits (64 for fp64 parameters) or in 8.
//
//   c = min(1, M / (|g| + 1e-6)),  g' = c g                     (|g| over all tensors, in fp64)
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
//   k_adamw_begin   the step count, each group's coefficients (fp64, once) and the sums of g^2 of
//                   the workgroups, at most kNormParts of them
//   k_adamw         adds the sums in a fixed order (the norm), then one pass over p, g, m, v
//
// Tensors are cut into tiles, so that a small one costs one workgroup; a launch takes kTensors
// tensors of one type, their addresses in the kernel's arguments (a captured graph keeps them, and
// nothing is copied to the device), or kFewTensors in less of them.  A lane holds the first tile of one
// or two tensors, and the tile's tensor is the number of those that are not behind it.
//
// Moments in 8 bits go by blocks of 256 consecutive elements, each with a power of two for m and one
// for v: codes that have exponents of their own lose nothing by a power of two where a free scale
// would keep their mantissas, and scaling is exact.  m is e4m3, the block's largest in [128, 256).
// v >= 0 has five bits of exponent and three of mantissa, the block's largest in [1, 2): code c in
// 1..254 is the fp32 number whose bits are (c + 770) << 20, 2^-31 * 1.375 to 2; 255 is NaN.  Only 0
// is held as 0: the root of v divides, and an element whose v were lost under its neighbours' would
// make a step of m / eps.
//
// An average that moves by less than half a step of its codes stays where it is when it is rounded to the
// nearest, which is (1 - b2) |g^2 - v| < v / 18 falling (codes are up to 1/9 apart) and v / 16 rising:
// with a b2 of 0.9 v stays within 2.25 times of where it belongs, above 17/18 it need not fall at all.
// Rounded at random, up with the probability of its distance from the code below, it is
// right on average (b2 = 0.999, gradients of one size: after 3000 steps the mean v is 0.02 of the true one
// by the nearest and 1.00 at random, steps 4.8 and 1.00 times theirs).  The random numbers are a hash of
// the step count, the tile and the element, by the finalizer of MurmurHash3 (Appleby), one word for the
// 16 bits of m and of v each: 200 M bf16 391 us instead of 356 (with the norm 577, 468), 100 M fp32 287
// as by the nearest.
//
// Bound by memory: 100 M fp32 elements 530 us without the norm (5.3 TB/s), 200 M bf16 with moments in 8
// bits 356 (5.6; with 77 % of what the VALU can do in that time); the norm's pass 15 to 20 us per 76 MB.  Small tensors are the host's: two launches of 3.5 us each.
#include "storage.h"

#include <algorithm>

namespace cl {
namespace {

constexpr int kOptThreads = 256;
constexpr int kTile = 2048;        // elements; whole blocks
constexpr int kNormTile = 8192;
constexpr int kFewTensors = 16, kTensors = 128;  // of a launch
constexpr int kGroups = 32;
constexpr int kHeld = 256;         // elements of a block
constexpr int kNormParts = 512;
constexpr int kCoefs = 8;

// A group's coefficients as the first kernel leaves them (fp64), and behind those of all groups the step's
// key to its random numbers.
enum { kDecay, kSize, kInvRoot, kB1, kRest1, kB2, kRest2, kEps };
constexpr int kCoefSpace = kGroups * kCoefs + 1;

template <typename D>
__device__ __forceinline__ auto random_key(D* coefs) {
    using Word = std::conditional_t<std::is_const_v<D>, const uint32_t, uint32_t>;
    return reinterpret_cast<Word*>(coefs + kGroups * kCoefs);
}

template <int N>
struct Tensors {
    int n;
    uint32_t tiles;
    uint32_t first[N];  // first tile; those of no tensor: UINT32_MAX
    int64_t numel[N];
    void* param[N];
    void* grad[N];
    void* m[N];
    void* v[N];
    uint8_t* power[N];  // 8 bits: exponents + 127 of the blocks, m's and then v's
    uint32_t number[N]; // of the tensor's first tile among all of the call
    uint8_t group[N];
};

template <int N>
struct Grads {
    int n;
    uint32_t tiles;
    uint32_t first[N];
    int64_t numel[N];
    const void* grad[N];
};

// x mixed: every bit of the result hangs on every bit of x.
__device__ __forceinline__ uint32_t mixed(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x85EBCA6Bu;
    x = (x ^ (x >> 13)) * 0xC2B2AE35u;
    return x ^ (x >> 16);
}

struct Groups {
    int n;
    double lr[kGroups], b1[kGroups], b2[kGroups], eps[kGroups], decay[kGroups];
};

// The tensor that a tile lies in, the same in all lanes.
template <int N>
__device__ __forceinline__ int tensor_of(const uint32_t (&first)[N], uint32_t tile) {
    static_assert(N <= 64 || N == 128, "tensors of a launch");
    const int l = lane_id();
    int n = int(__builtin_popcountll(__ballot(l < N && first[l < N ? l : 0] <= tile)));
    if constexpr (N == 128) n += int(__builtin_popcountll(__ballot(first[64 + l] <= tile)));
    return n - 1;
}

// Sum over the workgroup, the same bits in every thread.
__device__ __forceinline__ double group_total(double v, double* red) {
    v = wave_total(v);
    if (lane_id() == 0) red[wave_id()] = v;
    __syncthreads();
    double s = red[0];
#pragma unroll
    for (int i = 1; i < kOptThreads / 64; ++i) s += red[i];
    return s;
}

template <typename T, int N>
__global__ __launch_bounds__(kOptThreads) void k_adamw_begin(Grads<N> ts, double* __restrict__ parts,
                                                             Groups groups,
                                                             double* __restrict__ step,
                                                             double* __restrict__ coefs) {
    constexpr int VEC = wide_vec<T>(), NV = kNormTile / kOptThreads / VEC;
    __shared__ double red[kOptThreads / 64];
    if (groups.n > 0 && blockIdx.x == 0 && wave_id() == 0) {
        const double t = step[0] + 1.0;
        const int i = threadIdx.x;
        if (i < groups.n) {
            double* c = coefs + i * kCoefs;
            const double b1 = groups.b1[i], b2 = groups.b2[i], lr = groups.lr[i];
            c[kDecay] = 1.0 - lr * groups.decay[i];
            c[kSize] = lr / (1.0 - pow(b1, t));
            c[kInvRoot] = 1.0 / sqrt(1.0 - pow(b2, t));
            c[kB1] = b1;
            c[kRest1] = 1.0 - b1;
            c[kB2] = b2;
            c[kRest2] = 1.0 - b2;
            c[kEps] = groups.eps[i];
        }
        if (i == 0) {
            step[0] = t;
            const uint64_t count = uint64_t(t);
            *random_key(coefs) = mixed(uint32_t(count) ^ mixed(uint32_t(count >> 32) + 0x9E3779B9u));
        }
    }
    if (ts.n == 0) return;
    double s = 0.0;
    for (uint32_t tile = blockIdx.x; tile < ts.tiles; tile += gridDim.x) {
        const int k = tensor_of(ts.first, tile);
        const int64_t i0 = int64_t(tile - ts.first[k]) * kNormTile, n = ts.numel[k] - i0;
        const T* g = static_cast<const T*>(ts.grad[k]) + i0;
        if (n >= kNormTile) {
            Pack<T, VEC> v[NV];
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = pload<T, VEC>(g + (j * kOptThreads + threadIdx.x) * VEC);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) s = fma(double(v[j].v[e]), double(v[j].v[e]), s);
        } else {
            const int packs = int(n) / VEC, rest = int(n) - packs * VEC;
            for (int j = threadIdx.x; j < packs; j += kOptThreads) {
                const Pack<T, VEC> v = pload<T, VEC>(g + j * VEC);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s = fma(double(v.v[e]), double(v.v[e]), s);
            }
            if (int(threadIdx.x) < rest) {
                const double v = double(g[packs * VEC + threadIdx.x]);
                s = fma(v, v, s);
            }
        }
    }
    s = group_total(s, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

// ---- the update of one element.  m and v are rounded product by product, so that an 8-bit code does
// not depend on what a compiler fuses; the quotient, which only p takes, by the hardware's square
// root and reciprocal, each within a unit in the last place (fp32).  The IEEE forms take some 20
// instructions more of about 60.  Both take a number below 2^-126 for 0, which would make a step of
// m / 0 where eps is 0 or that small too: for a v below it, both sides of the division times 2^32.
template <typename A>
struct Coefs {
    A scale;  // of the gradient
    A decay, size, inv_root, b1, rest1, b2, rest2, eps;
};

__device__ __forceinline__ float quotient(float m, float v, const Coefs<float>& c) {
    const bool low = v < 0x1p-126f;
    const float root = __builtin_amdgcn_sqrtf(low ? v * 0x1p64f : v);
    const float up = low ? 0x1p32f : 1.0f;
    const float d = __builtin_fmaf(root, c.inv_root, c.eps * up);
    return m * up * __builtin_amdgcn_rcpf(d);
}
__device__ __forceinline__ double quotient(double m, double v, const Coefs<double>& c) {
    return m / (sqrt(v) * c.inv_root + c.eps);
}

template <typename A>
__device__ __forceinline__ void moments_step(A g, A& m, A& v, const Coefs<A>& c) {
#pragma clang fp contract(off)
    g = g * c.scale;
    const A q = g * g;
    m = m * c.b1 + g * c.rest1;
    v = v * c.b2 + q * c.rest2;
}

template <typename A>
__device__ __forceinline__ A param_step(A p, A m, A v, const Coefs<A>& c) {
    return fma(p, c.decay, -(c.size * quotient(m, v, c)));
}

// Every workgroup adds the same sums in the same order.  (A NaN scales nothing.)
template <typename A>
__device__ __forceinline__ Coefs<A> load_coefs(const double* __restrict__ parts, int nparts,
                                               double max_norm, const double* __restrict__ coefs,
                                               int group, double* red) {
    const double* c = coefs + group * kCoefs;
    Coefs<A> r;
    r.decay = A(c[kDecay]);
    r.size = A(c[kSize]);
    r.inv_root = A(c[kInvRoot]);
    r.b1 = A(c[kB1]);
    r.rest1 = A(c[kRest1]);
    r.b2 = A(c[kB2]);
    r.rest2 = A(c[kRest2]);
    r.eps = A(c[kEps]);
    r.scale = A(1);
    if (nparts > 0) {
        // by one wave: as much work as some two elements of each thread, and done once instead of by four
        if (wave_id() == 0) {
            double s = 0.0;
#pragma unroll 8
            for (int i = lane_id(); i < nparts; i += 64) s += parts[i];
            const double k = max_norm / (sqrt(wave_total(s)) + 1e-6);
            if (lane_id() == 0) red[0] = k < 1.0 ? k : 1.0;
        }
        __syncthreads();
        r.scale = A(red[0]);
    }
    return r;
}

// ---- 8 bits.  A block of 256 lies in 32 lanes of 8 elements.
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
    v = max(v, dpp_move<0xB1>(v));   // quad_perm [1,0,3,2]
    v = max(v, dpp_move<0x4E>(v));   // quad_perm [2,3,0,1]
    v = max(v, dpp_move<0x141>(v));  // row_half_mirror
    v = max(v, dpp_move<0x140>(v));  // row_mirror
    return max(v, xor_lane<16>(v));
}

constexpr uint32_t kInfBits = 0x7F800000u, kMagnitude = 0x7FFFFFFFu;
constexpr uint32_t kFirstCode = 770;

__device__ __forceinline__ uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float float_of(uint32_t x) { return __builtin_bit_cast(float, x); }

struct Codes {
    uint2 m, v;
};

struct Powers {
    int m, v;
};

// 2^k for k in -127..127
__device__ __forceinline__ float power_of_two(int k) { return __builtin_amdgcn_ldexpf(1.0f, k); }

// Exponents of the block, from its largest finite magnitude, and the codes of this lane's elements.
// A code of what is not finite is NaN, whatever the block's other elements are.  An infinite m comes
// with a v that is not finite (the exponential average of finite numbers does not overflow); a NaN
// is left out of a maximum and is converted to one.
//
// RANDOM: by the random words of elements `place` on under `key`, the lower half for m and the upper for v.
// e4m3 has the same step below 2^-6, its smallest normal number, as above it: 2^-6 more, and the bits of
// any number hold its code and 20 bits behind it.
template <bool RANDOM>
__device__ __forceinline__ Codes encode(float (&m)[8], float (&v)[8], Powers& power, uint32_t key = 0,
                                        uint32_t place = 0) {
    float top = 0.0f;
    uint32_t top_v = 0;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        top = __builtin_fmaxf(__builtin_fmaxf(top, __builtin_fabsf(m[e])), __builtin_fabsf(m[e + 1]));
        top_v = max(max(top_v, bits_of(v[e])), bits_of(v[e + 1]));
    }
    uint32_t top_m = block_max(bits_of(top));
    top_v = block_max(top_v);
    const bool odd = max(top_m, top_v) >= kInfBits;
    uint32_t no_m = 0, no_v = 0;
    if (odd) {  // the same in the 32 lanes of a block
        top_m = top_v = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t a = bits_of(m[e]) & kMagnitude, b = bits_of(v[e]) & kMagnitude;
            if (a >= kInfBits) {
                no_m |= 1u << e;
                m[e] = 0.0f;
            } else {
                top_m = max(top_m, a);
            }
            if (b >= kInfBits) {
                no_v |= 1u << e;
                v[e] = 0.0f;
            } else {
                top_v = max(top_v, b);
            }
        }
        top_m = block_max(top_m);
        top_v = block_max(top_v);
    }
    power.m = max(int(top_m >> 23) - 134, -126);
    power.v = max(int(top_v >> 23) - 127, -126);
    const float to_m = power_of_two(-power.m), to_v = power_of_two(-power.v);
    Codes c;
    uint32_t pm[2], pv[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = m[4 * h + e] * to_m;
        uint32_t word[4];
        if constexpr (RANDOM) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                word[e] = mixed(key + (place + uint32_t(4 * h + e)) * 0x9E3779B9u);
                const float size = __builtin_fabsf(u[e]), more = size < 0x1p-6f ? 0x1p-6f : 0.0f;
                const uint32_t up = ((word[e] & 0xFFFFu) << 4) + 8;
                u[e] = __builtin_copysignf(float_of((bits_of(size + more) + up) & 0xFFF00000u) - more, u[e]);
            }
        }
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], 0, false);
        pm[h] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], w, true));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t b = bits_of(v[4 * h + e] * to_v);
            const uint32_t up = RANDOM ? ((word[e] >> 16) << 4) + 8 : 0x7FFFFu + ((b >> 20) & 1);
            const int r = int(b + up - (kFirstCode << 20)) >> 20;
            // the middle one of r, 1 and a number that is 0 for v = 0 (r is then below 0) and else not
            // below r, nor 0 where scaling lost v
            const int some = int(b | bits_of(v[4 * h + e]));
            const int code = max(min(r, 1), min(max(r, 1), some));
            pv[h] |= uint32_t(code) << (8 * e);
        }
    }
    if (odd) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int s = 8 * (e & 3);
            if (no_m >> e & 1) pm[e >> 2] |= 0x7Fu << s;
            if (no_v >> e & 1) pv[e >> 2] |= 0xFFu << s;
        }
    }
    c.m = make_uint2(pm[0], pm[1]);
    c.v = make_uint2(pv[0], pv[1]);
    return c;
}

__device__ __forceinline__ void decode(const Codes& c, const Powers& power, float (&m)[8],
                                       float (&v)[8]) {
    const float of_m = power_of_two(power.m), of_v = power_of_two(power.v);
    const uint32_t wm[2] = {c.m.x, c.m.y}, wv[2] = {c.v.x, c.v.y};
    uint32_t least = 0xFF, most = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        typedef float pair __attribute__((ext_vector_type(2)));
        const pair lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(wm[h]), false);
        const pair hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(wm[h]), true);
        const float u[4] = {lo.x, lo.y, hi.x, hi.y};
        uint32_t code[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[4 * h + e] = u[e] * of_m;
            code[e] = (wv[h] >> (8 * e)) & 0xFFu;
            v[4 * h + e] = float_of((code[e] << 20) + (kFirstCode << 20)) * of_v;
        }
        least = min(min(least, min(code[0], code[1])), min(code[2], code[3]));
        most = max(max(most, max(code[0], code[1])), max(code[2], code[3]));
    }
    if (least == 0 || most == 0xFF) {  // 0 and NaN have no bits of that kind
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t code = (wv[e >> 2] >> (8 * (e & 3))) & 0xFFu;
            if (code == 0) v[e] = 0.0f;
            if (code == 0xFF) v[e] = __builtin_nanf("");
        }
    }
}

// Codes of eight elements, the last ones of a tensor one by one.
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int count) {
    if (count >= 8) {
        typedef uint32_t words __attribute__((ext_vector_type(2), aligned(1)));
        const words w = *reinterpret_cast<const words*>(p);
        return make_uint2(w.x, w.y);
    }
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (e < count) w[e >> 2] |= uint32_t(p[e]) << (8 * (e & 3));
    return make_uint2(w[0], w[1]);
}

template <bool THROUGH>
__device__ __forceinline__ void store_codes(uint8_t* p, uint2 c, int count) {
    if (count >= 8) {
        typedef uint32_t words __attribute__((ext_vector_type(2), aligned(1)));
        if constexpr (THROUGH)
            __builtin_nontemporal_store(words{c.x, c.y}, reinterpret_cast<words*>(p));
        else
            *reinterpret_cast<words*>(p) = words{c.x, c.y};
        return;
    }
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (e < count) p[e] = uint8_t(w[e >> 2] >> (8 * (e & 3)));
}

template <typename T>
struct Eight {
    T v[8];
};

template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int count) {
    Eight<T> r;
    if (count >= 8) return __builtin_bit_cast(Eight<T>, pload<T, 8>(p));
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = e < count ? p[e] : T(0);
    return r;
}

template <bool THROUGH, typename T>
__device__ __forceinline__ void store_eight(T* p, const Eight<T>& r, int count) {
    if (count >= 8) {
        pstore<T, 8, THROUGH>(p, __builtin_bit_cast(Pack<T, 8>, r));
        return;
    }
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (e < count) p[e] = r.v[e];
}

// Eight elements of a tile per thread, kHeld in 32 lanes; every lane takes part, those past the tensor's end
// with a count of 0 (and zeros).
static_assert(kTile == kOptThreads * 8);

struct Place {
    int64_t at, left;   // first element, and the tensor's from there on
    int64_t block, blocks;
    __device__ __forceinline__ Place(uint32_t tile, int64_t numel) {
        at = int64_t(tile) * kTile + threadIdx.x * 8;
        left = numel - at;
        block = at / kHeld;
        blocks = (numel + kHeld - 1) / kHeld;
    }
    // WHOLE: the tile lies inside of the tensor.  That is asked once, not at every access: where a whole
    // access and one by elements meet, the loads before them would be waited for.
    template <bool WHOLE>
    __device__ __forceinline__ int count() const {
        return WHOLE || left >= 8 ? 8 : left > 0 ? int(left) : 0;
    }
    __device__ __forceinline__ bool whole() const { return left + threadIdx.x * 8 >= kTile; }
};

__device__ __forceinline__ Powers load_powers(const uint8_t* power, const Place& at, int count) {
    if (count == 0) return {0, 0};
    const uint8_t* p = power + at.block;
    return {int(p[0]) - 127, int(p[at.blocks]) - 127};
}

__device__ __forceinline__ void store_powers(uint8_t* power, const Place& at, int count, const Powers& v) {
    if (count > 0 && (threadIdx.x & 31) == 0) {
        uint8_t* p = power + at.block;
        p[0] = uint8_t(v.m + 127);
        p[at.blocks] = uint8_t(v.v + 127);
    }
}

template <typename T, bool WHOLE, bool THROUGH, bool RANDOM, int N>
__device__ __forceinline__ void step_tile8(const Tensors<N>& ts, int k, const Place& at,
                                           const double* __restrict__ parts, int nparts,
                                           double max_norm, const double* __restrict__ coefs,
                                           double* red, uint32_t tile) {
    T* p = static_cast<T*>(ts.param[k]) + at.at;
    const T* d = static_cast<const T*>(ts.grad[k]) + at.at;
    uint8_t* pm = static_cast<uint8_t*>(ts.m[k]) + at.at;
    uint8_t* pv = static_cast<uint8_t*>(ts.v[k]) + at.at;
    const int count = at.count<WHOLE>();
    Eight<T> w = load_eight(p, count);
    const Eight<T> g = load_eight(d, count);
    const Codes held{load_codes(pm, count), load_codes(pv, count)};
    Powers power = load_powers(ts.power[k], at, count);
    uint32_t key = 0;
    if constexpr (RANDOM) key = mixed(ts.number[k] + tile + *random_key(coefs));
    const Coefs<float> c = load_coefs<float>(parts, nparts, max_norm, coefs, ts.group[k], red);
    float m[8], v[8];
    decode(held, power, m, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        moments_step(float(g.v[e]), m[e], v[e], c);
        w.v[e] = T(param_step(float(w.v[e]), m[e], v[e], c));
    }
    const Codes next = encode<RANDOM>(m, v, power, key, threadIdx.x * 8);
    store_eight<THROUGH>(p, w, count);
    store_codes<THROUGH>(pm, next.m, count);
    store_codes<THROUGH>(pv, next.v, count);
    store_powers(ts.power[k], at, count, power);
}

template <typename T, int N, bool THROUGH, bool RANDOM>
__global__ __launch_bounds__(kOptThreads) void k_adamw8(Tensors<N> ts, const double* __restrict__ parts,
                                                        int nparts, double max_norm,
                                                        const double* __restrict__ coefs) {
    __shared__ double red[kOptThreads / 64];
    const uint32_t tile = uint32_t(group_index());
    if (tile >= ts.tiles) return;
    const int k = tensor_of(ts.first, tile);
    const uint32_t own = tile - ts.first[k];
    const Place at(own, ts.numel[k]);
    if (at.whole())
        step_tile8<T, true, THROUGH, RANDOM>(ts, k, at, parts, nparts, max_norm, coefs, red, own);
    else
        step_tile8<T, false, THROUGH, RANDOM>(ts, k, at, parts, nparts, max_norm, coefs, red, own);
}

template <typename T, int N>
__global__ __launch_bounds__(kOptThreads) void k_adamw(Tensors<N> ts, const double* __restrict__ parts,
                                                       int nparts, double max_norm,
                                                       const double* __restrict__ coefs) {
    using A = wide_t<T>;
    constexpr int VEC = wide_vec<T>(), NV = kTile / kOptThreads / VEC;
    __shared__ double red[kOptThreads / 64];
    const uint32_t tile = uint32_t(group_index());
    if (tile >= ts.tiles) return;
    const int k = tensor_of(ts.first, tile);
    const int64_t i0 = int64_t(tile - ts.first[k]) * kTile, n = ts.numel[k] - i0;
    T* p = static_cast<T*>(ts.param[k]) + i0;
    const T* g = static_cast<const T*>(ts.grad[k]) + i0;
    A* pm = static_cast<A*>(ts.m[k]) + i0;
    A* pv = static_cast<A*>(ts.v[k]) + i0;
    if (n >= kTile) {
        Pack<T, VEC> w[NV], d[NV];
        Pack<A, VEC> m[NV], v[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = (j * kOptThreads + threadIdx.x) * VEC;
            w[j] = pload<T, VEC>(p + i);
            d[j] = pload<T, VEC>(g + i);
            m[j] = pload<A, VEC>(pm + i);
            v[j] = pload<A, VEC>(pv + i);
        }
        const Coefs<A> c = load_coefs<A>(parts, nparts, max_norm, coefs, ts.group[k], red);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = (j * kOptThreads + threadIdx.x) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                moments_step(A(d[j].v[e]), m[j].v[e], v[j].v[e], c);
                w[j].v[e] = T(param_step(A(w[j].v[e]), m[j].v[e], v[j].v[e], c));
            }
            pstore<T, VEC>(p + i, w[j]);
            pstore<A, VEC>(pm + i, m[j]);
            pstore<A, VEC>(pv + i, v[j]);
        }
    } else {
        const Coefs<A> c = load_coefs<A>(parts, nparts, max_norm, coefs, ts.group[k], red);
        for (int i = threadIdx.x; i < int(n); i += kOptThreads) {
            A m = pm[i], v = pv[i];
            moments_step(A(g[i]), m, v, c);
            p[i] = T(param_step(A(p[i]), m, v, c));
            pm[i] = m;
            pv[i] = v;
        }
    }
}

// What 8 bits hold, in bf16 (which holds it all from 2^-130 on), and 8 bits from fp32.  param: exp_avg, grad:
// exp_avg_sq as they are outside.
template <bool WHOLE, bool THROUGH, int N>
__device__ __forceinline__ void read_tile8(const Tensors<N>& ts, int k, const Place& at) {
    const int count = at.count<WHOLE>();
    const Codes held{load_codes(static_cast<uint8_t*>(ts.m[k]) + at.at, count),
                     load_codes(static_cast<uint8_t*>(ts.v[k]) + at.at, count)};
    const Powers power = load_powers(ts.power[k], at, count);
    float m[8], v[8];
    decode(held, power, m, v);
    Eight<bf16_t> a, b;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        a.v[e] = bf16_t(m[e]);
        b.v[e] = bf16_t(v[e]);
    }
    store_eight<THROUGH>(static_cast<bf16_t*>(ts.param[k]) + at.at, a, count);
    store_eight<THROUGH>(static_cast<bf16_t*>(ts.grad[k]) + at.at, b, count);
}

template <int N, bool THROUGH>
__global__ __launch_bounds__(kOptThreads) void k_adamw8_read(Tensors<N> ts) {
    const uint32_t tile = uint32_t(group_index());
    if (tile >= ts.tiles) return;
    const int k = tensor_of(ts.first, tile);
    const Place at(tile - ts.first[k], ts.numel[k]);
    if (at.whole())
        read_tile8<true, THROUGH>(ts, k, at);
    else
        read_tile8<false, THROUGH>(ts, k, at);
}

template <bool WHOLE, int N>
__device__ __forceinline__ void write_tile8(const Tensors<N>& ts, int k, const Place& at) {
    const int count = at.count<WHOLE>();
    const Eight<float> a = load_eight(static_cast<const float*>(ts.param[k]) + at.at, count);
    const Eight<float> b = load_eight(static_cast<const float*>(ts.grad[k]) + at.at, count);
    float m[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        m[e] = __builtin_isfinite(a.v[e]) ? a.v[e] : __builtin_nanf("");
        v[e] = b.v[e] < 0.0f ? __builtin_nanf("") : b.v[e] + 0.0f;  // no -0
    }
    Powers power;
    const Codes c = encode<false>(m, v, power);
    store_codes<false>(static_cast<uint8_t*>(ts.m[k]) + at.at, c.m, count);
    store_codes<false>(static_cast<uint8_t*>(ts.v[k]) + at.at, c.v, count);
    store_powers(ts.power[k], at, count, power);
}

template <int N>
__global__ __launch_bounds__(kOptThreads) void k_adamw8_write(Tensors<N> ts) {
    const uint32_t tile = uint32_t(group_index());
    if (tile >= ts.tiles) return;
    const int k = tensor_of(ts.first, tile);
    const Place at(tile - ts.first[k], ts.numel[k]);
    if (at.whole())
        write_tile8<true>(ts, k, at);
    else
        write_tile8<false>(ts, k, at);
}

// ---- tensors into launches
struct Batch {
    int n = 0;
    int64_t tiles = 0;
    const cl_adamw_tensor* t[kTensors];
    uint32_t number[kTensors];

    void add(const cl_adamw_tensor& tensor, int64_t first) {
        number[n] = uint32_t(first);
        t[n++] = &tensor;
        tiles += ceil_div(tensor.numel, kTile);
    }
    dim3 grid() const { return wide_grid(tiles); }
    template <int N>
    Tensors<N> tensors() const {
        Tensors<N> ts;
        ts.n = n;
        ts.tiles = 0;
        for (int i = 0; i < N; ++i) {
            ts.first[i] = i < n ? ts.tiles : UINT32_MAX;
            if (i >= n) continue;
            ts.numel[i] = t[i]->numel;
            ts.param[i] = t[i]->param;
            ts.grad[i] = t[i]->grad;
            ts.m[i] = t[i]->exp_avg;
            ts.v[i] = t[i]->exp_avg_sq;
            ts.power[i] = t[i]->powers;
            ts.number[i] = number[i];
            ts.group[i] = uint8_t(t[i]->group);
            ts.tiles += uint32_t(ceil_div(t[i]->numel, kTile));
        }
        return ts;
    }
    template <int N>
    Grads<N> grads() const {
        Grads<N> g;
        g.n = n;
        g.tiles = 0;
        for (int i = 0; i < N; ++i) {
            g.first[i] = i < n ? g.tiles : UINT32_MAX;
            if (i >= n) continue;
            g.numel[i] = t[i]->numel;
            g.grad[i] = t[i]->grad;
            g.tiles += uint32_t(ceil_div(t[i]->numel, kNormTile));
        }
        return g;
    }
};

// Runs the statement block with N bound to the tensors that a launch for n of them has room for.
#define CL_ADAMW_ROOM(n, ...)              \
    do {                                   \
        if ((n) <= kFewTensors) {          \
            constexpr int N = kFewTensors; \
            __VA_ARGS__                    \
        } else {                           \
            constexpr int N = kTensors;    \
            __VA_ARGS__                    \
        }                                  \
    } while (0)

// What must be the same within a launch: the type of the gradients; that, the bits of the moments (kinds
// from 4 on: 8 bits) and how they are rounded (from 8 on: at random); nothing.
enum class Alike { kDtype, kDtypeAndBits, kAll };
constexpr int kKinds = 12;

// From so many bytes on what a call with moments in 8 bits writes goes past the 256 MiB cache, where it
// would push out what the next one reads (37.8 M bf16 elements, each step followed by giving the moments
// back: 80 -> 65 us, the norm 20 -> 15, the moments 39 -> 35).  Steps alone, of more than the cache holds,
// take the same time either way, and so do those with moments in 32 bits.
constexpr double kThrough = 96 << 20;

int kind_of(const cl_adamw_tensor& t, Alike alike) {
    if (alike == Alike::kAll) return 0;
    if (alike == Alike::kDtype || t.bits != 8) return t.dtype;
    return t.dtype + (t.rounding == CL_ADAMW_AT_RANDOM ? 8 : 4);
}

// Calls f(kind, batch) for the launches that the tensors make, kind by kind.
template <typename F>
int each_batch(const cl_adamw_tensor* t, int64_t n, Alike alike, F&& f) {
    for (int kind = 0; kind < kKinds; ++kind) {
        Batch b;
        int64_t first = 0, next = 0;  // tiles of the tensors before this one, and with it
        for (int64_t i = 0; i < n; ++i, first = next) {
            next = first + ceil_div(t[i].numel, kTile);
            if (t[i].numel == 0 || kind_of(t[i], alike) != kind) continue;
            if (b.n == kTensors) {
                if (int rc = f(kind, b)) return rc;
                b = Batch();
            }
            b.add(t[i], first);
        }
        if (b.n)
            if (int rc = f(kind, b)) return rc;
    }
    return CL_OK;
}

int check_tensor(const cl_adamw_tensor& t, int64_t i, int64_t num_groups, bool values) {
    CL_ARG(t.numel >= 0, "negative tensor size at index %lld", (long long)i);
    CL_ARG(ceil_div(t.numel, kTile) < (int64_t(1) << 31) - 1, "tensor %lld is too long",
           (long long)i);
    CL_ARG(t.bits == 8 || (!values && t.bits == 32), "moments are held in 32 or 8 bits");
    CL_ARG(t.numel == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq &&
                            (t.bits == 32 || t.powers)),
           "null tensor pointer at index %lld", (long long)i);
    if (values) return CL_OK;
    CL_ARG(t.dtype >= CL_DTYPE_F32 && t.dtype <= CL_DTYPE_BF16,
           "unsupported dtype code %d (expected F32, F64, F16 or BF16)", int(t.dtype));
    CL_ARG(t.bits == 32 || t.dtype != CL_DTYPE_F64, "fp64 parameters have no moments in 8 bits");
    CL_ARG(t.group >= 0 && t.group < num_groups, "no group %d", int(t.group));
    CL_ARG(t.rounding == CL_ADAMW_NEAREST || t.rounding == CL_ADAMW_AT_RANDOM, "unknown rounding %d",
           int(t.rounding));
    return CL_OK;
}

// Sums that a launch of the norm leaves: a workgroup for each tile, but no more than its share of
// kNormParts by its elements' tiles, or kTensors (of many small tensors, one workgroup would have to
// go through some dozens).
int64_t norm_parts(int64_t norm_tiles, int64_t tiles, int64_t all) {
    int64_t share = tiles * kNormParts / all;
    if (share < kTensors) share = kTensors;
    return share < norm_tiles ? share : norm_tiles;
}

}  // namespace
}  // namespace cl

using namespace cl;

extern "C" int cl_adamw_workspace(int64_t num_tensors, int64_t* bytes) {
    clear_error();
    CL_ARG(bytes, "null pointer argument");
    CL_ARG(num_tensors >= 0, "negative number of tensors");
    // coefficients, and the norm's sums: kNormParts, and at most kTensors more for each launch, of which
    // there are those that hold kTensors and one of each type
    const int64_t launches = std::min<int64_t>(num_tensors, num_tensors / kTensors + 4);
    *bytes = 8 * (kCoefSpace + kNormParts + kTensors * launches);
    return CL_OK;
}

extern "C" int cl_adamw_step(int64_t num_tensors, const cl_adamw_tensor* tensors,
                             int64_t num_groups, const cl_adamw_group* groups, double max_norm,
                             double* step, void* workspace, int64_t workspace_bytes,
                             void* stream) {
    clear_error();
    CL_ARG(num_tensors >= 0 && num_groups >= 0, "negative count");
    CL_ARG(num_groups <= kGroups, "at most %d parameter groups", kGroups);
    CL_ARG((num_tensors == 0 || tensors) && (num_groups == 0 || groups), "null pointer argument");
    CL_ARG(step, "null step pointer");
    Groups gs{};
    gs.n = int(num_groups);
    for (int i = 0; i < gs.n; ++i) {
        const cl_adamw_group& g = groups[i];
        CL_ARG(g.lr >= 0 && g.beta1 >= 0 && g.beta1 < 1 && g.beta2 >= 0 && g.beta2 < 1 &&
                   g.eps >= 0 && g.weight_decay >= 0,
               "invalid AdamW hyper-parameters");
        gs.lr[i] = g.lr;
        gs.b1[i] = g.beta1;
        gs.b2[i] = g.beta2;
        gs.eps[i] = g.eps;
        gs.decay[i] = g.weight_decay;
    }
    int64_t all = 0;
    double written = 0;
    for (int64_t i = 0; i < num_tensors; ++i) {
        if (int rc = check_tensor(tensors[i], i, num_groups, false)) return rc;
        const int size = tensors[i].dtype == CL_DTYPE_F32 ? 4 : 2;
        if (tensors[i].bits == 8) written += double(tensors[i].numel) * (size + 2);
        all += ceil_div(tensors[i].numel, kTile);
        CL_ARG(all < (int64_t(1) << 31), "too many elements for one call");
    }
    int64_t need = 0;
    if (int rc = cl_adamw_workspace(num_tensors, &need)) return rc;
    CL_ARG(workspace && workspace_bytes >= need, "workspace of %lld bytes needed (cl_adamw_workspace)",
           (long long)need);
    CL_ARG(aligned(workspace, 8), "workspace must be aligned to 8 bytes");
    const bool through = written >= kThrough;
    hipStream_t s = as_stream(stream);
    double* coefs = static_cast<double*>(workspace);
    double* parts = coefs + kCoefSpace;
    int64_t nparts = 0;
    bool begun = false;
    auto begin = [&](int kind, const Batch& b) -> int {
        Groups now = gs;
        if (begun) now.n = 0;
        begun = true;
        unsigned grid = 1;
        CL_ADAMW_ROOM(b.n, {
            const Grads<N> g = b.grads<N>();
            if (b.n) grid = unsigned(norm_parts(g.tiles, b.tiles, all));
            CL_STORAGE_SWITCH(kind, {
                k_adamw_begin<scalar_t, N><<<grid, kOptThreads, 0, s>>>(g, parts + nparts, now, step,
                                                                       coefs);
            });
        });
        if (b.n) nparts += grid;
        return check_launch("cl_adamw_step(begin)");
    };
    if (gs.n == 0) gs.n = 1;  // the kernel counts the step along with the first group
    if (max_norm > 0 && all > 0) {
        if (int rc = each_batch(tensors, num_tensors, Alike::kDtype, begin)) return rc;
    } else {
        if (int rc = begin(CL_DTYPE_F32, Batch())) return rc;
    }
    return each_batch(tensors, num_tensors, Alike::kDtypeAndBits, [&](int kind, const Batch& b) -> int {
        CL_ADAMW_ROOM(b.n, {
            const Tensors<N> ts = b.tensors<N>();
            CL_STORAGE_SWITCH(kind & 3, {
                if (kind < 4) {
                    k_adamw<scalar_t, N><<<b.grid(), kOptThreads, 0, s>>>(ts, parts, int(nparts),
                                                                         max_norm, coefs);
                } else if constexpr (!std::is_same_v<scalar_t, double>) {
                    (kind < 8 ? through ? k_adamw8<scalar_t, N, true, false> : k_adamw8<scalar_t, N, false, false>
                     : through ? k_adamw8<scalar_t, N, true, true> : k_adamw8<scalar_t, N, false, true>)
                        <<<b.grid(), kOptThreads, 0, s>>>(ts, parts, int(nparts), max_norm, coefs);
                }
            });
        });
        return check_launch("cl_adamw_step");
    });
}

namespace {

int moments(const char* what, bool read, int64_t num_tensors, const cl_adamw_tensor* tensors,
            void* stream) {
    clear_error();
    CL_ARG(num_tensors >= 0, "negative count");
    CL_ARG(num_tensors == 0 || tensors, "null pointer argument");
    int64_t tiles = 0;
    for (int64_t i = 0; i < num_tensors; ++i) {
        if (int rc = check_tensor(tensors[i], i, 0, true)) return rc;
        tiles += ceil_div(tensors[i].numel, kTile);
        CL_ARG(tiles < (int64_t(1) << 31), "too many elements for one call");
    }
    const bool through = double(tiles) * kTile * 4 >= kThrough;
    hipStream_t s = as_stream(stream);
    return each_batch(tensors, num_tensors, Alike::kAll, [&](int, const Batch& b) -> int {
        CL_ADAMW_ROOM(b.n, {
            const Tensors<N> ts = b.tensors<N>();
            if (read)
                (through ? k_adamw8_read<N, true> : k_adamw8_read<N, false>)
                    <<<b.grid(), kOptThreads, 0, s>>>(ts);
            else
                k_adamw8_write<N><<<b.grid(), kOptThreads, 0, s>>>(ts);
        });
        return check_launch(what);
    });
}

}  // namespace

extern "C" int cl_adamw_moments_read(int64_t num_tensors, const cl_adamw_tensor* tensors,
                                     void* stream) {
    return moments("cl_adamw_moments_read", true, num_tensors, tensors, stream);
}

extern "C" int cl_adamw_moments_write(int64_t num_tensors, const cl_adamw_tensor* tensors,
                                      void* stream) {
    return moments("cl_adamw_moments_write", false, num_tensors, tensors, stream);
}

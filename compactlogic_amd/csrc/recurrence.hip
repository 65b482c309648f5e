// A gated linear recurrence over sequences, per batch entry and feature,
//   h_t = g_t h_(t-1) + b_t,   b_t = (1 - g_t) x_t ("mix") or x_t ("add"),
// and its gradients: with G_t = dy_t + c_t, c_(t-1) = g_t G_t (c of the last step: its state's gradient),
//   dx_t = (1 - g_t) G_t or G_t,   dg_t = G_t (h_(t-1) - x_t) or G_t h_(t-1),   dh_(-1) = c_(-1).
//
// A run of steps is a map h -> a h + b, and two maps in a row are one: (a2 a1, a2 b1 + b2).  So a
// workgroup takes a stretch of time at once: every thread the map of a few steps of its own, a scan
// over the threads' maps, then each thread's steps again from the state it starts with.  Both sweeps
// read the registers; memory is read once.  The backward goes through the stretches from the last one,
// makes their states again from the state each one began with (which the forward leaves, one per
// stretch) and scans the gradients' maps, c -> a c + q with the same a, the other way.
//
// A gate of exactly 0 drops what came before and one of exactly 1 leaves x unread, NaN and infinities
// too: a * h is not formed where a is 0, and a product of gates that are not 0 is kept from becoming 0.
//
// Gates may be of any magnitude.  A product of gates that passes the range says nothing about a state of
// 0, or a small one, that it is applied to: where a thread's product does (or, in a scan, is above
// kGrowth, so that sixteen of them may), the threads' steps are walked one after the other instead, and
// the maps of segments have factors with an exponent of their own.
//
// Where there are too few sequences for the chip, time is cut into segments: a first pass finds the
// map of each (reading everything once more), and every segment starts from the maps before it.
//
// Two layouts: features (or, for one step, the batch) contiguous, lanes beside each other; or time
// contiguous, as a LogicLayer gives batch * time samples, lanes one after the other in time.
// Arithmetic and states in fp32 (fp64 for fp64), each result rounded once.
#include "storage.h"

#include <algorithm>

namespace cl {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxSegments = 64;

__device__ __forceinline__ float least(float) { return 1.401298464324817e-45f; }
__device__ __forceinline__ double least(double) { return 4.9406564584124654e-324; }

// a h + b, h dropped by an a of 0
template <typename A>
__device__ __forceinline__ A apply(A a, A h, A b) {
    return a == A(0) ? b : fma(a, h, b);
}

// A product of factors other than 0 that is not 0 either.
template <typename A>
__device__ __forceinline__ A kept_product(A a, A b) {
    const A r = a * b;
    return r == A(0) && a != A(0) && b != A(0) ? least(r) : r;
}

__device__ __forceinline__ float least_magnitude(float a, float b) {
    return __builtin_fminf(a, __builtin_fabsf(b));
}
__device__ __forceinline__ double least_magnitude(double a, double b) {
    return __builtin_fmin(a, __builtin_fabs(b));
}

__device__ __forceinline__ float greatest_magnitude(float a, float b) {
    return __builtin_fmaxf(a, __builtin_fabsf(b));
}
__device__ __forceinline__ double greatest_magnitude(double a, double b) {
    return __builtin_fmax(a, __builtin_fabs(b));
}

// One step.  The rules of the ends of the gate differ from plain arithmetic only where something is
// not finite, and what is not finite stays so (0 * inf and 0 * NaN are NaN): a walk is taken in plain
// arithmetic, and again by the rules (EXACT) if its last value is not finite.  That saves three of some
// ten instructions an element, and the scalar registers of a mask for each.
template <bool EXACT, bool MIX, typename A>
__device__ __forceinline__ A step(A g, A x, A h) {
    A in = x;
    if constexpr (MIX) in = EXACT && g == A(1) ? A(0) : (A(1) - g) * x;
    if constexpr (EXACT) return apply(g, h, in);
    return fma(g, h, in);
}

// The gradient that goes on to the step before.
template <bool EXACT, typename A>
__device__ __forceinline__ A back_of(A g, A whole) {
    return EXACT && g == A(0) ? A(0) : g * whole;
}

template <bool EXACT, bool MIX, typename A>
__device__ __forceinline__ void gradients(A g, A x, A before, A whole, A& gx, A& gg) {
    if constexpr (MIX) {
        gx = EXACT && g == A(1) ? A(0) : (A(1) - g) * whole;
        gg = whole * (before - x);
    } else {
        gx = whole;
        gg = whole * before;
    }
}

template <typename A>
__device__ __forceinline__ bool finite(A v) {
    return __builtin_isfinite(v);
}

// A product of gates, m 2^e: it neither leaves the range nor becomes 0.  |m| <= 1, and e is kept to where
// sums of it and a type's exponents fit 32 bits.
__device__ __forceinline__ float mantissa(float v) { return __builtin_amdgcn_frexp_mantf(v); }
__device__ __forceinline__ double mantissa(double v) { return __builtin_amdgcn_frexp_mant(v); }
__device__ __forceinline__ int exponent(float v) { return __builtin_amdgcn_frexp_expf(v); }
__device__ __forceinline__ int exponent(double v) { return __builtin_amdgcn_frexp_exp(v); }
__device__ __forceinline__ float scaled(float m, int e) { return __builtin_amdgcn_ldexpf(m, e); }
__device__ __forceinline__ double scaled(double m, int e) { return __builtin_amdgcn_ldexp(m, e); }

constexpr float kSmall = 1.0f / 32768.0f;  // eight of them are a normal number

template <typename A>
struct Product {
    A m = A(1);
    int e = 0;
    // (at most 126 of them before the next `even`)
    __device__ __forceinline__ void by(A m2, int e2) {
        m = m == A(0) || m2 == A(0) ? A(0) : m * m2;
        e += e2;
    }
    __device__ __forceinline__ void by(A gate) { by(mantissa(gate), exponent(gate)); }
    __device__ __forceinline__ void even() {
        constexpr int most = 1 << 24;
        const int k = e + exponent(m);
        e = k < -most ? -most : k > most ? most : k;
        m = mantissa(m);
    }
    // An exponent of 0 where the product is a normal number (or 0, infinite, NaN).
    __device__ __forceinline__ void plain() {
        constexpr int most = sizeof(A) == 4 ? 127 : 1023;
        even();
        if (m == A(0) || !__builtin_isfinite(m) || (e > 1 - most && e <= most)) {
            m = scaled(m, e);
            e = 0;
        }
    }
    // m 2^e h + b: only the result may leave the range
    __device__ __forceinline__ A applied(A h, A b) const {
        const A r = scaled(mantissa(h) * m, exponent(h) + e) + b;
        return m == A(0) ? b : r;
    }
};

// |v| as a whole number, less one: 0 is above all others, and not among the small ones.
__device__ __forceinline__ uint32_t size_bits(float v) {
    return __builtin_bit_cast(uint32_t, __builtin_fabsf(v)) - 1;
}
__device__ __forceinline__ uint64_t size_bits(double v) {
    return __builtin_bit_cast(uint64_t, __builtin_fabs(v)) - 1;
}

// Each product of f by the gates of N <= 8 steps at its place, at once where they are neither small nor
// infinite, nor NaN.
template <int N, int VEC, typename A, typename V>
__device__ __forceinline__ void by_steps(Product<A> (&f)[VEC], const V (&gs)[N]) {
    static_assert(N <= 8);
    A p[VEC], rest = A(0);
    auto low = size_bits(A(0));
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        A lowest = A(1);
        p[e] = A(1);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            p[e] *= A(gs[k][e]);
            lowest = least_magnitude(lowest, A(gs[k][e]));
        }
        low = std::min(low, size_bits(lowest));
        rest = fma(p[e], A(0), fma(f[e].m, A(0), rest));
    }
    if (low >= size_bits(A(kSmall)) && rest == A(0)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            f[e].m *= mantissa(p[e]);
            f[e].e += exponent(p[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
#pragma unroll
            for (int k = 0; k < N; ++k) f[e].by(A(gs[k][e]));
    }
}

// The first `count` of the maps (f, b) applied to h in turn: in one instruction each where no factor has
// an exponent, in five else.
template <int N, typename A>
__device__ __forceinline__ A all_applied(const Product<A> (&f)[N], const A (&b)[N], int count, A h) {
    int e = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) e |= f[k].e;
    if (e == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < count) h = apply(f[k].m, h, b[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < count) h = f[k].applied(h, b[k]);
    }
    return h;
}

// The map of consecutive steps.
template <typename A>
struct Map {
    A a = A(1), b = A(0), lowest = A(1);  // lowest: of the gates' magnitudes
    template <bool EXACT, bool MIX>
    __device__ __forceinline__ void then(A g, A x) {
        b = step<EXACT, MIX>(g, x, b);
        factor_by(g);
    }
    __device__ __forceinline__ void factor_by(A g) {
        a *= g;
        lowest = least_magnitude(lowest, g);
    }
    // 0 only by a gate of 0
    __device__ __forceinline__ A factor() const {
        return lowest == A(0) ? A(0) : a == A(0) ? least(a) : a;
    }
    // Of a factor that has not left the range a product on the way may have, below it, if one of the
    // gates was small.
    __device__ __forceinline__ bool small() const { return size_bits(lowest) < size_bits(A(kSmall)); }
};

// From where on a lane's factor is not multiplied with its neighbours': sixteen of this one are 2^64, and
// what a product below the smallest number leaves of a state, by as much, is below 2^-80 of it.
constexpr float kGrowth = 16.0f;

// N elements of an access of 8 or 16 bytes at any address that is a multiple of the element size.  They
// stay as they were loaded until they are used: unpacked where the loads of a partial access and of a
// whole one meet, each load of 16-bit elements would be waited for by itself (a stretch of 16 loads
// took 11 us).
typedef uint32_t pair2 __attribute__((ext_vector_type(2), aligned(2)));

template <typename T, int N>
struct Few {
    using Access = std::conditional_t<
        N == 1, std::conditional_t<sizeof(T) == 2, uint16_t,
                                   std::conditional_t<sizeof(T) == 4, uint32_t, uint64_t>>,
        std::conditional_t<N * sizeof(T) == 8, pair2, quad_of<T>>>;
    struct Elements {
        T v[N];
    };
    Access w;

    __device__ __forceinline__ T operator[](int e) const {
        return __builtin_bit_cast(Elements, w).v[e];
    }
    __device__ __forceinline__ static Few of(const Elements& e) {
        return {__builtin_bit_cast(Access, e)};
    }
    __device__ __forceinline__ static Few all(T v) {
        Elements e;
#pragma unroll
        for (int k = 0; k < N; ++k) e.v[k] = v;
        return of(e);
    }
};

template <typename T, int N>
__device__ __forceinline__ Few<T, N> load_whole(const T* p) {
    return {*reinterpret_cast<const typename Few<T, N>::Access*>(p)};
}

template <typename T, int N>
__device__ __forceinline__ Few<T, N> load_part(const T* p, int count, T fill) {
    if (count >= N) return load_whole<T, N>(p);
    typename Few<T, N>::Elements r;
#pragma unroll
    for (int e = 0; e < N; ++e) r.v[e] = e < count ? p[e] : fill;
    return Few<T, N>::of(r);
}

// THROUGH: past the caches (non-temporal)
template <typename T, int N, bool THROUGH = false>
__device__ __forceinline__ void store_whole(T* p, const typename Few<T, N>::Elements& r) {
    auto* const to = reinterpret_cast<typename Few<T, N>::Access*>(p);
    if constexpr (THROUGH)
        __builtin_nontemporal_store(Few<T, N>::of(r).w, to);
    else
        *to = Few<T, N>::of(r).w;
}

template <typename T, int N>
__device__ __forceinline__ void store_part(T* p, const typename Few<T, N>::Elements& r, int count) {
    if (count >= N) {
        store_whole<T, N>(p, r);
        return;
    }
#pragma unroll
    for (int e = 0; e < N - 1; ++e)
        if (e < count) p[e] = r.v[e];
}

// A tensor [outer, time, inner] by its strides, and states [outer, inner] by theirs.
template <typename T>
struct Seq {
    T* p;
    int64_t so, st, si;
};

template <typename A>
struct States {
    A* p;  // may be null
    int64_t so, si;
    __device__ __forceinline__ A& at(int64_t o, int64_t i) const { return p[o * so + i * si]; }
};

template <typename T>
struct Args {
    using A = wide_t<T>;
    Seq<const T> x, g;
    Seq<T> y;                // forward
    Seq<const T> gy;         // backward; p may be null
    Seq<T> gx, gg;           // p may be null
    States<A> h0, last;      // last: the last state, or its gradient; h0: p may be null (0)
    States<A> gh0;
    A* starts;               // states at the stretches' starts [stretch, outer, inner]; may be null
    A* maps;                 // [segment][a, b][outer, inner]; null: one segment
    int* exps;               // of a, [segment][outer, inner]
    int64_t outer, time, inner;
    int segments;
    int64_t per_segment;     // stretches
    FastDiv tiles, outers;   // rows: workgroups of an outer place, outer places
    int64_t groups;
};

// The place of this workgroup's work: consecutive workgroups go to the 8 XCDs in turn, each with an L2 of
// its own, so each XCD gets a run of neighbours.  Tiles that share lines of memory otherwise fetch them
// twice (8 x 4096 x 2048 bf16 in tiles of 64 bytes: forward 126 -> 106 us; 65521 x 251 fp32, whose rows
// are off every line: 56 -> 35).
__device__ __forceinline__ int64_t neighbour_index(int64_t groups) {
    const uint32_t b = uint32_t(group_index()), n = uint32_t(groups);
    if (b >= n) return b;
    const uint32_t x = b & 7, rest = n & 7;
    return x * (n >> 3) + (x < rest ? x : rest) + (b >> 3);
}

// ---------------------------------------------------------------- inner contiguous
//
// FL lanes side by side, of VEC places, TG groups of C steps each one after the other: a stretch is
// TG * C steps.  Long sequences take 16 lanes (128 bytes of 16-bit elements; 64 bytes were slower, 128
// and 106 us became 99 and 88) and 32 groups of 8 steps, or of 4 in the backward, whose 8 spill: 8 x
// 4096 x 2048 bf16 88 us forward (4.6 TB/s) and 130 backward (5.2), VALU 22 and 32 % busy; what is
// missing to 6.2 is the latency of a stretch with one workgroup a CU.  The groups' maps go through LDS; one thread per inner place scans them.  While a
// stretch is worked on, the loads of the next one are under way.
//
// Every access is a whole one: the last lane of a row starts VEC places before its end, beside (and
// doing again) what its neighbour does, steps behind the last one are read from it and then replaced
// by ones that change nothing.  Rows of fewer than four places take one place a lane.
template <typename T, int FL, int TG, int C, int VEC>
struct Tile {
    using A = wide_t<T>;
    using V = Few<T, VEC>;
    static constexpr int NT = FL * TG;
    static constexpr int PLACES = FL * VEC;
    static constexpr int STRETCH = TG * C;
    static constexpr int PER = (PLACES + NT - 1) / NT;  // places of a scanning thread

    int fl, tg;
    int64_t segment, o, i0, i;
    bool live, writes;

    __device__ __forceinline__ Tile(const Args<T>& a) {
        const int64_t group = neighbour_index(a.groups);
        live = group < a.groups;
        const uint32_t rest = fast_div(uint32_t(group), a.tiles);
        segment = fast_div(rest, a.outers);
        o = rest - uint32_t(segment) * a.outers.d;
        i0 = int64_t(uint32_t(group) - rest * a.tiles.d) * PLACES;
        fl = threadIdx.x % FL;
        tg = threadIdx.x / FL;
        i = at(fl, a.inner);
        writes = i0 + fl * VEC < a.inner;
    }
    __device__ __forceinline__ int64_t at(int lane, int64_t inner) const {
        const int64_t first = i0 + lane * VEC;
        return first < inner - VEC ? first : inner - VEC;
    }
    // The inner place that place p of the tile stands for, and whether it is one of the tensor's.
    __device__ __forceinline__ int64_t place(int p, int64_t inner) const {
        return at(p / VEC, inner) + p % VEC;
    }
    __device__ __forceinline__ bool scans(int p, int64_t inner) const {
        return p < PLACES && i0 + p / VEC * VEC < inner;
    }
    // A thread's steps of stretch s; those behind the last one as `fill`.
    __device__ __forceinline__ void load(V (&v)[C], const Seq<const T>& from, int64_t s, int64_t time,
                                         T fill) const {
        const T* p = from.p + o * from.so + i;
        const int64_t t = s * STRETCH + tg * C;
        if ((s + 1) * STRETCH <= time) {
            p += t * from.st;
#pragma unroll
            for (int c = 0; c < C; ++c, p += from.st) v[c] = load_whole<T, VEC>(p);
        } else if (t < time) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int64_t row = t + c < time ? t + c : time - 1;
                v[c] = load_whole<T, VEC>(p + row * from.st);
            }
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (t + c >= time) v[c] = V::all(fill);
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = V::all(fill);
        }
    }
};

// Between two sweeps: 16-bit elements stay packed as they were loaded.  Without this the compiler keeps
// them widened, in twice the registers.
template <typename V, int C>
__device__ __forceinline__ void keep_packed(V (&v)[C]) {
    if constexpr (sizeof(v[0][0]) == 2 && sizeof(V) == 8) {
        typedef uint32_t words __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int c = 0; c < C; ++c) {
            words w = __builtin_bit_cast(words, v[c]);
            asm volatile("" : "+v"(w));
            v[c] = __builtin_bit_cast(V, w);
        }
    }
}

// State that segment `segment` starts with, or the gradient that it ends with (from the other side).
template <bool BACK, typename T>
__device__ __forceinline__ wide_t<T> segment_start(const Args<T>& a, int64_t segment, int64_t o,
                                                   int64_t i) {
    using A = wide_t<T>;
    const States<A>& from = BACK ? a.last : a.h0;
    A h = from.p ? from.at(o, i) : A(0);
    if (!a.maps) return h;
    const int64_t n = a.outer * a.inner;
    const A* m = a.maps + o * a.inner + i;
    const int* exps = a.exps + o * a.inner + i;
    constexpr int U = 16;  // loads under way at once: one by one, 63 maps took 40 us
    const int count = int(BACK ? a.segments - 1 - segment : segment);
    for (int k0 = 0; k0 < count; k0 += U) {
        Product<A> f[U];
        A b[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int j = k0 + k < count ? k0 + k : count - 1;
            const int64_t s = BACK ? a.segments - 1 - j : j;
            f[k] = {m[2 * s * n], exps[s * n]};
            b[k] = m[(2 * s + 1) * n];
        }
        h = all_applied(f, b, count - k0, h);
    }
    return h;
}

// The maps of a thread's C steps, place by place.
template <bool EXACT, bool MIX, typename A, typename V, int C, int VEC>
__device__ __forceinline__ void walk_maps(const V (&gs)[C], const V (&xs)[C], Map<A> (&m)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        m[e] = Map<A>();
#pragma unroll
        for (int c = 0; c < C; ++c) m[e].template then<EXACT, MIX>(A(gs[c][e]), A(xs[c][e]));
    }
}

template <bool MIX, typename A, typename V, int C, int VEC>
__device__ __forceinline__ void maps_of(const V (&gs)[C], const V (&xs)[C], Map<A> (&m)[VEC]) {
    walk_maps<false, MIX>(gs, xs, m);
    bool fine = true;
#pragma unroll
    for (int e = 0; e < VEC; ++e) fine = fine && finite(m[e].b);
    if (!fine) walk_maps<true, MIX>(gs, xs, m);
}

// What the gradients of a thread's steps make of 0 behind them.
template <typename A, typename V, int C, int VEC>
__device__ __forceinline__ void backs_of(const V (&gs)[C], const V (&ds)[C], A (&q)[VEC]) {
    bool fine = true;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        q[e] = A(0);
#pragma unroll
        for (int c = C - 1; c >= 0; --c) q[e] = back_of<false>(A(gs[c][e]), A(ds[c][e]) + q[e]);
        fine = fine && finite(q[e]);
    }
    if (!fine) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            q[e] = A(0);
#pragma unroll
            for (int c = C - 1; c >= 0; --c) q[e] = back_of<true>(A(gs[c][e]), A(ds[c][e]) + q[e]);
        }
    }
}

// Joins the groups' maps of place p in turn (BACK: from the last one): from `h` on, `to` gets what each
// group starts with.
template <bool BACK, int TG, int PLACES, typename A>
__device__ __forceinline__ A join_groups(const A (&fac)[TG][PLACES], A (&to)[TG][PLACES], int p, A h) {
    constexpr int U = TG < 16 ? TG : 16;
#pragma unroll
    for (int q0 = 0; q0 < TG; q0 += U) {
        A f[U], b[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int q = BACK ? TG - 1 - q0 - k : q0 + k;
            f[k] = fac[q][p];
            b[k] = to[q][p];
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int q = BACK ? TG - 1 - q0 - k : q0 + k;
            to[q][p] = h;
            h = apply(f[k], h, b[k]);
        }
    }
    return h;
}

// Whether a thread's steps have to be walked, where factors f of its maps have left the range, or have
// come back to it: by gates of a magnitude above 2.
template <typename A, typename V, int C, int VEC>
__device__ __forceinline__ bool any_walked(const Map<A> (&m)[VEC], const A (&f)[VEC], const V (&gs)[C]) {
    auto low = size_bits(A(0));
    A top = A(0);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        low = std::min(low, size_bits(m[e].lowest));
        top = greatest_magnitude(top, f[e]);
    }
    if (low >= size_bits(A(kSmall)) && !__builtin_isinf(top)) return false;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        odd = odd || __builtin_isinf(f[e]);
#pragma unroll
        for (int c = 0; c < C; ++c) odd = odd || A(gs[c][e]) > A(2) || A(gs[c][e]) < A(-2);
    }
    return odd;
}

// What a group's steps make of the states h at its places, and `starts` gets what they were.
template <bool MIX, typename A, typename V, int C, int VEC>
__device__ __forceinline__ void walk_group(const V (&gs)[C], const V (&xs)[C], A* h, A* starts) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        A v = h[e];
        starts[e] = v;
#pragma unroll
        for (int c = 0; c < C; ++c) v = step<true, MIX>(A(gs[c][e]), A(xs[c][e]), v);
        h[e] = v;
    }
}

// And of the gradients behind it.
template <typename A, typename V, int C, int VEC>
__device__ __forceinline__ void walk_group_back(const V (&gs)[C], const V (&ds)[C], A* q, A* ends) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        A v = q[e];
        ends[e] = v;
#pragma unroll
        for (int c = C - 1; c >= 0; --c) v = back_of<true>(A(gs[c][e]), A(ds[c][e]) + v);
        q[e] = v;
    }
}

// A forward's stretch may be STARTS of the backward's, and leaves a start for each.
template <typename T, bool MIX, int FL, int TG, int C, int VEC, int STARTS, bool THROUGH = false>
__global__ __launch_bounds__(FL * TG, sizeof(T) == 2 && FL == 32 ? 4 : 1) void k_rows_forward(Args<T> a) {
    using A = wide_t<T>;
    using W = Tile<T, FL, TG, C, VEC>;
    __shared__ A fac[2][TG][W::PLACES], sum[2][TG][W::PLACES];
    __shared__ int walks[2][W::NT / 64];  // a wave's steps of the stretch have to be
    const W w(a);
    if (!w.live) return;
    const int64_t s0 = w.segment * a.per_segment / STARTS;
    const int64_t s1 = std::min((w.segment + 1) * a.per_segment / STARTS,
                                (a.time + W::STRETCH - 1) / W::STRETCH);
    T* const y = a.y.p + w.o * a.y.so + w.i;
    Few<T, VEC> xn[C], gn[C];
    w.load(xn, a.x, s0, a.time, T(0));
    w.load(gn, a.g, s0, a.time, T(1));
    A carry[W::PER];
#pragma unroll
    for (int k = 0; k < W::PER; ++k) {
        const int p = threadIdx.x + k * W::NT;
        carry[k] = w.scans(p, a.inner)
                       ? segment_start<false>(a, w.segment, w.o, w.place(p, a.inner)) : A(0);
    }
    int buf = 0;
    for (int64_t s = s0; s < s1; ++s, buf ^= 1) {
        Few<T, VEC> xs[C], gs[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            xs[c] = xn[c];
            gs[c] = gn[c];
        }
        if (s + 1 < s1) {
            w.load(xn, a.x, s + 1, a.time, T(0));
            w.load(gn, a.g, s + 1, a.time, T(1));
        }
        Map<A> m[VEC];
        maps_of<MIX>(gs, xs, m);
        keep_packed(gs);
        keep_packed(xs);
        A f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            f[e] = m[e].factor();
            fac[buf][w.tg][w.fl * VEC + e] = f[e];
            sum[buf][w.tg][w.fl * VEC + e] = m[e].b;
        }
        const bool walked = __any(any_walked(m, f, gs));
        if (lane_id() == 0) walks[buf][wave_id()] = walked;
        keep_packed(gs);
        __syncthreads();
        A begin[W::PER];
#pragma unroll
        for (int k = 0; k < W::PER; ++k) {
            const int p = threadIdx.x + k * W::NT;
            begin[k] = carry[k];
            if (p < W::PLACES) carry[k] = join_groups<false>(fac[buf], sum[buf], p, carry[k]);
        }
        int walk = 0;
#pragma unroll
        for (int i = 0; i < W::NT / 64; ++i) walk |= walks[buf][i];
        walk = __builtin_amdgcn_readfirstlane(walk);
        if (walk) {
            __syncthreads();
            A* const now = fac[buf][0];
#pragma unroll
            for (int k = 0; k < W::PER; ++k) {
                const int p = threadIdx.x + k * W::NT;
                if (p < W::PLACES) now[p] = begin[k];
            }
            for (int q = 0; q < TG; ++q) {
                __syncthreads();
                if (w.tg == q)
                    walk_group<MIX, A, Few<T, VEC>, C, VEC>(gs, xs, now + w.fl * VEC,
                                                            &sum[buf][q][w.fl * VEC]);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < W::PER; ++k) {
                const int p = threadIdx.x + k * W::NT;
                if (p < W::PLACES) carry[k] = now[p];
            }
        }
#pragma unroll
        for (int k = 0; k < W::PER; ++k) {
            const int p = threadIdx.x + k * W::NT;
            if (a.starts && w.scans(p, a.inner)) {
                const int64_t i = w.place(p, a.inner);
#pragma unroll
                for (int j = 0; j < STARTS; ++j)
                    if (j == 0 || (s * STARTS + j) * (W::STRETCH / STARTS) < a.time)
                        a.starts[((s * STARTS + j) * a.outer + w.o) * a.inner + i] =
                            sum[buf][TG / STARTS * j][p];
            }
        }
        __syncthreads();
        const int64_t t = s * W::STRETCH + w.tg * C;
        const int steps = w.writes ? int(std::min<int64_t>(C, a.time - t)) : 0;
        auto sweep = [&](auto exact) {
            bool fine = true;
            A h[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[e] = sum[buf][w.tg][w.fl * VEC + e];
            T* to = y + t * a.y.st;
#pragma unroll
            for (int c = 0; c < C; ++c, to += a.y.st) {
                typename Few<T, VEC>::Elements out;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    h[e] = step<decltype(exact)::value, MIX>(A(gs[c][e]), A(xs[c][e]), h[e]);
                    out.v[e] = T(h[e]);
                }
                if (c < steps) store_whole<T, VEC, THROUGH>(to, out);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) fine = fine && finite(h[e]);
            return fine;
        };
        if (!sweep(std::false_type{})) sweep(std::true_type{});
    }
    if (w.segment == a.segments - 1) {
#pragma unroll
        for (int k = 0; k < W::PER; ++k) {
            const int p = threadIdx.x + k * W::NT;
            if (w.scans(p, a.inner)) a.last.at(w.o, w.place(p, a.inner)) = carry[k];
        }
    }
}

template <typename T, bool MIX, int FL, int TG, int C, int VEC, bool THROUGH = false>
__global__ __launch_bounds__(FL * TG, 2) void k_rows_backward(Args<T> a) {
    using A = wide_t<T>;
    using W = Tile<T, FL, TG, C, VEC>;
    __shared__ A fac[2][TG][W::PLACES], sum[2][TG][W::PLACES], back[2][TG][W::PLACES];
    __shared__ int walks[2][W::NT / 64];  // as in the forward
    const W w(a);
    if (!w.live) return;
    const int64_t s0 = w.segment * a.per_segment;
    const int64_t s1 = std::min((w.segment + 1) * a.per_segment,
                                (a.time + W::STRETCH - 1) / W::STRETCH);
    T* const gx = a.gx.p + w.o * a.gx.so + w.i;
    T* const gg = a.gg.p + w.o * a.gg.so + w.i;
    Few<T, VEC> xn[C], gn[C], dn[C];
    A start[W::PER];  // states that the stretch begins with
    auto load = [&](int64_t s) {
        w.load(xn, a.x, s, a.time, T(0));
        w.load(gn, a.g, s, a.time, T(1));
        if (a.gy.p) w.load(dn, a.gy, s, a.time, T(0));
#pragma unroll
        for (int k = 0; k < W::PER; ++k) {
            const int p = threadIdx.x + k * W::NT;
            start[k] = A(0);
            if (w.scans(p, a.inner)) {
                const int64_t i = w.place(p, a.inner);
                if (a.starts)
                    start[k] = a.starts[(s * a.outer + w.o) * a.inner + i];
                else if (a.h0.p)
                    start[k] = a.h0.at(w.o, i);
            }
        }
    };
    if (!a.gy.p) {
#pragma unroll
        for (int c = 0; c < C; ++c) dn[c] = Few<T, VEC>::all(T(0));
    }
    load(s1 - 1);
    // the states by the first threads, the gradients by the last ones
    const int rev = W::NT - 1 - int(threadIdx.x);
    A carry[W::PER];
#pragma unroll
    for (int k = 0; k < W::PER; ++k) {
        const int p = rev + k * W::NT;
        carry[k] = w.scans(p, a.inner)
                       ? segment_start<true>(a, w.segment, w.o, w.place(p, a.inner)) : A(0);
    }
    int buf = 0;
    for (int64_t s = s1 - 1; s >= s0; --s, buf ^= 1) {
        Few<T, VEC> xs[C], gs[C], ds[C];
        A begin[W::PER];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            xs[c] = xn[c];
            gs[c] = gn[c];
            ds[c] = dn[c];
        }
#pragma unroll
        for (int k = 0; k < W::PER; ++k) begin[k] = start[k];
        if (s > s0) load(s - 1);
        Map<A> m[VEC];
        A q[VEC];
        maps_of<MIX>(gs, xs, m);
        keep_packed(gs);
        keep_packed(xs);
        backs_of(gs, ds, q);
        keep_packed(gs);
        keep_packed(ds);
        A f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            f[e] = m[e].factor();
            fac[buf][w.tg][w.fl * VEC + e] = f[e];
            sum[buf][w.tg][w.fl * VEC + e] = m[e].b;
            back[buf][w.tg][w.fl * VEC + e] = q[e];
        }
        const bool walked = __any(any_walked(m, f, gs));
        if (lane_id() == 0) walks[buf][wave_id()] = walked;
        keep_packed(gs);
        __syncthreads();
        A behind[W::PER];
#pragma unroll
        for (int k = 0; k < W::PER; ++k) {
            const int p = threadIdx.x + k * W::NT;
            if (p < W::PLACES) join_groups<false>(fac[buf], sum[buf], p, begin[k]);
            const int r = rev + k * W::NT;
            behind[k] = carry[k];
            if (r < W::PLACES) carry[k] = join_groups<true>(fac[buf], back[buf], r, carry[k]);
        }
        int walk = 0;
#pragma unroll
        for (int i = 0; i < W::NT / 64; ++i) walk |= walks[buf][i];
        walk = __builtin_amdgcn_readfirstlane(walk);
        __syncthreads();
        if (walk) {
            A* const now = fac[buf][0];
            A* const later = fac[buf][1];
#pragma unroll
            for (int k = 0; k < W::PER; ++k) {
                const int p = threadIdx.x + k * W::NT, r = rev + k * W::NT;
                if (p < W::PLACES) now[p] = begin[k];
                if (r < W::PLACES) later[r] = behind[k];
            }
            for (int q = 0; q < TG; ++q) {
                __syncthreads();
                if (w.tg == q)
                    walk_group<MIX, A, Few<T, VEC>, C, VEC>(gs, xs, now + w.fl * VEC,
                                                            &sum[buf][q][w.fl * VEC]);
                if (w.tg == TG - 1 - q)
                    walk_group_back<A, Few<T, VEC>, C, VEC>(gs, ds, later + w.fl * VEC,
                                                            &back[buf][w.tg][w.fl * VEC]);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < W::PER; ++k) {
                const int r = rev + k * W::NT;
                if (r < W::PLACES) carry[k] = later[r];
            }
        }
        const int64_t t = s * W::STRETCH + w.tg * C;
        const int steps = w.writes ? int(std::min<int64_t>(C, a.time - t)) : 0;
        auto sweep = [&](auto exact) {
            constexpr bool EXACT = decltype(exact)::value;
            bool fine = true;
            A before[C][VEC], c_in[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                A h = sum[buf][w.tg][w.fl * VEC + e];
                c_in[e] = back[buf][w.tg][w.fl * VEC + e];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    before[c][e] = h;
                    h = step<EXACT, MIX>(A(gs[c][e]), A(xs[c][e]), h);
                }
                fine = fine && finite(h);
            }
            T* to_x = gx + (t + C - 1) * a.gx.st;
            T* to_g = gg + (t + C - 1) * a.gg.st;
#pragma unroll
            for (int c = C - 1; c >= 0; --c, to_x -= a.gx.st, to_g -= a.gg.st) {
                typename Few<T, VEC>::Elements ox, og;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A gate = A(gs[c][e]), whole = A(ds[c][e]) + c_in[e];
                    A dx, dg;
                    gradients<EXACT, MIX>(gate, A(xs[c][e]), before[c][e], whole, dx, dg);
                    ox.v[e] = T(dx);
                    og.v[e] = T(dg);
                    c_in[e] = back_of<EXACT>(gate, whole);
                }
                if (c < steps) {
                    if (a.gx.p) store_whole<T, VEC, THROUGH>(to_x, ox);
                    if (a.gg.p) store_whole<T, VEC, THROUGH>(to_g, og);
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) fine = fine && finite(c_in[e]);
            return fine;
        };
        if (!sweep(std::false_type{})) sweep(std::true_type{});
    }
    if (w.segment == 0 && a.gh0.p) {
#pragma unroll
        for (int k = 0; k < W::PER; ++k) {
            const int p = rev + k * W::NT;
            if (w.scans(p, a.inner)) a.gh0.at(w.o, w.place(p, a.inner)) = carry[k];
        }
    }
}

// The map of each segment: a group's steps lie one behind the other here.
template <typename T, bool MIX, bool BACK, int FL, int TG, int VEC>
__global__ __launch_bounds__(FL * TG) void k_rows_maps(Args<T> a, int stretch) {
    using A = wide_t<T>;
    using W = Tile<T, FL, TG, 1, VEC>;
    constexpr int U = 8;
    __shared__ A fac[TG][W::PLACES], sum[TG][W::PLACES];
    __shared__ int exp[TG][W::PLACES];
    const W w(a);
    if (!w.live) return;
    const int64_t t0 = w.segment * a.per_segment * stretch;
    const int64_t t1 = std::min(a.time, t0 + a.per_segment * stretch);
    const int64_t each = (t1 - t0 + TG - 1) / TG;
    const int64_t b0 = std::min(t1, t0 + w.tg * each), b1 = std::min(t1, b0 + each);
    const T* g = a.g.p + w.o * a.g.so + w.i;
    const Seq<const T>& in = BACK ? a.gy : a.x;
    const T* d = in.p + w.o * in.so + w.i;
    const bool some = !BACK || in.p;
    A h[VEC] = {};
    Product<A> f[VEC];
    Few<T, VEC> gs[U], ds[U];
#pragma unroll
    for (int u = 0; u < U; ++u) ds[u] = Few<T, VEC>::all(T(0));
    for (int64_t n = 0; n < b1 - b0; n += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = n + u < b1 - b0 ? n + u : b1 - b0 - 1;
            const int64_t t = BACK ? b1 - 1 - k : b0 + k;
            gs[u] = load_whole<T, VEC>(g + t * a.g.st);
            if (some) ds[u] = load_whole<T, VEC>(d + t * in.st);
        }
        if (b1 - b0 - n < U) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (n + u >= b1 - b0) {
                    gs[u] = Few<T, VEC>::all(T(1));
                    ds[u] = Few<T, VEC>::all(T(0));
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const A gate = A(gs[u][e]), v = A(ds[u][e]);
                if constexpr (BACK)
                    h[e] = back_of<true>(gate, v + h[e]);
                else
                    h[e] = step<true, MIX>(gate, v, h[e]);
            }
        }
        by_steps(f, gs);
        if ((n & 63) == 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e].even();
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        f[e].plain();
        fac[w.tg][w.fl * VEC + e] = f[e].m;
        exp[w.tg][w.fl * VEC + e] = f[e].e;
        sum[w.tg][w.fl * VEC + e] = h[e];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W::PER; ++k) {
        const int p = threadIdx.x + k * W::NT;
        if (!w.scans(p, a.inner)) continue;
        Product<A> all;
        A b = A(0);
        constexpr int N = 8;
#pragma unroll
        for (int q0 = 0; q0 < TG; q0 += N) {
            Product<A> f[N];
            A h[N];
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const int r = BACK ? TG - 1 - q0 - q : q0 + q;
                f[q] = {fac[r][p], exp[r][p]};
                h[q] = sum[r][p];
            }
            b = all_applied(f, h, N, b);
#pragma unroll
            for (int q = 0; q < N; ++q) all.by(mantissa(f[q].m), exponent(f[q].m) + f[q].e);
            all.even();
        }
        all.plain();
        const int64_t n = a.outer * a.inner, at = w.o * a.inner + w.place(p, a.inner);
        A* to = a.maps + 2 * w.segment * n + at;
        to[0] = all.m;
        to[n] = b;
        a.exps[w.segment * n + at] = all.e;
    }
}

// A few steps, at most N: a thread walks through them, VEC places side by side.
template <typename T, bool MIX, bool BACK, int N>
__global__ __launch_bounds__(kThreads) void k_rows_few(Args<T> a) {
    using A = wide_t<T>;
    constexpr int VEC = wide_vec<T>();
    // the threads of a workgroup go on to the next outer place where a row has fewer lanes
    const int64_t lanes = (a.inner + VEC - 1) / VEC;
    const int64_t item = neighbour_index(a.groups) * kThreads + threadIdx.x;
    if (item >= a.outer * lanes) return;
    int64_t o, lane;
    if (a.outer * lanes < (int64_t(1) << 31)) {
        o = fast_div(uint32_t(item), a.tiles);
        lane = uint32_t(item) - uint32_t(o) * a.tiles.d;
    } else {
        o = item / lanes;
        lane = item - o * lanes;
    }
    const int64_t i = lane * VEC;
    const int count = int(std::min<int64_t>(VEC, a.inner - i));
    auto states = [&](const States<A>& s, A (&h)[VEC]) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[e] = s.p && e < count ? s.at(o, i + e) : A(0);
    };
    auto put = [&](const States<A>& s, const A (&h)[VEC]) {
        if (!s.p) return;
        if (s.si == 1 && count == VEC) {
            Pack<A, VEC> all;
#pragma unroll
            for (int e = 0; e < VEC; ++e) all.v[e] = h[e];
            pstore<A, VEC>(&s.at(o, i), all);
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e < count) s.at(o, i + e) = h[e];
    };
    auto from = [&](const Seq<const T>& s, Few<T, VEC> (&v)[N]) {
        const T* p = s.p + o * s.so + i;
#pragma unroll
        for (int t = 0; t < N; ++t, p += s.st)
            if (t < a.time) v[t] = load_part<T, VEC>(p, s.p ? count : 0, T(0));
    };
    Few<T, VEC> xs[N], gs[N];
    from(a.x, xs);
    from(a.g, gs);
    A h[VEC];
    states(a.h0, h);
    if constexpr (!BACK) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            if (t >= a.time) break;
            typename Few<T, VEC>::Elements out;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[e] = step<true, MIX>(A(gs[t][e]), A(xs[t][e]), h[e]);
                out.v[e] = T(h[e]);
            }
            store_part<T, VEC>(a.y.p + o * a.y.so + t * a.y.st + i, out, count);
        }
        put(a.last, h);
    } else {
        A before[N][VEC], c[VEC];
        Few<T, VEC> ds[N];
        from(a.gy, ds);
        states(a.last, c);
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                before[t][e] = h[e];
                if (t + 1 < a.time) h[e] = step<true, MIX>(A(gs[t][e]), A(xs[t][e]), h[e]);
            }
#pragma unroll
        for (int t = N - 1; t >= 0; --t) {
            if (t >= a.time) continue;
            typename Few<T, VEC>::Elements ox, og;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const A gate = A(gs[t][e]), whole = A(ds[t][e]) + c[e];
                A dx, dg;
                gradients<true, MIX>(gate, A(xs[t][e]), before[t][e], whole, dx, dg);
                ox.v[e] = T(dx);
                og.v[e] = T(dg);
                c[e] = back_of<true>(gate, whole);
            }
            if (a.gx.p) store_part<T, VEC>(a.gx.p + o * a.gx.so + t * a.gx.st + i, ox, count);
            if (a.gg.p) store_part<T, VEC>(a.gg.p + o * a.gg.so + t * a.gg.st + i, og, count);
        }
        put(a.gh0, c);
    }
}
constexpr int64_t kFew = 8;

// ---------------------------------------------------------------- time contiguous
//
// L lanes of 16 bytes of one sequence one after the other: a stretch is L * VEC steps, scanned across
// the lanes; 64 lanes for long sequences (32 for some), which go through their stretches one by one,
// 4 to 32 where one stretch of those is enough.  Bound by memory: 64 x 64 x 12000 fp32 109 us forward (5.4 TB/s) and
// 170 backward (5.8), VALU 69 and 66 % busy; 64 x 129 x 12000 bf16, half of whose lanes have no steps, 241
// and 388, VALU 99 and 93 %.

// The value k lanes before (after: BACK) in the 16 lanes of a DPP row, `none` where there is none.
template <bool BACK, int K, typename A>
__device__ __forceinline__ A beside(A v, A none) {
    constexpr int ctrl = (BACK ? 0x100 : 0x110) | K;  // row_shl / row_shr
    if constexpr (sizeof(A) == 4) {
        return __builtin_bit_cast(
            A, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                           ctrl, 0xF, 0xF, false));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v), n = __builtin_bit_cast(uint64_t, none);
        const uint32_t lo = __builtin_amdgcn_update_dpp(int(uint32_t(n)), int(uint32_t(u)), ctrl, 0xF,
                                                        0xF, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(int(uint32_t(n >> 32)), int(uint32_t(u >> 32)),
                                                        ctrl, 0xF, 0xF, false);
        return __builtin_bit_cast(A, (uint64_t(hi) << 32) | lo);
    }
}

template <int L, bool BACK, int K, typename A>
__device__ __forceinline__ void scan_step(A& a, A& b, int l) {
    A pa = beside<BACK, K>(a, A(1)), pb = beside<BACK, K>(b, A(0));
    if constexpr (L < 16) {
        const bool none = BACK ? l + K >= L : l < K;
        if (none) {
            pa = A(1);
            pb = A(0);
        }
    }
    b = apply(a, pb, b);
    a = kept_product(pa, a);
}

// From the lanes' maps and the state `carry` that the stretch starts with (BACK: from its end), the
// state that each lane starts with; carry becomes the one after the stretch where L is 32 or 64.
template <int L, bool BACK, typename A>
__device__ __forceinline__ A scan_lanes(A a, A b, A& carry) {
    const int l = lane_id() & (L - 1);
    scan_step<L, BACK, 1>(a, b, l);
    scan_step<L, BACK, 2>(a, b, l);
    if constexpr (L >= 8) scan_step<L, BACK, 4>(a, b, l);
    if constexpr (L >= 16) scan_step<L, BACK, 8>(a, b, l);
    A pa = beside<BACK, 1>(a, A(1)), pb = beside<BACK, 1>(b, A(0));
    if constexpr (L < 16) {
        if (BACK ? l + 1 >= L : l < 1) {
            pa = A(1);
            pb = A(0);
        }
    }
    A from = carry;
    if constexpr (L == 32) {  // the state after the row of 16 before, in the lane's own half of the wave
        constexpr int ends[2] = {BACK ? 16 : 15, BACK ? 0 : 31};
        const bool high = lane_id() >= 32;
        auto after = [&](A h, int end) {
            const A la = read_lane(a, end), lb = read_lane(b, end);
            const A ha = read_lane(a, end + 32), hb = read_lane(b, end + 32);
            return apply(high ? ha : la, h, high ? hb : lb);
        };
        const A h = after(carry, ends[0]);
        if (BACK ? l < 16 : l >= 16) from = h;
        carry = after(h, ends[1]);
    }
    if constexpr (L == 64) {
        constexpr int ends[4] = {BACK ? 48 : 15, BACK ? 32 : 31, BACK ? 16 : 47, BACK ? 0 : 63};
        const int row = BACK ? 3 - (l >> 4) : l >> 4;
        A h = carry;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r > 0 && row == r) from = h;
            h = apply(read_lane(a, ends[r]), h, read_lane(b, ends[r]));
        }
        carry = h;
    }
    return apply(pa, from, pb);
}

// The same where maps are not joined (MIX as in step; in: x, or the gradients of the outputs): from the
// state, or the gradient, that the stretch starts with the lanes walk their steps one after the other.
template <int L, bool MIX, bool BACK, typename A, typename V>
__device__ __forceinline__ A walk_lanes(const V& g, const V& in, A& carry) {
    constexpr int VEC = sizeof(V) / sizeof(g[0]);
    const int l = lane_id() & (L - 1);
    A h = carry, from = h;
#pragma unroll 1
    for (int k = 0; k < L; ++k) {
        const int q = BACK ? L - 1 - k : k;
        if (l == q) from = h;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if constexpr (BACK)
                h = back_of<true>(A(g[VEC - 1 - e]), A(in[VEC - 1 - e]) + h);
            else
                h = step<true, MIX>(A(g[e]), A(in[e]), h);
        }
        h = __shfl(h, q, L);
    }
    carry = h;
    return from;
}

// Whether the factor f of any lane's map is none, or none to be multiplied with others; the same in all
// lanes.
template <typename A, typename V>
__device__ __forceinline__ bool lanes_walked(const Map<A>& m, A f, const V& g) {
    constexpr int VEC = sizeof(V) / sizeof(g[0]);
    bool odd = greatest_magnitude(A(0), f) > A(kGrowth);
    if (m.small()) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) odd = odd || A(g[e]) > A(2) || A(g[e]) < A(-2);
    }
    return __any(odd);
}

// A product by a lane's gates, as by_steps has it.
template <typename A, typename V>
__device__ __forceinline__ void by_gates(Product<A>& f, const V& g) {
    constexpr int VEC = sizeof(V) / sizeof(g[0]);
    A p = A(1), lowest = A(1);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        p *= A(g[e]);
        lowest = least_magnitude(lowest, A(g[e]));
    }
    if (lowest >= A(kSmall) && finite(p)) {
        f.by(p);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f.by(A(g[e]));
    }
}

template <typename T, int L, bool BACK>
struct Line {
    static constexpr int VEC = wide_vec<T>();
    static constexpr int STRETCH = L * VEC;
    static constexpr int ROWS = kThreads / L;
    int64_t row, o, i, segment;
    int l;
    bool live;

    __device__ __forceinline__ Line(const Args<T>& a) {
        const int64_t rows = a.outer * a.inner;
        // (backward 176 us with the workgroups in turn, 171 by neighbours; forward 106 and 121)
        int64_t group = BACK ? neighbour_index(a.groups) : group_index();
        live = group < a.groups;
        segment = 0;
        if (a.segments > 1) {  // then groups < 2^31
            segment = fast_div(uint32_t(group), a.tiles);
            group -= segment * a.tiles.d;
        }
        row = group * ROWS + threadIdx.x / L;
        l = threadIdx.x % L;
        live = live && row < rows;
        if (rows < (int64_t(1) << 31)) {
            o = fast_div(uint32_t(row), a.outers);
        } else {
            o = row / a.inner;
        }
        i = row - o * a.inner;
    }
    __device__ __forceinline__ int count(int64_t t, int64_t time) const {
        const int64_t left = time - t;
        return !live || left <= 0 ? 0 : left >= VEC ? VEC : int(left);
    }
};

// The map of a lane's steps.
template <bool MIX, typename A, typename V>
__device__ __forceinline__ void line_map(const V& g, const V& x, Map<A>& m) {
    constexpr int VEC = sizeof(V) / sizeof(g[0]);
    m = Map<A>();
#pragma unroll
    for (int e = 0; e < VEC; ++e) m.template then<false, MIX>(A(g[e]), A(x[e]));
    if (!finite(m.b)) {
        m = Map<A>();
#pragma unroll
        for (int e = 0; e < VEC; ++e) m.template then<true, MIX>(A(g[e]), A(x[e]));
    }
}

// MORE: more than one stretch
template <typename T, bool MIX, int L, bool MORE = L == 64>
__global__ __launch_bounds__(kThreads) void k_lines_forward(Args<T> a) {
    using A = wide_t<T>;
    using W = Line<T, L, false>;
    constexpr int VEC = W::VEC;
    const W w(a);
    const T* x = a.x.p + w.o * a.x.so + w.i * a.x.si;
    const T* g = a.g.p + w.o * a.g.so + w.i * a.g.si;
    T* y = a.y.p + w.o * a.y.so + w.i * a.y.si;
    const int64_t t0 = w.segment * a.per_segment * W::STRETCH;
    const int64_t t1 = std::min(a.time, t0 + a.per_segment * W::STRETCH);
    int64_t t = t0 + w.l * VEC;
    int count = w.count(t, a.time);
    Few<T, VEC> xs = load_part<T, VEC>(x + t, count, T(0)), gs = load_part<T, VEC>(g + t, count, T(1));
    A carry = w.live ? segment_start<false>(a, w.segment, w.o, w.i) : A(0);
    A h = carry;
    for (int64_t s = t0; s < t1; s += W::STRETCH) {
        const Few<T, VEC> xn = xs, gn = gs;
        const int now = count;
        const int64_t at = t;
        if constexpr (MORE) {  // the next stretch's loads are under way during this one's scan
            if (s + W::STRETCH < t1) {
                t += W::STRETCH;
                count = w.count(t, a.time);
                xs = load_part<T, VEC>(x + t, count, T(0));
                gs = load_part<T, VEC>(g + t, count, T(1));
            }
            if (a.starts && w.l == 0 && w.live)
                a.starts[s / W::STRETCH * (a.outer * a.inner) + w.row] = carry;
        }
        Map<A> m;
        line_map<MIX>(gn, xn, m);
        const A f = m.factor();
        const A begin = lanes_walked(m, f, gn) ? walk_lanes<L, MIX, false>(gn, xn, carry)
                                            : scan_lanes<L, false>(f, m.b, carry);
        auto sweep = [&](auto exact) {
            typename Few<T, VEC>::Elements out;
            h = begin;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h = step<decltype(exact)::value, MIX>(A(gn[e]), A(xn[e]), h);
                out.v[e] = T(h);
            }
            store_part<T, VEC>(y + at, out, now);
        };
        sweep(std::false_type{});
        if (!finite(h)) sweep(std::true_type{});
    }
    if (w.live && w.segment == a.segments - 1 && w.l == L - 1) a.last.at(w.o, w.i) = h;
}

template <typename T, bool MIX, int L, bool MORE = L == 64>
__global__ __launch_bounds__(kThreads) void k_lines_backward(Args<T> a) {
    using A = wide_t<T>;
    using W = Line<T, L, true>;
    constexpr int VEC = W::VEC;
    const W w(a);
    const T* x = a.x.p + w.o * a.x.so + w.i * a.x.si;
    const T* g = a.g.p + w.o * a.g.so + w.i * a.g.si;
    const T* gy = a.gy.p + w.o * a.gy.so + w.i * a.gy.si;
    T* gx = a.gx.p + w.o * a.gx.so + w.i * a.gx.si;
    T* gg = a.gg.p + w.o * a.gg.so + w.i * a.gg.si;
    const int64_t s0 = w.segment * a.per_segment;
    const int64_t s1 = std::min(s0 + a.per_segment, (a.time + W::STRETCH - 1) / W::STRETCH);
    int64_t t = (s1 - 1) * W::STRETCH + w.l * VEC;
    int count = 0;
    Few<T, VEC> xs, gs, ds;
    A start = A(0);
    auto load = [&](int64_t s) {
        count = w.count(t, a.time);
        xs = load_part<T, VEC>(x + t, count, T(0));
        gs = load_part<T, VEC>(g + t, count, T(1));
        ds = load_part<T, VEC>(gy + t, a.gy.p ? count : 0, T(0));
        if (w.live) {
            if (MORE && a.starts)
                start = a.starts[s * (a.outer * a.inner) + w.row];
            else if (a.h0.p)
                start = a.h0.at(w.o, w.i);
        }
    };
    load(s1 - 1);
    A carry = w.live ? segment_start<true>(a, w.segment, w.o, w.i) : A(0);
    A c = carry;
    for (int64_t s = s1 - 1; s >= s0; --s) {
        const Few<T, VEC> xn = xs, gn = gs, dn = ds;
        const int now = count;
        const int64_t at = t;
        A begin = start;
        if constexpr (MORE) {
            if (s > s0) {
                t -= W::STRETCH;
                load(s - 1);
            }
        }
        Map<A> m;
        line_map<MIX>(gn, xn, m);
        A q = A(0);
#pragma unroll
        for (int e = VEC - 1; e >= 0; --e) q = back_of<false>(A(gn[e]), A(dn[e]) + q);
        if (!finite(q)) {
            q = A(0);
#pragma unroll
            for (int e = VEC - 1; e >= 0; --e) q = back_of<true>(A(gn[e]), A(dn[e]) + q);
        }
        const A f = m.factor();
        const bool walk = lanes_walked(m, f, gn);
        const A h0 = walk ? walk_lanes<L, MIX, false>(gn, xn, begin) : scan_lanes<L, false>(f, m.b, begin);
        const A c0 = walk ? walk_lanes<L, MIX, true>(gn, dn, carry) : scan_lanes<L, true>(f, q, carry);
        auto sweep = [&](auto exact) {
            constexpr bool EXACT = decltype(exact)::value;
            A h = h0, before[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                before[e] = h;
                h = step<EXACT, MIX>(A(gn[e]), A(xn[e]), h);
            }
            c = c0;
            typename Few<T, VEC>::Elements ox, og;
#pragma unroll
            for (int e = VEC - 1; e >= 0; --e) {
                const A gate = A(gn[e]), whole = A(dn[e]) + c;
                A dx, dg;
                gradients<EXACT, MIX>(gate, A(xn[e]), before[e], whole, dx, dg);
                ox.v[e] = T(dx);
                og.v[e] = T(dg);
                c = back_of<EXACT>(gate, whole);
            }
            if (a.gx.p) store_part<T, VEC>(gx + at, ox, now);
            if (a.gg.p) store_part<T, VEC>(gg + at, og, now);
            return finite(h) && finite(c);
        };
        if (!sweep(std::false_type{})) sweep(std::true_type{});
    }
    if (w.live && w.segment == 0 && w.l == 0 && a.gh0.p) a.gh0.at(w.o, w.i) = c;
}

// The map of each segment, stretch by stretch.
template <typename T, bool MIX, bool BACK>
__global__ __launch_bounds__(kThreads) void k_lines_maps(Args<T> a) {
    using A = wide_t<T>;
    using W = Line<T, 64, BACK>;
    constexpr int VEC = W::VEC;
    const W w(a);
    const T* g = a.g.p + w.o * a.g.so + w.i * a.g.si;
    const Seq<const T>& src = BACK ? a.gy : a.x;
    const T* d = src.p + w.o * src.so + w.i * src.si;
    const bool some = !BACK || src.p;
    const int64_t s0 = w.segment * a.per_segment;
    const int64_t s1 = std::min(s0 + a.per_segment, (a.time + W::STRETCH - 1) / W::STRETCH);
    Few<T, VEC> gs, ds;
    auto load = [&](int64_t k) {
        const int64_t t = (BACK ? s1 - 1 - k : s0 + k) * W::STRETCH + w.l * VEC;
        const int count = w.count(t, a.time);
        gs = load_part<T, VEC>(g + t, count, T(1));
        ds = load_part<T, VEC>(d + t, some ? count : 0, T(0));
    };
    load(0);
    Product<A> f;
    A b = A(0);
    for (int64_t k = 0; k < s1 - s0; ++k) {
        const Few<T, VEC> gn = gs, dn = ds;
        if (k + 1 < s1 - s0) load(k + 1);
        Map<A> m;
        if constexpr (BACK) {
#pragma unroll
            for (int e = VEC - 1; e >= 0; --e) {
                m.b = back_of<true>(A(gn[e]), A(dn[e]) + m.b);
                m.factor_by(A(gn[e]));
            }
        } else {
            line_map<MIX>(gn, dn, m);
        }
        A fac = m.factor(), sum = m.b;
        if (lanes_walked(m, fac, gn)) {
            walk_lanes<64, MIX, BACK>(gn, dn, b);
        } else {
            scan_step<64, BACK, 1>(fac, sum, w.l);
            scan_step<64, BACK, 2>(fac, sum, w.l);
            scan_step<64, BACK, 4>(fac, sum, w.l);
            scan_step<64, BACK, 8>(fac, sum, w.l);
            constexpr int ends[4] = {BACK ? 48 : 15, BACK ? 32 : 31, BACK ? 16 : 47, BACK ? 0 : 63};
#pragma unroll
            for (int r = 0; r < 4; ++r)
                b = apply(read_lane(fac, ends[r]), b, read_lane(sum, ends[r]));
        }
        by_gates(f, gn);  // the lane's own steps of every stretch
        f.even();
    }
    // over the lanes: rows of 16, as wave_total goes, then the rows
    f.by(dpp_move<0xB1>(f.m), dpp_move<0xB1>(f.e));
    f.by(dpp_move<0x4E>(f.m), dpp_move<0x4E>(f.e));
    f.by(dpp_move<0x124>(f.m), dpp_move<0x124>(f.e));
    f.by(dpp_move<0x128>(f.m), dpp_move<0x128>(f.e));
    const Product<A> one = f;
    f = Product<A>();
#pragma unroll
    for (int r = 0; r < 64; r += 16) f.by(read_lane(one.m, r), read_lane(one.e, r));
    f.plain();
    if (w.live && w.l == 0) {
        const int64_t n = a.outer * a.inner;
        A* to = a.maps + 2 * w.segment * n + w.row;
        to[0] = f.m;
        to[n] = b;
        a.exps[w.segment * n + w.row] = f.e;
    }
}

// ---------------------------------------------------------------- launches

// How a call goes: which kernels, and into how many segments of how many stretches.
enum Way { kRowsFew, kRowsHalf, kRowsShort, kRowsLong, kRowsNarrow, kLines4, kLines8, kLines16, kLines32, kLines64 };

struct Route {
    Way way;
    int64_t stretch;      // steps
    int64_t stretches;
    int segments;
    int64_t per_segment;  // stretches
    int64_t units;        // workgroups of one segment
    int64_t tiles;        // rows: workgroups (kRowsFew: lanes) of an outer place
};

// Segments where there are fewer workgroups than would fill the chip's 256 CUs: as many as bring
// them to 1024 (two to four a CU), the first pass costing two thirds of another forward.
void cut(Route& r) {
    int64_t n = 1;
    if (r.units < 256) n = std::min<int64_t>({1024 / r.units, r.stretches / 2, kMaxSegments});
    if (n < 1) n = 1;
    r.per_segment = (ceil_div(r.stretches, n) + 1) / 2 * 2;  // (a forward may take two at once)
    r.segments = int(ceil_div(r.stretches, r.per_segment));
}

// Places of a lane of the kernels for inner contiguous.
int64_t places_of(int dtype) { return dtype == CL_DTYPE_F64 ? 2 : 4; }
int64_t vec_of(int dtype) { return dtype == CL_DTYPE_F64 ? 2 : dtype == CL_DTYPE_F32 ? 4 : 8; }

// time contiguous: outer * inner lines; else inner contiguous
Route route_of(int dtype, bool lines, int64_t outer, int64_t time, int64_t inner) {
    Route r{};
    const int64_t vec = vec_of(dtype), places = places_of(dtype);
    if (lines) {
        // As few lanes a sequence as hold it; where 32 do not, 32 with two stretches, of 16-bit values
        // three, or 64.  With 64 one stretch has no next one whose loads cover its scan, and many lanes
        // have no steps: 64 x T x 12000, 32 lanes against 64, forward / backward in us:
        //   fp32 T 129  271 / 429  367 / 522      bf16 T 300  360 / 686  461 / 940
        //   fp32 T 200  323 / 575  380 / 566      bf16 T 500  468 / 794  499 / 1030
        //   fp32 T 300  516 / 976  565 / 872      bf16 T 600  570 / 945  659 / 1220
        //   fp32 T 500  985 / 1640 793 / 1411     bf16 T 1000 x 2000  164 / 286  140 / 246
        // Few sequences take 64, and one stretch rather than two.
        int way = kLines4, l = 4;
        while (l < 32 && l * vec < time) l *= 2, ++way;
        const bool many = outer * inner >= 256 * (kThreads / 32);
        if (l * vec < time && !(many && time <= (vec == 8 ? 3 : 2) * 32 * vec)) l = 64, ++way;
        r.way = Way(way);
        r.stretch = l * vec;
        r.units = ceil_div(outer * inner, kThreads / l);
    } else if (time <= kFew) {
        r.way = kRowsFew;
        r.stretch = kFew;
        r.tiles = ceil_div(inner, vec);
        r.units = ceil_div(outer * r.tiles, kThreads);
    } else {
        // 32 lanes side by side and 8 groups (4) of 4 steps, whose workgroups are small and fill the chip
        // without a long time, or 16 and 32 (a forward: of 8), whose stretches are fewer.  Measured,
        // the first against the second, forward / backward in us:
        //   256 x 64 x 1000 fp16   20 / 34   32 / 75      256 x 96 x 1000 fp32   48 / 102   59 / 115
        //   64 x 64 x 12000 fp32  109 / 193 126 / 282     256 x 256 x 1000 fp16  73 / 155   95 / 196
        //   64 x 1000 x 1024 fp32 148 / 260 152 / 260     16 x 4000 x 2048 fp16 183 / 270  165 / 275
        // (The first is never cut into segments: up to 96 steps or with 512 workgroups.)
        const int64_t broad = ceil_div(inner, 32 * places);
        if (inner < places) {
            r.way = kRowsNarrow;
            r.tiles = 1;
            r.stretch = 256;
        } else if (time <= 96 || (time <= 512 && outer * broad >= 512)) {
            // Stretches of 16, by 4 groups, where they leave fewer groups without steps: one instead of 32
            // for 512 x 16 x 4000 fp16 58 / 170 -> 34 / 70, two for 512 x 24 x 4000 fp16 82 / 187 ->
            // 63 / 144, three for 256 x 48 x 1000 fp32 27 / 56 -> 24 / 40 (four 66 -> 69 backward; where
            // there is no other workgroup to hide it, each further one costs 2 us).
            const bool half = time <= 16 || (time <= 48 && outer * broad >= 512);
            r.way = half ? kRowsHalf : kRowsShort;
            r.tiles = broad;
            r.stretch = half ? 16 : 32;
        } else {
            r.way = kRowsLong;
            r.tiles = ceil_div(inner, 16 * places);
            r.stretch = 128;
        }
        r.units = outer * r.tiles;
    }
    r.stretches = ceil_div(time, r.stretch);
    cut(r);
    return r;
}

template <typename T>
int route_args(Args<T>& a, const Route& r, bool lines, void* workspace) {
    a.segments = r.segments;
    a.per_segment = r.per_segment;
    a.maps = r.segments > 1 ? static_cast<wide_t<T>*>(workspace) : nullptr;
    a.exps = a.maps ? reinterpret_cast<int*>(a.maps + 2 * r.segments * a.outer * a.inner) : nullptr;
    if (r.stretches <= 1) a.starts = nullptr;
    a.groups = r.units * r.segments;
    CL_ARG(a.groups < (int64_t(1) << 31), "too many sequences for one call");
    const int64_t most = INT32_MAX;
    a.tiles = make_fastdiv(uint32_t(std::min(lines ? r.units : r.tiles, most)));
    a.outers = make_fastdiv(uint32_t(std::min(lines ? a.inner : a.outer, most)));
    return CL_OK;
}

template <typename T, bool MIX, bool BACK>
int launch_recurrence(const Args<T>& a, const Route& r, hipStream_t s) {
    constexpr int P = sizeof(T) == 8 ? 2 : 4;
    const dim3 grid = wide_grid(a.groups);
    // Long sequences: outputs past the 256 MiB cache from 96 MiB each on, where what comes next would
    // not find them in it (134 MB each: forward 94 -> 86 us, backward 135 -> 128; 66 MB: 62 -> 66).
    const bool through = double(a.outer) * a.time * a.inner * sizeof(T) >= double(96 << 20);
    if (r.segments > 1) {
        if (r.way == kLines64)
            k_lines_maps<T, MIX, BACK><<<grid, kThreads, 0, s>>>(a);
        else if (r.way == kRowsNarrow)
            k_rows_maps<T, MIX, BACK, 8, 32, 1><<<grid, kThreads, 0, s>>>(a, int(r.stretch));
        else
            k_rows_maps<T, MIX, BACK, 16, 16, P><<<grid, kThreads, 0, s>>>(a, int(r.stretch));
        if (int rc = check_launch("cl_recurrence(maps)")) return rc;
    }
    switch (r.way) {
        case kRowsFew:
            if (a.time <= 2)
                k_rows_few<T, MIX, BACK, 2><<<grid, kThreads, 0, s>>>(a);
            else
                k_rows_few<T, MIX, BACK, int(kFew)><<<grid, kThreads, 0, s>>>(a);
            break;
        case kRowsHalf:
            if constexpr (BACK)
                k_rows_backward<T, MIX, 32, 4, 4, P><<<grid, 128, 0, s>>>(a);
            else
                k_rows_forward<T, MIX, 32, 4, 4, P, 1><<<grid, 128, 0, s>>>(a);
            break;
        case kRowsShort:  // (the forward past the cache: 256 x 256 x 1000 fp16 89 -> 71 us; no gain in the backward)
            if constexpr (BACK)
                k_rows_backward<T, MIX, 32, 8, 4, P><<<grid, kThreads, 0, s>>>(a);
            else if (through)
                k_rows_forward<T, MIX, 32, 8, 4, P, 1, true><<<grid, kThreads, 0, s>>>(a);
            else
                k_rows_forward<T, MIX, 32, 8, 4, P, 1><<<grid, kThreads, 0, s>>>(a);
            break;
        case kRowsLong:
            if constexpr (BACK) {
                if (through)
                    k_rows_backward<T, MIX, 16, 32, 4, P, true><<<grid, 512, 0, s>>>(a);
                else
                    k_rows_backward<T, MIX, 16, 32, 4, P><<<grid, 512, 0, s>>>(a);
            } else if (r.stretches == 1) {
                k_rows_forward<T, MIX, 16, 32, 4, P, 1><<<grid, 512, 0, s>>>(a);
            } else if (through) {
                k_rows_forward<T, MIX, 16, 32, 8, P, 2, true><<<grid, 512, 0, s>>>(a);
            } else {
                k_rows_forward<T, MIX, 16, 32, 8, P, 2><<<grid, 512, 0, s>>>(a);
            }
            break;
        case kRowsNarrow:
            if constexpr (BACK)
                k_rows_backward<T, MIX, 8, 32, 8, 1><<<grid, kThreads, 0, s>>>(a);
            else
                k_rows_forward<T, MIX, 8, 32, 8, 1, 1><<<grid, kThreads, 0, s>>>(a);
            break;
        case kLines4:
            if constexpr (BACK)
                k_lines_backward<T, MIX, 4><<<grid, kThreads, 0, s>>>(a);
            else
                k_lines_forward<T, MIX, 4><<<grid, kThreads, 0, s>>>(a);
            break;
        case kLines8:
            if constexpr (BACK)
                k_lines_backward<T, MIX, 8><<<grid, kThreads, 0, s>>>(a);
            else
                k_lines_forward<T, MIX, 8><<<grid, kThreads, 0, s>>>(a);
            break;
        case kLines16:
            if constexpr (BACK)
                k_lines_backward<T, MIX, 16><<<grid, kThreads, 0, s>>>(a);
            else
                k_lines_forward<T, MIX, 16><<<grid, kThreads, 0, s>>>(a);
            break;
        case kLines32:  // (one stretch by the other kernel, 64 x 200 x 12000 bf16: backward 427, 349 us)
            if constexpr (BACK) {
                if (r.stretches > 1)
                    k_lines_backward<T, MIX, 32, true><<<grid, kThreads, 0, s>>>(a);
                else
                    k_lines_backward<T, MIX, 32><<<grid, kThreads, 0, s>>>(a);
            } else {
                if (r.stretches > 1)
                    k_lines_forward<T, MIX, 32, true><<<grid, kThreads, 0, s>>>(a);
                else
                    k_lines_forward<T, MIX, 32><<<grid, kThreads, 0, s>>>(a);
            }
            break;
        case kLines64:
            if constexpr (BACK)
                k_lines_backward<T, MIX, 64><<<grid, kThreads, 0, s>>>(a);
            else
                k_lines_forward<T, MIX, 64><<<grid, kThreads, 0, s>>>(a);
            break;
    }
    return check_launch("cl_recurrence");
}

// The dimensions as the kernels name them: which of batch and features is the outer one.
struct Dims {
    int64_t outer, time, inner;
    bool lines;
    int o, i;  // the strides' places of outer and inner in (batch, time, features)
};

int dims_of(int order, int64_t batch, int64_t time, int64_t features, Dims& d) {
    CL_ARG(batch >= 0 && time >= 0 && features >= 0, "negative shape");
    switch (order) {
        case CL_RECURRENCE_FEATURES:
            d = {batch, time, features, false, 0, 2};
            return CL_OK;
        case CL_RECURRENCE_TIME_BATCH:
            d = {batch, time, features, true, 0, 2};
            return CL_OK;
        case CL_RECURRENCE_TIME_FEATURES:
            d = {features, time, batch, true, 2, 0};
            return CL_OK;
        case CL_RECURRENCE_BATCH:
            CL_ARG(time <= 1, "the batch is contiguous for one step only");
            d = {features, time, batch, false, 2, 0};
            return CL_OK;
        default:
            set_error("unknown order %d", order);
            return CL_ERR_INVALID_ARGUMENT;
    }
}

template <typename T>
int sequence(Seq<T>& s, const char* name, const void* p, const int64_t* strides, const Dims& d,
             bool optional) {
    s = {static_cast<T*>(const_cast<void*>(p)), 0, 0, 0};
    if (!p && optional) return CL_OK;
    CL_ARG(p && strides, "null pointer argument");
    s.so = strides[d.o];
    s.st = strides[1];
    s.si = strides[d.i];
    CL_ARG(s.so >= 0 && s.st >= 0 && s.si >= 0, "negative strides are not supported");
    if (d.lines)
        CL_ARG(s.st == 1 || d.time <= 1, "%s is not contiguous along its time", name);
    else
        CL_ARG(s.si == 1 || d.inner <= 1, "%s is not contiguous along its inner dimension", name);
    return CL_OK;
}

template <typename A>
int states(States<A>& s, const void* p, const int64_t* strides, const Dims& d, bool optional) {
    s = {static_cast<A*>(const_cast<void*>(p)), 0, 0};
    if (!p && optional) return CL_OK;
    CL_ARG(p && strides, "null pointer argument");
    s.so = strides[d.o == 0 ? 0 : 1];
    s.si = strides[d.i == 0 ? 0 : 1];
    CL_ARG(s.so >= 0 && s.si >= 0, "negative strides are not supported");
    return CL_OK;
}

int sizes(int dtype, int order, int64_t batch, int64_t time, int64_t features, Dims& d, Route& r,
          int64_t& starts, int64_t& bytes) {
    CL_ARG(dtype >= CL_DTYPE_F32 && dtype <= CL_DTYPE_BF16,
           "unsupported dtype code %d (expected F32, F64, F16 or BF16)", dtype);
    if (int rc = dims_of(order, batch, time, features, d)) return rc;
    starts = bytes = 0;
    if (batch == 0 || time == 0 || features == 0) return CL_OK;
    r = route_of(dtype, d.lines, d.outer, d.time, d.inner);
    const int64_t n = batch * features;
    starts = r.stretches > 1 ? r.stretches * n : 0;
    bytes = r.segments > 1 ? r.segments * n * (2 * (dtype == CL_DTYPE_F64 ? 8 : 4) + 4) : 0;
    return CL_OK;
}

}  // namespace
}  // namespace cl

using namespace cl;

extern "C" int cl_recurrence_sizes(int dtype, int order, int64_t batch, int64_t time, int64_t features,
                                   int64_t* starts, int64_t* workspace_bytes) {
    clear_error();
    CL_ARG(starts && workspace_bytes, "null pointer argument");
    Dims d;
    Route r;
    return sizes(dtype, order, batch, time, features, d, r, *starts, *workspace_bytes);
}

extern "C" int cl_recurrence_forward(int dtype, int order, int form, const void* x,
                                     const int64_t* x_strides, const void* gate,
                                     const int64_t* gate_strides, const void* state,
                                     const int64_t* state_strides, int64_t batch, int64_t time,
                                     int64_t features, void* y, const int64_t* y_strides, void* last,
                                     const int64_t* last_strides, void* starts, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    clear_error();
    CL_ARG(form == CL_RECURRENCE_MIX || form == CL_RECURRENCE_ADD, "unknown form %d", form);
    Dims d;
    Route r;
    int64_t n = 0, need = 0;
    if (int rc = sizes(dtype, order, batch, time, features, d, r, n, need)) return rc;
    CL_ARG(time > 0, "a recurrence of no steps");
    if (batch == 0 || features == 0) return CL_OK;
    CL_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 8)),
           "workspace of %lld bytes needed (cl_recurrence_sizes)", (long long)need);
    hipStream_t s = as_stream(stream);
    CL_STORAGE_SWITCH(dtype, {
        Args<scalar_t> a{};
        a.outer = d.outer;
        a.time = time;
        a.inner = d.inner;
        a.starts = static_cast<wide_t<scalar_t>*>(starts);
        if (int rc = sequence(a.x, "x", x, x_strides, d, false)) return rc;
        if (int rc = sequence(a.g, "gate", gate, gate_strides, d, false)) return rc;
        if (int rc = sequence(a.y, "y", y, y_strides, d, false)) return rc;
        if (int rc = states(a.h0, state, state_strides, d, true)) return rc;
        if (int rc = states(a.last, last, last_strides, d, false)) return rc;
        if (int rc = route_args(a, r, d.lines, workspace)) return rc;
        return form == CL_RECURRENCE_MIX ? launch_recurrence<scalar_t, true, false>(a, r, s)
                                         : launch_recurrence<scalar_t, false, false>(a, r, s);
    });
}

extern "C" int cl_recurrence_backward(int dtype, int order, int form, const void* x,
                                      const int64_t* x_strides, const void* gate,
                                      const int64_t* gate_strides, const void* state,
                                      const int64_t* state_strides, const void* starts,
                                      const void* grad_y, const int64_t* grad_y_strides,
                                      const void* grad_last, const int64_t* grad_last_strides,
                                      int64_t batch, int64_t time, int64_t features, void* grad_x,
                                      const int64_t* grad_x_strides, void* grad_gate,
                                      const int64_t* grad_gate_strides, void* grad_state,
                                      const int64_t* grad_state_strides, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    clear_error();
    CL_ARG(form == CL_RECURRENCE_MIX || form == CL_RECURRENCE_ADD, "unknown form %d", form);
    Dims d;
    Route r;
    int64_t n = 0, need = 0;
    if (int rc = sizes(dtype, order, batch, time, features, d, r, n, need)) return rc;
    CL_ARG(time > 0, "a recurrence of no steps");
    if (batch == 0 || features == 0) return CL_OK;
    CL_ARG(n == 0 || starts, "the forward's starts are needed (cl_recurrence_sizes)");
    CL_ARG(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 8)),
           "workspace of %lld bytes needed (cl_recurrence_sizes)", (long long)need);
    hipStream_t s = as_stream(stream);
    CL_STORAGE_SWITCH(dtype, {
        Args<scalar_t> a{};
        a.outer = d.outer;
        a.time = time;
        a.inner = d.inner;
        a.starts = static_cast<wide_t<scalar_t>*>(const_cast<void*>(starts));
        if (int rc = sequence(a.x, "x", x, x_strides, d, false)) return rc;
        if (int rc = sequence(a.g, "gate", gate, gate_strides, d, false)) return rc;
        if (int rc = sequence(a.gy, "grad_y", grad_y, grad_y_strides, d, true)) return rc;
        if (int rc = sequence(a.gx, "grad_x", grad_x, grad_x_strides, d, true)) return rc;
        if (int rc = sequence(a.gg, "grad_gate", grad_gate, grad_gate_strides, d, true)) return rc;
        if (int rc = states(a.h0, state, state_strides, d, true)) return rc;
        if (int rc = states(a.last, grad_last, grad_last_strides, d, true)) return rc;
        if (int rc = states(a.gh0, grad_state, grad_state_strides, d, true)) return rc;
        if (int rc = route_args(a, r, d.lines, workspace)) return rc;
        return form == CL_RECURRENCE_MIX ? launch_recurrence<scalar_t, true, true>(a, r, s)
                                         : launch_recurrence<scalar_t, false, true>(a, r, s);
    });
}

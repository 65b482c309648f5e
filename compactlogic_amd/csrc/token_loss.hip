// Losses on the log-probability of one chosen class or token per row of logits: the
// log-probability itself, the clipped policy loss with a KL term, and the preference loss of
// paired sequences, each with the logits' gradient.
//
// Row n of logits x[n, 0..V) with action a:  m = max x,  s = sum exp(x - m),
//   lp = (x_a - m) - log s,   p_j = exp(x_j - m) / s,   d lp / d x_j = [j = a] - p_j.
// Every loss is a function of the rows' lp, so its gradient is a number per row, the slope,
// times [j = a] - p_j.  The forward leaves per row (m, 1 / s, 1 - p_a, slope) and the backward
// forms the gradient from them (1 - p_a from the fp64 lp, rounded once).
//
// The row's scalars (lp and what the losses make of it) are taken in fp64: rows lie next to the
// borders of the clipped range, and the preference loss subtracts sums over whole sequences.
#include "row_loss.h"
#include "storage.h"

#include <algorithm>

namespace cl {
namespace {

template <typename T>
struct RowArgs {
    const T* x;
    int64_t stride;
    int64_t rows;
    int64_t cols;
    const int64_t* actions;
    int64_t ignore;
    wide_t<T>* lp;
    RowState<wide_t<T>>* state;
    // Logits and gradient past the 256 MiB cache, by their size.  A gradient from 96 MiB on would
    // push out the logits that the cache still holds (131 MB of bf16, policy loss and gradient 60
    // -> 55 us with the stores past it, 192 MB 96 -> 71, 262 MB of fp32 121 -> 100; at 38 MB
    // nothing changes, and what comes next finds it).  Logits larger than the cache are not found
    // again in it (328 MB 151 -> 126 us with the loads past it as well, 537 MB 237 -> 203; at 262
    // MB they cost 17 us).
    bool through_load, through_store;
};

template <typename A>
__device__ __forceinline__ A nan_value() {
    return A(__builtin_nan(""));
}

// ---- what each loss makes of a row's lp.  `load` fetches the row's own inputs early; e[1] and
// e[2] are the exponentials of arg(1) and arg(2), taken by neighbouring lanes at once; `counted`
// writes the loss's outputs (one lane) and returns the slope.
struct RowInputs {
    double old_lp, adv, ref;
};

template <typename A>
struct LogProbOp {
    __device__ __forceinline__ RowInputs load(int64_t) const { return {}; }
    __device__ __forceinline__ double arg(int, double lp, const RowInputs&) const { return lp; }
    __device__ __forceinline__ double counted(int64_t, double lp, const RowInputs&, const double*,
                                              bool) const {
        return lp == lp ? 1.0 : lp;
    }
    __device__ __forceinline__ void ignored(int64_t, bool) const {}
};

// term = kl (exp(g) - g - 1) - clip(r) adv with r = exp(lp - old) clipped from above where adv
// is positive and from below where it is negative (the smaller of the clipped and the free
// product), g = ref - lp.
template <typename A>
struct PolicyOp {
    const A* old_lp;
    const A* adv;
    const A* ref;
    double low, high, kl;
    A* terms;
    __device__ __forceinline__ RowInputs load(int64_t n) const {
        return {double(old_lp[n]), double(adv[n]), ref ? double(ref[n]) : 0.0};
    }
    __device__ __forceinline__ double arg(int i, double lp, const RowInputs& in) const {
        return i == 1 ? lp - in.old_lp : in.ref - lp;
    }
    __device__ __forceinline__ double counted(int64_t n, double lp, const RowInputs& in,
                                              const double* e, bool write) const {
        const double a = in.adv, r = e[1];
        double term, slope;
        if (a >= 0) {
            term = -(r > high ? high : r) * a;
            slope = r > high ? 0.0 : -a * r;
        } else {
            term = -(r < low ? low : r) * a;
            slope = r < low ? 0.0 : -a * r;
        }
        if (ref) {
            term += kl * ((e[2] - 1.0) - (in.ref - lp));
            slope -= kl * (e[2] - 1.0);
        }
        if (write) terms[n] = A(term);
        return slope;
    }
    __device__ __forceinline__ void ignored(int64_t n, bool write) const {
        if (write) terms[n] = A(0);
    }
};

// gap = lp - ref, summed over sequences by pair_terms.
template <typename A>
struct PreferenceOp {
    const A* ref;
    double* gaps;
    int32_t* row_seq;
    __device__ __forceinline__ RowInputs load(int64_t n) const {
        return {0.0, 0.0, ref ? double(ref[n]) : 0.0};
    }
    __device__ __forceinline__ double arg(int, double lp, const RowInputs&) const { return lp; }
    __device__ __forceinline__ double counted(int64_t n, double lp, const RowInputs& in,
                                              const double*, bool write) const {
        if (write) {
            gaps[n] = lp - in.ref;
            row_seq[n] = -1;
        }
        return 1.0;
    }
    __device__ __forceinline__ void ignored(int64_t n, bool write) const {
        if (write) {
            gaps[n] = 0.0;
            row_seq[n] = -1;
        }
    }
};

// ---- exponentials and reductions
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return __builtin_fmax(a, b); }

// Where a part of a row saw nothing but -inf its maximum is -inf, and differences are taken from
// 0 instead: its sum is 0, or NaN if a NaN came by.
template <typename A>
__device__ __forceinline__ A base_of(A m) {
    return m == -A(__builtin_inf()) ? A(0) : m;
}

// Over the TPR lanes of a row (16: a DPP row, 64: the wave), the same bits in each of them: every
// step exchanges with a mirror image, whose partial sum is the same two numbers the other way
// round.
template <int TPR, typename A>
__device__ __forceinline__ A lanes_max(A v) {
    v = max_of(v, dpp_move<0xB1>(v));   // quad_perm [1,0,3,2]
    v = max_of(v, dpp_move<0x4E>(v));   // quad_perm [2,3,0,1]
    v = max_of(v, dpp_move<0x141>(v));  // row_half_mirror
    v = max_of(v, dpp_move<0x140>(v));  // row_mirror
    if constexpr (TPR == 64)
        v = max_of(max_of(read_lane(v, 0), read_lane(v, 16)),
                   max_of(read_lane(v, 32), read_lane(v, 48)));
    return v;
}

template <int TPR, typename A>
__device__ __forceinline__ A lanes_sum(A v) {
    if constexpr (TPR == 64) return wave_total(v);
    v += dpp_move<0xB1>(v);
    v += dpp_move<0x4E>(v);
    v += dpp_move<0x141>(v);
    v += dpp_move<0x140>(v);
    return v;
}

// Running maximum m and sum s of exp(x - m) over the lanes of a row.
template <int LANES, typename A>
__device__ __forceinline__ void join_lanes(A& m, A& s) {
    // no product fused into the first addition: one lane would add it unrounded, its partner not
#pragma clang fp contract(off)
    const A all = lanes_max<LANES>(m), base = base_of(all);
    s = lanes_sum<LANES>(s * exp_diff(m - base));
    m = all;
}

// The same over the waves of a workgroup that share a row; every wave ends with the row's m and s.
template <int WAVES, typename A>
__device__ __forceinline__ void join_waves(A& m, A& s, A (*part)[2]) {
    join_lanes<64>(m, s);
    if constexpr (WAVES > 1) {
        if (lane_id() == 0) {
            part[wave_id()][0] = m;
            part[wave_id()][1] = s;
        }
        __syncthreads();
        const int l = lane_id();
        m = l < WAVES ? part[l][0] : -A(__builtin_inf());
        s = l < WAVES ? part[l][1] : A(0);
        join_lanes<64>(m, s);
    }
}

// ---- the row's scalars from m and s, by all lanes of one wave (or of a 16-lane row); the lane
// with write set stores them.
template <int LANES, typename T, typename Op>
__device__ __forceinline__ RowState<wide_t<T>> finish_row(const RowArgs<T>& a, const Op& op,
                                                          int64_t n, int64_t act, wide_t<T> xa,
                                                          const RowInputs& in, wide_t<T> m,
                                                          wide_t<T> s, bool write) {
    using A = wide_t<T>;
    RowState<A> st{m, A(1) / s, A(0), A(0)};
    if (act == a.ignore) {
        op.ignored(n, write);
        if (write) a.lp[n] = A(0);
    } else {
        double lp = (double(xa) - double(m)) - log(double(s));
        if (act < 0 || act >= a.cols) lp = nan_value<double>();
        const int l = lane_id() & (LANES - 1);
        const double mine = exp(l == 1 || l == 2 ? op.arg(l, lp, in) : lp);
        const double e[3] = {__shfl(mine, 0, LANES), __shfl(mine, 1, LANES),
                             __shfl(mine, 2, LANES)};
        if (write) a.lp[n] = A(lp);
        st.rest = A(1.0 - e[0]);
        st.slope = A(op.counted(n, lp, in, e, write));
    }
    if (write) a.state[n] = st;
    return st;
}

// The action as a place among the cols elements from j0 on, -1 where it is none of them.
__device__ __forceinline__ int action_place(int64_t act, int64_t j0, int cols) {
    const uint64_t place = uint64_t(act) - uint64_t(j0);
    return place < uint64_t(cols) ? int(place) : -1;
}

template <typename T>
__device__ __forceinline__ wide_t<T> action_logit(const RowArgs<T>& a, const T* x, int64_t act) {
    return act >= 0 && act < a.cols ? wide_t<T>(x[act]) : wide_t<T>(0);
}

// ---- gradient of one logit: c ([j = a] - p_j) as exp(x - m) * k, k = -c / s; the action's own,
// c (1 - p_a), is written over it by the thread that wrote it.  A result of 16 bits takes log2 e as
// one number, off by some 2^-20 of the result; fp32 takes it as the loss does.
template <typename T>
struct RowGrad {
    using A = wide_t<T>;
    A m, k, own;
    __device__ __forceinline__ RowGrad(const RowState<A>& st, A c)
        : m(st.m), k(-c * st.inv_s), own(c * st.rest) {}
    __device__ __forceinline__ T operator()(T x) const {
        if constexpr (sizeof(T) == 2)
            return T(__builtin_amdgcn_exp2f((A(x) - m) * 1.44269504088896340736f) * k);
        else
            return T(exp_diff(A(x) - m) * k);
    }
};

// ---- a row cut where its memory is: the elements before the first whole line of ALIGN bytes, the
// vectors of 16 bytes from there on, the elements after them.  The first and last ones ("loose")
// are taken one per thread.  Rows of odd lengths start anywhere; accesses of 16 bytes work there
// too, but each wave's then end inside two lines: 4096 rows of 50021 bf16, loss and gradient in
// one pass, took 200 us so, 162 us cut at 16 bytes and 155 us at 128.
template <typename T>
struct Cut {
    static constexpr int VEC = wide_vec<T>();
    int head, nvec, loose;

    template <int ALIGN>
    static __device__ __forceinline__ Cut at(const T* p, int cols) {
        Cut c;
        const int off = int(-reinterpret_cast<uintptr_t>(p) & (ALIGN - 1)) / int(sizeof(T));
        c.head = off < cols ? off : cols;
        c.nvec = (cols - c.head) / VEC;
        c.loose = cols - c.nvec * VEC;
        return c;
    }
    __device__ __forceinline__ int place(int i) const {  // of loose element i
        return i < head ? i : i + nvec * VEC;
    }
};

// Lines that a row's accesses are cut at: a workgroup has threads enough for the loose elements of
// a 128-byte line, 16 lanes only for those of 16 bytes.
template <int TPR>
constexpr int kLine = TPR >= 256 ? 128 : 16;

// ---- a row held in registers: NV vectors and one loose element per thread.  Maximum and sum take
// two sweeps over registers instead of a running maximum: one exponential per element.
template <typename T, int TPR, int NV>
struct Held {
    static constexpr int VEC = wide_vec<T>();
    Pack<T, VEC> v[NV];
    T one;
    Cut<T> cut;

    // x: the row; at: where its accesses are cut (the row itself, or the gradient that will be
    // written)
    __device__ __forceinline__ void load(const T* x, const T* at, int cols, int t, bool through) {
        cut = Cut<T>::template at<kLine<TPR>>(at, cols);
        if (t < cut.loose) one = x[cut.place(t)];
        x += cut.head;
        if (through)
            load_vecs<true>(x, t);
        else
            load_vecs<false>(x, t);
    }

    template <bool THROUGH>
    __device__ __forceinline__ void load_vecs(const T* x, int t) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * TPR + t < cut.nvec) v[i] = pload<T, VEC, THROUGH>(x + (i * TPR + t) * VEC);
    }

    // Between two sweeps: the row stays as it was loaded.  Without this the compiler keeps 16-bit
    // elements widened from one sweep to the next, in twice the registers (64 KB of bf16 by 512
    // threads: 103 registers and half the waves).
    __device__ __forceinline__ void keep_packed() {
        if constexpr (sizeof(T) == 2) {
            typedef uint32_t words __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                words w = __builtin_bit_cast(words, v[i]);
                asm volatile("" : "+v"(w));
                using Vector = Pack<T, VEC>;
                v[i] = __builtin_bit_cast(Vector, w);
            }
        }
    }

    __device__ __forceinline__ void reduce(int t, wide_t<T>& m, wide_t<T>& s) {
        using A = wide_t<T>;
        m = -A(__builtin_inf());
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * TPR + t < cut.nvec) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) m = max_of(m, A(v[i].v[e]));
            }
        if (t < cut.loose) m = max_of(m, A(one));
        const A base = base_of(m);
        keep_packed();
        s = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * TPR + t < cut.nvec) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) s += exp_diff(A(v[i].v[e]) - base);
            }
        if (t < cut.loose) s += exp_diff(A(one) - base);
    }

    template <bool THROUGH>
    __device__ __forceinline__ void store_vecs(T* g, int t, const RowGrad<T>& rg) const {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * TPR + t < cut.nvec) {
                Pack<T, VEC> r;
#pragma unroll
                for (int e = 0; e < VEC; ++e) r.v[e] = rg(v[i].v[e]);
                pstore<T, VEC, THROUGH>(g + (i * TPR + t) * VEC, r);
            }
    }

    __device__ __forceinline__ void store_grad(T* g, int t, int act, const RowGrad<T>& rg,
                                               bool through) const {
        if (through)
            store_vecs<true>(g + cut.head, t, rg);
        else
            store_vecs<false>(g + cut.head, t, rg);
        if (t < cut.loose) g[cut.place(t)] = rg(one);
        // the action's own gradient, by the thread that has just written its vector or its loose
        // element: a thread's own stores stay in order
        const int body = cut.nvec * VEC, in = act - cut.head;
        const int owner = in >= 0 && in < body ? (in / VEC) % TPR
                          : in < 0             ? act
                                               : act - body;
        if (act >= 0 && t == owner) g[act] = T(rg.own);
    }

    static __device__ __forceinline__ void store_zero(T* g, int cols, int t, bool through) {
        const Cut<T> c = Cut<T>::template at<kLine<TPR>>(g, cols);
        const Pack<T, VEC> z{};
        T* body = g + c.head;
        if (through) {
            for (int i = t; i < c.nvec; i += TPR) pstore<T, VEC, true>(body + i * VEC, z);
        } else {
            for (int i = t; i < c.nvec; i += TPR) pstore<T, VEC>(body + i * VEC, z);
        }
        if (t < c.loose) g[c.place(t)] = T(0);
    }
};

constexpr int kRowBlock = 256;

// ---- the gradient out of the forward, for an upstream gradient of 1: the row is still in
// registers.  grad: null where the forward only takes the loss.
template <typename T>
struct GradOut {
    T* grad;
    const wide_t<T>* count;  // what a mean divides by, or null
    __device__ __forceinline__ wide_t<T> slope(wide_t<T> s) const {
        if (s == wide_t<T>(0)) return wide_t<T>(0);
        return count ? s * (wide_t<T>(1) / count[0]) : s;
    }
};

template <typename T, int TPR, int NV>
__device__ __forceinline__ void emit_grad(const RowArgs<T>& a, const GradOut<T>& out, int64_t n,
                                          int64_t act, int t, const Held<T, TPR, NV>& row,
                                          const RowState<wide_t<T>>& st) {
    const wide_t<T> c = out.slope(st.slope);
    T* g = out.grad + n * a.cols;
    if (c == wide_t<T>(0))
        row.store_zero(g, int(a.cols), t, a.through_store);
    else
        row.store_grad(g, t, action_place(act, 0, int(a.cols)), RowGrad<T>(st, c), a.through_store);
}

// ---- short rows: TPR lanes (16 or 64) of a wave per row, several rows per workgroup, no LDS.  A
// launch and the chain action -> logits -> fp64 scalars bound it: 128 x 10 or 1024 x 200 fp32 take
// 3.4 us.
template <typename T, int TPR, int NV, typename Op, bool GRAD>
__global__ __launch_bounds__(kRowBlock) void k_rows_short(RowArgs<T> a, Op op, GradOut<T> out) {
    using A = wide_t<T>;
    const int64_t n = group_index() * (kRowBlock / TPR) + threadIdx.x / TPR;
    if (n >= a.rows) return;
    const int t = threadIdx.x % TPR;
    const int64_t act = a.actions[n];
    const T* x = a.x + n * a.stride;
    const RowInputs in = op.load(n);
    const A xa = action_logit(a, x, act);
    Held<T, TPR, NV> row;
    row.load(x, GRAD ? out.grad + n * a.cols : x, int(a.cols), t, a.through_load);
    A m, s;
    row.reduce(t, m, s);
    join_lanes<TPR>(m, s);
    const RowState<A> st = finish_row<TPR>(a, op, n, act, xa, in, m, s, t == 0);
    if constexpr (GRAD) emit_grad<T, TPR, NV>(a, out, n, act, t, row, st);
}

// ---- a row per workgroup, held in its registers between the loss and the gradient.  Bound by
// memory: 8192 x 32768 bf16, a quarter of the rows ignored (403 MB read, 537 written), 155 us = 6.0
// TB/s; 2047 x 32003 fp32, a tenth ignored (236 MB read, 262 written), 83 us.  Eight waves per SIMD
// (64 registers, four of them spilled round the fp64 scalars) let two workgroups or more of a CU
// take turns at loading and storing: the step on 8192 x 32768 took 247 us at four waves, 236 at
// eight, before the choices of cut and cache below and above.
template <typename T, int TPR, int NV, typename Op>
__global__ __launch_bounds__(TPR, 8) void k_rows_held(RowArgs<T> a, Op op, GradOut<T> out) {
    using A = wide_t<T>;
    __shared__ A part[TPR / 64][2];
    __shared__ RowState<A> shared;
    const int64_t n = group_index();
    if (n >= a.rows) return;
    const int t = threadIdx.x;
    const int64_t act = a.actions[n];
    Held<T, TPR, NV> row;
    RowState<A> st{A(0), A(1), A(0), A(0)};
    if (act == a.ignore) {
        if (wave_id() == 0) finish_row<64>(a, op, n, act, A(0), RowInputs{}, A(0), A(1), t == 0);
    } else {
        const T* x = a.x + n * a.stride;
        const RowInputs in = op.load(n);
        const A xa = action_logit(a, x, act);
        row.load(x, out.grad + n * a.cols, int(a.cols), t, a.through_load);
        A m, s;
        row.reduce(t, m, s);
        row.keep_packed();
        join_waves<TPR / 64>(m, s, part);
        if (wave_id() == 0) {
            st = finish_row<64>(a, op, n, act, xa, in, m, s, t == 0);
            if (t == 0) shared = st;
        }
        __syncthreads();
        st = shared;
    }
    emit_grad<T, TPR, NV>(a, out, n, act, t, row, st);
}

// ---- a row per workgroup, read once with a running maximum and sum; ignored rows are not read.
// One exponential per element and one per 32 for the running maximum.  Bound by memory: 8192 x
// 32000 bf16 81 us = 6.4 TB/s.
constexpr int kStreamUnroll = 4;  // vectors in flight per thread

// Vectors lo..hi-1 of a row, and its loose elements with `loose`.
template <typename T, bool THROUGH = false>
__device__ __forceinline__ void stream_part(const T* x, const Cut<T>& cut, int lo, int hi,
                                            bool loose, wide_t<T>& m, wide_t<T>& s) {
    using A = wide_t<T>;
    constexpr int VEC = wide_vec<T>(), U = kStreamUnroll;
    const T* body = x + cut.head;
    m = -A(__builtin_inf());
    s = 0;
    for (int i = lo + int(threadIdx.x); i < hi; i += U * kRowBlock) {
        Pack<T, VEC> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * kRowBlock < hi)
                v[u] = pload<T, VEC, THROUGH>(body + (i + u * kRowBlock) * VEC);
        A top = m;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * kRowBlock < hi) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) top = max_of(top, A(v[u].v[e]));
            }
        const A base = base_of(top);
        A add = 0;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * kRowBlock < hi) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) add += exp_diff(A(v[u].v[e]) - base);
            }
        s = s * exp_diff(m - base) + add;
        m = top;
    }
    if (loose && int(threadIdx.x) < cut.loose) {
        const A v = A(x[cut.place(threadIdx.x)]), top = max_of(m, v), base = base_of(top);
        s = s * exp_diff(m - base) + exp_diff(v - base);
        m = top;
    }
}

template <typename T, typename Op>
__global__ __launch_bounds__(kRowBlock) void k_rows_stream(RowArgs<T> a, Op op) {
    using A = wide_t<T>;
    __shared__ A part[kRowBlock / 64][2];
    const int64_t n = group_index();
    if (n >= a.rows) return;
    const int64_t act = a.actions[n];
    A m = 0, s = 1, xa = 0;
    RowInputs in{};
    if (act != a.ignore) {
        const T* x = a.x + n * a.stride;
        in = op.load(n);
        xa = action_logit(a, x, act);
        const Cut<T> cut = Cut<T>::template at<kLine<kRowBlock>>(x, int(a.cols));
        if (a.through_load)
            stream_part<T, true>(x, cut, 0, cut.nvec, true, m, s);
        else
            stream_part<T>(x, cut, 0, cut.nvec, true, m, s);
        join_waves<kRowBlock / 64>(m, s, part);
    }
    if (wave_id() == 0) finish_row<64>(a, op, n, act, xa, in, m, s, lane_id() == 0);
}

// ---- few long rows: (row, part) workgroups, the parts joined by one wave per row.  16 rows of
// 131072 fp16: 3.6 + 3.0 us, where one workgroup per row took 108 us.
template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_rows_split(RowArgs<T> a, int parts, int per,
                                                          wide_t<T>* __restrict__ ws) {
    using A = wide_t<T>;
    __shared__ A part[kRowBlock / 64][2];
    const int64_t n = blockIdx.y;
    const int p = blockIdx.x;
    if (a.actions[n] == a.ignore) return;
    const T* x = a.x + n * a.stride;
    const Cut<T> cut = Cut<T>::template at<kLine<kRowBlock>>(x, int(a.cols));
    A m, s;
    stream_part<T>(x, cut, p * per, std::min(cut.nvec, (p + 1) * per), p == parts - 1, m, s);
    join_waves<kRowBlock / 64>(m, s, part);
    if (threadIdx.x == 0) {
        ws[(n * parts + p) * 2] = m;
        ws[(n * parts + p) * 2 + 1] = s;
    }
}

template <typename T, typename Op>
__global__ __launch_bounds__(kRowBlock) void k_rows_joined(RowArgs<T> a, Op op, int parts,
                                                           const wide_t<T>* __restrict__ ws) {
    using A = wide_t<T>;
    const int64_t n = int64_t(blockIdx.x) * (kRowBlock / 64) + wave_id();
    if (n >= a.rows) return;
    const int64_t act = a.actions[n];
    A m = -A(__builtin_inf()), s = 0, xa = 0;
    RowInputs in{};
    if (act != a.ignore) {
        in = op.load(n);
        xa = action_logit(a, a.x + n * a.stride, act);
        if (lane_id() < parts) {
            m = ws[(n * parts + lane_id()) * 2];
            s = ws[(n * parts + lane_id()) * 2 + 1];
        }
        join_lanes<64>(m, s);
    }
    finish_row<64>(a, op, n, act, xa, in, m, s, lane_id() == 0);
}

// ---- the gradient in a pass of its own.  Rows whose slope is 0 are written without being read:
// ignored, clipped, or of no sequence.  Bound by memory: 8192 x 32000 bf16 165 us = 6.3 TB/s.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(kRowBlock) void k_grad_short(RowArgs<T> a, Upstream<wide_t<T>> up,
                                                          T* __restrict__ grad) {
    using A = wide_t<T>;
    const int64_t n = group_index() * (kRowBlock / TPR) + threadIdx.x / TPR;
    if (n >= a.rows) return;
    const int t = threadIdx.x % TPR;
    const RowState<A> st = a.state[n];
    const int64_t act = a.actions[n];
    const A c = up(n, st.slope);
    T* g = grad + n * a.cols;
    Held<T, TPR, NV> row;
    if (c == A(0)) {
        row.store_zero(g, int(a.cols), t, a.through_store);
        return;
    }
    row.load(a.x + n * a.stride, g, int(a.cols), t, a.through_load);
    row.store_grad(g, t, action_place(act, 0, int(a.cols)), RowGrad<T>(st, c), a.through_store);
}

constexpr int kGradVecs = 4;  // vectors per thread

template <typename T>
__device__ __forceinline__ void grad_chunk(const RowArgs<T>& a, const Upstream<wide_t<T>>& up,
                                           T* grad, int64_t n, int64_t chunk) {
    using A = wide_t<T>;
    constexpr int CHUNK = kRowBlock * kGradVecs * wide_vec<T>();
    const int64_t j0 = chunk * CHUNK;
    const int cols = int(std::min<int64_t>(CHUNK, a.cols - j0));
    const RowState<A> st = a.state[n];
    const int64_t act = a.actions[n];
    const A c = up(n, st.slope);
    T* g = grad + n * a.cols + j0;
    Held<T, kRowBlock, kGradVecs> row;
    if (c == A(0)) {
        row.store_zero(g, cols, threadIdx.x, a.through_store);
        return;
    }
    row.load(a.x + n * a.stride + j0, g, cols, threadIdx.x, a.through_load);
    row.store_grad(g, threadIdx.x, action_place(act, j0, cols), RowGrad<T>(st, c), a.through_store);
}

template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_grad_long(RowArgs<T> a, Upstream<wide_t<T>> up,
                                                         T* __restrict__ grad, uint32_t chunks) {
    const uint32_t i = uint32_t(group_index()), n = i / chunks;
    if (n < a.rows) grad_chunk<T>(a, up, grad, n, i % chunks);
}

// A gradient that the forward left for an upstream gradient of 1: nothing to do where it is 1,
// else formed again, but for the rows where it is 0 anyway.  Few workgroups, which walk the chunks
// (4096: nothing to do costs what it does with 1024, 4.8 us between two kernels; 8192 x 32768 bf16,
// a quarter ignored, loss and an upstream gradient of 0.5 take 302 us, 313 with 1024).
constexpr int64_t kAgainGroups = 4096;

template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_grad_again(RowArgs<T> a, Upstream<wide_t<T>> up,
                                                          T* __restrict__ grad, uint32_t chunks) {
    if (up.scalar[0] == wide_t<T>(1)) return;
    for (int64_t i = blockIdx.x; i < a.rows * chunks; i += gridDim.x) {
        const int64_t n = i / chunks;
        if (a.state[n].slope != wide_t<T>(0))  // (else it is 0 already)
            grad_chunk<T>(a, up, grad, n, i % chunks);
    }
}

// ---- sums in a fixed order by one workgroup, in fp64
constexpr int kSumThreads = 1024;

// Over the workgroup, by lanes and then waves; the result in every thread of wave 0.
__device__ __forceinline__ double group_sum(double v, double* red) {
    v = wave_total(v);
    if (lane_id() == 0) red[wave_id()] = v;
    __syncthreads();
    const int waves = int(blockDim.x) >> 6;
    return wave_total(lane_id() < waves ? red[lane_id()] : 0.0);
}

// Where there are more rows than one workgroup adds in a few microseconds, workgroups first add
// kSumRows each into partial sums, which the last one adds in order: a policy step on 10^6 rows of
// 10 classes takes 213 us instead of 346, on 10^5 rows 39 instead of 47.
constexpr int64_t kSumRows = 16384;

struct RowSums {
    double term, count;
};

template <typename A>
__device__ __forceinline__ RowSums sum_rows(const A* terms, const int64_t* actions, int64_t from,
                                            int64_t to, int64_t ignore,
                                            double (*red)[kSumThreads / 64]) {
    double t = 0;
    int c = 0;
#pragma unroll 8
    for (int64_t n = from + threadIdx.x; n < to; n += kSumThreads) {
        if (terms) t += double(terms[n]);
        c += actions[n] != ignore;
    }
    RowSums r{0.0, group_sum(double(c), red[0])};
    if (terms) r.term = group_sum(t, red[1]);
    return r;
}

__device__ __forceinline__ RowSums sum_parts(const RowSums* parts, int64_t n,
                                             double (*red)[kSumThreads / 64]) {
    double t = 0, c = 0;
    for (int64_t i = threadIdx.x; i < n; i += kSumThreads) {
        t += parts[i].term;
        c += parts[i].count;
    }
    c = group_sum(c, red[0]);
    t = group_sum(t, red[1]);
    return {t, c};
}

template <typename A>
__global__ __launch_bounds__(kSumThreads) void k_sum_parts(const A* __restrict__ terms,
                                                           const int64_t* __restrict__ actions,
                                                           int64_t rows, int64_t ignore,
                                                           RowSums* __restrict__ parts) {
    __shared__ double red[2][kSumThreads / 64];
    const int64_t from = int64_t(blockIdx.x) * kSumRows;
    const RowSums r = sum_rows(terms, actions, from, std::min(rows, from + kSumRows), ignore, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = r;
}

// The number of rows that count, and, with terms, their sum or mean as the loss; from the rows or
// from nparts partial sums.
template <typename A>
__global__ __launch_bounds__(kSumThreads) void k_sum(const A* __restrict__ terms,
                                                     const int64_t* __restrict__ actions,
                                                     int64_t rows, int64_t ignore,
                                                     const RowSums* __restrict__ parts,
                                                     int64_t nparts, int mean, A* __restrict__ loss,
                                                     A* __restrict__ count) {
    __shared__ double red[2][kSumThreads / 64];
    const RowSums r = nparts ? sum_parts(parts, nparts, red)
                             : sum_rows(terms, actions, 0, rows, ignore, red);
    if (threadIdx.x != 0) return;
    // no counted row: 0 / 0 = NaN, the mean of nothing
    if (terms) loss[0] = A(mean ? r.term / r.count : r.term);
    count[0] = A(r.count);
}

template <typename A>
struct PairArgs {
    const double* gaps;
    const int64_t* offsets;
    int64_t rows, pairs;
    double beta, smooth;
    RowState<A>* state;
    int32_t* row_seq;
    A* seq_slope;
    A* margins;
    A* terms;
};

// Pair i by LANES threads: a DPP row (16), a wave (64) or a workgroup (then all of its threads come
// here): the sums over both sequences, the margin h, the loss term
//   -(1 - e) log sigma(h) - e log sigma(-h)
// and its slope by the chosen sequence's sum; the rejected one's is the negative.
template <int LANES, typename A>
__device__ __forceinline__ double pair_term(const PairArgs<A>& a, int64_t i, double* red) {
    const int t0 = int(threadIdx.x) % LANES;
    double d[2];
    bool bad = false;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const int64_t q = i + side * a.pairs;
        int64_t b = a.offsets[q], e = a.offsets[q + 1];
        bad |= b < 0 || e < b || e > a.rows;
        // Rows inside of a decrease may lie in several sequences, whose stores of row_seq then race:
        // their gradient is NaN whichever comes last.
        for (int64_t n = std::max<int64_t>(e, 0) + t0; n < std::min(b, a.rows); n += LANES)
            if (a.state[n].slope != A(0)) a.state[n].slope = nan_value<A>();
        b = std::min(std::max<int64_t>(b, 0), a.rows);
        e = std::min(std::max(e, b), a.rows);
        double t = 0;
        // eight loads at a time, in row order
        for (int64_t n = b + t0; n < e; n += 8 * LANES) {
            double v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = n + u * LANES < e ? a.gaps[n + u * LANES] : 0.0;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                t += v[u];
                if (n + u * LANES < e) a.row_seq[n + u * LANES] = int32_t(q);
            }
        }
        if constexpr (LANES > 64)
            d[side] = group_sum(t, red + side * (LANES / 64));
        else
            d[side] = lanes_sum<LANES>(t);
    }
    double h = a.beta * (d[0] - d[1]);
    if (bad) h = nan_value<double>();
    // with u = exp(-|h|): log sigma(h) = min(h, 0) - log(1 + u), sigma(h) = 1 / (1 + u) or
    // u / (1 + u)
    const double u = exp(-fabs(h)), tail = log1p(u), inv = 1.0 / (1.0 + u);
    const double away = tail - (h < 0 ? h : 0.0), near = tail + (h > 0 ? h : 0.0);
    const double yes = h >= 0 ? inv : u * inv, no = h >= 0 ? u * inv : inv;  // sigma(h), sigma(-h)
    const double slope = a.beta * (a.smooth * yes - (1 - a.smooth) * no);
    const double term = (1 - a.smooth) * away + a.smooth * near;
    if (t0 == 0) {
        a.margins[i] = A(h);
        a.terms[i] = A(term);
        a.seq_slope[i] = A(slope);
        a.seq_slope[i + a.pairs] = A(-slope);
    }
    return double(A(term));
}

template <typename A>
__global__ __launch_bounds__(kRowBlock) void k_pref_pairs(PairArgs<A> a) {
    const int64_t i = group_index() * (kRowBlock / 64) + wave_id();
    if (i < a.pairs) pair_term<64>(a, i, nullptr);
}

template <typename A>
__global__ __launch_bounds__(kSumThreads) void k_pref_long(PairArgs<A> a) {
    __shared__ double red[2 * kSumThreads / 64];
    pair_term<kSumThreads>(a, blockIdx.x, red);
}

template <typename A>
__global__ __launch_bounds__(kSumThreads) void k_pref_sum(const A* __restrict__ terms,
                                                          int64_t pairs, int mean,
                                                          A* __restrict__ loss,
                                                          A* __restrict__ count) {
    __shared__ double red[kSumThreads / 64];
    double t = 0;
    for (int64_t i = threadIdx.x; i < pairs; i += blockDim.x) t += double(terms[i]);
    t = group_sum(t, red);
    if (threadIdx.x == 0) {
        loss[0] = A(mean ? t / double(pairs) : t);
        count[0] = A(pairs);
    }
}

// Both in one launch, 16 lanes per pair: for batches of at most 64 pairs of about 128 rows, each
// pair's loads then in flight together.
template <typename A>
__global__ __launch_bounds__(kSumThreads) void k_pref_small(PairArgs<A> a, int mean,
                                                            A* __restrict__ loss,
                                                            A* __restrict__ count) {
    __shared__ double red[kSumThreads / 64];
    double t = 0;
    for (int64_t i = threadIdx.x / 16; i < a.pairs; i += kSumThreads / 16) {
        const double term = pair_term<16>(a, i, nullptr);
        t += threadIdx.x % 16 == 0 ? term : 0.0;
    }
    if (!loss) return;
    t = group_sum(t, red);
    if (threadIdx.x == 0) {
        loss[0] = A(mean ? t / double(a.pairs) : t);
        count[0] = A(a.pairs);
    }
}

int check_logits(const void* logits, int64_t row_stride, int64_t rows, int64_t cols,
                 const int64_t* actions, const void* state) {
    CL_ARG(rows >= 0 && rows < (int64_t(1) << 31), "rows must be in [0, 2^31)");
    CL_ARG(cols >= 1 && cols < (int64_t(1) << 31), "cols must be in [1, 2^31), got %lld",
           (long long)cols);
    CL_ARG(row_stride >= 0, "negative strides are not supported");
    CL_ARG(rows == 0 || (logits && actions && state), "null pointer argument");
    return CL_OK;
}

template <typename T>
RowArgs<T> row_args(const void* logits, int64_t row_stride, int64_t rows, int64_t cols,
                    const int64_t* actions, int64_t ignore, void* lp, const void* state) {
    RowArgs<T> a;
    a.x = static_cast<const T*>(logits);
    a.stride = row_stride;
    a.rows = rows;
    a.cols = cols;
    a.actions = actions;
    a.ignore = ignore;
    a.lp = static_cast<wide_t<T>*>(lp);
    a.state = const_cast<RowState<wide_t<T>>*>(static_cast<const RowState<wide_t<T>>*>(state));
    const int64_t bytes = rows * cols * int64_t(sizeof(T));
    a.through_store = bytes >= (int64_t(96) << 20);
    a.through_load = bytes >= (int64_t(256) << 20);
    return a;
}

// Rows up to 256 bytes stay in registers of 16 lanes, up to 4 KB of a wave; longer ones take a
// workgroup, or several where the rows alone would not fill the card.  Chosen log-probabilities and
// gradient: 20000 x 64 fp32 16 us on 16 lanes, 22 on 64; 12000 x 1000 fp32 32 us on a wave, 42 on a
// workgroup; 16 x 131072 see k_rows_split.
constexpr int64_t kPrefSmallPairs = 64;
constexpr int64_t kPrefSmallRows = 128, kPrefLongRows = 2048;  // of a pair, on average
constexpr int64_t kSplitBlocks = 1024;  // workgroups wanted
constexpr int kMaxParts = 64;           // joined by the lanes of one wave

template <typename T>
int row_parts(int64_t rows, int64_t cols) {
    const int64_t per_block = int64_t(kRowBlock) * kStreamUnroll;  // vectors of one sweep
    const int64_t nvec = cols / wide_vec<T>();
    if (rows <= 0 || rows > kSplitBlocks / 2 || nvec < 2 * per_block) return 1;
    return int(std::min<int64_t>(std::min<int64_t>(nvec / per_block, kMaxParts),
                                 ceil_div(kSplitBlocks, rows)));
}

// (few rows are split, many are summed in parts: never both)
template <typename T>
int64_t rows_workspace(int64_t rows, int64_t cols) {
    const int parts = row_parts<T>(rows, cols);
    if (parts > 1) return rows * parts * 2 * int64_t(sizeof(wide_t<T>));
    return rows > kSumRows ? ceil_div(rows, kSumRows) * int64_t(sizeof(RowSums)) : 0;
}

// The loss and the number of counted rows; without terms that number alone.
template <typename A>
int launch_sum(const A* terms, const int64_t* actions, int64_t rows, int64_t ignore, bool mean,
               A* loss, A* count, void* workspace, int64_t workspace_bytes, hipStream_t s) {
    const int64_t nparts = rows > kSumRows ? ceil_div(rows, kSumRows) : 0;
    auto* parts = static_cast<RowSums*>(workspace);
    if (nparts) {
        CL_ARG(workspace && workspace_bytes >= nparts * int64_t(sizeof(RowSums)),
               "workspace of %lld bytes needed (cl_token_loss_workspace)",
               (long long)(nparts * int64_t(sizeof(RowSums))));
        k_sum_parts<A><<<unsigned(nparts), kSumThreads, 0, s>>>(terms, actions, rows, ignore,
                                                               parts);
        if (int rc = check_launch("sums in parts")) return rc;
    }
    k_sum<A><<<1, kSumThreads, 0, s>>>(terms, actions, rows, ignore, parts, nparts, mean, loss,
                                       count);
    return check_launch("sum");
}

template <typename T, int TPR, int NV, bool GRAD, typename Op>
void launch_rows_short(const RowArgs<T>& a, const Op& op, const GradOut<T>& out, hipStream_t s) {
    k_rows_short<T, TPR, NV, Op, GRAD>
        <<<wide_grid(ceil_div(a.rows, kRowBlock / TPR)), kRowBlock, 0, s>>>(a, op, out);
}

template <bool GRAD, typename T, typename Op>
bool launch_short(const RowArgs<T>& a, const Op& op, const GradOut<T>& out, hipStream_t s) {
    const int64_t bytes = a.cols * int64_t(sizeof(T));
    if (bytes <= 256)
        launch_rows_short<T, 16, 1, GRAD>(a, op, out, s);
    else if (bytes <= 1024)
        launch_rows_short<T, 64, 1, GRAD>(a, op, out, s);
    else if (bytes <= 4096)
        launch_rows_short<T, 64, 4, GRAD>(a, op, out, s);
    else
        return false;
    return true;
}

// The largest row, in bytes, that one workgroup holds, and the fewest logits, in bytes, for which
// the loss and its gradient are taken in one pass (67 MB of fp32 36 us, 43 in two; 34 MB of bf16 31
// and 30, the one pass having two launches more).  It is taken for an upstream gradient of 1: 8192
// x 32768 bf16 178 us instead of 218, for another one 302.  fp16 keeps two: a gradient formed before the
// upstream one is known may vanish in half's range, which a scaled loss is meant to prevent.  fp64
// rows are not worth their registers.
constexpr int64_t kHeldRow = 131072;
constexpr int64_t kHeldLogits = int64_t(48) << 20;

template <typename T>
constexpr bool kPrefillType = std::is_same_v<T, float> || std::is_same_v<T, bf16_t>;

template <typename T>
bool policy_prefills(int64_t rows, int64_t cols) {
    const int64_t bytes = cols * int64_t(sizeof(T));
    return kPrefillType<T> && bytes <= kHeldRow && rows * bytes >= kHeldLogits;
}

// The rows' terms and, for an upstream gradient of 1, the logits' gradient.
template <typename T, typename Op>
int launch_rows_grad(const RowArgs<T>& a, const Op& op, const GradOut<T>& out, hipStream_t s) {
    if constexpr (kPrefillType<T>) {
        const int64_t bytes = a.cols * int64_t(sizeof(T));
        const dim3 grid = wide_grid(a.rows);
        if (a.rows == 0) return CL_OK;
        if (launch_short<true>(a, op, out, s)) {
        } else if (bytes <= 16384) {
            k_rows_held<T, 256, 4, Op><<<grid, 256, 0, s>>>(a, op, out);
        } else if (bytes <= 32768) {
            k_rows_held<T, 512, 4, Op><<<grid, 512, 0, s>>>(a, op, out);
        } else if (bytes <= 65536) {
            k_rows_held<T, 512, 8, Op><<<grid, 512, 0, s>>>(a, op, out);
        } else {
            CL_ARG(bytes <= kHeldRow, "rows of %lld bytes are not held", (long long)bytes);
            k_rows_held<T, 1024, 8, Op><<<grid, 1024, 0, s>>>(a, op, out);
        }
        return check_launch("rows and gradient");
    } else {
        CL_ARG(false, "the gradient of this type is not taken by the forward");
    }
}

template <typename T, typename Op>
int launch_rows(const RowArgs<T>& a, const Op& op, void* workspace, int64_t workspace_bytes,
                hipStream_t s) {
    if (a.rows == 0) return CL_OK;
    const int parts = row_parts<T>(a.rows, a.cols);
    if (launch_short<false>(a, op, GradOut<T>{}, s)) {
    } else if (parts > 1) {
        CL_ARG(workspace && workspace_bytes >= rows_workspace<T>(a.rows, a.cols),
               "workspace of %lld bytes needed (cl_token_loss_workspace)",
               (long long)rows_workspace<T>(a.rows, a.cols));
        auto* ws = static_cast<wide_t<T>*>(workspace);
        const int per = int(ceil_div(a.cols / wide_vec<T>(), parts));
        k_rows_split<T><<<dim3(unsigned(parts), unsigned(a.rows)), kRowBlock, 0, s>>>(a, parts,
                                                                                    per, ws);
        if (int rc = check_launch("row parts")) return rc;
        k_rows_joined<T, Op><<<unsigned(ceil_div(a.rows, kRowBlock / 64)), kRowBlock, 0, s>>>(
            a, op, parts, ws);
    } else {
        k_rows_stream<T, Op><<<wide_grid(a.rows), kRowBlock, 0, s>>>(a, op);
    }
    return check_launch("rows");
}

template <typename T>
int launch_logit_grad(const RowArgs<T>& a, const Upstream<wide_t<T>>& up, void* grad,
                      hipStream_t s, bool prefilled = false) {
    if (a.rows == 0) return CL_OK;
    const int64_t bytes = a.cols * int64_t(sizeof(T));
    T* g = static_cast<T*>(grad);
    if (prefilled) {
        if constexpr (kPrefillType<T>) {
            const int64_t chunks = ceil_div(a.cols, kRowBlock * kGradVecs * wide_vec<T>());
            const int64_t grid = std::min<int64_t>(a.rows * chunks, kAgainGroups);
            k_grad_again<T><<<unsigned(grid), kRowBlock, 0, s>>>(a, up, g, uint32_t(chunks));
        } else {
            CL_ARG(false, "the gradient of this type is not taken by the forward");
        }
    } else if (bytes <= 256) {
        k_grad_short<T, 16, 1><<<wide_grid(ceil_div(a.rows, kRowBlock / 16)), kRowBlock, 0, s>>>(
            a, up, g);
    } else if (bytes <= 1024) {
        k_grad_short<T, 64, 1><<<wide_grid(ceil_div(a.rows, kRowBlock / 64)), kRowBlock, 0, s>>>(
            a, up, g);
    } else if (bytes <= 4096) {
        k_grad_short<T, 64, 4><<<wide_grid(ceil_div(a.rows, kRowBlock / 64)), kRowBlock, 0, s>>>(
            a, up, g);
    } else {
        const int64_t chunks = ceil_div(a.cols, kRowBlock * kGradVecs * wide_vec<T>());
        CL_ARG(a.rows * chunks < (int64_t(1) << 31), "too many logits for one call");
        k_grad_long<T><<<wide_grid(a.rows * chunks), kRowBlock, 0, s>>>(a, up, g,
                                                                      uint32_t(chunks));
    }
    return check_launch("logit gradient");
}

}  // namespace
}  // namespace cl

using namespace cl;

extern "C" int cl_token_loss_workspace(int dtype, int64_t rows, int64_t cols, int64_t* bytes) {
    clear_error();
    CL_ARG(bytes, "null pointer argument");
    CL_ARG(rows >= 0 && rows < (int64_t(1) << 31) && cols >= 1 && cols < (int64_t(1) << 31),
           "bad shape");
    CL_STORAGE_SWITCH(dtype, { *bytes = rows_workspace<scalar_t>(rows, cols); });
    return CL_OK;
}

extern "C" int cl_selected_log_prob_forward(int dtype, const void* logits, int64_t row_stride,
                                            int64_t rows, int64_t cols, const int64_t* actions,
                                            int64_t ignore_index, void* log_probs, void* row_state,
                                            void* workspace, int64_t workspace_bytes,
                                            void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || log_probs, "null pointer argument");
    if (rows == 0) return CL_OK;
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        return launch_rows(row_args<T>(logits, row_stride, rows, cols, actions, ignore_index,
                                       log_probs, row_state),
                           LogProbOp<wide_t<T>>{}, workspace, workspace_bytes, as_stream(stream));
    });
}

extern "C" int cl_selected_log_prob_backward(int dtype, const void* logits, int64_t row_stride,
                                             int64_t rows, int64_t cols, const int64_t* actions,
                                             const void* row_state, const void* grad_log_probs,
                                             void* grad_logits, void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || (grad_log_probs && grad_logits), "null pointer argument");
    if (rows == 0) return CL_OK;
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        using A = wide_t<T>;
        Upstream<A> up{};
        up.rows = static_cast<const A*>(grad_log_probs);
        return launch_logit_grad(row_args<T>(logits, row_stride, rows, cols, actions, 0, nullptr,
                                      row_state),
                          up, grad_logits, as_stream(stream));
    });
}

extern "C" int cl_policy_loss_prefills(int dtype, int64_t rows, int64_t cols, int* yes) {
    clear_error();
    CL_ARG(yes, "null pointer argument");
    CL_ARG(rows >= 0 && cols >= 1, "bad shape");
    CL_STORAGE_SWITCH(dtype, { *yes = policy_prefills<scalar_t>(rows, cols) ? 1 : 0; });
    return CL_OK;
}

extern "C" int cl_policy_loss_forward(int dtype, const void* logits, int64_t row_stride,
                                      int64_t rows, int64_t cols, const int64_t* actions,
                                      int64_t ignore_index, const void* old_log_probs,
                                      const void* advantages, const void* ref_log_probs,
                                      double clip_low, double clip_high, double kl_coef,
                                      int reduction, void* log_probs, void* row_state,
                                      void* terms, void* loss, void* count, void* grad_logits,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || (old_log_probs && advantages && log_probs && terms),
           "null pointer argument");
    CL_ARG(!grad_logits || reduction == CL_REDUCE_SUM || reduction == CL_REDUCE_MEAN,
           "the forward takes the gradient of a scalar loss only");
    CL_ARG(clip_low >= 0 && clip_high >= 0, "the clipped range must contain 1");
    CL_ARG(kl_coef == 0 || ref_log_probs, "a KL term needs the reference's log-probabilities");
    CL_ARG(reduction >= CL_REDUCE_NONE && reduction <= CL_REDUCE_MEAN, "unknown reduction %d",
           reduction);
    CL_ARG(reduction == CL_REDUCE_NONE || (loss && count), "null pointer argument");
    hipStream_t s = as_stream(stream);
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        using A = wide_t<T>;
        PolicyOp<A> op;
        op.old_lp = static_cast<const A*>(old_log_probs);
        op.adv = static_cast<const A*>(advantages);
        op.ref = kl_coef != 0 ? static_cast<const A*>(ref_log_probs) : nullptr;
        op.low = 1.0 - clip_low;
        op.high = 1.0 + clip_high;
        op.kl = kl_coef;
        op.terms = static_cast<A*>(terms);
        const RowArgs<T> a = row_args<T>(logits, row_stride, rows, cols, actions, ignore_index,
                                         log_probs, row_state);
        if (grad_logits) {
            const bool mean = reduction == CL_REDUCE_MEAN;
            if (mean)
                if (int rc = launch_sum<A>(nullptr, actions, rows, ignore_index, true, nullptr,
                                           static_cast<A*>(count), workspace, workspace_bytes, s))
                    return rc;
            const GradOut<T> out{static_cast<T*>(grad_logits),
                                 mean ? static_cast<const A*>(count) : nullptr};
            if (int rc = launch_rows_grad(a, op, out, s)) return rc;
        } else if (int rc = launch_rows(a, op, workspace, workspace_bytes, s)) {
            return rc;
        }
        if (reduction == CL_REDUCE_NONE) return CL_OK;
        return launch_sum<A>(op.terms, actions, rows, ignore_index, reduction == CL_REDUCE_MEAN,
                             static_cast<A*>(loss), static_cast<A*>(count), workspace,
                             workspace_bytes, s);
    });
}

extern "C" int cl_policy_loss_backward(int dtype, const void* logits, int64_t row_stride,
                                       int64_t rows, int64_t cols, const int64_t* actions,
                                       const void* row_state, int reduction, const void* grad_loss,
                                       const void* count, int prefilled, void* grad_logits,
                                       void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || (grad_loss && grad_logits), "null pointer argument");
    CL_ARG(reduction >= CL_REDUCE_NONE && reduction <= CL_REDUCE_MEAN, "unknown reduction %d",
           reduction);
    CL_ARG(reduction != CL_REDUCE_MEAN || count, "null pointer argument");
    CL_ARG(!prefilled || reduction != CL_REDUCE_NONE, "only a scalar loss's gradient is prefilled");
    if (rows == 0) return CL_OK;
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        using A = wide_t<T>;
        Upstream<A> up{};
        if (reduction == CL_REDUCE_NONE)
            up.rows = static_cast<const A*>(grad_loss);
        else
            up.scalar = static_cast<const A*>(grad_loss);
        if (reduction == CL_REDUCE_MEAN) up.count = static_cast<const A*>(count);
        return launch_logit_grad(row_args<T>(logits, row_stride, rows, cols, actions, 0, nullptr,
                                      row_state),
                          up, grad_logits, as_stream(stream), prefilled != 0);
    });
}

extern "C" int cl_preference_loss_forward(int dtype, const void* logits, int64_t row_stride,
                                          int64_t rows, int64_t cols, const int64_t* actions,
                                          int64_t ignore_index, const void* ref_log_probs,
                                          const int64_t* offsets, int64_t pairs, double beta,
                                          double label_smoothing, int reduction, void* log_probs,
                                          void* row_state, double* gaps, int32_t* row_seq,
                                          void* seq_slope, void* margins, void* terms, void* loss,
                                          void* count, void* workspace, int64_t workspace_bytes,
                                          void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || (log_probs && gaps && row_seq), "null pointer argument");
    CL_ARG(pairs >= 0 && pairs < (int64_t(1) << 30), "pairs must be in [0, 2^30)");
    CL_ARG(pairs == 0 || (offsets && seq_slope && margins && terms), "null pointer argument");
    CL_ARG(label_smoothing >= 0 && label_smoothing <= 1, "label_smoothing must be in [0, 1]");
    CL_ARG(reduction >= CL_REDUCE_NONE && reduction <= CL_REDUCE_MEAN, "unknown reduction %d",
           reduction);
    CL_ARG(reduction == CL_REDUCE_NONE || (loss && count), "null pointer argument");
    hipStream_t s = as_stream(stream);
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        using A = wide_t<T>;
        PreferenceOp<A> op{static_cast<const A*>(ref_log_probs), gaps, row_seq};
        if (int rc = launch_rows(row_args<T>(logits, row_stride, rows, cols, actions,
                                             ignore_index, log_probs, row_state),
                                 op, workspace, workspace_bytes, s))
            return rc;
        const PairArgs<A> pa{gaps, offsets, rows, pairs, beta, label_smoothing,
                             static_cast<RowState<A>*>(row_state), row_seq,
                             static_cast<A*>(seq_slope), static_cast<A*>(margins),
                             static_cast<A*>(terms)};
        const int mean = reduction == CL_REDUCE_MEAN;
        A* out = reduction != CL_REDUCE_NONE ? static_cast<A*>(loss) : nullptr;
        // Steps on 64 classes: 64 pairs of 1 + 1 rows take 19.6 us in one launch and 20.1 in two,
        // of 128 + 128 21.7 and 20.6; one pair of 32768 rows each 43 us by a workgroup (8192 rows
        // at a time), 86 by a wave (512).
        const int64_t each = pairs > 0 ? rows / pairs : 0;
        if (pairs <= kPrefSmallPairs && each <= kPrefSmallRows) {
            if (pairs > 0 || out)
                k_pref_small<A><<<1, kSumThreads, 0, s>>>(pa, mean, out, static_cast<A*>(count));
            return check_launch("cl_preference_loss_forward(pairs)");
        }
        const bool longs = each > kPrefLongRows;
        if (longs)
            k_pref_long<A><<<unsigned(pairs), kSumThreads, 0, s>>>(pa);
        else if (pairs > 0)
            k_pref_pairs<A><<<wide_grid(ceil_div(pairs, kRowBlock / 64)), kRowBlock, 0, s>>>(pa);
        if (int rc = check_launch("cl_preference_loss_forward(pairs)")) return rc;
        if (out) {
            const int64_t threads = std::min<int64_t>(kSumThreads, ceil_div(pairs, 64) * 64);
            k_pref_sum<A><<<1, unsigned(threads), 0, s>>>(static_cast<const A*>(terms), pairs,
                                                          mean, out, static_cast<A*>(count));
        }
    });
    return check_launch("cl_preference_loss_forward(sum)");
}

extern "C" int cl_preference_loss_backward(int dtype, const void* logits, int64_t row_stride,
                                           int64_t rows, int64_t cols, const int64_t* actions,
                                           const void* row_state, const int32_t* row_seq,
                                           const void* seq_slope, int64_t pairs, int reduction,
                                           const void* grad_loss, const void* count,
                                           void* grad_logits, void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || (row_seq && grad_logits), "null pointer argument");
    CL_ARG(pairs >= 0 && pairs < (int64_t(1) << 30), "pairs must be in [0, 2^30)");
    CL_ARG(rows == 0 || pairs == 0 || (seq_slope && grad_loss), "null pointer argument");
    CL_ARG(reduction >= CL_REDUCE_NONE && reduction <= CL_REDUCE_MEAN, "unknown reduction %d",
           reduction);
    CL_ARG(reduction != CL_REDUCE_MEAN || count, "null pointer argument");
    if (rows == 0) return CL_OK;
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        using A = wide_t<T>;
        Upstream<A> up{};
        up.row_seq = row_seq;
        up.seq_slope = static_cast<const A*>(seq_slope);
        up.pairs = pairs;
        if (reduction == CL_REDUCE_NONE)
            up.pair_grad = static_cast<const A*>(grad_loss);
        else
            up.scalar = static_cast<const A*>(grad_loss);
        if (reduction == CL_REDUCE_MEAN) up.count = static_cast<const A*>(count);
        return launch_logit_grad(row_args<T>(logits, row_stride, rows, cols, actions, 0, nullptr,
                                      row_state),
                          up, grad_logits, as_stream(stream));
    });
}

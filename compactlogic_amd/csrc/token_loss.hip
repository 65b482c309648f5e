// Losses on the log-probability of one chosen class or token per row of logits: the
// log-probability itself, the clipped policy loss with a KL term, and the preference loss of
// paired sequences, each with the logits' gradient.
//
// Row n of logits x[n, 0..V) with action a:  m = max x,  s = sum exp(x - m),
//   lp = (x_a - m) - log s,   p_j = exp(x_j - m) / s,   d lp / d x_j = [j = a] - p_j.
// Every loss is a function of the rows' lp, so its gradient is a number per row, the slope,
// times [j = a] - p_j.  The forward leaves per row (m, 1 / s, 1 - p_a, slope) and the backward
// forms the gradient from them (1 - p_a is -expm1(lp), rounded once).
//
// The row's scalars (lp and what the losses make of it) are taken in fp64: rows lie next to the
// borders of the clipped range, and the preference loss subtracts sums over whole sequences.
#include "storage.h"

#include <algorithm>

namespace cl {
namespace {

constexpr int kRowThreads = 256;

// What the backward needs of a row.
template <typename A>
struct alignas(4 * sizeof(A)) RowState {
    A m;      // largest logit
    A inv_s;  // 1 / sum exp(x - m)
    A rest;   // 1 - p of the action
    A slope;  // d loss term / d lp, 0 for a row that does not count
};

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
};

// ---- what each loss makes of a row's lp: writes its own outputs, returns the slope
template <typename A>
struct LogProbOp {
    __device__ __forceinline__ A counted(int64_t, double lp) const {
        return lp == lp ? A(1) : A(lp);
    }
    __device__ __forceinline__ void ignored(int64_t) const {}
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
    __device__ __forceinline__ A counted(int64_t n, double lp) const {
        const double a = double(adv[n]);
        const double r = exp(lp - double(old_lp[n]));
        double term, slope;
        if (a >= 0) {
            term = -(r > high ? high : r) * a;
            slope = r > high ? 0.0 : -a * r;
        } else {
            term = -(r < low ? low : r) * a;
            slope = r < low ? 0.0 : -a * r;
        }
        if (ref) {
            const double g = double(ref[n]) - lp;
            const double e = expm1(g);
            term += kl * (e - g);
            slope -= kl * e;
        }
        terms[n] = A(term);
        return A(slope);
    }
    __device__ __forceinline__ void ignored(int64_t n) const { terms[n] = A(0); }
};

// gap = lp - ref, summed over sequences by k_pref_pairs.
template <typename A>
struct PreferenceOp {
    const A* ref;
    double* gaps;
    int32_t* row_seq;
    __device__ __forceinline__ A counted(int64_t n, double lp) const {
        gaps[n] = lp - (ref ? double(ref[n]) : 0.0);
        row_seq[n] = -1;
        return A(1);
    }
    __device__ __forceinline__ void ignored(int64_t n) const {
        gaps[n] = 0.0;
        row_seq[n] = -1;
    }
};

template <typename A>
__device__ __forceinline__ A nan_value() {
    return A(__builtin_nan(""));
}

// Running maximum and sum of a softmax: two partial rows joined.  A part that saw nothing but
// -inf has m = -inf; its sum is then kept as it is (0, or NaN if a NaN came by).
template <typename A>
__device__ __forceinline__ void join(A& m, A& s, A m2, A s2) {
    const A mm = m2 > m ? m2 : m;
    const A base = mm == -A(__builtin_inf()) ? A(0) : mm;
    s = s * exp(m - base) + s2 * exp(m2 - base);
    m = mm;
}

// The row's scalars, by one thread.
template <typename T, typename Op>
__device__ __forceinline__ void finish_row(const RowArgs<T>& a, const Op& op, int64_t n,
                                           wide_t<T> m, wide_t<T> s) {
    using A = wide_t<T>;
    const int64_t act = a.actions[n];
    RowState<A> st{m, A(1) / s, A(0), A(0)};
    if (act == a.ignore) {
        op.ignored(n);
        a.lp[n] = A(0);
    } else {
        double lp = nan_value<double>();
        if (act >= 0 && act < a.cols)
            lp = (double(a.x[n * a.stride + act]) - double(m)) - log(double(s));
        a.lp[n] = A(lp);
        st.rest = A(-expm1(lp));
        st.slope = op.counted(n, lp);
    }
    a.state[n] = st;
}

template <typename T, typename Op>
__global__ __launch_bounds__(kRowThreads) void k_rows(RowArgs<T> a, Op op) {
    using A = wide_t<T>;
    __shared__ A sm[kRowThreads], ss[kRowThreads];
    const int64_t n = blockIdx.x;
    const T* x = a.x + n * a.stride;
    A m = -A(__builtin_inf()), s = 0;
    for (int64_t j = threadIdx.x; j < a.cols; j += kRowThreads) join(m, s, A(x[j]), A(1));
    sm[threadIdx.x] = m;
    ss[threadIdx.x] = s;
    __syncthreads();
    for (int h = kRowThreads / 2; h > 0; h >>= 1) {
        if (int(threadIdx.x) < h)
            join(sm[threadIdx.x], ss[threadIdx.x], sm[threadIdx.x + h], ss[threadIdx.x + h]);
        __syncthreads();
    }
    if (threadIdx.x == 0) finish_row(a, op, n, sm[0], ss[0]);
}

// ---- the upstream gradient of a row's slope
template <typename A>
struct Upstream {
    const A* rows;           // a gradient per row, or null
    const A* scalar;         // the gradient of a scalar loss, or null
    const A* count;          // what a mean divides by, or null
    const int32_t* row_seq;  // preference: the row's sequence (-1: none), else null
    const A* seq_slope;      // per sequence; sequence q belongs to pair q % pairs
    const A* pair_grad;      // a gradient per pair, or null
    int64_t pairs;
    __device__ __forceinline__ A operator()(int64_t n, A slope) const {
        if (slope == A(0)) return A(0);
        A g = slope;
        if (row_seq) {
            const int64_t q = row_seq[n];
            if (q < 0) return A(0);
            g *= seq_slope[q];
            if (pair_grad) g *= pair_grad[q < pairs ? q : q - pairs];
        }
        if (rows) g *= rows[n];
        if (scalar) g *= count ? scalar[0] / count[0] : scalar[0];
        return g;
    }
};

template <typename T>
__global__ __launch_bounds__(kRowThreads) void k_logit_grad(RowArgs<T> a, Upstream<wide_t<T>> up,
                                                            T* __restrict__ grad) {
    using A = wide_t<T>;
    const int64_t n = blockIdx.x;
    const RowState<A> st = a.state[n];
    const A c = up(n, st.slope);
    const int64_t act = a.actions[n];
    const T* x = a.x + n * a.stride;
    T* g = grad + n * a.cols;
    for (int64_t j = threadIdx.x; j < a.cols; j += kRowThreads) {
        A v = 0;
        if (c != A(0)) v = j == act ? c * st.rest : -c * (exp(A(x[j]) - st.m) * st.inv_s);
        g[j] = T(v);
    }
}

// ---- sums in a fixed order by one workgroup, in fp64
constexpr int kSumThreads = 1024;

__device__ __forceinline__ double group_sum(double v, double* red) {
    red[threadIdx.x] = v;
    __syncthreads();
    for (int h = int(blockDim.x) / 2; h > 0; h >>= 1) {
        if (int(threadIdx.x) < h) red[threadIdx.x] += red[threadIdx.x + h];
        __syncthreads();
    }
    const double r = red[0];
    __syncthreads();
    return r;
}

// loss = sum of the rows' terms, divided by the number of counted rows for a mean.
template <typename A>
__global__ __launch_bounds__(kSumThreads) void k_policy_sum(const A* __restrict__ terms,
                                                            const int64_t* __restrict__ actions,
                                                            int64_t rows, int64_t ignore, int mean,
                                                            A* __restrict__ loss,
                                                            A* __restrict__ count) {
    __shared__ double red[kSumThreads];
    double t = 0, c = 0;
    for (int64_t n = threadIdx.x; n < rows; n += kSumThreads) {
        t += double(terms[n]);
        c += actions[n] != ignore ? 1.0 : 0.0;
    }
    t = group_sum(t, red);
    c = group_sum(c, red);
    if (threadIdx.x == 0) {
        loss[0] = A(mean ? t / c : t);  // no counted row: 0 / 0 = NaN, the mean of nothing
        count[0] = A(c);
    }
}

// One workgroup per pair: the sums over both sequences, the margin h, the loss term
//   -(1 - e) log sigma(h) - e log sigma(-h)
// and its slope by the chosen sequence's sum; the rejected one's is the negative.
template <typename A>
__global__ __launch_bounds__(kRowThreads) void k_pref_pairs(const double* __restrict__ gaps,
                                                            const int64_t* __restrict__ offsets,
                                                            int64_t rows, int64_t pairs,
                                                            double beta, double smooth,
                                                            int32_t* __restrict__ row_seq,
                                                            A* __restrict__ seq_slope,
                                                            A* __restrict__ margins,
                                                            A* __restrict__ terms) {
    __shared__ double red[kRowThreads];
    const int64_t i = blockIdx.x;
    double d[2];
    bool bad = false;
    for (int side = 0; side < 2; ++side) {
        const int64_t q = i + side * pairs;
        int64_t b = offsets[q], e = offsets[q + 1];
        bad |= b < 0 || e < b || e > rows;
        b = std::min(std::max<int64_t>(b, 0), rows);
        e = std::min(std::max(e, b), rows);
        double t = 0;
        for (int64_t n = b + threadIdx.x; n < e; n += kRowThreads) {
            t += gaps[n];
            row_seq[n] = int32_t(q);
        }
        d[side] = group_sum(t, red);
    }
    if (threadIdx.x != 0) return;
    double h = beta * (d[0] - d[1]);
    if (bad) h = nan_value<double>();
    const double tail = log1p(exp(-fabs(h)));
    const double away = tail - (h < 0 ? h : 0.0);  // -log sigma(h)
    const double near = tail + (h > 0 ? h : 0.0);  // -log sigma(-h)
    const double slope = beta * (smooth / (1 + exp(-h)) - (1 - smooth) / (1 + exp(h)));
    margins[i] = A(h);
    terms[i] = A((1 - smooth) * away + smooth * near);
    seq_slope[i] = A(slope);
    seq_slope[i + pairs] = A(-slope);
}

template <typename A>
__global__ __launch_bounds__(kSumThreads) void k_pref_sum(const A* __restrict__ terms,
                                                          int64_t pairs, int mean,
                                                          A* __restrict__ loss,
                                                          A* __restrict__ count) {
    __shared__ double red[kSumThreads];
    double t = 0;
    for (int64_t i = threadIdx.x; i < pairs; i += kSumThreads) t += double(terms[i]);
    t = group_sum(t, red);
    if (threadIdx.x == 0) {
        loss[0] = A(mean ? t / double(pairs) : t);
        count[0] = A(pairs);
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
    return a;
}

template <typename T, typename Op>
void launch_rows(const RowArgs<T>& a, const Op& op, hipStream_t s) {
    if (a.rows > 0) k_rows<T, Op><<<unsigned(a.rows), kRowThreads, 0, s>>>(a, op);
}

template <typename T>
void launch_logit_grad(const RowArgs<T>& a, const Upstream<wide_t<T>>& up, void* grad,
                       hipStream_t s) {
    if (a.rows > 0)
        k_logit_grad<T><<<unsigned(a.rows), kRowThreads, 0, s>>>(a, up, static_cast<T*>(grad));
}

}  // namespace
}  // namespace cl

using namespace cl;

extern "C" int cl_selected_log_prob_forward(int dtype, const void* logits, int64_t row_stride,
                                            int64_t rows, int64_t cols, const int64_t* actions,
                                            int64_t ignore_index, void* log_probs, void* row_state,
                                            void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || log_probs, "null pointer argument");
    if (rows == 0) return CL_OK;
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        launch_rows(row_args<T>(logits, row_stride, rows, cols, actions, ignore_index, log_probs,
                                row_state),
                    LogProbOp<wide_t<T>>{}, as_stream(stream));
    });
    return check_launch("cl_selected_log_prob_forward");
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
        launch_logit_grad(row_args<T>(logits, row_stride, rows, cols, actions, 0, nullptr,
                                      row_state),
                          up, grad_logits, as_stream(stream));
    });
    return check_launch("cl_selected_log_prob_backward");
}

extern "C" int cl_policy_loss_forward(int dtype, const void* logits, int64_t row_stride,
                                      int64_t rows, int64_t cols, const int64_t* actions,
                                      int64_t ignore_index, const void* old_log_probs,
                                      const void* advantages, const void* ref_log_probs,
                                      double clip_low, double clip_high, double kl_coef,
                                      int reduction, void* log_probs, void* row_state,
                                      void* terms, void* loss, void* count, void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || (old_log_probs && advantages && log_probs && terms),
           "null pointer argument");
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
        launch_rows(row_args<T>(logits, row_stride, rows, cols, actions, ignore_index, log_probs,
                                row_state),
                    op, s);
        if (int rc = check_launch("cl_policy_loss_forward(rows)")) return rc;
        if (reduction != CL_REDUCE_NONE)
            k_policy_sum<A><<<1, kSumThreads, 0, s>>>(op.terms, actions, rows, ignore_index,
                                                      reduction == CL_REDUCE_MEAN,
                                                      static_cast<A*>(loss),
                                                      static_cast<A*>(count));
    });
    return check_launch("cl_policy_loss_forward(sum)");
}

extern "C" int cl_policy_loss_backward(int dtype, const void* logits, int64_t row_stride,
                                       int64_t rows, int64_t cols, const int64_t* actions,
                                       const void* row_state, int reduction, const void* grad_loss,
                                       const void* count, void* grad_logits, void* stream) {
    clear_error();
    if (int rc = check_logits(logits, row_stride, rows, cols, actions, row_state)) return rc;
    CL_ARG(rows == 0 || (grad_loss && grad_logits), "null pointer argument");
    CL_ARG(reduction >= CL_REDUCE_NONE && reduction <= CL_REDUCE_MEAN, "unknown reduction %d",
           reduction);
    CL_ARG(reduction != CL_REDUCE_MEAN || count, "null pointer argument");
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
        launch_logit_grad(row_args<T>(logits, row_stride, rows, cols, actions, 0, nullptr,
                                      row_state),
                          up, grad_logits, as_stream(stream));
    });
    return check_launch("cl_policy_loss_backward");
}

extern "C" int cl_preference_loss_forward(int dtype, const void* logits, int64_t row_stride,
                                          int64_t rows, int64_t cols, const int64_t* actions,
                                          int64_t ignore_index, const void* ref_log_probs,
                                          const int64_t* offsets, int64_t pairs, double beta,
                                          double label_smoothing, int reduction, void* log_probs,
                                          void* row_state, double* gaps, int32_t* row_seq,
                                          void* seq_slope, void* margins, void* terms, void* loss,
                                          void* count, void* stream) {
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
        launch_rows(row_args<T>(logits, row_stride, rows, cols, actions, ignore_index, log_probs,
                                row_state),
                    op, s);
        if (int rc = check_launch("cl_preference_loss_forward(rows)")) return rc;
        if (pairs > 0)
            k_pref_pairs<A><<<unsigned(pairs), kRowThreads, 0, s>>>(
                gaps, offsets, rows, pairs, beta, label_smoothing, row_seq,
                static_cast<A*>(seq_slope), static_cast<A*>(margins), static_cast<A*>(terms));
        if (int rc = check_launch("cl_preference_loss_forward(pairs)")) return rc;
        if (reduction != CL_REDUCE_NONE)
            k_pref_sum<A><<<1, kSumThreads, 0, s>>>(static_cast<const A*>(terms), pairs,
                                                    reduction == CL_REDUCE_MEAN,
                                                    static_cast<A*>(loss), static_cast<A*>(count));
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
        launch_logit_grad(row_args<T>(logits, row_stride, rows, cols, actions, 0, nullptr,
                                      row_state),
                          up, grad_logits, as_stream(stream));
    });
    return check_launch("cl_preference_loss_backward");
}

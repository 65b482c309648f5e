// Verification of drafted tokens against the target's probabilities.  Sequence s has K drafted tokens
// x_i, drawn from the draft's probabilities q_i, and the target's p_0 .. p_K, all as logits, and K + 1
// uniform numbers.  Token i is accepted while
//   u_i q_i(x_i) < p_i(x_i);
// at the first one that is not, a token is drawn from max(p_i - q_i, 0), and behind the last one from
// p_i, by the last number r: the first j whose sum of weights up to j is above r times their sum.  What
// comes out is distributed as the target's own tokens are, whatever the draft was.
//
// The tests take a maximum and a sum in fp32 (fp64 for fp64) over each row, as the losses do: a number
// within some 10^-7 of its border is tested as the order of the sums goes.  The draw takes a sum in fp64 of
// exponentials in fp64, of one row of each: next to some 10^5 borders between tokens, fp32 sums would draw
// a neighbour once in 10^3 draws.
//
//   k_small    one workgroup a sequence does it all, for rows of at most kSmall elements
// else
//   k_stats    (m, s) of every part of the rows, kPart elements each
//   k_decide   joins them and takes the tests
//   k_sums     the fp64 sums of a chunk, kChunk elements, of the two rows
//   k_weights  the sum of max(p - q, 0) of its chunk
//   k_pick     the chunk that the number falls into, and the place in it
// Chunks are short because k_pick takes one by one workgroup (8192 elements of two rows took 11 us).  256
// sequences of 4 drafts of 10: 9 us, latency.  64 of 5 of 50021 bf16: statistics 16 us (4.4 TB/s), sums,
// weights and place 9 to 10 each, tests 4.5.  These four are latency too, of launches that wait for one
// another and of each one's loads, scans and exponentials in a row: VALU 28 % busy in sums and weights, 2 %
// in the tests and the place.
#include "row_loss.h"
#include "storage.h"

namespace cl {
namespace {

constexpr int kRun = 8;                  // elements of a thread, one behind the other
constexpr int kThreads = 512;            // k_small, k_decide
constexpr int kSmall = kThreads * kRun;
constexpr int kDrawThreads = 256;        // of a chunk
constexpr int kChunk = kDrawThreads * kRun;
constexpr int kStatThreads = 256;
constexpr int kPart = 8192;

template <typename A>
struct Stat {
    A m, s;
};

// What the tests leave for the draw.
struct Draw {
    double mp, mq;   // largest logits of the two rows
    int64_t n;       // accepted tokens
    int64_t refused; // one was drafted there: the draft's row counts
};

template <typename T>
struct Args {
    using A = wide_t<T>;
    const T *p, *q;                  // q may be null: the draft was sure of its tokens
    int64_t p_seq, p_row, q_seq, q_row;
    const int64_t* tokens;
    const void* uniforms;
    bool uniforms64;
    int64_t ignore;
    int64_t seqs, drafts, cols;
    int64_t* out;
    int64_t* accepted;
    A* lp;
    // workspace, where a row has several chunks
    int parts, chunks;
    Stat<A>* stats;                  // [seq][2 drafts + 1][part], the target's rows first
    Draw* draws;
    double* sums;                    // [seq][chunk][p, q]
    double* weights;                 // [seq][chunk]

    __device__ __forceinline__ double uniform(int64_t seq, int64_t i) const {
        const int64_t at = seq * (drafts + 1) + i;
        return uniforms64 ? static_cast<const double*>(uniforms)[at]
                          : double(static_cast<const float*>(uniforms)[at]);
    }
    __device__ __forceinline__ const T* row(int64_t seq, int64_t i, bool draft) const {
        return draft ? q + seq * q_seq + i * q_row : p + seq * p_seq + i * p_row;
    }
    __device__ __forceinline__ Stat<A>* stat(int64_t seq, int64_t i, bool draft) const {
        return stats + (seq * (2 * drafts + 1) + i + (draft ? drafts + 1 : 0)) * parts;
    }
    __device__ __forceinline__ bool holds(int64_t token) const { return token >= 0 && token < cols; }
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_part(const T* p, int64_t count) {
    if (count >= N) return pload<T, N>(p);
    Pack<T, N> r;
#pragma unroll
    for (int e = 0; e < N; ++e) r.v[e] = e < count ? p[e] : T(-__builtin_inff());
    return r;
}

// ---- maximum and sum of exp(x - m).  Where there was nothing but -inf, differences are taken from 0.
template <typename A>
__device__ __forceinline__ A base_of(A m) {
    return m == -A(__builtin_inf()) ? A(0) : m;
}
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return __builtin_fmax(a, b); }

template <int LANES, typename A>
__device__ __forceinline__ Stat<A> join(Stat<A> st) {
    A m = st.m;
    m = max_of(m, dpp_move<0xB1>(m));   // quad_perm [1,0,3,2]
    m = max_of(m, dpp_move<0x4E>(m));   // quad_perm [2,3,0,1]
    m = max_of(m, dpp_move<0x141>(m));  // row_half_mirror
    m = max_of(m, dpp_move<0x140>(m));  // row_mirror
    if constexpr (LANES == 64)
        m = max_of(max_of(read_lane(m, 0), read_lane(m, 16)),
                   max_of(read_lane(m, 32), read_lane(m, 48)));
    A s = st.s * exp_diff(st.m - base_of(m));
    if constexpr (LANES == 64) {
        s = wave_total(s);
    } else {
        s += dpp_move<0xB1>(s);
        s += dpp_move<0x4E>(s);
        s += dpp_move<0x141>(s);
        s += dpp_move<0x140>(s);
    }
    return {m, s};
}

template <typename A>
__device__ __forceinline__ void add(Stat<A>& st, const Stat<A>& more) {
    const A m = max_of(st.m, more.m), base = base_of(m);
    st.s = st.s * exp_diff(st.m - base) + more.s * exp_diff(more.m - base);
    st.m = m;
}

template <typename T>
__global__ __launch_bounds__(kStatThreads) void k_stats(Args<T> a) {
    using A = wide_t<T>;
    constexpr int VEC = wide_vec<T>(), NV = kPart / kStatThreads / VEC;
    __shared__ Stat<A> part[kStatThreads / 64];
    const int64_t rows = 2 * a.drafts + 1;
    const int64_t group = group_index();  // below 2^31
    if (group >= a.seqs * rows * a.parts) return;
    const uint32_t row = uint32_t(group) / uint32_t(a.parts);
    const int at_part = int(uint32_t(group) - row * uint32_t(a.parts));
    const int64_t seq = row / uint32_t(rows), r = row - seq * rows;
    const bool draft = r > a.drafts;
    const int64_t i = draft ? r - a.drafts - 1 : r;
    if (draft && !a.q) return;
    // a row behind the end of the drafts is not read
    bool ended = false;
    for (int64_t j = 0; j < (draft ? i + 1 : i); ++j) ended |= a.tokens[seq * a.drafts + j] == a.ignore;
    if (ended) return;
    const int64_t j0 = int64_t(at_part) * kPart;
    const T* x = a.row(seq, i, draft) + j0;
    const int64_t n = a.cols - j0;
    Pack<T, VEC> v[NV];
    if (n >= kPart) {  // (no branch between the loads: each would be waited for)
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = pload<T, VEC>(x + (k * kStatThreads + threadIdx.x) * VEC);
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t at = (k * kStatThreads + threadIdx.x) * VEC;
            v[k] = load_part<T, VEC>(x + at, n - at);
        }
    }
    Stat<A> st{-A(__builtin_inf()), A(0)};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) st.m = max_of(st.m, A(v[k].v[e]));
    const A base = base_of(st.m);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) st.s += exp_diff(A(v[k].v[e]) - base);
    st = join<64>(st);
    if (lane_id() == 0) part[wave_id()] = st;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kStatThreads / 64; ++w) add(st, part[w]);
        a.stat(seq, i, draft)[at_part] = st;
    }
}

// ---- the tests, kThreads / LANES rows at a time: position i's target and draft beside each other.
// Every thread returns with the outcome.  rows(seq, i, draft) gives a row's (m, s) to its lanes.
template <int LANES>
struct Round {
    static constexpr int N = kThreads / LANES / 2;  // positions
    double prob[N][2], m[N][2], lp[N];
    int first;
};

template <int LANES, typename T, typename F>
__device__ __forceinline__ Draw decide(const Args<T>& a, int64_t seq, Round<LANES>& sh, F&& rows) {
    using A = wide_t<T>;
    constexpr int N = Round<LANES>::N;
    const int g = threadIdx.x / LANES;
    for (int64_t i0 = 0;; i0 += N) {
        const bool draft = g & 1;
        const int64_t i = i0 + g / 2;
        const int64_t token = i < a.drafts ? a.tokens[seq * a.drafts + i] : a.ignore;
        const bool given = i < a.drafts && token != a.ignore;
        // by the first wave, in time for the tests
        const int64_t mine_at = i0 + threadIdx.x;
        const bool tests = threadIdx.x < N && mine_at < a.drafts;
        const int64_t mine = tests ? a.tokens[seq * a.drafts + mine_at] : a.ignore;
        const double u = tests ? a.uniform(seq, mine_at) : 0.0;
        if (draft ? given && a.q : i <= a.drafts) {
            const Stat<A> st = rows(seq, i, draft);
            double pr = 0.0, lp = -__builtin_inf();
            if (given && a.holds(token)) {
                const double d = double(a.row(seq, i, draft)[token]) - double(st.m);
                pr = exp(d) / double(st.s);
                lp = d - log(double(st.s));
            }
            if (threadIdx.x % LANES == 0) {
                sh.prob[g / 2][draft] = pr;
                sh.m[g / 2][draft] = double(st.m);
                if (!draft) sh.lp[g / 2] = lp;
            }
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const int l = threadIdx.x;
            const int64_t at = i0 + l;
            bool stop = false;
            if (l < N && at <= a.drafts) {
                stop = true;
                if (mine != a.ignore) stop = !(u * (a.q ? sh.prob[l][1] : 1.0) < sh.prob[l][0]);
            }
            const uint64_t stops = __ballot(stop);
            const int first = stops ? __builtin_ctzll(stops) : N;
            if (l < first) {
                a.out[seq * (a.drafts + 1) + at] = mine;
                a.lp[seq * (a.drafts + 1) + at] = A(sh.lp[l]);
            }
            if (l == 0) sh.first = first;
        }
        __syncthreads();
        const int first = sh.first;
        if (first < N) {
            const int64_t n = i0 + first;
            const bool refused = n < a.drafts && a.tokens[seq * a.drafts + n] != a.ignore;
            for (int64_t k = n + 1 + threadIdx.x; k <= a.drafts; k += kThreads) {
                a.out[seq * (a.drafts + 1) + k] = a.ignore;
                a.lp[seq * (a.drafts + 1) + k] = A(0);
            }
            if (threadIdx.x == 0) a.accepted[seq] = n;
            return {sh.m[first][0], refused && a.q ? sh.m[first][1] : 0.0, n, refused};
        }
        __syncthreads();
    }
}

// ---- fp64 sums over a workgroup
// Sum up to and with each lane's v: within rows of 16 lanes by shifts (0 comes in from outside), then
// the rows' sums in turn.
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_move<0x111>(v);  // row_shr:1
    v += dpp_move<0x112>(v);
    v += dpp_move<0x114>(v);
    v += dpp_move<0x118>(v);
    const double a = read_lane(v, 15), b = a + read_lane(v, 31), c = b + read_lane(v, 47);
    const int row = lane_id() >> 4;
    return v + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? b : c);
}

// Sum up to and with each thread's v; `total`: of all.
template <int WAVES>
__device__ __forceinline__ double group_scan(double v, double* red, double& total) {
    v = wave_scan(v);
    if (lane_id() == 63) red[wave_id()] = v;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave_id()) before = total;
        total += red[w];
    }
    __syncthreads();
    return before + v;
}

// exp of x <= 0 within some 2^-52, without the cases of the library's (30 instructions to 20):
// 2^n exp(r), n the integer next to x log2 e, ln 2 in two parts as fdlibm's exp has them (after Cody and
// Waite: the first one times n is exact), exp(r) by its series to r^13 / 13!.  |r| < 0.35: what is left out,
// r^14 / 14! and on, is below 2^-57, and of exp(r) >= 0.7 below 2^-56; the last roundings are the rest.
__device__ __forceinline__ double exp_below(double x) {
    x = x < -800.0 ? -800.0 : x;  // (0; NaN stays)
    const double n = __builtin_rint(x * 1.4426950408889634);
    const double r = fma(n, -1.9082149292705877e-10, fma(n, -0.6931471803691238, x));
    double s = 1.0 / 6227020800.0;
    s = fma(s, r, 1.0 / 479001600.0);
    s = fma(s, r, 1.0 / 39916800.0);
    s = fma(s, r, 1.0 / 3628800.0);
    s = fma(s, r, 1.0 / 362880.0);
    s = fma(s, r, 1.0 / 40320.0);
    s = fma(s, r, 1.0 / 5040.0);
    s = fma(s, r, 1.0 / 720.0);
    s = fma(s, r, 1.0 / 120.0);
    s = fma(s, r, 1.0 / 24.0);
    s = fma(s, r, 1.0 / 6.0);
    s = fma(s, r, 0.5);
    s = fma(s, r, 1.0);
    s = fma(s, r, 1.0);
    return __builtin_ldexp(s, int(n));
}

// ---- the draw.  A thread's elements of a chunk of NT threads: `run` of them from `at` on.
template <typename T, int NT>
struct Place {
    int64_t at;
    int count;
    __device__ __forceinline__ Place(int64_t j0, int64_t cols) {
        constexpr int VEC = wide_vec<T>();
        const int64_t n = cols - j0 < NT * kRun ? cols - j0 : NT * kRun;
        const int run = int((n + NT * VEC - 1) / (NT * VEC)) * VEC;
        at = j0 + int64_t(threadIdx.x) * run;
        const int64_t left = j0 + n - at;
        count = left >= run ? run : left > 0 ? int(left) : 0;
    }
};

// exp(x - m) of the thread's elements in fp64, 0 behind them (whose logits are -inf: asking for each
// whether it is there, one exponential would wait for the other); returns their sum.
template <typename T, int NT>
__device__ __forceinline__ double exponentials(const T* row, const Place<T, NT>& w, double m,
                                               double (&e)[kRun]) {
    constexpr int VEC = wide_vec<T>();
    Pack<T, VEC> v[kRun / VEC];
#pragma unroll
    for (int k = 0; k < kRun / VEC; ++k)
        v[k] = load_part<T, VEC>(row + w.at + k * VEC, w.count - k * VEC);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        e[k] = exp_below(double(v[k / VEC].v[k % VEC]) - m);
        sum += e[k];
    }
    return sum;
}

template <typename T>
struct Rows {
    const T *p, *q;   // q null: no draft counts, or it was sure of `token`
    int64_t token;
    bool sure;
    __device__ __forceinline__ Rows(const Args<T>& a, int64_t seq, const Draw& d) {
        p = a.row(seq, d.n, false);
        q = d.refused && a.q ? a.row(seq, d.n, true) : nullptr;
        sure = d.refused && !a.q;
        token = sure ? a.tokens[seq * a.drafts + d.n] : 0;
    }
};

// Weights where a draft was refused, max(p - q, 0), of the thread's exponentials e and f of the two rows;
// returns their sum.
template <typename T, int NT>
__device__ __forceinline__ double over(const Rows<T>& r, const Place<T, NT>& w, const double (&e)[kRun],
                                       const double (&f)[kRun], double inv_sp, double inv_sq,
                                       double (&v)[kRun]) {
    // equal rows leave nothing: both products are rounded (and both sums taken alike)
#pragma clang fp contract(off)
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
        double d = e[k] * inv_sp;
        if (r.q)
            d -= f[k] * inv_sq;
        else if (w.at + k == r.token)
            d = 0.0;
        v[k] = d > 0.0 || d != d ? d : 0.0;
        sum += v[k];
    }
    return sum;
}

// Draws the first token up to and with which the sum of the weights v is above `goal`, `before` counted
// in; the last one with a weight above 0 if rounding leaves none.  mine, upto: the thread's sum of v, and
// that up to and with it; e: its exponentials of the target's row, whose sum is sp.  The thread that
// holds the token writes it, with its log-probability; where p is no probability, or no weight is above
// 0, none is drawn.
template <typename T, int NT>
__device__ __forceinline__ void draw(const Args<T>& a, int64_t seq, const Draw& d, const T* row,
                                     const Place<T, NT>& w,
                                     const double (&v)[kRun], const double (&e)[kRun], double sp,
                                     double mine, double upto, double before, double goal, int* sh) {
    using A = wide_t<T>;
    if (threadIdx.x == 0) {
        sh[0] = NT;
        sh[1] = -1;
    }
    __syncthreads();
    if (mine > 0.0) {
        if (before + upto > goal) atomicMin(&sh[0], int(threadIdx.x));
        atomicMax(&sh[1], int(threadIdx.x));
    }
    __syncthreads();
    const bool hit = sh[0] < NT;
    const int owner = !(sp > 0.0) ? -1 : hit ? sh[0] : sh[1];
    const int64_t to = seq * (a.drafts + 1) + d.n;
    if (int(threadIdx.x) == owner) {
        double c = before + (upto - mine), chosen = 0.0;
        int at = 0;
        bool found = false;
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
            c += v[k];
            if (v[k] > 0.0 && !found) {
                at = k;
                chosen = e[k];
                found = hit && c > goal;
            }
        }
        a.out[to] = w.at + at;
        // (the logit itself where its exponential has lost bits)
        const double z = chosen > 1e-280 ? log(chosen) : double(row[w.at + at]) - d.mp;
        a.lp[to] = A(z - log(sp));
    } else if (owner < 0 && threadIdx.x == 0) {
        a.out[to] = a.ignore;
        a.lp[to] = A(__builtin_nan(""));
    }
}

template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void k_small(Args<T> a) {
    using A = wide_t<T>;
    constexpr int VEC = wide_vec<T>(), WAVES = kThreads / 64;
    __shared__ Round<LANES> round;
    __shared__ double red[WAVES];
    __shared__ int ends[2];
    const int64_t seq = group_index();
    if (seq >= a.seqs) return;
    const double u = a.uniform(seq, a.drafts);
    const Draw d = decide<LANES>(a, seq, round, [&](int64_t s, int64_t i, bool draft) {
        const T* x = a.row(s, i, draft);
        Stat<A> st{-A(__builtin_inf()), A(0)};
        for (int64_t j = (threadIdx.x % LANES) * VEC; j < a.cols; j += LANES * VEC) {
            const Pack<T, VEC> v = load_part<T, VEC>(x + j, a.cols - j);
            A m = st.m;
#pragma unroll
            for (int e = 0; e < VEC; ++e) m = max_of(m, A(v.v[e]));
            const A base = base_of(m);
            st.s *= exp_diff(st.m - base);
#pragma unroll
            for (int e = 0; e < VEC; ++e) st.s += exp_diff(A(v.v[e]) - base);
            st.m = m;
        }
        return join<LANES>(st);
    });
    const Rows<T> r(a, seq, d);
    const Place<T, kThreads> w(0, a.cols);
    double e[kRun], f[kRun] = {}, total;
    double mine = exponentials(r.p, w, d.mp, e);
    const double mine_q = r.q ? exponentials(r.q, w, d.mq, f) : 0.0;
    double upto = group_scan<WAVES>(mine, red, total);
    const double sp = total;
    double v[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) v[k] = e[k];
    if (d.refused) {
        double sq = 1.0, total_v;
        if (r.q) group_scan<WAVES>(mine_q, red, sq);
        const double mine_v = over(r, w, e, f, 1.0 / sp, 1.0 / sq, v);
        const double upto_v = group_scan<WAVES>(mine_v, red, total_v);
        if (total_v > 0.0) {
            mine = mine_v;
            upto = upto_v;
            total = total_v;
        } else {  // nothing is above the draft: the target's own
#pragma unroll
            for (int k = 0; k < kRun; ++k) v[k] = e[k];
        }
    }
    draw(a, seq, d, r.p, w, v, e, sp, mine, upto, 0.0, u * total, ends);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_decide(Args<T> a) {
    using A = wide_t<T>;
    __shared__ Round<16> round;
    const int64_t seq = group_index();
    if (seq >= a.seqs) return;
    const Draw d = decide<16>(a, seq, round, [&](int64_t s, int64_t i, bool draft) {
        const Stat<A>* part = a.stat(s, i, draft);
        Stat<A> st{-A(__builtin_inf()), A(0)};
        for (int c = threadIdx.x & 15; c < a.parts; c += 16) add(st, part[c]);
        return join<16>(st);
    });
    if (threadIdx.x == 0) a.draws[seq] = d;
}

template <typename T>
__global__ __launch_bounds__(kDrawThreads) void k_sums(Args<T> a) {
    constexpr int WAVES = kDrawThreads / 64;
    __shared__ double red[WAVES];
    const int64_t group = group_index();  // below 2^31
    if (group >= a.seqs * a.chunks) return;
    const int64_t seq = uint32_t(group) / uint32_t(a.chunks);
    const int64_t chunk = group - seq * a.chunks;
    const Draw d = a.draws[seq];
    const Rows<T> r(a, seq, d);
    const Place<T, kDrawThreads> w(chunk * kChunk, a.cols);
    double e[kRun], f[kRun], total;
    const double mine = exponentials(r.p, w, d.mp, e);
    const double mine_q = r.q ? exponentials(r.q, w, d.mq, f) : 0.0;
    group_scan<WAVES>(mine, red, total);  // as k_pick will have it
    if (threadIdx.x == 0) a.sums[2 * group] = total;
    if (r.q) {
        group_scan<WAVES>(mine_q, red, total);
        if (threadIdx.x == 0) a.sums[2 * group + 1] = total;
    }
}

// The sum of the chunks' sums, the same in every thread; stride: of them.
__device__ __forceinline__ double chunks_total(const double* sums, int stride, int chunks) {
    double s = 0.0;
    for (int c = lane_id(); c < chunks; c += 64) s += sums[int64_t(c) * stride];
    return wave_total(s);
}

template <typename T>
__global__ __launch_bounds__(kDrawThreads) void k_weights(Args<T> a) {
    constexpr int WAVES = kDrawThreads / 64;
    __shared__ double red[WAVES];
    const int64_t group = group_index();
    if (group >= a.seqs * a.chunks) return;
    const int64_t seq = uint32_t(group) / uint32_t(a.chunks);
    const Draw d = a.draws[seq];
    if (!d.refused) return;
    const int64_t chunk = group - seq * a.chunks;
    const Rows<T> r(a, seq, d);
    const Place<T, kDrawThreads> w(chunk * kChunk, a.cols);
    double e[kRun], f[kRun] = {}, v[kRun], total;
    exponentials(r.p, w, d.mp, e);
    if (r.q) exponentials(r.q, w, d.mq, f);
    const double* sums = a.sums + 2 * seq * a.chunks;
    const double sp = chunks_total(sums, 2, a.chunks);
    const double sq = r.q ? chunks_total(sums + 1, 2, a.chunks) : 1.0;
    group_scan<WAVES>(over(r, w, e, f, 1.0 / sp, 1.0 / sq, v), red, total);
    if (threadIdx.x == 0) a.weights[group] = total;
}

template <typename T>
__global__ __launch_bounds__(kDrawThreads) void k_pick(Args<T> a) {
    constexpr int WAVES = kDrawThreads / 64;
    __shared__ double red[WAVES];
    __shared__ int ends[2];
    const int64_t seq = group_index();
    if (seq >= a.seqs) return;
    // a lane's chunks are read before anything is known of them (weights of a sequence that refused no
    // token were not written, and are not used)
    const double* sums = a.sums + 2 * seq * a.chunks;
    const double* weights = a.weights + seq * a.chunks;
    const Draw d = a.draws[seq];
    const double u = a.uniform(seq, a.drafts);
    const int l = lane_id();
    double first_p = 0.0, first_q = 0.0, first_w = 0.0;
    if (l < a.chunks) {
        first_p = sums[2 * l];
        first_q = sums[2 * l + 1];
        first_w = weights[l];
    }
    const Rows<T> r(a, seq, d);
    double sp = first_p, sq = r.q ? first_q : 0.0, total = d.refused ? first_w : 0.0;
    for (int c = l + 64; c < a.chunks; c += 64) {
        sp += sums[2 * int64_t(c)];
        if (r.q) sq += sums[2 * int64_t(c) + 1];
        if (d.refused) total += weights[c];
    }
    sp = wave_total(sp);
    sq = r.q ? wave_total(sq) : 1.0;
    total = wave_total(total);
    const bool own = !(total > 0.0);  // the target's own: no draft was refused, or nothing is above it
    if (own) total = sp;
    // the chunk, as draw finds a place in it; every wave alike
    const double goal = u * total;
    int chosen = -1, last = -1;
    double before = 0.0, at_last = 0.0, carry = 0.0;
    for (int c0 = 0; c0 < a.chunks && chosen < 0; c0 += 64) {
        const int c = c0 + l;
        double mine = own ? first_p : first_w;
        if (c0 > 0) mine = c >= a.chunks ? 0.0 : own ? sums[2 * int64_t(c)] : weights[c];
        const double v = wave_scan(mine);
        const uint64_t some = __ballot(mine > 0.0);
        const uint64_t hit = __ballot(mine > 0.0 && carry + v > goal);
        const double start = __shfl_up(v, 1, 64);
        const double prior = carry + (l == 0 ? 0.0 : start);
        if (hit) {
            const int h = __builtin_ctzll(hit);
            chosen = c0 + h;
            before = read_lane(prior, h);
        } else if (some) {
            const int h = 63 - __builtin_clzll(some);
            last = c0 + h;
            at_last = read_lane(prior, h);
        }
        carry += read_lane(v, 63);
    }
    if (chosen < 0) {
        chosen = last;
        before = at_last;
    }
    // (where no chunk has a weight, or NaN, the first one finds the same)
    const Place<T, kDrawThreads> w(int64_t(chosen < 0 ? 0 : chosen) * kChunk, a.cols);
    // (one copy of the code for either kind of weights: a workgroup alone waits for its instructions too)
    double e[kRun], f[kRun] = {}, v[kRun], sum;
    double mine = exponentials(r.p, w, d.mp, e);
#pragma unroll
    for (int k = 0; k < kRun; ++k) v[k] = e[k];
    if (!own) {
        if (r.q) exponentials(r.q, w, d.mq, f);
        mine = over(r, w, e, f, 1.0 / sp, 1.0 / sq, v);
    }
    const double upto = group_scan<WAVES>(mine, red, sum);
    draw(a, seq, d, r.p, w, v, e, sp, mine, upto, before, goal, ends);
}

// Parts and chunks of a row, and the arrays of the workspace behind each other on 16 bytes.
struct Layout {
    bool small;
    int64_t parts, chunks, draws, sums, weights, total;
};

int layout_of(int dtype, int64_t seqs, int64_t drafts, int64_t cols, Layout& l) {
    CL_ARG(dtype >= CL_DTYPE_F32 && dtype <= CL_DTYPE_BF16,
           "unsupported dtype code %d (expected F32, F64, F16 or BF16)", dtype);
    CL_ARG(seqs >= 0 && drafts >= 0 && cols >= 1, "bad shape: %lld sequences, %lld drafts, %lld classes",
           (long long)seqs, (long long)drafts, (long long)cols);
    l.small = cols <= kSmall;
    l.parts = ceil_div(cols, kPart);
    l.chunks = ceil_div(cols, kChunk);
    const double most = double(int64_t(1) << 31);
    CL_ARG(double(seqs) * (2.0 * double(drafts) + 1) * double(l.parts) < most &&
               double(seqs) * double(l.chunks) < most && double(drafts) < most && double(l.chunks) < most,
           "too many logits for one call");
    l.draws = l.sums = l.weights = l.total = 0;
    if (l.small) return CL_OK;
    const int64_t wide = dtype == CL_DTYPE_F64 ? 8 : 4;
    l.draws = ceil_div(2 * wide * seqs * (2 * drafts + 1) * l.parts, 16) * 16;
    l.sums = l.draws + int64_t(sizeof(Draw)) * seqs;
    l.weights = l.sums + 16 * seqs * l.chunks;
    l.total = l.weights + 8 * seqs * l.chunks;
    return CL_OK;
}

}  // namespace
}  // namespace cl

using namespace cl;

extern "C" int cl_verify_drafts_workspace(int dtype, int64_t sequences, int64_t drafts, int64_t cols,
                                          int64_t* bytes) {
    clear_error();
    CL_ARG(bytes, "null pointer argument");
    Layout l;
    if (int rc = layout_of(dtype, sequences, drafts, cols, l)) return rc;
    *bytes = l.total;
    return CL_OK;
}

extern "C" int cl_verify_drafts(int dtype, const void* logits, int64_t seq_stride, int64_t row_stride,
                                const void* draft_logits, int64_t draft_seq_stride,
                                int64_t draft_row_stride, const int64_t* draft_tokens,
                                int64_t ignore_index, const void* uniforms, int uniforms_dtype,
                                int64_t sequences, int64_t drafts, int64_t cols, int64_t* tokens,
                                int64_t* accepted, void* log_probs, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    clear_error();
    Layout l;
    if (int rc = layout_of(dtype, sequences, drafts, cols, l)) return rc;
    CL_ARG(uniforms_dtype == CL_DTYPE_F32 || uniforms_dtype == CL_DTYPE_F64,
           "the uniform numbers must be F32 or F64");
    CL_ARG(seq_stride >= 0 && row_stride >= 0 && draft_seq_stride >= 0 && draft_row_stride >= 0,
           "negative strides are not supported");
    if (sequences == 0) return CL_OK;
    CL_ARG(logits && uniforms && tokens && accepted && log_probs && (drafts == 0 || draft_tokens),
           "null pointer argument");
    CL_ARG(l.total == 0 || (workspace && workspace_bytes >= l.total && aligned(workspace, 16)),
           "workspace of %lld bytes needed (cl_verify_drafts_workspace)", (long long)l.total);
    hipStream_t s = as_stream(stream);
    CL_STORAGE_SWITCH(dtype, {
        using T = scalar_t;
        Args<T> a{};
        a.p = static_cast<const T*>(logits);
        a.q = static_cast<const T*>(draft_logits);
        a.p_seq = seq_stride;
        a.p_row = row_stride;
        a.q_seq = draft_seq_stride;
        a.q_row = draft_row_stride;
        a.tokens = draft_tokens;
        a.uniforms = uniforms;
        a.uniforms64 = uniforms_dtype == CL_DTYPE_F64;
        a.ignore = ignore_index;
        a.seqs = sequences;
        a.drafts = drafts;
        a.cols = cols;
        a.out = tokens;
        a.accepted = accepted;
        a.lp = static_cast<wide_t<T>*>(log_probs);
        a.parts = int(l.parts);
        a.chunks = int(l.chunks);
        const dim3 each = wide_grid(sequences);
        if (l.small) {
            // rows of up to 32 elements a lane: more positions at once
            if (cols <= 512)
                k_small<T, 16><<<each, kThreads, 0, s>>>(a);
            else
                k_small<T, 64><<<each, kThreads, 0, s>>>(a);
            return check_launch("cl_verify_drafts");
        }
        char* ws = static_cast<char*>(workspace);
        a.stats = reinterpret_cast<Stat<wide_t<T>>*>(ws);
        a.draws = reinterpret_cast<Draw*>(ws + l.draws);
        a.sums = reinterpret_cast<double*>(ws + l.sums);
        a.weights = reinterpret_cast<double*>(ws + l.weights);
        const dim3 grid = wide_grid(sequences * l.chunks);
        k_stats<T><<<wide_grid(sequences * (2 * drafts + 1) * l.parts), kStatThreads, 0, s>>>(a);
        if (int rc = check_launch("cl_verify_drafts(stats)")) return rc;
        k_decide<T><<<each, kThreads, 0, s>>>(a);
        if (int rc = check_launch("cl_verify_drafts(decide)")) return rc;
        k_sums<T><<<grid, kDrawThreads, 0, s>>>(a);
        if (int rc = check_launch("cl_verify_drafts(sums)")) return rc;
        k_weights<T><<<grid, kDrawThreads, 0, s>>>(a);
        if (int rc = check_launch("cl_verify_drafts(weights)")) return rc;
        k_pick<T><<<each, kDrawThreads, 0, s>>>(a);
        return check_launch("cl_verify_drafts");
    });
}

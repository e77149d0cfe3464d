// Log probabilities of given classes, entropies and the likeliest classes of every position, and the gradient of all three.
//
// With m the largest logit x_c of a position, d_c = x_c - m, S = sum exp(d_c) and T = sum exp(d_c) d_c over its classes:
//     log p_c = d_c - log S,   H = log S - T / S,   the likeliest by falling x, equal ones by index
//     dx_c = -p_c (g_label + sum g_top) - p_c g_H (log p_c + H), and + g_label, + g_top at the classes that they belong to
// One pass over the logits: m, S and T are carried along, and S and T brought to a new m when one comes up.  What goes into the backward pass is
// m, log S and H of every position, so that it reads the logits once more and writes as much.
//
// Logits of -infinity are classes that cannot be: exp(-infinity) = 0, and d is held at kFar in T, where exp(d) is 0 already.  Where all are, the
// answer is log p = -infinity, H = 0, dx = 0.  A NaN, and an infinity by d = infinity - infinity, makes S a NaN and with it every answer of the position.
#include "kernels.cuh"

namespace simnets {
namespace {

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

template <typename T> __device__ __forceinline__ T infinity() { return T(CUDART_INF_F); }
// exp(kFar) = 0 in both types
template <typename T> __device__ __forceinline__ T far_below() { return sizeof(T) == 4 ? T(-200) : T(-800); }

// m, S and T of the classes seen so far; NaNs are not in m, they are in S
template <typename T>
struct Sums {
    T m, s, t;
    __device__ __forceinline__ void clear() { m = -infinity<T>(); s = T(0); t = T(0); }
    // (from -infinity: S is 0, or NaN and stays one)
    __device__ __forceinline__ void raise(T to) {
        const T by = larger(m - to, far_below<T>()), r = exp_of(by);
        t = r * (t + s * by);
        s *= r;
        m = to;
    }
    // (where nothing can be, m stays -infinity and is no base for differences; what comes together is added up by itself first, which
    // makes the chains of roundings U times shorter)
    template <int U>
    __device__ __forceinline__ void add(const T (&x)[U]) {
        T hi = x[0];
#pragma unroll
        for (int u = 1; u < U; ++u) hi = larger(hi, x[u]);
        if (hi > m) raise(hi);
        const T base = m > -infinity<T>() ? m : T(0);
        T more_s = T(0), more_t = T(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const T d = x[u] - base, e = exp_of(d);
            more_s += e;
            more_t += e * larger(d, far_below<T>());
        }
        s += more_s;
        t += more_t;
    }
    __device__ __forceinline__ void join(Sums o) {
        if (o.m > m) raise(o.m);
        else if (m > -infinity<T>()) o.raise(m);
        s += o.s;
        t += o.t;
    }
};

// the answers of a position: log p_c = (x_c - m) - log_s; nothing: no class can be
template <typename T>
struct Answer {
    T m, log_s, entropy;
    bool nothing;
    __device__ __forceinline__ explicit Answer(const Sums<T>& a) {
        nothing = a.m == -infinity<T>() && a.s == T(0);
        m = a.m;
        log_s = log_of(a.s);
        entropy = nothing ? T(0) : log_s - a.t / a.s;
    }
    __device__ __forceinline__ T of(T x) const { return nothing ? -infinity<T>() : (x - m) - log_s; }
};

// the N largest so far, largest first; equal ones keep the order in which they came, NaN and -infinity are above nothing
template <typename T, int N>
struct Largest {
    T v[N];
    int i[N];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < N; ++j) { v[j] = -infinity<T>(); i[j] = -1; }
    }
    __device__ __forceinline__ void offer(T x, int c) {
        bool above = false;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            above = above || x > v[j];
            const T ov = v[j];
            const int oi = i[j];
            v[j] = above ? x : ov; i[j] = above ? c : oi;
            x = above ? ov : x; c = above ? oi : c;
        }
    }
};
template <typename T>
struct Largest<T, 0> {
    T v[1];
    int i[1];
    __device__ __forceinline__ void clear() {}
    __device__ __forceinline__ void offer(T, int) {}
};

struct Logits {
    long long batch, positions, stride_batch, stride_class, stride_position;
    int classes, top_k, top_last;
    __host__ __device__ long long count() const { return batch * positions; }
    __device__ __forceinline__ long long at(long long q) const { return (q / positions) * stride_batch + (q % positions) * stride_position; }
    // of the place j of the likeliest of position q
    __device__ __forceinline__ long long top_at(long long q, int j) const {
        return top_last ? q * top_k + j : ((q / positions) * top_k + j) * positions + q % positions;
    }
};

// What a position's answers go to; any may be null but stats and the others together.  stats: m, log S, H, each of all positions; where no class can
// be m is +infinity, so that exp(x - m) is 0 whatever x.
template <typename T>
struct Answers {
    const T* logits;
    const long long* labels;
    T *label, *entropy, *top, *stats;
    int* top_index;
};

template <typename T>
__device__ __forceinline__ void write_position(const Logits& g, const Answers<T>& a, long long q, const T* x, const Answer<T>& w) {
    if (a.label) {
        const long long c = a.labels[q];
        a.label[q] = c >= 0 && c < g.classes ? w.of(x[c * g.stride_class]) : T(0);
    }
    if (a.entropy) a.entropy[q] = w.entropy;
    if (a.stats) {
        const long long n = g.count();
        a.stats[q] = w.nothing ? infinity<T>() : w.m;
        a.stats[n + q] = w.nothing ? T(0) : w.log_s;
        a.stats[2 * n + q] = w.entropy;
    }
}

// ---------------------------------------------------------------------------------------------------- a lane a position
constexpr int kAhead = 8;        // loads that a lane has under way

template <typename T, int TOP>
__global__ void __launch_bounds__(128) answer_lanes(Logits g, Answers<T> a) {
    stream_order();
    const long long q = (long long)blockIdx.x * 128 + threadIdx.x;
    if (q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    Sums<T> sums;
    Largest<T, TOP> top;
    sums.clear();
    top.clear();
    for (int c = 0; c < g.classes; c += kAhead) {
        T v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = c + u < g.classes ? x[(c + u) * g.stride_class] : -infinity<T>();
        sums.add(v);
        if (TOP > 0) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) top.offer(v[u], c + u);
        }
    }
    const Answer<T> w(sums);
    write_position(g, a, q, x, w);
#pragma unroll
    for (int j = 0; j < TOP; ++j) {
        if (j >= g.top_k) break;
        a.top_index[g.top_at(q, j)] = top.i[j];
        a.top[g.top_at(q, j)] = top.i[j] < 0 ? -infinity<T>() : w.of(top.v[j]);
    }
}

// What comes in for a position; any of the gradients may be null
template <typename T>
struct Gradients {
    const T* logits;
    const long long* labels;
    const T* stats;
    const int* top_index;
    const T *label, *entropy, *top;
    T* dlogits;
    long long out_batch, out_class, out_position;
};

// a position's share: dx_c = -p_c (taken + g_entropy (log p_c + H)), and what is given to single classes
template <typename T>
struct Share {
    T m, log_s, entropy, g_label, g_entropy, taken;
    long long label;
    bool nothing;
    __device__ __forceinline__ Share(const Logits& g, const Gradients<T>& a, long long q) {
        const long long n = g.count();
        m = a.stats[q];
        log_s = a.stats[n + q];
        entropy = a.stats[2 * n + q];
        nothing = m == infinity<T>() && log_s == T(0);
        label = a.label ? a.labels[q] : -1;
        if (label >= g.classes) label = -1;
        g_label = label >= 0 ? a.label[q] : T(0);
        g_entropy = a.entropy ? a.entropy[q] : T(0);
        taken = g_label;
        if (a.top)
            for (int j = 0; j < g.top_k; ++j)
                if (a.top_index[g.top_at(q, j)] >= 0) taken += a.top[g.top_at(q, j)];
    }
    __device__ __forceinline__ T of(T x) const {
        const T l = (x - m) - log_s, p = exp_of(l);
        return -p * (taken + g_entropy * (larger(l, far_below<T>()) + entropy));
    }
};

template <typename T>
__global__ void __launch_bounds__(128) gradient_lanes(Logits g, Gradients<T> a) {
    stream_order();
    const long long q = (long long)blockIdx.x * 128 + threadIdx.x;
    if (q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    T* dx = a.dlogits + (q / g.positions) * a.out_batch + (q % g.positions) * a.out_position;
    const Share<T> share(g, a, q);
    for (int c = 0; c < g.classes; c += kAhead) {
        T v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = c + u < g.classes ? x[(c + u) * g.stride_class] : -infinity<T>();
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c + u < g.classes) dx[(c + u) * a.out_class] = share.nothing ? T(0) : share.of(v[u]) + (c + u == share.label ? share.g_label : T(0));
    }
    if (a.top && !share.nothing)
        for (int j = 0; j < g.top_k; ++j) {
            const int c = a.top_index[g.top_at(q, j)];
            if (c >= 0 && c < g.classes) dx[c * a.out_class] += a.top[g.top_at(q, j)];
        }
}

Logits logits_of(const simnets_likelihood_desc& d) {
    return {d.batch, d.positions, d.stride_batch, d.stride_class, d.stride_position, d.classes, d.top_k, d.top_last};
}

template <typename T, int TOP>
cudaError_t answer_lanes_of(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    in_stream_order(answer_lanes<T, TOP>, unsigned((g.count() + 127) / 128), 128, 0, s)(g, a);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t answer_as(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    if (g.top_k == 0) return answer_lanes_of<T, 0>(g, a, s);
    if (g.top_k == 1) return answer_lanes_of<T, 1>(g, a, s);
    if (g.top_k <= 4) return answer_lanes_of<T, 4>(g, a, s);
    if (g.top_k <= 8) return answer_lanes_of<T, 8>(g, a, s);
    return answer_lanes_of<T, 16>(g, a, s);
}

template <typename T>
cudaError_t gradient_as(const Logits& g, const Gradients<T>& a, cudaStream_t s) {
    in_stream_order(gradient_lanes<T>, unsigned((g.count() + 127) / 128), 128, 0, s)(g, a);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_log_probabilities(const simnets_likelihood_desc& d, const void* logits, const long long* labels, void* label, void* entropy, int* top_index,
                                     void* top, void* stats, cudaStream_t s) {
    const Logits g = logits_of(d);
    if (g.count() == 0) return cudaSuccess;
    if (d.dtype == SIMNETS_F64)
        return answer_as<double>(g, {(const double*)logits, labels, (double*)label, (double*)entropy, (double*)top, (double*)stats, top_index}, s);
    return answer_as<float>(g, {(const float*)logits, labels, (float*)label, (float*)entropy, (float*)top, (float*)stats, top_index}, s);
}

cudaError_t launch_log_probabilities_gradient(const simnets_likelihood_desc& d, const void* logits, const long long* labels, const void* stats, const int* top_index,
                                              const void* g_label, const void* g_entropy, const void* g_top, void* dlogits, cudaStream_t s) {
    const Logits g = logits_of(d);
    if (g.count() == 0) return cudaSuccess;
    // dlogits is dense in the order of the logits: the classes of a position together where they are, else the positions of a class
    const bool rows = d.stride_class == 1;
    const long long ob = (long long)d.classes * d.positions, oc = rows ? 1 : d.positions, op = rows ? d.classes : 1;
    if (d.dtype == SIMNETS_F64)
        return gradient_as<double>(g, {(const double*)logits, labels, (const double*)stats, top_index, (const double*)g_label, (const double*)g_entropy, (const double*)g_top,
                                       (double*)dlogits, ob, oc, op}, s);
    return gradient_as<float>(g, {(const float*)logits, labels, (const float*)stats, top_index, (const float*)g_label, (const float*)g_entropy, (const float*)g_top,
                                  (float*)dlogits, ob, oc, op}, s);
}

}  // namespace simnets

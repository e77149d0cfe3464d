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
#include <cooperative_groups.h>
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
    // the largest of U more classes, which are added.  (Where nothing can be, m stays -infinity and is no base for differences; what comes together is added up by itself first, which
    // makes the chains of roundings U times shorter)
    template <int U>
    __device__ __forceinline__ T add(const T (&x)[U]) {
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
        return hi;
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

// `x` the logits of position q, `of_label` that of its label
template <typename T>
__device__ __forceinline__ void write_position(const Logits& g, const Answers<T>& a, long long q, T of_label, bool labelled, const Answer<T>& w) {
    if (a.label) a.label[q] = labelled ? w.of(of_label) : T(0);
    if (a.entropy) a.entropy[q] = w.entropy;
    if (a.stats) {
        const long long n = g.count();
        a.stats[q] = w.nothing ? infinity<T>() : w.m;
        a.stats[n + q] = w.nothing ? T(0) : w.log_s;
        a.stats[2 * n + q] = w.entropy;
    }
}

constexpr int kAhead = 8;        // loads that a lane has under way

// ---------------------------------------------------------------------------------------------------- a lane a position
// For maps, whose positions lie side by side, and for rows of so few classes that a warp's rows are a few lines of memory.  Where there
// are few positions several warps share 32 of them, each a run of the classes; what they found is joined pair by pair, lower classes first.
template <typename T, int TOP>
struct Found {
    Sums<T> sums;
    Largest<T, TOP> top;
    static constexpr size_t kBytes = 32 * (3 * sizeof(T) + TOP * (sizeof(T) + sizeof(int)));
    __device__ __forceinline__ void put(char* to, int lane) const {
        T* v = reinterpret_cast<T*>(to) + lane;
        v[0] = sums.m; v[32] = sums.s; v[64] = sums.t;
        int* i = reinterpret_cast<int*>(reinterpret_cast<T*>(to) + 32 * (3 + TOP)) + lane;
#pragma unroll
        for (int j = 0; j < TOP; ++j) { v[32 * (3 + j)] = top.v[j]; i[32 * j] = top.i[j]; }
    }
    __device__ __forceinline__ void join(const char* from, int lane) {
        const T* v = reinterpret_cast<const T*>(from) + lane;
        sums.join({v[0], v[32], v[64]});
        const int* i = reinterpret_cast<const int*>(reinterpret_cast<const T*>(from) + 32 * (3 + TOP)) + lane;
#pragma unroll
        for (int j = 0; j < TOP; ++j) {
            const T x = v[32 * (3 + j)];
            if (!__any_sync(0xffffffffu, x > top.v[TOP - 1])) break;
            top.offer(x, i[32 * j]);
        }
    }
};

// position of a lane, the same for all threads of a column; beyond the last one it is that one again, and nothing is written
__device__ __forceinline__ long long lane_position(const Logits& g, bool* mine) {
    const long long q = ((long long)blockIdx.x * blockDim.z + threadIdx.z) * 32 + threadIdx.x, n = g.count();
    *mine = q < n;
    return q < n ? q : n - 1;
}
// the classes [begin, end) of a warp
__device__ __forceinline__ void warp_classes(const Logits& g, int* begin, int* end) {
    const int share = (g.classes + int(blockDim.y) - 1) / int(blockDim.y);
    *begin = min(g.classes, int(threadIdx.y) * share);
    *end = min(g.classes, *begin + share);
}

template <typename T, int TOP>
__global__ void __launch_bounds__(512) answer_lanes(Logits g, Answers<T> a) {
    stream_order();
    extern __shared__ __align__(16) char room[];
    bool mine;
    const long long q = lane_position(g, &mine);
    const T* x = a.logits + g.at(q);
    const long long label = a.label && threadIdx.y == 0 ? a.labels[q] : -1;
    const bool labelled = label >= 0 && label < g.classes;
    const T of_label = labelled ? x[label * g.stride_class] : T(0);
    Found<T, TOP> f;
    f.sums.clear();
    f.top.clear();
    int begin, end;
    warp_classes(g, &begin, &end);
    for (int c = begin; c < end; c += kAhead) {
        T v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = c + u < end ? x[(c + u) * g.stride_class] : -infinity<T>();
        const T hi = f.sums.add(v);
        if (TOP > 0 && __any_sync(0xffffffffu, hi > f.top.v[TOP > 0 ? TOP - 1 : 0])) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) f.top.offer(v[u], c + u);
        }
    }
    char* at = room + (threadIdx.z * blockDim.y + threadIdx.y) * Found<T, TOP>::kBytes;
    for (int d = 1; d < int(blockDim.y); d *= 2) {
        if (threadIdx.y % (2 * d) == d) f.put(at, threadIdx.x);
        __syncthreads();
        if (threadIdx.y % (2 * d) == 0 && threadIdx.y + d < blockDim.y) f.join(at + d * Found<T, TOP>::kBytes, threadIdx.x);
    }
    if (threadIdx.y != 0 || !mine) return;
    const Answer<T> w(f.sums);
    write_position(g, a, q, of_label, labelled, w);
#pragma unroll
    for (int j = 0; j < TOP; ++j) {
        if (j >= g.top_k) break;
        a.top_index[g.top_at(q, j)] = f.top.i[j];
        a.top[g.top_at(q, j)] = f.top.i[j] < 0 ? -infinity<T>() : w.of(f.top.v[j]);
    }
}

// ----------------------------------------------------------------------------------------------- several lanes a position
// For rows, whose classes lie side by side: a warp, a CTA or a cluster of CTAs a row.  The largest so far are a list of the warp, the j-th of them in
// lane j; a class is compared with the last one that counts, and only one above it moves the list.
template <typename T>
struct WarpList {
    T v, last;               // this lane's value; the value of place top_k - 1
    int i;
    __device__ __forceinline__ void clear() { v = last = -infinity<T>(); i = -1; }
    __device__ __forceinline__ void insert(T x, int c, int top_k) {
        // (a free place is -infinity and -1, the largest of unsigned indices)
        const unsigned behind = __ballot_sync(0xffffffffu, x > v || (x == v && unsigned(c) < unsigned(i)));
        const T up = __shfl_up_sync(0xffffffffu, v, 1);
        const int up_i = __shfl_up_sync(0xffffffffu, i, 1);
        const int lane = threadIdx.x % 32, place = __ffs(behind) - 1;
        if (behind && lane >= place) { v = lane == place ? x : up; i = lane == place ? c : up_i; }
        last = __shfl_sync(0xffffffffu, v, top_k - 1);
    }
    // one value of each lane, of class `first` + lane; those in the list are of lower classes, or of these
    __device__ __forceinline__ void offer(T x, int first, int top_k) {
        unsigned who = __ballot_sync(0xffffffffu, x > last);
        while (who) {
            const int from = __ffs(who) - 1;
            insert(__shfl_sync(0xffffffffu, x, from), first + from, top_k);
            who &= ~(1u << from) & __ballot_sync(0xffffffffu, x > last);
        }
    }
    // another list, place j of it in lane j
    __device__ __forceinline__ void join(T x, int c, int top_k) {
        for (int j = 0; j < top_k; ++j) {
            const T xj = __shfl_sync(0xffffffffu, x, j);
            if (!(xj >= last) || xj == -infinity<T>()) break;
            insert(xj, __shfl_sync(0xffffffffu, c, j), top_k);
        }
    }
};

template <typename T>
__device__ __forceinline__ Sums<T> over_warp(Sums<T> a) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const Sums<T> o = {__shfl_xor_sync(0xffffffffu, a.m, d), __shfl_xor_sync(0xffffffffu, a.s, d), __shfl_xor_sync(0xffffffffu, a.t, d)};
        a.join(o);
    }
    return a;
}

// what a warp, and then a CTA, found
template <typename T>
struct RowFound {
    Sums<T> sums;
    T top[16];
    int top_index[16];
};

// WARPS = 1: a warp a row, kRowWarps rows a CTA; else a cluster of gridDim.y CTAs of WARPS warps a row
constexpr int kRowWarps = 8;
template <typename T, bool TOP, int WARPS>
__global__ void __launch_bounds__(32 * (WARPS == 1 ? kRowWarps : WARPS)) answer_rows(Logits g, Answers<T> a) {
    stream_order();
    __shared__ RowFound<T> found[WARPS == 1 ? 1 : WARPS];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const long long q = WARPS == 1 ? (long long)blockIdx.x * kRowWarps + warp : blockIdx.x;
    if (WARPS == 1 && q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    const long long label = a.label ? a.labels[q] : -1;
    const bool labelled = label >= 0 && label < g.classes;
    const T of_label = labelled ? x[label] : T(0);
    Sums<T> sums;
    WarpList<T> list;
    sums.clear();
    list.clear();
    constexpr int kStep = 32 * WARPS;
    const int span = kStep * kAhead;
    for (long long c0 = (WARPS == 1 ? 0LL : (long long)blockIdx.y * span) + 32 * (WARPS == 1 ? 0 : warp); c0 < g.classes; c0 += (long long)span * gridDim.y) {
        T v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = c0 + u * kStep + lane < g.classes ? x[c0 + u * kStep + lane] : -infinity<T>();
        const T hi = sums.add(v);
        if (TOP && __any_sync(0xffffffffu, hi > list.last)) {
#pragma unroll 1
            for (int u = 0; u < kAhead; ++u) {
                T x_u = v[0];
#pragma unroll
                for (int w = 1; w < kAhead; ++w) x_u = u == w ? v[w] : x_u;
                list.offer(x_u, int(c0) + u * kStep, g.top_k);
            }
        }
    }
    sums = over_warp(sums);
    if (WARPS > 1) {
        // the warps of the CTA, then the CTAs of the cluster, into the first of them
        const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        RowFound<T>& own = found[warp];
        if (lane == 0) own.sums = sums;
        if (TOP && lane < 16) { own.top[lane] = list.v; own.top_index[lane] = list.i; }
        __syncthreads();
        if (warp == 0) {
            if (TOP)
                for (int w = 1; w < WARPS; ++w) list.join(lane < 16 ? found[w].top[lane] : -infinity<T>(), lane < 16 ? found[w].top_index[lane] : -1, g.top_k);
            sums.clear();
            if (lane < WARPS) sums = found[lane].sums;
            sums = over_warp(sums);
        }
        if (gridDim.y > 1) {
            __syncwarp();
            if (warp == 0 && lane == 0) own.sums = sums;
            if (TOP && warp == 0 && lane < 16) { own.top[lane] = list.v; own.top_index[lane] = list.i; }
            cluster.sync();
            if (warp == 0 && blockIdx.y == 0) {
                sums.clear();
                if (lane < int(gridDim.y)) sums = cluster.map_shared_rank(found, lane)->sums;
                sums = over_warp(sums);
                if (TOP)
                    for (int r = 1; r < int(gridDim.y); ++r) {
                        const RowFound<T>* other = cluster.map_shared_rank(found, r);
                        list.join(lane < 16 ? other->top[lane] : -infinity<T>(), lane < 16 ? other->top_index[lane] : -1, g.top_k);
                    }
            }
            cluster.sync();
        }
        if (warp != 0 || blockIdx.y != 0) return;
    }
    const Answer<T> w(sums);
    if (lane == 0) write_position(g, a, q, of_label, labelled, w);
    if (TOP && lane < g.top_k) {
        a.top_index[g.top_at(q, lane)] = list.i;
        a.top[g.top_at(q, lane)] = list.i < 0 ? -infinity<T>() : w.of(list.v);
    }
}

// ----------------------------------------------------------------------------------------------------------- the gradient
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
    __device__ __forceinline__ T of(T x, long long c) const {
        const T l = (x - m) - log_s, p = exp_of(l);
        const T dx = -p * (taken + g_entropy * (larger(l, far_below<T>()) + entropy));
        return nothing ? T(0) : c == label ? dx + g_label : dx;
    }
};

template <typename T>
__global__ void __launch_bounds__(512) gradient_lanes(Logits g, Gradients<T> a) {
    stream_order();
    bool mine;
    const long long q = lane_position(g, &mine);
    if (!mine) return;
    const T* x = a.logits + g.at(q);
    T* dx = a.dlogits + (q / g.positions) * a.out_batch + (q % g.positions) * a.out_position;
    const Share<T> share(g, a, q);
    int begin, end;
    warp_classes(g, &begin, &end);
    for (int c = begin; c < end; c += kAhead) {
        T v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = c + u < end ? x[(c + u) * g.stride_class] : -infinity<T>();
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c + u < end) dx[(c + u) * a.out_class] = share.of(v[u], c + u);
    }
    if (a.top && !share.nothing)
        for (int j = 0; j < g.top_k; ++j) {
            const int c = a.top_index[g.top_at(q, j)];
            if (c >= begin && c < end) dx[c * a.out_class] += a.top[g.top_at(q, j)];
        }
}

// WARPS = 1: a warp a row; else CTAs of WARPS warps share a row, blockIdx.y of them each kSegment classes
template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * (WARPS == 1 ? kRowWarps : WARPS)) gradient_rows(Logits g, Gradients<T> a) {
    stream_order();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const long long q = WARPS == 1 ? (long long)blockIdx.x * kRowWarps + warp : blockIdx.x;
    if (WARPS == 1 && q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    T* dx = a.dlogits + (q / g.positions) * a.out_batch + (q % g.positions) * a.out_position;
    const Share<T> share(g, a, q);
    constexpr int kStep = 32 * WARPS;
    const long long segment = ((g.classes + gridDim.y - 1) / gridDim.y + 31) / 32 * 32;
    const long long begin = blockIdx.y * segment, end = begin + segment < g.classes ? begin + segment : g.classes;
    for (long long c0 = begin + (WARPS == 1 ? lane : threadIdx.x); c0 < end; c0 += kStep * kAhead) {
        T v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) v[u] = c0 + u * kStep < end ? x[c0 + u * kStep] : -infinity<T>();
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c0 + u * kStep < end) dx[c0 + u * kStep] = share.of(v[u], c0 + u * kStep);
    }
    if (a.top) {
        if (WARPS == 1) __syncwarp();
        else __syncthreads();
        if (!share.nothing && (WARPS == 1 || warp == 0) && lane < g.top_k) {
            const int c = a.top_index[g.top_at(q, lane)];
            if (c >= begin && c < end) dx[c] += a.top[g.top_at(q, lane)];
        }
    }
}

// --------------------------------------------------------------------------------------------------------------- launches
Logits logits_of(const simnets_likelihood_desc& d) {
    return {d.batch, d.positions, d.stride_batch, d.stride_class, d.stride_position, d.classes, d.top_k, d.top_last};
}

// rows of more classes than this are read by several lanes
bool by_rows(const Logits& g) { return g.stride_class == 1 && g.classes > 32; }

// warps that share 32 positions
int warps_of_lanes(const Logits& g, size_t bytes_a_warp) {
    const long long tiles = (g.count() + 31) / 32;
    int w = 1;
    while (w < 16 && tiles * w < 32LL * device_sm_count() && g.classes >= 2 * w * kAhead && 2 * w * bytes_a_warp <= 48 * 1024) w *= 2;
    return w;
}

template <class Kernel, class A>
cudaError_t launch_lanes(Kernel* kernel, const Logits& g, const A& a, int warps, size_t bytes_a_warp, cudaStream_t s) {
    const int tiles = warps < 4 ? 4 / warps : 1;
    const unsigned grid = unsigned((g.count() + 32 * tiles - 1) / (32 * tiles));
    in_stream_order(kernel, grid, dim3(32, warps, tiles), warps > 1 ? bytes_a_warp * warps * tiles : 0, s)(g, a);
    count_launch();
    return cudaGetLastError();
}

template <typename T, int TOP>
cudaError_t answer_lanes_of(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    return launch_lanes(answer_lanes<T, TOP>, g, a, warps_of_lanes(g, Found<T, TOP>::kBytes), Found<T, TOP>::kBytes, s);
}

template <typename T, bool TOP>
cudaError_t answer_rows_of(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    if (g.classes <= 1024) {
        in_stream_order(answer_rows<T, TOP, 1>, unsigned((g.count() + kRowWarps - 1) / kRowWarps), 32 * kRowWarps, 0, s)(g, a);
    } else {
        int cluster = 1;
        while (cluster < 8 && g.count() * cluster < 2LL * device_sm_count() && g.classes > 2048 * cluster) cluster *= 2;
        const dim3 grid(unsigned(g.count()), cluster);
        if (cluster > 1) in_stream_order(answer_rows<T, TOP, 32>, grid, 1024, 0, s, cluster)(g, a);
        else in_stream_order(answer_rows<T, TOP, 8>, grid, 256, 0, s)(g, a);
    }
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t answer_as(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    if (by_rows(g)) return g.top_k > 0 ? answer_rows_of<T, true>(g, a, s) : answer_rows_of<T, false>(g, a, s);
    if (g.top_k == 0) return answer_lanes_of<T, 0>(g, a, s);
    if (g.top_k == 1) return answer_lanes_of<T, 1>(g, a, s);
    if (g.top_k <= 4) return answer_lanes_of<T, 4>(g, a, s);
    if (g.top_k <= 8) return answer_lanes_of<T, 8>(g, a, s);
    return answer_lanes_of<T, 16>(g, a, s);
}

template <typename T>
cudaError_t gradient_as(const Logits& g, const Gradients<T>& a, cudaStream_t s) {
    if (!by_rows(g)) return launch_lanes(gradient_lanes<T>, g, a, warps_of_lanes(g, 0), 0, s);
    if (g.classes <= 1024) {
        in_stream_order(gradient_rows<T, 1>, unsigned((g.count() + kRowWarps - 1) / kRowWarps), 32 * kRowWarps, 0, s)(g, a);
    } else {
        const dim3 grid(unsigned(g.count()), (g.classes + 8191) / 8192 < 65535 ? (g.classes + 8191) / 8192 : 65535);
        in_stream_order(gradient_rows<T, 8>, grid, 256, 0, s)(g, a);
    }
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

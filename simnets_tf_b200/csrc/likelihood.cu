// Log probabilities of given classes, entropies and the likeliest classes of every position, and the gradient of all three.
//
// With m the largest logit x_c of a position, d_c = x_c - m, S = sum exp(d_c) and T = sum exp(d_c) d_c over its classes:
//     log p_c = d_c - log S,   H = log S - T / S,   the likeliest by falling x, equal ones by index
//     dx_c = -p_c (g_label + sum g_top) - p_c g_H (log p_c + H), and + g_label, + g_top at the classes that they belong to
// One pass over the logits: m, S and T are carried along, and S and T brought to a new m when one comes up.  What goes into the backward pass is
// m, log S and H of every position, so that it reads the logits once more and writes as much.
//
// Logits of -infinity are classes that cannot be: exp(-infinity) = 0, and in T d is held where exp(d) is 0 already.  Where all are, the
// answer is log p = -infinity, H = 0, dx = 0.  A NaN, and an infinity by d = infinity - infinity, makes S a NaN and with it every answer of the position.
#include <cooperative_groups.h>
#include "kernels.cuh"

namespace simnets {
namespace {

__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

template <typename T> __device__ __forceinline__ T infinity() { return T(CUDART_INF_F); }

// Exponents are counted in units in which an exponential is one instruction: float32 in powers of two, whose instruction is off by up to 2^-22 of the
// value, as much as rounding a difference of 4 nats; float64 in nats.
template <typename T> struct Unit;
template <> struct Unit<float> {
    static __device__ __forceinline__ float per_nat() { return 1.4426950408889634f; }
    static __device__ __forceinline__ float nats() { return 0.6931471805599453f; }
    static __device__ __forceinline__ float exp(float u) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(u)); return r; }
    // exp of it is 0
    static __device__ __forceinline__ float far_below() { return -300.f; }
};
template <> struct Unit<double> {
    static __device__ __forceinline__ double per_nat() { return 1.0; }
    static __device__ __forceinline__ double nats() { return 1.0; }
    static __device__ __forceinline__ double exp(double u) { return ::exp(u); }
    static __device__ __forceinline__ double far_below() { return -800.0; }
};

// Two values that one instruction adds, multiplies, or multiplies and adds (float32; float64 in two).
template <typename T> struct Pair { T x, y; };
__device__ __forceinline__ unsigned long long bits(Pair<float> p) { unsigned long long r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(p.x), "f"(p.y)); return r; }
__device__ __forceinline__ Pair<float> pair(unsigned long long b) { Pair<float> p; asm("mov.b64 {%0, %1}, %2;" : "=f"(p.x), "=f"(p.y) : "l"(b)); return p; }
__device__ __forceinline__ Pair<float> add2(Pair<float> a, Pair<float> b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ Pair<float> mul2(Pair<float> a, Pair<float> b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ Pair<float> fma2(Pair<float> a, Pair<float> b, Pair<float> c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return pair(r);
}
__device__ __forceinline__ Pair<double> add2(Pair<double> a, Pair<double> b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ Pair<double> mul2(Pair<double> a, Pair<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Pair<double> fma2(Pair<double> a, Pair<double> b, Pair<double> c) { return {::fma(a.x, b.x, c.x), ::fma(a.y, b.y, c.y)}; }
template <typename T> __device__ __forceinline__ Pair<T> both(T v) { return {v, v}; }
template <typename T> __device__ __forceinline__ Pair<T> exp_both(Pair<T> u) { return {Unit<T>::exp(u.x), Unit<T>::exp(u.y)}; }
template <typename T> __device__ __forceinline__ Pair<T> not_far(Pair<T> u) { return {larger(u.x, Unit<T>::far_below()), larger(u.y, Unit<T>::far_below())}; }

// m, S and T (in units) of the classes seen so far; NaNs are not in m, they are in S
template <typename T>
struct Sums {
    T m, s, t;
    __device__ __forceinline__ void clear() { m = -infinity<T>(); s = T(0); t = T(0); }
    // (from -infinity: S is 0, or NaN and stays one)
    __device__ __forceinline__ void raise(T to) {
        const T by = larger((m - to) * Unit<T>::per_nat(), Unit<T>::far_below()), r = Unit<T>::exp(by);
        t = r * (t + s * by);
        s *= r;
        m = to;
    }
    // the largest of U more classes, which are added.  (Where nothing can be, m stays -infinity and is no base for differences; what comes together
    // is added up by itself first, which makes the chains of roundings shorter.)
    template <int U>
    __device__ __forceinline__ T add(const T (&x)[U]) {
        T hi = x[0];
#pragma unroll
        for (int u = 1; u < U; ++u) hi = larger(hi, x[u]);
        if (hi > m) raise(hi);
        const Pair<T> base = both(m > -infinity<T>() ? -m : T(0)), unit = both(Unit<T>::per_nat());
        Pair<T> more_s = both(T(0)), more_t = both(T(0));
#pragma unroll
        for (int i = 0; i < U; i += 2) {
            const Pair<T> u = mul2(add2(Pair<T>{x[i], x[i + 1]}, base), unit), e = exp_both(u);
            more_s = add2(more_s, e);
            more_t = fma2(e, not_far(u), more_t);
        }
        s += more_s.x + more_s.y;
        t += more_t.x + more_t.y;
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
        entropy = nothing ? T(0) : log_s - Unit<T>::nats() * (a.t / a.s);
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

// kAhead classes from `at` on, which moves behind them; `left` of them are there
template <typename T>
__device__ __forceinline__ void load_classes(T (&v)[kAhead], const T*& at, long long stride, int left) {
    if (left >= kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) { v[u] = *at; at += stride; }
    } else {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) { v[u] = u < left ? *at : -infinity<T>(); at += u < left ? stride : 0; }
    }
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
    const T* at_class = x + begin * g.stride_class;
    for (int c = begin; c < end; c += kAhead) {
        T v[kAhead];
        load_classes(v, at_class, g.stride_class, end - c);
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
// For rows, whose classes lie side by side: a warp, a CTA or a cluster of CTAs a row, 16 bytes a load.  Rows start anywhere: chunks are counted from
// the 16-byte boundary in front of a row.
template <typename T> struct Bytes16;
template <> struct Bytes16<float> { using type = float4; };
template <> struct Bytes16<double> { using type = double2; };
template <typename T> constexpr int kWide = 16 / sizeof(T);

template <typename T>
__device__ __forceinline__ int in_front(const T* x) { return int(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)); }

// The share of thread `tid` of THREADS in the U * THREADS classes from `first` on; value u is class first + class_in_chunk(tid, u).
template <typename T, int THREADS>
__device__ __forceinline__ int class_in_chunk(int tid, int u) { return (u / kWide<T> * THREADS + tid) * kWide<T> + u % kWide<T>; }
template <typename T, int U, int THREADS>
__device__ __forceinline__ void load_chunk(T (&v)[U], const T* x, long long first, int classes, int tid) {
    const bool inside = first >= 0 && first + U * THREADS <= classes;
#pragma unroll
    for (int j = 0; j < U; j += kWide<T>) {
        const long long c = first + class_in_chunk<T, THREADS>(tid, j);
        if (inside || (c >= 0 && c + kWide<T> <= classes)) {
            *reinterpret_cast<typename Bytes16<T>::type*>(v + j) = *reinterpret_cast<const typename Bytes16<T>::type*>(x + c);
        } else {
#pragma unroll
            for (int e = 0; e < kWide<T>; ++e) v[j + e] = c + e >= 0 && c + e < classes ? x[c + e] : -infinity<T>();
        }
    }
}
template <typename T, int U, int THREADS>
__device__ __forceinline__ void store_chunk(const T (&v)[U], T* x, bool aligned, long long first, int classes, int tid) {
    const bool inside = aligned && first >= 0 && first + U * THREADS <= classes;
#pragma unroll
    for (int j = 0; j < U; j += kWide<T>) {
        const long long c = first + class_in_chunk<T, THREADS>(tid, j);
        if (inside || (aligned && c >= 0 && c + kWide<T> <= classes)) {
            *reinterpret_cast<typename Bytes16<T>::type*>(x + c) = *reinterpret_cast<const typename Bytes16<T>::type*>(v + j);
        } else {
#pragma unroll
            for (int e = 0; e < kWide<T>; ++e)
                if (c + e >= 0 && c + e < classes) x[c + e] = v[j + e];
        }
    }
}

// Numbers as unsigned ones in the same order (-0 as 0)
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float number(unsigned k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ unsigned long long ordered(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v + 0.0);
    return b ^ (b >> 63 ? ~0ULL : 1ULL << 63);
}
__device__ __forceinline__ double number(unsigned long long k) { return __longlong_as_double((long long)(k ^ (k >> 63 ? 1ULL << 63 : ~0ULL))); }
template <typename T> struct KeyOf;
template <> struct KeyOf<float> { using type = unsigned; };
template <> struct KeyOf<double> { using type = unsigned long long; };

__device__ __forceinline__ float warp_max(float v) { return number(__reduce_max_sync(0xffffffffu, ordered(v))); }
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = larger(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
// the k-th largest of the lanes' values
template <typename T>
__device__ __forceinline__ T warp_largest(T v, int k) {
    T best = -infinity<T>();
    for (int j = 0; j < k; ++j) {
        best = warp_max(v);
        const unsigned who = __ballot_sync(0xffffffffu, v == best);
        if (int(threadIdx.x % 32) == __ffs(who) - 1) v = -infinity<T>();
    }
    return best;
}

// The largest so far as a list of the warp, the j-th of them in lane j.  A class is compared with the last one that counts, and only one above it moves
// the list: a row of n classes in any order moves it about top_k log(n / top_k) times.
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
    // The classes of a chunk (see load_chunk), all behind those that were offered before, `hi` the lane's largest.  Those below `bound` are known not
    // to be among the top_k.
    template <int THREADS, int U>
    __device__ __forceinline__ void offer(const T (&x)[U], T hi, T bound, long long first, int top_k) {
        if (!__any_sync(0xffffffffu, hi > last && hi >= bound)) return;
        unsigned mine = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) mine |= x[u] > last && x[u] >= bound ? 1u << u : 0u;
        while (const unsigned who = __ballot_sync(0xffffffffu, mine)) {
            const int from = __ffs(who) - 1, u = __shfl_sync(0xffffffffu, __ffs(mine) - 1, from);
            T xu = x[0];
#pragma unroll
            for (int w = 1; w < U; ++w) xu = u == w ? x[w] : xu;
            xu = __shfl_sync(0xffffffffu, xu, from);
            if (xu >= last) insert(xu, int(first + class_in_chunk<T, THREADS>((THREADS == 32 ? 0 : int(threadIdx.x) / 32 * 32) + from, u)), top_k);
            if (int(threadIdx.x % 32) == from) mine &= mine - 1;
        }
    }
};

// what a warp, and then a CTA, found
template <typename T>
struct RowFound {
    Sums<T> sums;
    T top[16];
    int top_index[16];
};

// the best of the lanes' values, the lowest index of equal ones
__device__ __forceinline__ void warp_best(float& v, int& i) {
    const unsigned key = ordered(v), best = __reduce_max_sync(0xffffffffu, key);
    i = int(__reduce_min_sync(0xffffffffu, key == best ? unsigned(i) : 0xffffffffu));
    v = number(best);
}
__device__ __forceinline__ void warp_best(double& v, int& i) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const double ov = __shfl_xor_sync(0xffffffffu, v, d);
        const int oi = __shfl_xor_sync(0xffffffffu, i, d);
        if (ov > v || (ov == v && unsigned(oi) < unsigned(i))) { v = ov; i = oi; }
    }
}
// the lists of `count` rows of `found` (32 at most) as one: each lane looks at the front of one of them, and the best of these goes into the list
template <typename T>
__device__ __forceinline__ void join_lists(WarpList<T>& list, const RowFound<T>* found, int count, int top_k) {
    const int lane = threadIdx.x % 32;
    list.clear();
    int place = 0;
    T v = lane < count ? found[lane].top[0] : -infinity<T>();
    int i = lane < count ? found[lane].top_index[0] : -1;
    for (int j = 0; j < top_k; ++j) {
        T best = v;
        int best_i = i;
        warp_best(best, best_i);
        if (best_i < 0) break;
        if (lane == j) { list.v = best; list.i = best_i; }
        if (i == best_i) {
            ++place;
            v = place < top_k ? found[lane].top[place] : -infinity<T>();
            i = place < top_k ? found[lane].top_index[place] : -1;
        }
    }
}

template <typename T>
__device__ __forceinline__ Sums<T> over_warp(Sums<T> a) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const Sums<T> o = {__shfl_xor_sync(0xffffffffu, a.m, d), __shfl_xor_sync(0xffffffffu, a.s, d), __shfl_xor_sync(0xffffffffu, a.t, d)};
        a.join(o);
    }
    return a;
}

// WARPS = 1: a warp a row, kRowWarps rows a CTA; else a cluster of gridDim.y CTAs of WARPS warps a row
constexpr int kRowWarps = 8;
template <int WARPS> constexpr int kRowAhead = WARPS == 1 ? 4 : 8;
template <typename T, bool TOP, int WARPS>
__global__ void __launch_bounds__(32 * (WARPS == 1 ? kRowWarps : WARPS)) answer_rows(Logits g, Answers<T> a) {
    using Key = typename KeyOf<T>::type;
    stream_order();
    __shared__ RowFound<T> found[WARPS == 1 ? 1 : WARPS];
    __shared__ Key shared_bound;            // the largest value that a warp's list ends with
    constexpr int U = kRowAhead<WARPS>, kThreads = 32 * WARPS;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, tid = WARPS == 1 ? lane : int(threadIdx.x);
    const long long q = WARPS == 1 ? (long long)blockIdx.x * kRowWarps + warp : blockIdx.x;
    if (WARPS == 1 && q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    const bool writes = lane == 0 && (WARPS == 1 || (warp == 0 && blockIdx.y == 0));
    const long long label = a.label && writes ? a.labels[q] : -1;
    const bool labelled = label >= 0 && label < g.classes;
    const T of_label = labelled ? x[label] : T(0);
    Sums<T> sums;
    WarpList<T> list;
    sums.clear();
    list.clear();
    if (TOP && WARPS > 1) {
        if (threadIdx.x == 0) shared_bound = ordered(-infinity<T>());
        __syncthreads();
    }
    const long long step = (long long)kThreads * U * (WARPS == 1 ? 1 : gridDim.y);
    long long first = (WARPS == 1 ? 0LL : (long long)blockIdx.y * kThreads * U) - in_front(x);
    T v[U];
    if (first < g.classes) load_chunk<T, U, kThreads>(v, x, first, g.classes, tid);
    for (bool start = true; first < g.classes; first += step, start = false) {
        T next[U];
        if (first + step < g.classes) load_chunk<T, U, kThreads>(next, x, first + step, g.classes, tid);
        const T hi = sums.add(v);
        if (TOP) {
            // at the start at least top_k of the warp's classes are not below the k-th largest of the lanes' largest
            // (of a lane all of whose classes are NaN, hi is one too)
            T bound = start ? warp_largest(hi == hi ? hi : -infinity<T>(), g.top_k) : -infinity<T>();
            if (WARPS > 1) {
                if (start && lane == 0) atomicMax(&shared_bound, ordered(bound));
                bound = larger(bound, number(*static_cast<volatile Key*>(&shared_bound)));
            }
            const T before = list.last;
            list.template offer<kThreads>(v, hi, bound, first, g.top_k);
            if (WARPS > 1 && lane == 0 && list.last > before) atomicMax(&shared_bound, ordered(list.last));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
    }
    sums = over_warp(sums);
    if (WARPS > 1) {
        // the warps of the CTA, then the CTAs of the cluster, into the first of them
        if (lane == 0) found[warp].sums = sums;
        if (TOP && lane < 16) { found[warp].top[lane] = list.v; found[warp].top_index[lane] = list.i; }
        __syncthreads();
        if (warp == 0) {
            sums.clear();
            if (lane < WARPS) sums = found[lane].sums;
            sums = over_warp(sums);
            if (TOP) join_lists(list, found, WARPS, g.top_k);
        }
        if (gridDim.y > 1) {
            const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
            __syncwarp();
            if (warp == 0 && lane == 0) found[0].sums = sums;
            if (TOP && warp == 0 && lane < 16) { found[0].top[lane] = list.v; found[0].top_index[lane] = list.i; }
            cluster.sync();
            if (warp == 0 && blockIdx.y == 0) {
                const int others = int(gridDim.y);
                sums.clear();
                if (lane < others) sums = cluster.map_shared_rank(found, lane)->sums;
                sums = over_warp(sums);
                if (TOP) {
                    // (one list a warp of this CTA was joined already: their places take the other CTAs' lists)
                    for (int e = lane; e < others * 16; e += 32) {
                        const RowFound<T>* other = cluster.map_shared_rank(found, e / 16);
                        const T top = other->top[e % 16];
                        const int index = other->top_index[e % 16];
                        if (e >= 16) { found[e / 16].top[e % 16] = top; found[e / 16].top_index[e % 16] = index; }
                    }
                    __syncwarp();
                    join_lists(list, found, others, g.top_k);
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

// a position's share: -p_c (g_label + sum g_top + g_entropy (log p_c + H)) = p_c (fixed + by_log log p_c), and what is given to single classes
template <typename T>
struct Share {
    T m, log_s, fixed, by_log, g_label;
    long long label;
    bool nothing;
    __device__ __forceinline__ Share(const Logits& g, const Gradients<T>& a, long long q) {
        const long long n = g.count();
        m = a.stats[q];
        const T log_nats = a.stats[n + q];
        nothing = m == infinity<T>() && log_nats == T(0);
        log_s = log_nats * Unit<T>::per_nat();
        label = a.label ? a.labels[q] : -1;
        if (label < 0 || label >= g.classes || nothing) label = -1;
        g_label = label >= 0 ? a.label[q] : T(0);
        T taken = g_label;
        if (a.top)
            for (int j = 0; j < g.top_k; ++j)
                if (a.top_index[g.top_at(q, j)] >= 0) taken += a.top[g.top_at(q, j)];
        const T g_entropy = a.entropy ? a.entropy[q] : T(0);
        fixed = nothing ? T(0) : -(taken + g_entropy * a.stats[2 * n + q]);
        by_log = nothing ? T(0) : -g_entropy * Unit<T>::nats();
    }
    __device__ __forceinline__ Pair<T> of(Pair<T> x) const {
        const Pair<T> u = fma2(add2(x, both(-m)), both(Unit<T>::per_nat()), both(-log_s));
        return mul2(exp_both(u), fma2(both(by_log), not_far(u), both(fixed)));
    }
    template <int U>
    __device__ __forceinline__ void of(T (&x)[U]) const {
#pragma unroll
        for (int u = 0; u < U; u += 2) {
            const Pair<T> dx = of(Pair<T>{x[u], x[u + 1]});
            x[u] = dx.x;
            x[u + 1] = dx.y;
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(512) gradient_lanes(Logits g, Gradients<T> a) {
    stream_order();
    bool mine;
    const long long q = lane_position(g, &mine);
    if (!mine) return;
    T* dx = a.dlogits + (q / g.positions) * a.out_batch + (q % g.positions) * a.out_position;
    const Share<T> share(g, a, q);
    int begin, end;
    warp_classes(g, &begin, &end);
    const T* at_class = a.logits + g.at(q) + begin * g.stride_class;
    T* to = dx + begin * a.out_class;
    for (int c = begin; c < end; c += kAhead) {
        T v[kAhead];
        load_classes(v, at_class, g.stride_class, end - c);
        share.of(v);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u < end - c) { *to = v[u]; to += a.out_class; }
    }
    if (share.label >= begin && share.label < end) dx[share.label * a.out_class] += share.g_label;
    if (a.top && !share.nothing)
        for (int j = 0; j < g.top_k; ++j) {
            const int c = a.top_index[g.top_at(q, j)];
            if (c >= begin && c < end) dx[c * a.out_class] += a.top[g.top_at(q, j)];
        }
}

// WARPS = 1: a warp a row; else gridDim.y CTAs of WARPS warps share a row, a run of its classes each
template <typename T, int WARPS>
__global__ void __launch_bounds__(32 * (WARPS == 1 ? kRowWarps : WARPS)) gradient_rows(Logits g, Gradients<T> a) {
    stream_order();
    constexpr int U = kRowAhead<WARPS>, kThreads = 32 * WARPS;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, tid = WARPS == 1 ? lane : int(threadIdx.x);
    const long long q = WARPS == 1 ? (long long)blockIdx.x * kRowWarps + warp : blockIdx.x;
    if (WARPS == 1 && q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    T* dx = a.dlogits + (q / g.positions) * a.out_batch + (q % g.positions) * a.out_position;
    const Share<T> share(g, a, q);
    const int skip = in_front(x);
    const bool aligned = in_front(dx) == skip;
    // whole chunks a CTA
    const long long chunks = (g.classes + skip + kThreads * U - 1) / (kThreads * U), each = (chunks + gridDim.y - 1) / gridDim.y;
    const long long begin = blockIdx.y * each * kThreads * U - skip, end = begin + each * kThreads * U;
    // single classes, which get more: written once the others have been
    const int place = WARPS == 1 || warp == 0 ? lane : 32;
    long long single = -1;
    T add = T(0);
    if (place < 32) {
        const int c = place < g.top_k && a.top ? a.top_index[g.top_at(q, place)] : -1;
        const bool both_ways = __any_sync(0xffffffffu, c >= 0 && c == share.label);
        if (c >= 0) { single = c; add = (c == share.label ? share.g_label : T(0)); }
        if (place == 31 && share.label >= 0 && !both_ways) { single = share.label; add = share.g_label; }
        if (share.nothing || single >= g.classes || single < begin || single >= end) single = -1;
        if (single >= 0) {
            add += share.of(Pair<T>{x[single], x[single]}).x;
            if (c >= 0) add += a.top[g.top_at(q, place)];
        }
    }
    for (long long first = begin; first < end && first < g.classes; first += kThreads * U) {
        T v[U];
        load_chunk<T, U, kThreads>(v, x, first, g.classes, tid);
        share.of(v);
        store_chunk<T, U, kThreads>(v, dx, aligned, first, g.classes, tid);
    }
    if (WARPS == 1) __syncwarp();
    else __syncthreads();
    if (single >= 0) dx[single] = add;
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
        const dim3 grid(unsigned(g.count()), std::min((g.classes + 8191) / 8192, 65535));
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

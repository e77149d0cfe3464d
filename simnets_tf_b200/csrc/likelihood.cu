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

// Two values that one instruction adds, multiplies, or multiplies and adds (float32; float64 in two).  With / without, us: 2048 rows of 65537 classes with
// five alternatives 96 / 100, the gradient of 20000 rows of 500 20.3 / 22.9.  (Times here are of kernels back to back for some milliseconds, at 1.97 GHz; under the
// power limit, after some hundred milliseconds, the clock is 1.63 GHz and these 96 are 108.)
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
        entropy = log_s - Unit<T>::nats() * (a.t / a.s);
        if (nothing || entropy < T(0)) entropy = T(0);                // (of one class that is nearly sure, by rounding)
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
    __device__ __forceinline__ void offer(T x, int c) { put<false>(x, c); }
    // in any order: of equal ones the lowest index is the first (a free place has -1, the largest of unsigned ones)
    __device__ __forceinline__ void offer_any(T x, int c) { put<true>(x, c); }
    template <bool ANY>
    __device__ __forceinline__ void put(T x, int c) {
        bool above = false;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            above = above || x > v[j] || (ANY && x == v[j] && x > -infinity<T>() && unsigned(c) < unsigned(i[j]));
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
    // where position q = b * positions + p is in an array with these steps; the places of the likeliest of a position are top_step apart from
    // top_first on.  (A division of 64-bit numbers is a hundred instructions, as many as a dozen classes take.)
    __device__ __forceinline__ long long at(long long q, long long of_batch, long long of_position) const {
        if (batch == 1) return q * of_position;
        if ((unsigned long long)q >> 32 || (unsigned long long)positions >> 32) return (q / positions) * of_batch + (q % positions) * of_position;
        const unsigned b = unsigned(q) / unsigned(positions);
        return b * of_batch + (unsigned(q) - b * unsigned(positions)) * of_position;
    }
    __device__ __forceinline__ long long at(long long q) const { return at(q, stride_batch, stride_position); }
    __device__ __forceinline__ long long top_first(long long q) const { return top_last ? q * top_k : at(q, positions * top_k, 1); }
    __device__ __forceinline__ long long top_step() const { return top_last ? 1 : positions; }
};

// Where answers go; what is not wanted is null.  stats: m, log S, H, each of all positions; where no class can be m is +infinity, so that exp(x - m) is 0
// whatever x.
template <typename T>
struct Answers {
    const T* logits;
    const long long* labels;
    T *label, *entropy, *top, *stats;
    int* top_index;
};

// of_label: the logit of the label of position q
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

// 16 bytes a load where classes lie side by side
template <typename T> struct Bytes16;
template <> struct Bytes16<float> { using type = float4; };
template <> struct Bytes16<double> { using type = double2; };
template <typename T> constexpr int kWide = 16 / sizeof(T);
// (What they go to and come from is an array of T, which is bound to a multiple of its own size only wherever it is not in registers.)
template <typename T>
__device__ __forceinline__ void load_wide(T* v, const void* from) {
    const typename Bytes16<T>::type w = *static_cast<const typename Bytes16<T>::type*>(from);
    memcpy(v, &w, 16);
}
template <typename T>
__device__ __forceinline__ void store_wide(T* to, const T* v) {
    typename Bytes16<T>::type w;
    memcpy(&w, v, 16);
    *reinterpret_cast<typename Bytes16<T>::type*>(to) = w;
}

template <typename T>
__device__ __forceinline__ int in_front(const T* x) { return int(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)); }

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

// Classes that a lane loads at a time, the next ones on their way meanwhile.
constexpr int kLaneAhead = 8;

// The run [begin, end) of a position's classes that a warp has, U at a time from c on.  SIDE: classes lie side by side, and c is counted from the
// 16-byte boundary in front of the run, which may be in front of it.
template <typename T, bool SIDE>
struct Run {
    static_assert(kLaneAhead % kWide<T> == 0, "chunks start at 16-byte addresses");
    int begin, end, c;
    long long step;
    __device__ __forceinline__ Run(const Logits& g, const T* x, int warp) {
        const int share = (g.classes + int(blockDim.y) - 1) / int(blockDim.y);
        begin = min(g.classes, warp * share);
        end = min(g.classes, begin + share);
        c = begin - (SIDE ? in_front(x + begin) : 0);
        step = g.stride_class;
    }
    // the same for all lanes of a warp
    __device__ __forceinline__ int chunks(int u) const { return (end - begin + (SIDE ? kWide<T> - 1 : 0) + u - 1) / u; }
    // x: class c
    template <int U>
    __device__ __forceinline__ void load(T (&v)[U], const T* x) const {
        if (SIDE) {
#pragma unroll
            for (int j = 0; j < U; j += kWide<T>) {
                if (c + j >= begin && c + j + kWide<T> <= end) {
                    load_wide(v + j, x + j);
                } else {
#pragma unroll
                    for (int e = j; e < j + kWide<T>; ++e) v[e] = c + e >= begin && c + e < end ? x[e] : -infinity<T>();
                }
            }
        } else if (c + U <= end) {
#pragma unroll
            for (int u = 0; u < U; ++u) { v[u] = *x; x += step; }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                v[u] = c + u < end ? *x : -infinity<T>();
                if (c + u < end) x += step;
            }
        }
    }
    // to: class c, which `aligned` says lies to 16 bytes as the logits do
    template <int U>
    __device__ __forceinline__ void store(const T (&v)[U], T* to, long long to_step, bool aligned) const {
        if (SIDE) {
#pragma unroll
            for (int j = 0; j < U; j += kWide<T>) {
                if (aligned && c + j >= begin && c + j + kWide<T> <= end) {
                    store_wide(to + j, v + j);
                } else {
#pragma unroll
                    for (int e = j; e < j + kWide<T>; ++e)
                        if (c + e >= begin && c + e < end) to[e] = v[e];
                }
            }
        } else if (c + U <= end) {
#pragma unroll
            for (int u = 0; u < U; ++u) { *to = v[u]; to += to_step; }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (c + u < end) { *to = v[u]; to += to_step; }
        }
    }
};

// The likeliest classes: a list takes as many comparisons and choices a class as it has places, times five.  So what is listed are chunks by their largest,
// equal ones by their order (warp << kWarpShift | chunk of its run): the first top_k of them have the top_k largest classes, and only these
// are read again for it.
constexpr int kWarpShift = 27;          // (2^30 classes are 2^27 chunks)

// what a lane finds in its run; DIRECT: classes are listed, not chunks
template <typename T, int TOP, bool SIDE, bool DIRECT>
__device__ __forceinline__ Found<T, TOP> found_in_run(const Logits& g, const T* x) {
    constexpr int U = kLaneAhead;
    Run<T, SIDE> run(g, x, threadIdx.y);
    const T* from = x + run.c * run.step;
    T v[U];
    run.load(v, from);
    Found<T, TOP> f;
    f.sums.clear();
    f.top.clear();
    for (int n = run.chunks(U), i = int(threadIdx.y) << kWarpShift; n > 0; --n, ++i) {
        run.c += U;
        from += U * run.step;
        T next[U];
        if (n > 1) run.load(next, from);
        const T hi = f.sums.add(v);
        if (TOP > 0 && __any_sync(0xffffffffu, hi > f.top.v[TOP > 0 ? TOP - 1 : 0])) {
            if (DIRECT) {
#pragma unroll
                for (int u = 0; u < U; ++u) f.top.offer(v[u], run.c - U + u);
            } else {
                f.top.offer(hi, i);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
    }
    return f;
}
// a listed chunk of the logits x
template <typename T, bool SIDE>
__device__ __forceinline__ Run<T, SIDE> listed_chunk(const Logits& g, const T* x, int i) {
    Run<T, SIDE> chunk(g, x, i >> kWarpShift);
    chunk.c += (i & ((1 << kWarpShift) - 1)) * kLaneAhead;
    return chunk;
}

template <typename T, int TOP, bool SIDE, bool DIRECT>
__global__ void __launch_bounds__(128, sizeof(T) == 4 && TOP <= 4 ? 8 : 1) answer_lanes(Logits g, Answers<T> a) {
    constexpr int U = kLaneAhead;
    stream_order();
    extern __shared__ __align__(16) char room[];
    bool mine;
    const long long q = lane_position(g, &mine);
    const T* x = a.logits + g.at(q);
    const long long label = a.label && threadIdx.y == 0 ? a.labels[q] : -1;
    Found<T, TOP> f = found_in_run<T, TOP, SIDE, DIRECT>(g, x);
    const bool labelled = label >= 0 && label < g.classes;
    const T of_label = labelled ? x[label * g.stride_class] : T(0);
    char* at = room + (threadIdx.z * blockDim.y + threadIdx.y) * Found<T, TOP>::kBytes;
    for (int d = 1; d < int(blockDim.y); d *= 2) {
        if (threadIdx.y % (2 * d) == d) f.put(at, threadIdx.x);
        __syncthreads();
        if (threadIdx.y % (2 * d) == 0 && threadIdx.y + d < blockDim.y) f.join(at + d * Found<T, TOP>::kBytes, threadIdx.x);
    }
    if (threadIdx.y != 0) return;
    Largest<T, TOP> top = f.top;
    if constexpr (TOP > 0 && !DIRECT) {
        // the chunks in the order of the list, and every lane's classes not below its last chunk's largest one after the other
        top.clear();
        T bound = f.top.v[0];
#pragma unroll
        for (int j = 1; j < TOP; ++j) bound = j < g.top_k ? f.top.v[j] : bound;
#pragma unroll
        for (int j = 0; j < TOP; ++j) {
            const int i = f.top.i[j];
            const bool has = j < g.top_k && i >= 0;
            if (!__any_sync(0xffffffffu, has)) break;
            unsigned above = 0;
            int c = 0;
            T v[U];
            if (has) {
                const Run<T, SIDE> chunk = listed_chunk<T, SIDE>(g, x, i);
                c = chunk.c;
                chunk.load(v, x + chunk.c * chunk.step);
#pragma unroll
                for (int u = 0; u < U; ++u) above |= v[u] >= bound && v[u] > -infinity<T>() ? 1u << u : 0u;
            }
            while (__any_sync(0xffffffffu, above)) {
                const int u = __ffs(above) - 1;
                T xu = -infinity<T>();
#pragma unroll
                for (int w = 0; w < U; ++w) xu = u == w ? v[w] : xu;
                top.offer_any(xu, c + u);
                above &= above - 1;
            }
        }
    }
    if (!mine) return;
    const Answer<T> w(f.sums);
    write_position(g, a, q, of_label, labelled, w);
    long long to = TOP > 0 ? g.top_first(q) : 0;
#pragma unroll
    for (int j = 0; j < TOP; ++j) {
        if (j >= g.top_k) break;
        a.top_index[to] = top.i[j];
        a.top[to] = top.i[j] < 0 ? -infinity<T>() : w.of(top.v[j]);
        to += g.top_step();
    }
}

// ----------------------------------------------------------------------------------------------- several lanes a position
// For rows, whose classes lie side by side, 16 bytes a load.  Rows start anywhere: chunks are counted from the 16-byte boundary in front of a row.

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
            load_wide(v + j, x + c);
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
            store_wide(x + c, v + j);
        } else {
#pragma unroll
            for (int e = 0; e < kWide<T>; ++e)
                if (c + e >= 0 && c + e < classes) x[c + e] = v[j + e];
        }
    }
}

// float32 numbers as unsigned ones in the same order (-0 as 0), of which a warp finds the largest in one instruction
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float number(unsigned k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }

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

__device__ __forceinline__ float warp_max(float v) { return number(__reduce_max_sync(0xffffffffu, ordered(v))); }
__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = larger(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
// take(j, value, index) of the top_k best of all lanes' values, by falling value, equal ones by index; NaN and -infinity are none.  Every lane puts its own
// in order, and the best of the lanes' first ones is taken away again and again.
template <typename T, int N, class Take>
__device__ __forceinline__ void best_of_lanes(T (&v)[N], int (&i)[N], int top_k, Take take) {
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (!(v[e] > -infinity<T>())) { v[e] = -infinity<T>(); i[e] = -1; }
#pragma unroll
    for (int n = N - 1; n > 0; --n)
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const bool swap = v[e + 1] > v[e] || (v[e + 1] == v[e] && unsigned(i[e + 1]) < unsigned(i[e]));
            const T ov = v[e];
            const int oi = i[e];
            v[e] = swap ? v[e + 1] : ov; i[e] = swap ? i[e + 1] : oi;
            v[e + 1] = swap ? ov : v[e + 1]; i[e + 1] = swap ? oi : i[e + 1];
        }
#pragma unroll 1
    for (int j = 0; j < top_k; ++j) {
        T best = v[0];
        int at = i[0];
        warp_best(best, at);
        if (at < 0) break;
        take(j, best, at);
        const bool mine = i[0] == at;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            v[e] = mine ? (e + 1 < N ? v[e + 1 < N ? e + 1 : e] : -infinity<T>()) : v[e];
            i[e] = mine ? (e + 1 < N ? i[e + 1 < N ? e + 1 : e] : -1) : i[e];
        }
    }
}

// The largest so far as a list of the warp, the j-th of them in lane j.  A class is compared with the last one that counts, and only one in front of it
// moves the list: a row of n classes in any order moves it about top_k log(n / top_k) times.
template <typename T>
struct WarpList {
    T v, last;               // this lane's value; that of place top_k - 1
    int i;                   // (a free place is -infinity and -1, the largest of unsigned indices)
    __device__ __forceinline__ void clear() { v = last = -infinity<T>(); i = -1; }
    __device__ __forceinline__ unsigned last_i(int top_k) const { return unsigned(__shfl_sync(0xffffffffu, i, top_k - 1)); }
    __device__ __forceinline__ void insert(T x, int c, int top_k) {
        const unsigned behind = __ballot_sync(0xffffffffu, x > v || (x == v && unsigned(c) < unsigned(i)));
        const T up = __shfl_up_sync(0xffffffffu, v, 1);
        const int up_i = __shfl_up_sync(0xffffffffu, i, 1);
        const int lane = threadIdx.x % 32, place = __ffs(behind) - 1;
        if (behind && lane >= place) { v = lane == place ? x : up; i = lane == place ? c : up_i; }
        last = __shfl_sync(0xffffffffu, v, top_k - 1);
    }
    // one value of each lane that is in `who`.  (Where they are many most are not in front of the last any more: equal classes, 20000 rows of 500 zeros 361 us
    // if all are put in, 65 so.)
    __device__ __forceinline__ void insert_lanes(unsigned who, T x, int c, int top_k) {
        if (__popc(who) > 8) {
            const unsigned behind = last_i(top_k);
            who &= __ballot_sync(0xffffffffu, x > last || (x == last && x > -infinity<T>() && unsigned(c) < behind));
        }
        for (; who; who &= who - 1) {
            const T best = __shfl_sync(0xffffffffu, x, __ffs(who) - 1);
            if (best >= last) insert(best, __shfl_sync(0xffffffffu, c, __ffs(who) - 1), top_k);
        }
    }
    // The classes of a warp's chunk (see load_chunk) that are not below `bound`, all behind those that were offered before.
    template <int U>
    __device__ __forceinline__ void offer_above(const T (&x)[U], T bound, long long first, int top_k) {
        unsigned mine = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) mine |= x[u] > last && x[u] >= bound ? 1u << u : 0u;
        // one of each lane's at a time
        while (const unsigned who = __ballot_sync(0xffffffffu, mine)) {
            const int u = __ffs(mine) - 1, c = int(first + class_in_chunk<T, 32>(threadIdx.x % 32, u));
            T xu = x[0];
#pragma unroll
            for (int w = 1; w < U; ++w) xu = u == w ? x[w] : xu;
            mine &= mine - 1;
            insert_lanes(who, xu, c, top_k);
        }
    }
    // the top_k-th largest of the lanes' values, of which none is NaN
    static __device__ __forceinline__ T bound_of(T rest, int top_k) {
        T bound = rest;
        for (int j = 0; j < top_k; ++j) {
            bound = warp_max(rest);
            const unsigned who = __ballot_sync(0xffffffffu, rest == bound);
            if (int(threadIdx.x % 32) == __ffs(who) - 1) rest = -infinity<T>();
        }
        return bound;
    }
    // the first chunk, `hi` the lane's largest: at least top_k classes are not below the top_k-th largest of these
    template <int U>
    __device__ __forceinline__ void start(const T (&x)[U], T hi, long long first, int top_k) {
        clear();
        offer_above(x, bound_of(hi == hi ? hi : -infinity<T>(), top_k), first, top_k);           // (a lane all of whose classes are NaN)
    }
    // a further one; a bound is worth its search where most lanes have a candidate (classes in rising order: 4096 rows of 2000 187 us without, 38 with)
    template <int U>
    __device__ __forceinline__ void offer(const T (&x)[U], T hi, long long first, int top_k) {
        const unsigned lanes = __ballot_sync(0xffffffffu, hi > last);
        if (!lanes) return;
        offer_above(x, __popc(lanes) > 16 ? bound_of(hi > last ? hi : -infinity<T>(), top_k) : -infinity<T>(), first, top_k);
    }
};

// what a warp, and then a CTA, found
template <typename T>
struct RowFound {
    Sums<T> sums;
    T top[16];
    int top_index[16];
};

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
    const T m = warp_max(a.m);                      // (no NaN among them)
    if (m > -infinity<T>()) a.raise(m);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, d);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, d);
    }
    a.m = m;
    return a;
}

// the answers of position q by a whole warp, from what its label's logit is in lane 0
template <typename T, bool TOP>
__device__ __forceinline__ void write_row(const Logits& g, const Answers<T>& a, long long q, T of_label, bool labelled, const Sums<T>& sums, const WarpList<T>& list) {
    const int lane = threadIdx.x % 32;
    const Answer<T> w(sums);
    if (lane == 0) write_position(g, a, q, of_label, labelled, w);
    if (TOP && lane < g.top_k) {
        const long long to = g.top_first(q) + lane * g.top_step();
        a.top_index[to] = list.i;
        a.top[to] = list.i < 0 ? -infinity<T>() : w.of(list.v);
    }
}
// the label's logit of position q, in lane 0
template <typename T>
__device__ __forceinline__ T logit_of_label(const Logits& g, const Answers<T>& a, long long q, const T* x, bool* labelled) {
    const long long label = a.label && threadIdx.x % 32 == 0 ? a.labels[q] : -1;
    *labelled = label >= 0 && label < g.classes;
    return *labelled ? x[label] : T(0);
}

// Few positions whose classes are apart, by kGroupWarps warps a tile of 32: what the warps found is joined position by position, a warp each, its lanes
// over the listed chunks and then over their classes.
constexpr int kGroupWarps = 16;
// (the entries of a position lie in as many banks)
template <typename T, int TOP> constexpr size_t kGroupBytes = Found<T, TOP>::kBytes + 8;
template <typename T, int TOP>
__global__ void __launch_bounds__(32 * kGroupWarps, sizeof(T) == 4 ? 2 : 1) answer_groups(Logits g, Answers<T> a) {
    stream_order();
    extern __shared__ __align__(16) char room[];
    const int lane = threadIdx.x;
    bool mine;
    {
        const T* x = a.logits + g.at(lane_position(g, &mine));
        const Found<T, TOP> f = found_in_run<T, TOP, false, false>(g, x);
        f.put(room + threadIdx.y * kGroupBytes<T, TOP>, lane);
    }
    __syncthreads();
#pragma unroll 1
    for (int p = threadIdx.y; p < 32; p += kGroupWarps) {
        const long long q = (long long)blockIdx.x * 32 + p;
        if (q >= g.count()) break;
        const T* x = a.logits + g.at(q);
        const long long label = a.label && lane == 0 ? a.labels[q] : -1;
        const bool labelled = label >= 0 && label < g.classes;
        const T of_label = labelled ? x[label * g.stride_class] : T(0);
        auto values = [&](int warp) { return reinterpret_cast<const T*>(room + warp * kGroupBytes<T, TOP>) + p; };
        Sums<T> sums;
        sums.clear();
        if (lane < kGroupWarps) sums = {values(lane)[0], values(lane)[32], values(lane)[64]};
        sums = over_warp(sums);
        WarpList<T> list;
        list.clear();
        if constexpr (TOP > 0) {
            // (kGroupWarps * TOP entries, and then 8 classes of each chunk that is taken)
            constexpr int kEntries = (kGroupWarps * TOP + 31) / 32, kClasses = (TOP * kLaneAhead + 31) / 32;
            T v[kEntries];
            int i[kEntries], taken = -1;
#pragma unroll
            for (int e = 0; e < kEntries; ++e) {
                const int entry = e * 32 + lane, warp = entry % kGroupWarps, j = entry / kGroupWarps;
                const bool there = j < TOP;
                v[e] = there ? values(warp)[32 * (3 + j)] : -infinity<T>();
                i[e] = there ? reinterpret_cast<const int*>(values(warp) - p + 32 * (3 + TOP))[32 * j + p] : -1;
            }
            best_of_lanes(v, i, g.top_k, [&](int j, T, int at) { if (lane == j) taken = at; });
            T w[kClasses];
            int c[kClasses];
#pragma unroll
            for (int e = 0; e < kClasses; ++e) {
                const int entry = e * 32 + lane, j = entry / kLaneAhead, at = __shfl_sync(0xffffffffu, taken, j < 16 ? j : 0);
                w[e] = -infinity<T>();
                c[e] = -1;
                if (j < g.top_k && at >= 0) {
                    const Run<T, false> chunk = listed_chunk<T, false>(g, x, at);
                    const int here = chunk.c + entry % kLaneAhead;
                    if (here >= chunk.begin && here < chunk.end) { w[e] = x[here * chunk.step]; c[e] = here; }
                }
            }
            best_of_lanes(w, c, g.top_k, [&](int j, T best, int at) { if (lane == j) { list.v = best; list.i = at; } });
        }
        write_row<T, (TOP > 0)>(g, a, q, of_label, labelled, sums, list);
    }
}

// A warp a row, kRowWarps of them a CTA, U classes a lane and chunk.
constexpr int kRowWarps = 8;
template <typename T, bool TOP, int U>
__global__ void __launch_bounds__(32 * kRowWarps) answer_rows(Logits g, Answers<T> a) {
    stream_order();
    const int lane = threadIdx.x % 32;
    const long long q = (long long)blockIdx.x * kRowWarps + threadIdx.x / 32;
    if (q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    int first = -in_front(x);
    T v[U];
    load_chunk<T, U, 32>(v, x, first, g.classes, lane);
    bool labelled;
    const T of_label = logit_of_label(g, a, q, x, &labelled);
    Sums<T> sums;
    WarpList<T> list;
    sums.clear();
    T hi = sums.add(v);
    if (TOP) list.start(v, hi, first, g.top_k);
    for (first += 32 * U; first < g.classes; first += 32 * U) {
        load_chunk<T, U, 32>(v, x, first, g.classes, lane);
        hi = sums.add(v);
        if (TOP) list.offer(v, hi, first, g.top_k);
    }
    write_row<T, TOP>(g, a, q, of_label, labelled, over_warp(sums), list);
}

// Long rows: all rows' chunks in their order, in equal runs for the CTAs of one wave, which have the next ones on their way all the time, those of the
// next row as well: every thread copies what it reads itself into shared memory (cp.async), kStages - 1 chunks ahead, and waits for nobody else.
// More on the way at once is slower (2048 rows of 65537 classes with 5 alternatives / of 32000 without, us: 2 CTAs a multiprocessor with 2, 3, 4
// stages 116 / 55, 96 / 46, 101 / 47, 3 CTAs with 2, 3, 4 stages 97 / 47, 105 / 47, 109 / 51, 4 with 3 112 / 52; the memory's floor 82 / 40).
//
// The likeliest classes cost the streaming warps a few comparisons a chunk.  Every thread keeps the largest of its classes, the chunk in which it came up
// first, and the largest of its other chunks.  Of the threads by their largest, equal ones by its first class, the first top_k have all of the row's
// top_k: every other thread's classes have at least top_k in front of them.  Another warp, while the others go on, picks these threads and reads the
// chunks of theirs again that may have one, seldom more than one a thread.
//
// A run that has all of a row answers it; of others what it found goes to `parts`, two places a CTA (0: with its first chunk, 1: without), where join_parts
// finds it.
constexpr int kStreamWarps = 8, kStreamThreads = 32 * kStreamWarps, kStages = 3, kStreamCtas = 2;
template <typename T> constexpr int kStreamAhead = 64 / sizeof(T);
template <typename T> constexpr int kStreamChunk = kStreamThreads * kStreamAhead<T>;
constexpr int kStreamBytes = kStages * kStreamThreads * 64;

struct Runs {
    long long chunks;                               // of all rows
    int of_row, ctas;
    __host__ __device__ long long begin(int cta) const { return chunks / ctas * cta + (chunks % ctas) * cta / ctas; }
};

// 16 bytes from class c of row x on their way into shared memory, what is not of the row as classes that cannot be
template <typename T>
__device__ __forceinline__ void copy_wide(char* to, const T* x, long long c, bool inside, int classes) {
    constexpr int kBytes = int(sizeof(T));
    const unsigned at = unsigned(__cvta_generic_to_shared(to));
    if (inside || (c >= 0 && c + kWide<T> <= classes)) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(x + c) : "memory");
    } else {
#pragma unroll
        for (int e = 0; e < kWide<T>; ++e) {
            if (c + e >= 0 && c + e < classes) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at + e * kBytes), "l"(x + c + e), "n"(kBytes) : "memory");
            else reinterpret_cast<T*>(to)[e] = -infinity<T>();
        }
    }
}
// a thread's share of the chunk from `first` on: value u is class_in_chunk(threadIdx.x, u), 16 bytes of every kStreamThreads * 16
template <typename T>
__device__ __forceinline__ void copy_chunk(char* to, const T* x, long long first, int classes) {
    const bool inside = first >= 0 && first + kStreamChunk<T> <= classes;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        copy_wide(to + (j * kStreamThreads + threadIdx.x) * 16, x, first + class_in_chunk<T, kStreamThreads>(threadIdx.x, j * kWide<T>), inside, classes);
}

// What the streaming warps leave of (their part of) a row.
template <typename T>
struct Streamed {
    Sums<T> sums[kStreamWarps];
    T largest[kStreamThreads], second[kStreamThreads];          // (second: of the chunks' largest)
    int chunk[kStreamThreads];                                  // where the largest came up
};

// All warps but the waiting one come and go on (bar.arrive), or wait for it: 32 more threads than stream take part.
__device__ __forceinline__ void barrier_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kStreamThreads + 32) : "memory"); }
__device__ __forceinline__ void barrier_wait(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kStreamThreads + 32) : "memory"); }

// where the j-th 16 bytes of thread `tid` in the chunk from `first` on are
template <typename T>
__device__ __forceinline__ long long share_of(long long first, int tid, int j) { return first + class_in_chunk<T, kStreamThreads>(tid, j * kWide<T>); }

// the first class of thread `tid` in the chunk from `first` on that is `value` (there is one)
template <typename T>
__device__ __noinline__ int first_equal(const T* x, T value, long long first, int tid, int classes) {
#pragma unroll 1
    for (int u = 0; u < kStreamAhead<T>; ++u) {
        const long long c = first + class_in_chunk<T, kStreamThreads>(tid, u);
        if (c >= 0 && c < classes && x[c] == value) return int(c);
    }
    return 0x7fffffff;
}

// classes that may be among the likeliest
template <typename T>
struct Above {
    T top[32];
    int top_index[32];
};

// The top_k largest of the classes in chunks [begin, end) of row x, from what the threads kept of them; by one warp.
template <typename T>
__device__ __forceinline__ void pick(WarpList<T>& list, const Streamed<T>& kept, Above<T>& room, const T* x, int begin, int end, int classes, int top_k) {
    const int lane = threadIdx.x % 32, front = in_front(x);
    T rest[kStreamWarps], bound = -infinity<T>();
    int chunk[kStreamWarps], front_class[kStreamWarps];     // (front_class: the first class that is the thread's largest, where it was looked up)
#pragma unroll
    for (int w = 0; w < kStreamWarps; ++w) {
        rest[w] = kept.largest[w * 32 + lane];
        chunk[w] = kept.chunk[w * 32 + lane];
        front_class[w] = -1;
    }
    int picked = -1, last_chunk = -1, n = 0;                // lane j: the j-th thread; the last chunk of those picked for the same value
#pragma unroll 1
    for (; n < top_k; ++n) {
        T most = rest[0];
#pragma unroll
        for (int w = 1; w < kStreamWarps; ++w) most = larger(most, rest[w]);
        const T best = warp_max(most);
        if (best == -infinity<T>()) break;
        if (best != bound) last_chunk = -1;
        bound = best;
        int equal = 0, place = 0;
        unsigned soonest = 0xffffffffu;
#pragma unroll
        for (int w = kStreamWarps - 1; w >= 0; --w) {
            const bool is = rest[w] == best;
            equal += is;
            place = is ? w : place;
            soonest = is ? min(soonest, unsigned(chunk[w])) : soonest;
        }
        unsigned who = __ballot_sync(0xffffffffu, equal > 0);
        if (__reduce_add_sync(0xffffffffu, equal) > 1) {
            // of equal ones the first class decides, which is of those in the first chunk
            soonest = __reduce_min_sync(0xffffffffu, soonest);
            unsigned at = 0xffffffffu;
#pragma unroll
            for (int w = 0; w < kStreamWarps; ++w) {
                if (rest[w] == best && unsigned(chunk[w]) == soonest) {
                    if (front_class[w] < 0) front_class[w] = first_equal(x, best, (long long)chunk[w] * kStreamChunk<T> - front, w * 32 + lane, classes);
                    if (unsigned(front_class[w]) < at) { at = unsigned(front_class[w]); place = w; }
                }
            }
            who = __ballot_sync(0xffffffffu, at == __reduce_min_sync(0xffffffffu, at));
        }
        const int from = __ffs(who) - 1, tid = __shfl_sync(0xffffffffu, place * 32 + lane, from);
        if (lane == n) picked = tid;
        last_chunk = max(last_chunk, kept.chunk[tid]);
#pragma unroll
        for (int w = 0; w < kStreamWarps; ++w)
            if (w * 32 + lane == tid) rest[w] = -infinity<T>();
    }
    if (n < top_k) bound = -infinity<T>();                  // (all of the classes that can be are theirs)
    // First the chunks in which their largest came up, then all others of a thread whose second largest is above the bound, or those up to last_chunk where it is
    // the bound: of equal classes, those picked come before what is behind.  The classes that are not below the bound are hardly ever more
    // than the lanes of a warp: the best of these again and again; more, equal ones, are put in one by one.  (Loops that are not unrolled:
    // the code runs once a row, and would wait for its instructions.)
    list.clear();
    int count = 0;
    const T second = lane < n ? kept.second[picked] : -infinity<T>();
    const unsigned all = __ballot_sync(0xffffffffu, second > bound);
    unsigned passes = all | __ballot_sync(0xffffffffu, second == bound && second > -infinity<T>());
#pragma unroll 1
    for (int pass = -1;;) {
        const int total = pass < 0 ? 4 * n : 4 * ((all >> pass & 1 ? end : min(end, last_chunk + 1)) - begin);
#pragma unroll 1
        for (int from = 0; from < total; from += 32) {
            const int at = from + lane, tid = __shfl_sync(0xffffffffu, picked, pass < 0 ? min(at, total - 1) / 4 : pass), first = kept.chunk[tid], chunk = pass < 0 ? first : begin + at / 4;
            const long long c0 = share_of<T>((long long)chunk * kStreamChunk<T> - front, tid, at % 4);
            T v[kWide<T>];
#pragma unroll
            for (int e = 0; e < kWide<T>; ++e) v[e] = at < total && (pass < 0 || chunk != first) && c0 + e >= 0 && c0 + e < classes ? x[c0 + e] : -infinity<T>();
            unsigned mine = 0;
#pragma unroll
            for (int e = 0; e < kWide<T>; ++e) mine |= v[e] > -infinity<T>() && v[e] >= bound ? 1u << e : 0u;
#pragma unroll 1
            while (const unsigned who = __ballot_sync(0xffffffffu, mine)) {
                const int e = __ffs(mine) - 1, left = 32 - count, to = count + __popc(who & ((1u << lane) - 1)), c = int(c0) + e;
                T w = v[0];
#pragma unroll
                for (int k = 1; k < kWide<T>; ++k) w = e == k ? v[k] : w;
                if (mine && to < 32) { room.top[to] = w; room.top_index[to] = c; }
                mine &= mine - 1;
                count += __popc(who);
                // (what has no room)
                if (count > 32) list.insert_lanes(left <= 0 ? who : who & ~((2u << __fns(who, 0, left)) - 1), w, c, top_k);
            }
        }
        if (!passes) break;
        pass = __ffs(passes) - 1;
        passes &= passes - 1;
    }
    __syncwarp();
    T mine = lane < count ? room.top[lane] : -infinity<T>();
    int mine_i = lane < count ? room.top_index[lane] : -1;
    if (count > 32) {
        list.insert_lanes(0xffffffffu, mine, mine_i, top_k);
    } else {
#pragma unroll 1
        for (int j = 0; j < top_k; ++j) {
            T best = mine;
            int at = mine_i;
            warp_best(best, at);
            if (at < 0) break;
            if (lane == j) { list.v = best; list.i = at; }
            if (at == mine_i) { mine = -infinity<T>(); mine_i = -1; }
        }
    }
    __syncwarp();
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kStreamThreads + 32, kStreamCtas) answer_stream(Logits g, Answers<T> a, Runs runs, RowFound<T>* parts) {
    stream_order();
    constexpr int U = kStreamAhead<T>;
    extern __shared__ __align__(16) char stages[];
    __shared__ Streamed<T> kept[2];                         // (the warps that stream are at the next row meanwhile)
    __shared__ Above<T> above;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const long long begin = runs.begin(blockIdx.x), end = runs.begin(blockIdx.x + 1);
    if (begin >= end) return;
    long long q = begin / runs.of_row;
    int chunk = int(begin - q * runs.of_row), turn = 0;
    const T* x = a.logits + g.at(q);
    // barriers 1 and 2: a row is streamed, into kept[0] and kept[1]; 3 and 4: it is answered, and kept may be written again
    if (warp == kStreamWarps) {
        bool first_part = true;
        for (long long at = begin; at < end; turn ^= 1, ++q, chunk = 0, first_part = false) {
            const int last = int(min((long long)runs.of_row, chunk + (end - at)));
            const bool whole = chunk == 0 && last == runs.of_row;
            x = a.logits + g.at(q);
            bool labelled = false;
            const T of_label = whole ? logit_of_label(g, a, q, x, &labelled) : T(0);
            __syncwarp();                                   // (barriers are for whole warps)
            barrier_wait(1 + turn);
            Sums<T> sums;
            sums.clear();
            if (lane < kStreamWarps) sums = kept[turn].sums[lane];
            sums = over_warp(sums);
            WarpList<T> list;
            list.clear();
            if (TOP) pick(list, kept[turn], above, x, chunk, last, g.classes, g.top_k);
            at += last - chunk;
            // (the next row but one is there: who waits is sure to come)
            __threadfence_block();
            __syncwarp();
            if (end - at > runs.of_row) barrier_arrive(3 + turn);
            if (whole) {
                write_row<T, TOP>(g, a, q, of_label, labelled, sums, list);
            } else {
                RowFound<T>* const to = parts + 2 * blockIdx.x + (first_part ? 0 : 1);
                if (lane == 0) to->sums = sums;
                if (TOP && lane < 16) { to->top[lane] = list.v; to->top_index[lane] = list.i; }
            }
        }
        return;
    }
    // what is on its way
    long long q_ahead = q, ahead = begin;
    int chunk_ahead = chunk, stage = 0, stage_ahead = 0, rows = 0;
    const T* x_ahead = x;
    auto copy_next = [&] {
        if (ahead < end) {
            copy_chunk(stages + stage_ahead * (kStreamThreads * 64), x_ahead, (long long)chunk_ahead * kStreamChunk<T> - in_front(x_ahead), g.classes);
            ++ahead;
            if (++chunk_ahead == runs.of_row && ahead < end) {
                chunk_ahead = 0;
                x_ahead = a.logits + g.at(++q_ahead);
            }
        }
        stage_ahead = stage_ahead + 1 == kStages ? 0 : stage_ahead + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int s = 0; s + 1 < kStages; ++s) copy_next();
    Sums<T> sums;
    sums.clear();
    T largest = -infinity<T>(), second = largest;
    int largest_chunk = 0;
    for (long long at = begin; at < end; ++at) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        T v[U];
        const char* here = stages + stage * (kStreamThreads * 64) + threadIdx.x * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) load_wide(v + j * kWide<T>, here + j * kStreamThreads * 16);
        stage = stage + 1 == kStages ? 0 : stage + 1;
        copy_next();                                        // (into what was read an iteration ago)
        const T hi = sums.add(v);
        if (TOP) {
            second = larger(second, hi > largest ? largest : hi);
            if (hi > largest) { largest = hi; largest_chunk = chunk; }
        }
        const bool ends = ++chunk == runs.of_row;
        if (ends || at + 1 == end) {
            sums = over_warp(sums);
            __syncwarp();
            if (rows >= 2) barrier_wait(3 + turn);          // (the row before the last one has been answered)
            if (lane == 0) kept[turn].sums[warp] = sums;
            if (TOP) { kept[turn].largest[threadIdx.x] = largest; kept[turn].second[threadIdx.x] = second; kept[turn].chunk[threadIdx.x] = largest_chunk; }
            __threadfence_block();
            __syncwarp();
            barrier_arrive(1 + turn);
            ++rows;
            turn ^= 1;
            chunk = 0;
            sums.clear();
            largest = second = -infinity<T>();
        }
    }
}

// A warp for every border between two runs that is inside a row and the first one there: the row's parts, up to 32.
template <typename T, bool TOP>
__global__ void __launch_bounds__(32) join_parts(Logits g, Answers<T> a, Runs runs, const RowFound<T>* parts) {
    stream_order();
    __shared__ RowFound<T> found[32];
    const int lane = threadIdx.x, cta = int(blockIdx.x) + 1;
    const long long border = runs.begin(cta), q = border / runs.of_row, row = q * runs.of_row;
    if (border == row || runs.begin(cta - 1) > row) return;
    bool labelled;
    const T of_label = logit_of_label(g, a, q, a.logits + g.at(q), &labelled);
    // the run in front of the border has the row's first part, behind other rows' unless it starts with it
    const int mine = cta - 1 + lane;
    const bool has = mine < runs.ctas && (lane == 0 || runs.begin(mine) < row + runs.of_row);
    Sums<T> sums;
    sums.clear();
    if (has) {
        const RowFound<T>& part = parts[2 * mine + (lane == 0 && runs.begin(mine) < row ? 1 : 0)];
        sums = part.sums;
        if (TOP)
            for (int j = 0; j < g.top_k; ++j) { found[lane].top[j] = part.top[j]; found[lane].top_index[j] = part.top_index[j]; }
    }
    __syncwarp();
    WarpList<T> list;
    list.clear();
    if (TOP) join_lists(list, found, __popc(__ballot_sync(0xffffffffu, has)), g.top_k);
    write_row<T, TOP>(g, a, q, of_label, labelled, over_warp(sums), list);
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
    int label;
    bool nothing;
    // top: the sum of the gradients of the alternatives
    __device__ __forceinline__ Share(const Logits& g, const Gradients<T>& a, long long q, T top) {
        const long long n = g.count(), at = a.label ? a.labels[q] : -1;
        const T log_nats = a.stats[n + q], entropy = a.stats[2 * n + q], g_entropy = a.entropy ? a.entropy[q] : T(0), given = a.label ? a.label[q] : T(0);
        m = a.stats[q];
        nothing = m == infinity<T>() && log_nats == T(0);
        log_s = log_nats * Unit<T>::per_nat();
        label = at < 0 || at >= g.classes || nothing ? -1 : int(at);
        g_label = label >= 0 ? given : T(0);
        fixed = nothing ? T(0) : -(g_label + top + g_entropy * entropy);
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

template <typename T, bool SIDE>
__global__ void __launch_bounds__(512, sizeof(T) == 4 ? 2 : 1) gradient_lanes(Logits g, Gradients<T> a) {
    constexpr int U = kLaneAhead;
    stream_order();
    bool mine;
    const long long q = lane_position(g, &mine);
    if (!mine) return;
    const T* x = a.logits + g.at(q);
    T* dx = a.dlogits + g.at(q, a.out_batch, a.out_position);
    Run<T, SIDE> run(g, x, threadIdx.y), out = run;
    const T* from = x + run.c * run.step;
    T* to = dx + run.c * a.out_class;
    const bool aligned = in_front(x) == in_front(dx);
    T v[U], top = T(0);
    run.load(v, from);
    if (a.top) {
        long long at = g.top_first(q);
        for (int j = 0; j < g.top_k; ++j, at += g.top_step()) top += a.top_index[at] >= 0 ? a.top[at] : T(0);
    }
    const Share<T> share(g, a, q, top);
    for (int n = run.chunks(U); n > 0; --n) {
        run.c += U;
        from += U * run.step;
        T next[U];
        if (n > 1) run.load(next, from);
        share.of(v);
        out.store(v, to, a.out_class, aligned);
        out.c += U;
        to += U * a.out_class;
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
    }
    if (share.label >= run.begin && share.label < run.end) dx[share.label * a.out_class] += share.g_label;
    if (a.top && !share.nothing) {
        long long at = g.top_first(q);
        for (int j = 0; j < g.top_k; ++j, at += g.top_step()) {
            const int c = a.top_index[at];
            if (c >= run.begin && c < run.end) dx[c * a.out_class] += a.top[at];
        }
    }
}

// WARPS = 1: a warp a row, kRowWarps of them a CTA; else gridDim.y CTAs of WARPS warps share a row, a run of its chunks each.  U classes a thread and chunk.
template <typename T, int WARPS, int U>
__global__ void __launch_bounds__(32 * (WARPS == 1 ? kRowWarps : WARPS)) gradient_rows(Logits g, Gradients<T> a) {
    stream_order();
    constexpr int kThreads = 32 * WARPS;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, tid = WARPS == 1 ? lane : int(threadIdx.x);
    const long long q = WARPS == 1 ? (long long)blockIdx.x * kRowWarps + warp : blockIdx.x;
    if (WARPS == 1 && q >= g.count()) return;
    const T* x = a.logits + g.at(q);
    T* dx = a.dlogits + g.at(q, a.out_batch, a.out_position);
    const int skip = in_front(x);
    const bool aligned = in_front(dx) == skip;
    const long long chunks = ((long long)g.classes + skip + kThreads * U - 1) / (kThreads * U), each = WARPS == 1 ? chunks : (chunks + gridDim.y - 1) / gridDim.y;
    const long long begin = (WARPS == 1 ? 0 : blockIdx.y) * each * kThreads * U - skip;
    const int end = int(min((long long)g.classes, begin + each * kThreads * U));
    T v[U];
    if (begin < end) load_chunk<T, U, kThreads>(v, x, begin, g.classes, tid);
    // lane j of every warp has the j-th alternative
    int single = -1;
    T more = T(0), top = T(0);
    if (a.top) {
        const long long at = g.top_first(q) + lane * g.top_step();
        if (lane < g.top_k) { single = a.top_index[at]; more = a.top[at]; }
        top = single >= 0 ? more : T(0);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) top += __shfl_xor_sync(0xffffffffu, top, d);
        top = __shfl_sync(0xffffffffu, top, 0);
    }
    const Share<T> share(g, a, q, top);
    // single classes get more than the others: the alternatives, and by lane 31 the label unless it is one of them
    const bool is_label = single >= 0 && single == share.label;
    T more_label = is_label ? share.g_label : T(0), single_x = T(0);
    if (!__any_sync(0xffffffffu, is_label) && lane == 31) { single = share.label; more_label = share.g_label; }
    if (share.nothing || single < begin || single >= end || (WARPS > 1 && warp > 0)) single = -1;
    if (single >= 0) single_x = x[single];
    for (long long first = begin; first < end; first += kThreads * U) {
        T next[U];
        if (first + kThreads * U < end) load_chunk<T, U, kThreads>(next, x, first + kThreads * U, g.classes, tid);
        share.of(v);
        store_chunk<T, U, kThreads>(v, dx, aligned, first, g.classes, tid);
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
    }
    if (WARPS == 1) __syncwarp();
    else __syncthreads();
    if (single >= 0) dx[single] = share.of(Pair<T>{single_x, single_x}).x + more_label + more;
}

// --------------------------------------------------------------------------------------------------------------- launches
Logits logits_of(const simnets_likelihood_desc& d) {
    return {d.batch, d.positions, d.stride_batch, d.stride_class, d.stride_position, d.classes, d.top_k, d.top_last};
}

// Classes that lie side by side are read by several lanes where they are many or the rows are few.  Else a lane's loads of 16 bytes are a few lines of
// memory for the whole warp, and joining what lanes found costs more than the classes (lanes / warps of rows, us: 100000 rows of 100 with three
// alternatives 18 / 64 and their gradient 39 / 42, 60000 of 200 20 / 38 and 50 / 35, 3000 of 100 6.0 / 4.5 and 6.0 / 4.3).
bool by_rows(const Logits& g, int most) { return g.stride_class == 1 && (g.classes > most || (g.classes > 32 && g.count() < 16384)); }
constexpr int kMostByLanes = 256, kMostGradientByLanes = 128;

// Warps that share 32 positions: 4 or 2 where the tiles are then there all at once (by the CTAs of 4 warps that registers let be on a multiprocessor), and
// kGroupWarps where that many are as well and runs of so many classes are worth the join; of more classes two rounds of them are.  float64 answers of many
// classes are shared by 2 beyond that, and by 4 where those 2 would be a few more CTAs than are there at once.
// All sides, maps with four alternatives, us:
//     1 / 2 / 4 warps: 32768 positions of 150 classes 18.2 / 13.1 / 12.9, 49152 20.4 / 15.4 / 18.3, 98304 26.5 / 29.3 / 31.5, their gradients 20.5 / 14.2 / 11.4,
//         23.1 / 17.7 / 18.4, 34.8 / 34.1 / 32.7; float64 12288 of 64 12.6 / 8.8 / 7.4, 24576 15.1 / 11.1 / 13.8, 49152 18.6 / 20.1 / 24.0, 65536 29.2 / 26.5 /
//         30.4, of 32 15.6 / 16.3 / 21.5, 32768 of 300 62 / 66 / 60, the gradients of 64 10.2 / 7.5 / 5.9, 12.0 / 9.1 / 9.9, 15.9 / 17.5 / 16.3, 19.1 / 20.1 / 21.6
//     4 / 16: 8192 of 150 6.0 / 9.1, of 256 9.8 / 9.7, of 512 16.3 / 11.8, 16384 of 512 18.5 / 22.7, of 1000 33 / 31, gradients of 96 4.2 / 4.2, of 100 5.0 / 4.3, of
//         150 6.7 / 5.6, 16384 of 150 8.2 / 9.8, of 512 21.2 / 18.8; float64 4096 of 256 14.0 / 13.6, of 512 25 / 18, 8192 of 512 29 / 35, of 2000 97 / 79,
//         gradients of 64 4.6 / 4.9, of 100 5.6 / 4.9, 8192 of 256 13 / 13.6, of 512 22.0 / 20.5
// Rows, whose classes lie side by side, come here in such numbers only that 16 warps lose: 17500 of 128 8.4 / 16.9, of 256 12.6 / 20.5, the gradient of
// 128 10.7 / 16.0.
template <typename T, bool GRADIENT>
int warps_of_lanes(const Logits& g) {
    constexpr bool kDouble = sizeof(T) == 8, kAnswer64 = kDouble && !GRADIENT;
    constexpr int kCtas = !kDouble ? 8 : GRADIENT ? 4 : 3, kSixteen = GRADIENT ? 97 : 256, kSixteenTwice = GRADIENT ? (kDouble ? 512 : 256) : kDouble ? 1024 : 768;
    const long long tiles = (g.count() + 31) / 32, sms = device_sm_count(), groups = (kDouble ? 1 : 2) * sms;
    if (g.stride_class != 1 && g.classes >= kSixteen && tiles <= (g.classes >= kSixteenTwice ? 2 * groups : groups)) return kGroupWarps;
    if (g.classes >= 4 * kLaneAhead && tiles < kCtas * sms) return 4;
    if (kAnswer64 && g.classes >= 16 * kLaneAhead && tiles >= 2 * kCtas * sms && tiles < 8 * sms) return 4;
    return g.classes >= 2 * kLaneAhead && tiles < (kAnswer64 && g.classes >= 8 * kLaneAhead ? 16 : 2 * kCtas) * sms ? 2 : 1;
}

template <class Kernel, class A>
cudaError_t launch_lanes(Kernel* kernel, const Logits& g, const A& a, int warps, size_t bytes, cudaStream_t s) {
    const int tiles = warps < 4 ? 4 / warps : 1;
    const unsigned grid = unsigned((g.count() + 32 * tiles - 1) / (32 * tiles));
    in_stream_order(kernel, grid, dim3(32, warps, tiles), bytes, s)(g, a);
    count_launch();
    return cudaGetLastError();
}

template <typename T, int TOP, bool SIDE>
cudaError_t answer_lanes_of(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    const int warps = warps_of_lanes<T, false>(g);
    // a run of hardly more chunks than the list has places would be read twice (us, classes / chunks listed: 65536 rows of 10, three alternatives 4.4 / 7.6,
    // float64 maps of 37, four alternatives 7.3 / 9.5, 100000 rows of 100, three alternatives 20.7 / 16.9, a map of 150 36 / 27)
    const bool direct = g.classes <= 16 * TOP * warps;
    if constexpr (!SIDE) {
        if (warps == kGroupWarps) {
            constexpr int kBytes = int(kGroupWarps * kGroupBytes<T, TOP>);
            if (kBytes > 48 * 1024) {
                static SmemLimit limit;
                const cudaError_t e = limit.raise(answer_groups<T, TOP>, kBytes);
                if (e != cudaSuccess) return e;
            }
            return launch_lanes(answer_groups<T, TOP>, g, a, kGroupWarps, kBytes, s);
        }
    }
    return launch_lanes(direct || TOP == 0 ? answer_lanes<T, TOP, SIDE, true> : answer_lanes<T, TOP, SIDE, TOP == 0>, g, a, warps, warps > 1 ? 4 * Found<T, TOP>::kBytes : 0, s);
}

// A warp a row where a row is a chunk or two, or where rows are so many that their number hides how long a warp is at one, a quarter as many as classes;
// else streams.  float64 warps are longer at a row: half as many, or a quarter where they have 2^24 logits or more.  (Four alternatives, warps / streams,
// us: 100 rows of 2000 classes 7.5 / 4.6, 500 8.0 / 9.5, 1000 9.3 / 15.4; 500 of 8000 21.5 / 14.7, 1000 22.8 / 19.1, 2000 26.1 / 30.5; 10000 of 16000 120
// / 137; 2048 of 32000 72 / 52, 8000 187 / 169.  float64: 200 of 1000 12.6 / 8.4, 400 12.9 / 15.2; 500 of 2000 24.4 / 15.3, 1000 24.5 / 26.1; 1500 of 4000
// 47 / 45, 2000 48 / 55; 2000 of 8000 82 / 75, 3000 99 / 104; 4000 of 16000 221 / 230; 2048 of 32000 270 / 227.)
template <typename T>
bool by_warps(const Logits& g) {
    const long long rows = g.count();
    return g.classes <= 512 || 2 * rows >= g.classes || (4 * rows >= g.classes && (sizeof(T) == 4 || rows >= (1 << 24) / g.classes));
}

// runs of one wave, but a row no more than 32 parts (30 runs a row have 31 borders in it at most)
template <typename T>
Runs runs_of(const Logits& g) {
    Runs r;
    r.of_row = int(((long long)g.classes + kWide<T> - 1 + kStreamChunk<T> - 1) / kStreamChunk<T>);
    r.chunks = r.of_row * g.count();
    r.ctas = int(std::min({r.chunks, (long long)kStreamCtas * device_sm_count(), 30 * g.count()}));
    return r;
}

template <typename T, bool TOP, int U>
cudaError_t answer_rows_of(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    in_stream_order(answer_rows<T, TOP, U>, unsigned((g.count() + kRowWarps - 1) / kRowWarps), 32 * kRowWarps, 0, s)(g, a);
    count_launch();
    return cudaGetLastError();
}

template <typename T, bool TOP>
cudaError_t answer_stream_of(const Logits& g, const Answers<T>& a, void* ws, cudaStream_t s) {
    const Runs runs = runs_of<T>(g);
    RowFound<T>* parts = static_cast<RowFound<T>*>(ws);
    static SmemLimit limit;
    cudaError_t e = limit.raise(answer_stream<T, TOP>, kStreamBytes);
    if (e != cudaSuccess) return e;
    in_stream_order(answer_stream<T, TOP>, runs.ctas, kStreamThreads + 32, kStreamBytes, s)(g, a, runs, parts);
    count_launch();
    e = cudaGetLastError();
    if (e != cudaSuccess || runs.ctas == 1 || runs.chunks % runs.ctas == 0 && runs.chunks / runs.ctas % runs.of_row == 0) return e;     // (whole rows)
    in_stream_order(join_parts<T, TOP>, runs.ctas - 1, 32, 0, s)(g, a, runs, (const RowFound<T>*)parts);
    count_launch();
    return cudaGetLastError();
}

template <typename T, bool SIDE>
cudaError_t answer_by_lanes(const Logits& g, const Answers<T>& a, cudaStream_t s) {
    if (g.top_k == 0) return answer_lanes_of<T, 0, SIDE>(g, a, s);
    if (g.top_k == 1) return answer_lanes_of<T, 1, SIDE>(g, a, s);
    if (g.top_k <= 4) return answer_lanes_of<T, 4, SIDE>(g, a, s);
    if (g.top_k <= 8) return answer_lanes_of<T, 8, SIDE>(g, a, s);
    return answer_lanes_of<T, 16, SIDE>(g, a, s);
}

template <typename T>
cudaError_t answer_as(const Logits& g, const Answers<T>& a, void* ws, cudaStream_t s) {
    if (by_rows(g, kMostByLanes)) {
        if (!by_warps<T>(g)) return g.top_k > 0 ? answer_stream_of<T, true>(g, a, ws, s) : answer_stream_of<T, false>(g, a, ws, s);
        // (60000 rows of 200 classes with three alternatives 38 us with 8 a lane, 49 with 16, 20000 of 500 20 and 18; float64 3000 of 1500 24 with 4, 32 with 8)
        constexpr int kFew = sizeof(T) == 4 ? 8 : 4, kMany = sizeof(T) == 4 ? 16 : 4;
        if (g.classes <= 32 * kFew) return g.top_k > 0 ? answer_rows_of<T, true, kFew>(g, a, s) : answer_rows_of<T, false, kFew>(g, a, s);
        return g.top_k > 0 ? answer_rows_of<T, true, kMany>(g, a, s) : answer_rows_of<T, false, kMany>(g, a, s);
    }
    return g.stride_class == 1 ? answer_by_lanes<T, true>(g, a, s) : answer_by_lanes<T, false>(g, a, s);
}

template <typename T>
cudaError_t gradient_as(const Logits& g, const Gradients<T>& a, cudaStream_t s) {
    if (!by_rows(g, kMostGradientByLanes))
        return launch_lanes(g.stride_class == 1 ? gradient_lanes<T, true> : gradient_lanes<T, false>, g, a, warps_of_lanes<T, true>(g), 0, s);
    // A chunk should be no more than a row, and a row a few chunks (us, 3000 rows of 1000 with 4 classes a lane / 16 9.3 / 6.8, 60000 of 200 34 / 45;
    // 4096 rows of 2000 by a warp / 8 13.7 / 23.4; 3000 of 6000 by 4 warps / 8 26.9 / 31.0, 2048 of 32000 86.0 / 83.5).
    constexpr int U = kStreamAhead<T>;
    const unsigned rows = unsigned(g.count()), ctas = unsigned((g.count() + kRowWarps - 1) / kRowWarps);
    if (g.classes <= 512) in_stream_order(gradient_rows<T, 1, 4>, ctas, 32 * kRowWarps, 0, s)(g, a);
    else if (g.classes <= 4096) in_stream_order(gradient_rows<T, 1, U>, ctas, 32 * kRowWarps, 0, s)(g, a);
    else if (g.classes <= 16384) in_stream_order(gradient_rows<T, 4, U>, rows, 128, 0, s)(g, a);
    else in_stream_order(gradient_rows<T, 8, U>, dim3(rows, std::min((g.classes + 16383) / 16384, 65535)), 256, 0, s)(g, a);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_log_probabilities(const simnets_likelihood_desc& d, const void* logits, const long long* labels, void* label, void* entropy, int* top_index,
                                     void* top, void* stats, void* ws, cudaStream_t s) {
    const Logits g = logits_of(d);
    if (g.count() == 0) return cudaSuccess;
    if (d.dtype == SIMNETS_F64)
        return answer_as<double>(g, {(const double*)logits, labels, (double*)label, (double*)entropy, (double*)top, (double*)stats, top_index}, ws, s);
    return answer_as<float>(g, {(const float*)logits, labels, (float*)label, (float*)entropy, (float*)top, (float*)stats, top_index}, ws, s);
}

size_t log_probabilities_workspace_bytes(const simnets_likelihood_desc& d) {
    const Logits g = logits_of(d);
    if (g.count() == 0 || !by_rows(g, kMostByLanes)) return 0;
    if (d.dtype == SIMNETS_F64) return by_warps<double>(g) ? 0 : 2 * sizeof(RowFound<double>) * runs_of<double>(g).ctas;
    return by_warps<float>(g) ? 0 : 2 * sizeof(RowFound<float>) * runs_of<float>(g).ctas;
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

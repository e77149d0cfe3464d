// Routing of positions to components: of the k components of every position the top few by score, with weights that sum to one.
//
//     l = score + prior,  v = l + bias        the choice goes by v, the weights by l (a bias moves loads, not what is learned)
//     w_i = exp(l_i) / sum of the chosen, or sigmoid(l_i) / sum of the chosen
//
// Only the chosen are exponentiated, from the largest of them: no sum over all components is needed, and the choice is made of two
// additions in the type of the scores, so that it is the same wherever it is computed.  Components whose v is -infinity or NaN are out of the
// choice; a position with fewer than top_k others has index -1 and weight 0 in what is left.
//
// Loads are added up as integers and masses (sums of weights) from the written weights in a fixed order: the same on every run.
#include "kernels.cuh"
#include <atomic>

namespace simnets {
namespace {

// Keys hold up to 256 components: beyond, what their last bits tell apart is too little, and more positions do both passes (normal scores, 131072
// positions, index and weights, keys / values and indices: four of 256 53 / 58 us, four of 300 64 / 67, four of 512 109 / 108, four of 1024 222 / 206,
// 2048 493 / 401; eight of 300 92 / 115).
constexpr int kRouteThreads = 128, kKeyed = 256, kSums = 16 * 1024;

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float log1p_of(float v) { return log1pf(v); }
__device__ __forceinline__ double log1p_of(double v) { return log1p(v); }

template <typename T> __device__ __forceinline__ T below_all() { return -T(CUDART_INF_F); }

// the TK largest so far, largest first; equal ones keep the order in which they came
template <typename T, int TK>
struct Top {
    T v[TK];
    int i[TK];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < TK; ++t) { v[t] = below_all<T>(); i[t] = -1; }
    }
    // (a NaN and -infinity are above nothing; what makes room moves on in front of its equals)
    __device__ __forceinline__ void offer(T value, int index) {
        bool above = false;
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            above = above || value > v[t];
            const T ov = v[t];
            const int oi = i[t];
            v[t] = above ? value : ov; i[t] = above ? index : oi;
            value = above ? ov : value; index = above ? oi : index;
        }
    }
    // by falling value, equal ones by index, empty places last
    __device__ __forceinline__ void sort() {
#pragma unroll
        for (int n = TK - 1; n > 0; --n)
#pragma unroll
            for (int t = 0; t < n; ++t) {
                const bool swap = v[t + 1] > v[t] || (v[t + 1] == v[t] && unsigned(i[t + 1]) < unsigned(i[t]));
                const T ov = v[t];
                const int oi = i[t];
                v[t] = swap ? v[t + 1] : ov; i[t] = swap ? i[t + 1] : oi;
                v[t + 1] = swap ? ov : v[t + 1]; i[t + 1] = swap ? oi : i[t + 1];
            }
    }
    // the lists of the G lanes that share a position (RUN lanes apart) as one, the same in all of them; equal values by index
    template <int G, int RUN>
    __device__ __forceinline__ void merge() {
        if constexpr (G > 1) {
            Top all;
#pragma unroll
            for (int t = 0; t < TK; ++t) {
                T bv = v[0];
                unsigned bi = unsigned(i[0]);                            // (-1, nothing, is the largest)
#pragma unroll
                for (int d = RUN; d < 32; d <<= 1) {
                    const T ov = __shfl_xor_sync(0xffffffffu, bv, d);
                    const unsigned oi = __shfl_xor_sync(0xffffffffu, bi, d);
                    const bool other = ov > bv || (ov == bv && oi < bi);
                    bv = other ? ov : bv; bi = other ? oi : bi;
                }
                all.v[t] = bv; all.i[t] = int(bi);
                if (bi == unsigned(i[0])) {                              // it was this lane's: the next one comes up
#pragma unroll
                    for (int u = 0; u + 1 < TK; ++u) { v[u] = v[u + 1]; i[u] = i[u + 1]; }
                    v[TK - 1] = below_all<T>(); i[TK - 1] = -1;
                }
            }
            *this = all;
        }
    }
};

// The TK + 1 largest of float32 values whose last bits are replaced by the component: one key instead of a value and an index, so that a place of the
// list is a minimum and a maximum instead of five instructions.  What the bits decide, keys of one bucket, is looked at afterwards.
__device__ __forceinline__ float min_or_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
template <int TK>
struct Keys {
    float t[TK + 1], total;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i <= TK; ++i) t[i] = below_all<float>();
        total = 0.f;
    }
    // (-infinity becomes a NaN, which moves nothing; infinity and NaN show in the total, which is scaled so that numbers do not make an infinity)
    __device__ __forceinline__ void offer(float v, int c, uint32_t mask) {
        v += 0.f;                                                        // (-0 = 0)
        total = fmaf(v, 0x1p-13f, total);
        const float key = __uint_as_float((__float_as_uint(v) & ~mask) | uint32_t(c));
#pragma unroll
        for (int i = TK; i > 0; --i) t[i] = fmaxf(t[i], min_or_nan(t[i - 1], key));
        t[0] = fmaxf(t[0], key);
    }
    __device__ __forceinline__ bool empty(int i) const { return t[i] == below_all<float>(); }
    __device__ __forceinline__ int at(int i, uint32_t mask) const { return empty(i) ? -1 : int(__float_as_uint(t[i]) & mask); }
    __device__ __forceinline__ bool alike(int i, uint32_t mask) const { return !empty(i) && ((__float_as_uint(t[i - 1]) ^ __float_as_uint(t[i])) & ~mask) == 0; }
    // whether the first `top` are not known by the keys
    __device__ __forceinline__ bool unknown(int top, uint32_t mask) const {
        bool yes = !(total < CUDART_INF_F);
#pragma unroll
        for (int i = 1; i <= TK; ++i) yes = yes || (i == top && alike(i, mask));
        return yes;
    }
    // whether their order is not
    __device__ __forceinline__ bool unordered(int top, uint32_t mask) const {
        bool yes = false;
#pragma unroll
        for (int i = 1; i < TK; ++i) yes = yes || (i < top && alike(i, mask));
        return yes;
    }
};

struct RouteArgs {
    long long positions;         // of the whole batch
    long long N;                 // per sample
    FastDiv f_N;                 // where `positions` fits 31 bits
    int k, top, groups, size, top_groups;
    int turns;                   // in which the warps of a CTA add to their common sums
    uint32_t key_mask;           // last bits of a key that hold the component, 0 for no keys
    int sigmoid;
    double scale;
};
// sample and place inside it
__device__ __forceinline__ long long sample_of(const RouteArgs& a, long long p) { return a.f_N.d ? (long long)fast_div(uint32_t(p), a.f_N) : p / a.N; }

template <typename T> struct alignas(2 * sizeof(T)) Pair { T prior, bias; };

// f(v, c) for components from .. to, every G-th from `sub` on; `add`: prior and bias of every component, or null for none
template <int G, int kBatch, bool AHEAD = true, typename T, class F>
__device__ __forceinline__ void over_range(const T* __restrict__ s, long long N, const Pair<T>* add, int from, int to, int sub, F f) {
    int c = from + sub;
    const T* q = s + c * N;
    const long long step = G * N;
    T v[kBatch], w[kBatch];
    auto load = [&](T (&b)[kBatch]) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u, q += step) b[u] = __ldg(q);
    };
    auto give = [&](const T (&b)[kBatch]) {
        if (add)
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const Pair<T> both = add[c + G * u];
                f((b[u] + both.prior) + both.bias, c + G * u);
            }
        else
#pragma unroll
            for (int u = 0; u < kBatch; ++u) f(b[u], c + G * u);
        c += G * kBatch;
    };
    if (!AHEAD)
        for (; c + G * (kBatch - 1) < to;) { load(v); give(v); }
    int left = AHEAD && c < to ? ((to - c - 1) / G + 1) / kBatch : 0;             // whole batches, the next one under way while one is worked on
    if (left > 0) load(v);
    while (left > 0) {
        if (left > 1) load(w);
        give(v);
        if (left > 1) {
            if (left > 2) load(v);
            give(w);
        }
        left -= 2;
    }
    if (c < to) {
#pragma unroll
        for (int u = 0; u < kBatch - 1; ++u, q += step) v[u] = c + G * u < to ? __ldg(q) : T(0);
#pragma unroll
        for (int u = 0; u < kBatch - 1; ++u)
            if (c + G * u < to) f(add ? (v[u] + add[c + G * u].prior) + add[c + G * u].bias : v[u], c + G * u);
    }
}
// the largest of them, over the lanes of a position
template <int G, int kBatch, typename T>
__device__ __forceinline__ T best_of_range(const T* __restrict__ s, long long N, const Pair<T>* add, int from, int to, int sub) {
    T best = below_all<T>();
    over_range<G, kBatch>(s, N, add, from, to, sub, [&](T v, int) { best = v > best ? v : best; });
#pragma unroll
    for (int d = 32 / G; d < 32; d <<= 1) {
        const T other = __shfl_xor_sync(0xffffffffu, best, d);
        best = other > best ? other : best;
    }
    return best;
}

// Bound: HBM, the scores read once and, for the dense form, as much written (512 x 64 x 30 x 30 float32: 236 MB, 36 us).  The nearest one of
// 64 components takes 47 us (5.0 TB/s); cut to four 66: loads of a warp wait for the list of the ones in front (sparse 42, three of 24 components 22).
//
// G lanes share a position where positions are few, neighbouring lanes are neighbouring positions; a lane has eight scores in flight beside the eight
// that it puts into a sorted list of TK.  Up to 256 components lists are of keys (`Keys`; with values and indices 81 and 52 us); what keys do not
// tell, a tie at the end of the list or infinities, is done again with values and indices (scores rounded to integers, where every warp does both: 91 and
// 72), and ties inside the list are sorted.  (Also tried: a position's scores in the registers of four lanes, with lists of values only, 105 us; two
// passes, values alone in sorting networks and then who reaches the last of them, 100; registers held down to nine CTAs a multiprocessor, 87.)  192
// components in groups, 64 x 15 x 15, six of three of eight groups: 17 us with the maxima of four groups in flight (23 with one).
//
// With SUMS a CTA adds the weights up in shared memory: a column of sums per thread, or, where those would keep CTAs out, per two or four threads of
// different warps, which then take turns (78 -> 72 us).  As many CTAs as are resident by their registers too: more of them begin when the SMs run empty
// (72 -> 66).  The masses cost no second pass over the dense form, and come out the same on every run.
template <typename T, int TK, int G, bool SUMS, bool GROUPS>
__global__ void __launch_bounds__(kRouteThreads) route_choose(RouteArgs a, const T* __restrict__ scores, const T* __restrict__ prior, const T* __restrict__ bias,
                                                              int* __restrict__ index, T* __restrict__ weights, T* __restrict__ dense, T* __restrict__ part_mass,
                                                              unsigned* __restrict__ part_load) {
    stream_order();
    constexpr int RUN = 32 / G, PLACES = kRouteThreads / G;
    constexpr int kBatch = 8;                                                // scores of a position in flight (there are fewer warps beside the sums)
    extern __shared__ __align__(16) unsigned char route_smem[];
    const int columns = SUMS ? PLACES / a.turns : 0;
    T* const sums = reinterpret_cast<T*>(route_smem);                                    // [k][columns]
    Pair<T>* const add_s = reinterpret_cast<Pair<T>*>(sums + (size_t)a.k * columns);
    unsigned* const load = reinterpret_cast<unsigned*>(add_s + a.k);
    const int lane = threadIdx.x & 31, sub = lane / RUN, place = (threadIdx.x >> 5) * RUN + lane % RUN;
    for (int c = threadIdx.x; c < a.k; c += kRouteThreads) {
        load[c] = 0;
        add_s[c] = Pair<T>{prior ? prior[c] : T(0), bias ? bias[c] : T(0)};
    }
    if (SUMS) for (int i = threadIdx.x; i < a.k * columns; i += kRouteThreads) sums[i] = T(0);
    __syncthreads();
    const Pair<T>* const add = prior || bias ? add_s : nullptr;
    for (long long p0 = (long long)blockIdx.x * PLACES; p0 < a.positions; p0 += (long long)gridDim.x * PLACES) {
        const long long p = p0 + place;
        const bool live = p < a.positions;
        const long long n = sample_of(a, live ? p : p0), j = (live ? p : p0) - n * a.N;
        const T* s = scores + n * a.k * a.N + j;
        unsigned long long open = 0;                     // groups that are in the choice
        Top<T, TK> top;
        if constexpr (GROUPS) {
            top.clear();
            if (a.size <= G * kBatch) {                  // several groups in flight
                constexpr int S = 4;
                for (int g0 = 0; g0 < a.groups; g0 += S) {
                    T v[S][kBatch], best[S];
#pragma unroll
                    for (int j = 0; j < S; ++j)
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) {
                            const int c = sub + G * u;
                            v[j][u] = c < a.size && g0 + j < a.groups ? __ldg(s + ((g0 + j) * a.size + c) * a.N) : below_all<T>();
                        }
#pragma unroll
                    for (int j = 0; j < S; ++j) {
                        best[j] = below_all<T>();
#pragma unroll
                        for (int u = 0; u < kBatch; ++u) {
                            const int c = (g0 + j) * a.size + sub + G * u;
                            if (add && sub + G * u < a.size && g0 + j < a.groups) v[j][u] = (v[j][u] + add[c].prior) + add[c].bias;
                            best[j] = v[j][u] > best[j] ? v[j][u] : best[j];
                        }
#pragma unroll
                        for (int d = RUN; d < 32; d <<= 1) {
                            const T other = __shfl_xor_sync(0xffffffffu, best[j], d);
                            best[j] = other > best[j] ? other : best[j];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < S; ++j) top.offer(best[j], g0 + j);
                }
            } else {
                for (int g = 0; g < a.groups; ++g) top.offer(best_of_range<G, kBatch>(s, a.N, add, g * a.size, (g + 1) * a.size, sub), g);
            }
#pragma unroll
            for (int t = 0; t < TK; ++t) if (t < a.top_groups && top.i[t] >= 0) open |= 1ull << top.i[t];
        }
        top.clear();
        if constexpr (GROUPS) {
            for (; open; open &= open - 1) {             // (by rising index; every position has about as many)
                const int g = __ffsll((long long)open) - 1;
                over_range<G, kBatch>(s, a.N, add, g * a.size, (g + 1) * a.size, sub, [&](T v, int c) { top.offer(v, c); });
            }
            __syncwarp();
        } else {
            constexpr bool KEYS = sizeof(T) == 4 && TK > 1;
            bool whole = true;                           // values and indices are compared one by one
            if constexpr (KEYS) {
                const uint32_t mask = a.key_mask;
                if (mask) {
                    Keys<TK> keys;
                    keys.clear();
                    over_range<G, kBatch, (TK < 16 || G > 1)>(s, a.N, add, 0, a.k, sub, [&](T v, int c) { keys.offer(v, c, mask); });
                    whole = __any_sync(0xffffffffu, keys.unknown(a.top, mask));
                    if (!whole) {
#pragma unroll
                        for (int t = 0; t < TK; ++t) top.i[t] = t < a.top ? keys.at(t, mask) : -1;
                        const bool sort = __any_sync(0xffffffffu, keys.unordered(a.top, mask));
                        if (G > 1 || sort) {             // (sorted by value, then index)
#pragma unroll
                            for (int t = 0; t < TK; ++t) {
                                if (top.i[t] < 0) continue;
                                const T v = __ldg(s + top.i[t] * a.N);
                                top.v[t] = add ? (v + add[top.i[t]].prior) + add[top.i[t]].bias : v;
                            }
                            if (sort) top.sort();
                        }
                    }
                }
            }
            if (whole) over_range<G, kBatch, !KEYS || (G > 1)>(s, a.N, add, 0, a.k, sub, [&](T v, int c) { top.offer(v, c); });
        }
        top.template merge<G, RUN>();
        // weights of the chosen: they sum to one over them
        T l[TK], hi = below_all<T>(), sum = T(0);
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            l[t] = below_all<T>();
            if (t >= a.top || top.i[t] < 0) continue;
            l[t] = __ldg(s + top.i[t] * a.N);
            if (add) l[t] += add[top.i[t]].prior;
            if (a.sigmoid) l[t] = l[t] >= T(0) ? -log1p_of(exp_of(-l[t])) : l[t] - log1p_of(exp_of(l[t]));
            hi = l[t] > hi ? l[t] : hi;
        }
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            l[t] = t < a.top && top.i[t] >= 0 ? (l[t] == hi ? T(1) : exp_of(l[t] - hi)) : T(0);              // (infinities are equal too)
            sum += l[t];
        }
        const T scale = T(a.scale), inv = sum > T(0) ? T(1) / sum : T(0);
#pragma unroll
        for (int t = 0; t < TK; ++t) l[t] = scale * (l[t] * inv);
        if (live && dense) {
            T* d = dense + (n * a.k + sub) * a.N + j;
            const long long step = G * a.N;
            if constexpr (TK == 1) {                     // every value once
#pragma unroll 4
                for (int c = sub; c < a.k; c += G, d += step) __stcs(d, c == top.i[0] ? l[0] : T(0));
            } else {                                     // zeros, then the chosen (each by the lane that wrote its zero)
#pragma unroll 8
                for (int c = sub; c < a.k; c += G, d += step) *d = T(0);
#pragma unroll
                for (int t = 0; t < TK; ++t)
                    if (t < a.top && top.i[t] >= 0 && top.i[t] % G == sub) dense[(n * a.k + top.i[t]) * a.N + j] = l[t];
            }
        }
        if (live && sub == 0) {
#pragma unroll
            for (int t = 0; t < TK; ++t) {
                if (t >= a.top) continue;
                const long long at = (n * a.top + t) * a.N + j;
                if (index) index[at] = top.i[t];
                if (weights) weights[at] = l[t];
                if (top.i[t] < 0) continue;
                atomicAdd(load + top.i[t], 1u);
            }
        }
        if constexpr (SUMS)
            for (int turn = 0; turn < a.turns; ++turn) {
                if (turn == (threadIdx.x >> 5) * a.turns / (kRouteThreads / 32) && live && sub == 0) {
#pragma unroll
                    for (int t = 0; t < TK; ++t)
                        if (t < a.top && top.i[t] >= 0) sums[top.i[t] * columns + (place & (columns - 1))] += l[t];
                }
                if (a.turns > 1) __syncthreads();
            }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.k; c += kRouteThreads) part_load[(size_t)blockIdx.x * a.k + c] = load[c];
    if constexpr (SUMS)
        for (int c = threadIdx.x >> 5; c < a.k; c += kRouteThreads / 32) {
            T m = T(0);
            for (int i = lane; i < columns; i += 32) m += sums[c * columns + i];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) m += __shfl_xor_sync(0xffffffffu, m, d);
            if (lane == 0) part_mass[(size_t)blockIdx.x * a.k + c] = m;
        }
}

// part[split][c] = sum of the responsibilities of component c = blockIdx.x in the split's samples (for more components than shared memory has sums for)
template <typename T>
__global__ void __launch_bounds__(256) route_mass(RouteArgs a, long long batch, const T* __restrict__ dense, T* __restrict__ part) {
    stream_order();
    __shared__ T red[256];
    T sum = T(0);
    for (long long n = blockIdx.y; n < batch; n += gridDim.y) {
        const T* d = dense + (n * a.k + blockIdx.x) * a.N;
        for (long long j = threadIdx.x; j < a.N; j += 256) sum += d[j];
    }
    red[threadIdx.x] = sum;
    __syncthreads();
    for (int d = 128; d > 0; d >>= 1) {
        if (threadIdx.x < d) red[threadIdx.x] += red[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) part[(size_t)blockIdx.y * a.k + blockIdx.x] = red[0];
}

template <typename T>
__global__ void __launch_bounds__(128) route_totals(int ctas, int splits, int k, T weight, const unsigned* __restrict__ part_load, const T* __restrict__ part_mass,
                                                    long long* __restrict__ load, T* __restrict__ mass) {
    stream_order();
    __shared__ long long red[128];
    __shared__ T redm[128];
    long long n = 0;
    T m = T(0);
    for (int i = threadIdx.x; i < ctas; i += 128) n += part_load[(size_t)i * k + blockIdx.x];
    if (mass) for (int i = threadIdx.x; i < splits; i += 128) m += part_mass[(size_t)i * k + blockIdx.x];
    red[threadIdx.x] = n; redm[threadIdx.x] = m;
    __syncthreads();
    for (int d = 64; d > 0; d >>= 1) {
        if (threadIdx.x < d) { red[threadIdx.x] += red[threadIdx.x + d]; redm[threadIdx.x] += redm[threadIdx.x + d]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        load[blockIdx.x] = red[0];
        if (mass) mass[blockIdx.x] = splits > 0 ? redm[0] : weight * T(red[0]);
    }
}

// dscores of the weights' gradient:  dl_i = W_i (g_i - sum_j W_j g_j / scale), times 1 - sigmoid(l_i) where the values are sigmoids.
// Bound: HBM, the zeros of the others.  A thread has a position and a run of components (blockIdx.y): its zeros, then the chosen among them.
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) route_gradient(RouteArgs a, const T* __restrict__ scores, const T* __restrict__ prior, const int* __restrict__ index,
                                                                const T* __restrict__ weights, const T* __restrict__ grad, T* __restrict__ dscores) {
    stream_order();
    const T inv_scale = T(1.0 / a.scale);
    const int from = int((long long)a.k * blockIdx.y / gridDim.y), to = int((long long)a.k * (blockIdx.y + 1) / gridDim.y);
    for (long long p = (long long)blockIdx.x * kRouteThreads + threadIdx.x; p < a.positions; p += (long long)gridDim.x * kRouteThreads) {
        const long long n = sample_of(a, p), j = p - n * a.N, chosen = n * a.top * a.N + j;
        const T* s = scores + n * a.k * a.N + j;
        T* d = dscores + (n * a.k + from) * a.N + j;
#pragma unroll 8
        for (int c = from; c < to; ++c, d += a.N) *d = T(0);
        T sum = T(0);
        for (int t = 0; t < a.top; ++t)
            if (index[chosen + t * a.N] >= 0) sum += weights[chosen + t * a.N] * inv_scale * grad[chosen + t * a.N];
        for (int t = 0; t < a.top; ++t) {
            const int c = index[chosen + t * a.N];
            if (c < from || c >= to) continue;
            T v = weights[chosen + t * a.N] * (grad[chosen + t * a.N] - sum);
            if (a.sigmoid) {
                T l = s[c * a.N];
                if (prior) l += prior[c];
                v *= T(1) / (T(1) + exp_of(l));
            }
            dscores[(n * a.k + c) * a.N + j] = v;
        }
    }
}

RouteArgs args_of(const simnets_route_desc& d) {
    RouteArgs a;
    a.N = d.positions;
    a.positions = d.positions * d.batch;
    a.f_N = FastDiv{0, 0, 0};
    if (a.positions > 0 && a.positions <= 0x7fffffffLL) a.f_N = make_fastdiv(int(a.N));
    a.k = d.components; a.top = d.top_k; a.groups = d.groups; a.size = d.components / d.groups; a.top_groups = d.top_groups;
    a.turns = 1;
    a.key_mask = 0;
    if (a.k > 1 && a.k <= kKeyed)
        while (int(a.key_mask) < a.k - 1) a.key_mask = 2 * a.key_mask + 1;
    a.sigmoid = d.sigmoid != 0;
    a.scale = d.scale;
    return a;
}
// Lanes per position: eight where positions are few for their components (a lane each leaves the loads of a position in turn), where groups are
// chosen four (64 x 15 x 15, six of 192: 17 us; with eight, whose maxima go over one lane more each, 26), else one (no lists to merge).  Index and
// weights of scores that are not in L2, us with eight lanes / with one, over 4096, 14400 and 57600 positions:
//     two of 16      4.9 / 4.1     6.8 / 4.5    13.4 / 7.0        eight of 192   11.4 / 24.8    19.3 / 28.8    54.8 / 43.0
//     four of 64     6.3 / 7.2    11.3 / 9.5    22.2 / 13.1       four of 1024   18.2 / 105     33.2 / 107      100 / 133
//     four of 128    8.1 / 13.0   12.8 / 14.8   26.9 / 20.8       six of 192 in three of eight groups, four lanes / one   15.9 / 20.7  22.0 / 23.0  59.2 / 35.5
// They meet near 128 positions a component, with groups near 64; many components with the dense form earlier (1024: 14).
int route_lanes(const simnets_route_desc& d) {
    const bool groups = d.top_groups < d.groups;
    if (d.positions * d.batch >= std::min<long long>(512LL * device_sm_count(), (groups ? 64LL : 128LL) * d.components) || d.components < 8) return 1;
    return groups ? 4 : 8;
}
// a CTA's sums: a column per position, or for two or four of them one after the other where that leaves room for more CTAs
size_t sums_bytes(const simnets_route_desc& d, int turns) { return (d.dtype == SIMNETS_F64 ? 8 : 4) * (size_t)d.components * (kRouteThreads / route_lanes(d) / turns); }
int sums_turns(const simnets_route_desc& d) { return sums_bytes(d, 1) <= kSums ? 1 : sums_bytes(d, 2) <= kSums ? 2 : 4; }
size_t sums_bytes(const simnets_route_desc& d) { return sums_bytes(d, sums_turns(d)); }
bool route_sums(const simnets_route_desc& d) { return d.top_k > 1 && d.top_groups == d.groups && sums_bytes(d) <= 2 * kSums; }
size_t choose_bytes(const simnets_route_desc& d, bool sums) { return (sums ? sums_bytes(d) : 0) + (size_t)d.components * (2 * (d.dtype == SIMNETS_F64 ? 8 : 4) + sizeof(unsigned)); }
// as many CTAs as are resident together
int route_ctas(const simnets_route_desc& d, bool sums) {
    const long long places = kRouteThreads / route_lanes(d), tiles = (d.positions * d.batch + places - 1) / places;
    const long long resident = std::max<long long>(1, std::min<long long>(12, 220 * 1024 / (choose_bytes(d, sums) + 2048))) * device_sm_count();
    return int(std::max<long long>(1, std::min(tiles, resident)));
}
int most_ctas(const simnets_route_desc& d) { return std::max(route_ctas(d, false), route_ctas(d, route_sums(d))); }
int mass_splits(const simnets_route_desc& d) {
    if (route_sums(d)) return most_ctas(d);
    return int(std::max<long long>(1, std::min<long long>(d.batch, (8LL * device_sm_count() + d.components - 1) / d.components)));
}
size_t load_bytes(const simnets_route_desc& d) { return (sizeof(unsigned) * (size_t)most_ctas(d) * d.components + 255) & ~size_t(255); }

// CTAs of a kernel that the registers of a multiprocessor hold (its own answer, asked for once)
template <typename K>
int held_by_registers(K kernel, std::atomic<int>& known) {
    int n = known.load(std::memory_order_relaxed);
    if (n == 0) {
        cudaFuncAttributes at;
        n = cudaFuncGetAttributes(&at, kernel) == cudaSuccess && at.numRegs > 0 ? std::max(1, 65536 / (kRouteThreads * ((at.numRegs + 7) / 8 * 8))) : 4;
        known.store(n, std::memory_order_relaxed);
    }
    return n;
}

// `ctas`: how many it launched
template <typename T, int TK, int G, bool SUMS, bool GROUPS>
cudaError_t choose(int& ctas, const simnets_route_desc& d, const RouteArgs& a, const void* scores, const void* prior, const void* bias, int* index, void* weights, void* dense,
                   T* part_mass, unsigned* part_load, cudaStream_t s) {
    const size_t smem = choose_bytes(d, SUMS);
    static SmemLimit limit;
    if (smem > 32 * 1024) {
        const cudaError_t e = limit.raise(route_choose<T, TK, G, SUMS, GROUPS>, 160 * 1024);
        if (e != cudaSuccess) return e;
    }
    static std::atomic<int> held{0};
    ctas = std::min(route_ctas(d, SUMS), held_by_registers(route_choose<T, TK, G, SUMS, GROUPS>, held) * device_sm_count());
    in_stream_order(route_choose<T, TK, G, SUMS, GROUPS>, ctas, kRouteThreads, smem, s)(a, (const T*)scores, (const T*)prior, (const T*)bias, index, (T*)weights, (T*)dense, part_mass, part_load);
    return cudaSuccess;
}

template <typename T>
cudaError_t route(const simnets_route_desc& d, const void* scores, const void* prior, const void* bias, int* index, void* weights, void* dense, long long* load,
                  void* mass, void* ws, cudaStream_t s) {
    RouteArgs a = args_of(d);
    a.turns = sums_turns(d);
    const bool sums = dense && route_sums(d), one = route_lanes(d) == 1, counted = a.top == 1;      // (of one chosen the weight is the scale: the mass is that many of the load)
    int ctas = 0;
    const int want = std::max(a.top, a.top_groups < a.groups ? a.top_groups : 1);
    unsigned* part_load = static_cast<unsigned*>(ws);
    T* part_mass = reinterpret_cast<T*>(static_cast<char*>(ws) + load_bytes(d));
    cudaError_t e = cudaSuccess;
#define CHOOSE(TK, G, SUMS, GROUPS) choose<T, TK, G, SUMS, GROUPS>(ctas, d, a, scores, prior, bias, index, weights, dense, part_mass, part_load, s)
#define ROUTE(TK) e = sums ? (one ? CHOOSE(TK, 1, true, false) : CHOOSE(TK, 8, true, false))                                                            \
                           : a.top_groups < a.groups ? (one ? CHOOSE(TK, 1, false, true) : CHOOSE(TK, 4, false, true))                                   \
                                                     : (one ? CHOOSE(TK, 1, false, false) : CHOOSE(TK, 8, false, false))
    if (want <= 1) ROUTE(1);
    else if (sizeof(T) == 8 ? want <= 4 : false) ROUTE(4);               // (float64: fewer lengths of the list)
    else if constexpr (sizeof(T) == 4) { if (want <= 2) ROUTE(2); else if (want <= 4) ROUTE(4); else if (want <= 8) ROUTE(8); else ROUTE(16); }
    else ROUTE(16);
#undef CHOOSE
#undef ROUTE
    if (e != cudaSuccess) return e;
    const int splits = sums ? ctas : mass_splits(d);
    if (mass && !sums && !counted) in_stream_order(route_mass<T>, dim3(a.k, splits), 256, 0, s)(a, (long long)d.batch, (const T*)dense, part_mass);
    in_stream_order(route_totals<T>, a.k, 128, 0, s)(ctas, counted ? 0 : splits, a.k, T(a.scale), part_load, part_mass, load, (T*)mass);
    count_launch(mass && !sums && !counted ? 3 : 2);
    return cudaGetLastError();
}

}  // namespace

size_t route_workspace_bytes(const simnets_route_desc& d) { return load_bytes(d) + sizeof(double) * (size_t)mass_splits(d) * d.components; }

cudaError_t launch_route(const simnets_route_desc& d, const void* scores, const void* prior, const void* bias, int* index, void* weights, void* dense,
                         long long* load, void* mass, void* ws, cudaStream_t s) {
    return d.dtype == SIMNETS_F64 ? route<double>(d, scores, prior, bias, index, weights, dense, load, mass, ws, s)
                                  : route<float>(d, scores, prior, bias, index, weights, dense, load, mass, ws, s);
}

cudaError_t launch_route_gradient(const simnets_route_desc& d, const void* scores, const void* prior, const int* index, const void* weights, const void* grad,
                                  void* dscores, cudaStream_t s) {
    const RouteArgs a = args_of(d);
    if (a.positions == 0) return cudaSuccess;
    const long long tiles = (a.positions + kRouteThreads - 1) / kRouteThreads, resident = 12LL * device_sm_count();
    const dim3 ctas(unsigned(std::min(tiles, resident)), unsigned(std::max<long long>(1, std::min<long long>(a.k / 16, resident / tiles))));
    if (d.dtype == SIMNETS_F64)
        in_stream_order(route_gradient<double>, ctas, kRouteThreads, 0, s)(a, (const double*)scores, (const double*)prior, index, (const double*)weights, (const double*)grad, (double*)dscores);
    else
        in_stream_order(route_gradient<float>, ctas, kRouteThreads, 0, s)(a, (const float*)scores, (const float*)prior, index, (const float*)weights, (const float*)grad, (float*)dscores);
    count_launch();
    return cudaGetLastError();
}

}  // namespace simnets

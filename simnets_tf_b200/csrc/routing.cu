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

namespace simnets {
namespace {

constexpr int kRouteThreads = 128;

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

struct RouteArgs {
    long long positions;         // of the whole batch
    long long N;                 // per sample
    FastDiv f_N;                 // where `positions` fits 31 bits
    int k, top, groups, size, top_groups;
    int sigmoid;
    double scale;
};
// sample and place inside it
__device__ __forceinline__ long long sample_of(const RouteArgs& a, long long p) { return a.f_N.d ? (long long)fast_div(uint32_t(p), a.f_N) : p / a.N; }

template <typename T> struct alignas(2 * sizeof(T)) Pair { T prior, bias; };

// f(v, c) for components from .. to, every G-th from `sub` on; `add`: prior and bias of every component, or null for none
template <int G, int kBatch, typename T, class F>
__device__ __forceinline__ void over_range(const T* __restrict__ s, long long N, const Pair<T>* add, int from, int to, int sub, F f) {
    int c = from + sub;
    const T* q = s + c * N;
    const long long step = G * N;
    for (; c + G * (kBatch - 1) < to; c += G * kBatch) {
        T v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u, q += step) v[u] = __ldg(q);
        if (add)
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const Pair<T> both = add[c + G * u];
                f((v[u] + both.prior) + both.bias, c + G * u);
            }
        else
#pragma unroll
            for (int u = 0; u < kBatch; ++u) f(v[u], c + G * u);
    }
    if (c < to) {
        T v[kBatch - 1];
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
// 64 components takes 54 us (4.4 TB/s); cut to four 81: a place of the list is five instructions of the half-rate pipe per component (66 % busy).
//
// G lanes share a position (four where positions are few), neighbouring lanes are neighbouring positions; a lane has eight or sixteen scores in
// flight and keeps a sorted list of TK.  (A position's scores in the registers of four lanes, with lists of values only: 105 us; two passes, values
// alone in sorting networks and then who reaches the last of them: 100.)  192 components in groups, 64 x 15 x 15, six of three of eight groups: 17 us with the
// maxima of four groups in flight (23 with one).
// With SUMS every thread adds the weights that it gives to sums of its own in shared memory, one per component, which the CTA adds up at its
// end: the masses cost no second pass over the dense form, and come out the same on every run.
template <typename T, int TK, int G, bool SUMS, bool GROUPS>
__global__ void __launch_bounds__(kRouteThreads) route_choose(RouteArgs a, const T* __restrict__ scores, const T* __restrict__ prior, const T* __restrict__ bias,
                                                              int* __restrict__ index, T* __restrict__ weights, T* __restrict__ dense, T* __restrict__ part_mass,
                                                              unsigned* __restrict__ part_load) {
    stream_order();
    constexpr int RUN = 32 / G, PLACES = kRouteThreads / G;
    constexpr int kBatch = SUMS ? 16 : 8;                                                // scores of a position in flight (there are fewer warps beside the sums)
    extern __shared__ __align__(16) unsigned char route_smem[];
    T* const sums = reinterpret_cast<T*>(route_smem);                                    // [k][PLACES]
    Pair<T>* const add_s = reinterpret_cast<Pair<T>*>(sums + (SUMS ? (size_t)a.k * PLACES : 0));
    unsigned* const load = reinterpret_cast<unsigned*>(add_s + a.k);
    const int lane = threadIdx.x & 31, sub = lane / RUN, place = (threadIdx.x >> 5) * RUN + lane % RUN;
    for (int c = threadIdx.x; c < a.k; c += kRouteThreads) {
        load[c] = 0;
        add_s[c] = Pair<T>{prior ? prior[c] : T(0), bias ? bias[c] : T(0)};
    }
    if (SUMS) for (int i = threadIdx.x; i < a.k * PLACES; i += kRouteThreads) sums[i] = T(0);
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
            over_range<G, kBatch>(s, a.N, add, 0, a.k, sub, [&](T v, int c) { top.offer(v, c); });
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
                if (SUMS) sums[top.i[t] * PLACES + place] += l[t];
                atomicAdd(load + top.i[t], 1u);
            }
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.k; c += kRouteThreads) part_load[(size_t)blockIdx.x * a.k + c] = load[c];
    if constexpr (SUMS)
        for (int c = threadIdx.x >> 5; c < a.k; c += kRouteThreads / 32) {
            T m = T(0);
#pragma unroll
            for (int i = 0; i < PLACES; i += 32) m += sums[c * PLACES + i + lane];
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
    a.sigmoid = d.sigmoid != 0;
    a.scale = d.scale;
    return a;
}
// lanes per position: one where the positions fill the GPU
int route_lanes(const simnets_route_desc& d) { return d.positions * d.batch >= 512LL * device_sm_count() || d.components < 8 ? 1 : 4; }
// a CTA's sums fit the shared memory of a multiprocessor three times
size_t sums_bytes(const simnets_route_desc& d) { return (d.dtype == SIMNETS_F64 ? 8 : 4) * (size_t)d.components * (kRouteThreads / route_lanes(d)); }
bool route_sums(const simnets_route_desc& d) { return d.top_k > 1 && d.top_groups == d.groups && sums_bytes(d) <= 64 * 1024; }
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

template <typename T, int TK, int G, bool SUMS, bool GROUPS>
cudaError_t choose(const simnets_route_desc& d, const RouteArgs& a, const void* scores, const void* prior, const void* bias, int* index, void* weights, void* dense,
                   T* part_mass, unsigned* part_load, cudaStream_t s) {
    const size_t smem = choose_bytes(d, SUMS);
    static SmemLimit limit;
    if (smem > 32 * 1024) {
        const cudaError_t e = limit.raise(route_choose<T, TK, G, SUMS, GROUPS>, 160 * 1024);
        if (e != cudaSuccess) return e;
    }
    in_stream_order(route_choose<T, TK, G, SUMS, GROUPS>, route_ctas(d, SUMS), kRouteThreads, smem, s)(a, (const T*)scores, (const T*)prior, (const T*)bias, index, (T*)weights, (T*)dense, part_mass, part_load);
    return cudaSuccess;
}

template <typename T>
cudaError_t route(const simnets_route_desc& d, const void* scores, const void* prior, const void* bias, int* index, void* weights, void* dense, long long* load,
                  void* mass, void* ws, cudaStream_t s) {
    const RouteArgs a = args_of(d);
    const bool sums = dense && route_sums(d), one = route_lanes(d) == 1, counted = a.top == 1;      // (of one chosen the weight is the scale: the mass is that many of the load)
    const int ctas = route_ctas(d, sums), splits = sums ? ctas : mass_splits(d), want = std::max(a.top, a.top_groups < a.groups ? a.top_groups : 1);
    unsigned* part_load = static_cast<unsigned*>(ws);
    T* part_mass = reinterpret_cast<T*>(static_cast<char*>(ws) + load_bytes(d));
    cudaError_t e = cudaSuccess;
#define CHOOSE(TK, G, SUMS, GROUPS) choose<T, TK, G, SUMS, GROUPS>(d, a, scores, prior, bias, index, weights, dense, part_mass, part_load, s)
#define ROUTE(TK) e = sums ? (one ? CHOOSE(TK, 1, true, false) : CHOOSE(TK, 4, true, false))                                                            \
                           : a.top_groups < a.groups ? (one ? CHOOSE(TK, 1, false, true) : CHOOSE(TK, 4, false, true))                                   \
                                                     : (one ? CHOOSE(TK, 1, false, false) : CHOOSE(TK, 4, false, false))
    if (want <= 1) ROUTE(1);
    else if (sizeof(T) == 8 ? want <= 4 : false) ROUTE(4);               // (float64: fewer lengths of the list)
    else if constexpr (sizeof(T) == 4) { if (want <= 2) ROUTE(2); else if (want <= 4) ROUTE(4); else if (want <= 8) ROUTE(8); else ROUTE(16); }
    else ROUTE(16);
#undef CHOOSE
#undef ROUTE
    if (e != cudaSuccess) return e;
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

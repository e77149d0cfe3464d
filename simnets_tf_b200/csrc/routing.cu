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
    T v[TK], l[TK];
    int i[TK];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < TK; ++t) { v[t] = l[t] = below_all<T>(); i[t] = -1; }
    }
    __device__ __forceinline__ void offer(T value, T logit, int index, int want) {
        bool placed = false;                             // (a NaN and -infinity are above nothing)
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            if (t < want && (placed || value > v[t])) {
                const T ov = v[t], ol = l[t];
                const int oi = i[t];
                v[t] = value; l[t] = logit; i[t] = index;
                value = ov; logit = ol; index = oi;
                placed = true;
            }
        }
    }
};

// weights of the chosen from their l, in place: they sum to one over the chosen (all 0 if there are none)
template <typename T, int TK>
__device__ __forceinline__ void weigh(Top<T, TK>& top, int want, bool sigmoid) {
    T hi = below_all<T>();
#pragma unroll
    for (int t = 0; t < TK; ++t) {
        if (t >= want || top.i[t] < 0) continue;
        if (sigmoid) top.l[t] = top.l[t] >= T(0) ? -log1p_of(exp_of(-top.l[t])) : top.l[t] - log1p_of(exp_of(top.l[t]));
        hi = top.l[t] > hi ? top.l[t] : hi;
    }
    T sum = T(0);
#pragma unroll
    for (int t = 0; t < TK; ++t) {
        top.l[t] = t < want && top.i[t] >= 0 ? (top.l[t] == hi ? T(1) : exp_of(top.l[t] - hi)) : T(0);      // (infinities are equal too)
        sum += top.l[t];
    }
    const T inv = sum > T(0) ? T(1) / sum : T(0);
#pragma unroll
    for (int t = 0; t < TK; ++t) top.l[t] *= inv;
}

struct RouteArgs {
    long long positions;         // of the whole batch
    long long N;                 // per sample
    int k, top, groups, size, top_groups;
    int sigmoid;
    double scale;
};

template <typename T, int TK>
__global__ void __launch_bounds__(kRouteThreads) route_choose(RouteArgs a, const T* __restrict__ scores, const T* __restrict__ prior, const T* __restrict__ bias,
                                                              int* __restrict__ index, T* __restrict__ weights, T* __restrict__ dense,
                                                              unsigned* __restrict__ part_load) {
    stream_order();
    extern __shared__ unsigned load[];
    for (int c = threadIdx.x; c < a.k; c += kRouteThreads) load[c] = 0;
    __syncthreads();
    for (long long p = (long long)blockIdx.x * kRouteThreads + threadIdx.x; p < a.positions; p += (long long)gridDim.x * kRouteThreads) {
        const long long n = p / a.N, j = p - n * a.N;
        const T* s = scores + n * a.k * a.N + j;
        unsigned long long open = ~0ull;                 // groups that are in the choice
        Top<T, TK> top;
        if (a.top_groups < a.groups) {
            top.clear();
            for (int g = 0; g < a.groups; ++g) {
                T best = below_all<T>();
                for (int c = g * a.size; c < (g + 1) * a.size; ++c) {
                    T v = s[c * a.N];
                    if (prior) v += prior[c];
                    if (bias) v += bias[c];
                    best = v > best ? v : best;
                }
                top.offer(best, best, g, a.top_groups);
            }
            open = 0;
#pragma unroll
            for (int t = 0; t < TK; ++t) if (t < a.top_groups && top.i[t] >= 0) open |= 1ull << top.i[t];
        }
        top.clear();
        for (int g = 0; g < a.groups; ++g) {
            if (a.top_groups < a.groups && !(open >> g & 1)) continue;
            for (int c = g * a.size; c < (g + 1) * a.size; ++c) {
                T l = s[c * a.N];
                if (prior) l += prior[c];
                top.offer(bias ? l + bias[c] : l, l, c, a.top);
            }
        }
        weigh(top, a.top, a.sigmoid);
        T* d = dense ? dense + n * a.k * a.N + j : nullptr;
        if (d) for (int c = 0; c < a.k; ++c) d[c * a.N] = T(0);
#pragma unroll
        for (int t = 0; t < TK; ++t) {
            if (t >= a.top) continue;
            const long long at = (n * a.top + t) * a.N + j;
            const T w = T(a.scale) * top.l[t];
            if (index) index[at] = top.i[t];
            if (weights) weights[at] = w;
            if (top.i[t] < 0) continue;
            if (d) d[top.i[t] * a.N] = w;
            atomicAdd(load + top.i[t], 1u);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.k; c += kRouteThreads) part_load[(size_t)blockIdx.x * a.k + c] = load[c];
}

// part[split][c] = sum of the responsibilities of component c = blockIdx.x in the split's samples
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
__global__ void __launch_bounds__(128) route_totals(int ctas, int splits, int k, const unsigned* __restrict__ part_load, const T* __restrict__ part_mass,
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
        if (mass) mass[blockIdx.x] = redm[0];
    }
}

// dscores of the weights' gradient:  dl_i = W_i (g_i - sum_j W_j g_j / scale), times 1 - sigmoid(l_i) where the values are sigmoids
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) route_gradient(RouteArgs a, const T* __restrict__ scores, const T* __restrict__ prior, const int* __restrict__ index,
                                                                const T* __restrict__ weights, const T* __restrict__ grad, T* __restrict__ dscores) {
    stream_order();
    const T inv_scale = T(1.0 / a.scale);
    for (long long p = (long long)blockIdx.x * kRouteThreads + threadIdx.x; p < a.positions; p += (long long)gridDim.x * kRouteThreads) {
        const long long n = p / a.N, j = p - n * a.N, chosen = n * a.top * a.N + j;
        const T* s = scores + n * a.k * a.N + j;
        T* d = dscores + n * a.k * a.N + j;
        for (int c = 0; c < a.k; ++c) d[c * a.N] = T(0);
        T sum = T(0);
        for (int t = 0; t < a.top; ++t)
            if (index[chosen + t * a.N] >= 0) sum += weights[chosen + t * a.N] * inv_scale * grad[chosen + t * a.N];
        for (int t = 0; t < a.top; ++t) {
            const int c = index[chosen + t * a.N];
            if (c < 0) continue;
            T v = weights[chosen + t * a.N] * (grad[chosen + t * a.N] - sum);
            if (a.sigmoid) {
                T l = s[c * a.N];
                if (prior) l += prior[c];
                v *= T(1) / (T(1) + exp_of(l));
            }
            d[c * a.N] = v;
        }
    }
}

RouteArgs args_of(const simnets_route_desc& d) {
    RouteArgs a;
    a.N = d.positions;
    a.positions = d.positions * d.batch;
    a.k = d.components; a.top = d.top_k; a.groups = d.groups; a.size = d.components / d.groups; a.top_groups = d.top_groups;
    a.sigmoid = d.sigmoid != 0;
    a.scale = d.scale;
    return a;
}
int route_ctas(const simnets_route_desc& d) {
    const long long tiles = (d.positions * d.batch + kRouteThreads - 1) / kRouteThreads;
    return int(std::max<long long>(1, std::min<long long>(tiles, 8LL * device_sm_count())));
}
int mass_splits(const simnets_route_desc& d) { return int(std::max<long long>(1, std::min<long long>(d.batch, (8LL * device_sm_count() + d.components - 1) / d.components))); }
size_t load_bytes(const simnets_route_desc& d) { return (sizeof(unsigned) * (size_t)route_ctas(d) * d.components + 255) & ~size_t(255); }

template <typename T>
cudaError_t route(const simnets_route_desc& d, const void* scores, const void* prior, const void* bias, int* index, void* weights, void* dense, long long* load,
                  void* mass, void* ws, cudaStream_t s) {
    const RouteArgs a = args_of(d);
    const int ctas = route_ctas(d), splits = mass_splits(d), want = std::max(a.top, a.top_groups < a.groups ? a.top_groups : 1);
    unsigned* part_load = static_cast<unsigned*>(ws);
    T* part_mass = reinterpret_cast<T*>(static_cast<char*>(ws) + load_bytes(d));
#define ROUTE(TK) in_stream_order(route_choose<T, TK>, ctas, kRouteThreads, sizeof(unsigned) * a.k, s)(a, (const T*)scores, (const T*)prior, (const T*)bias, index, (T*)weights, (T*)dense, part_load)
    if (want <= 1) ROUTE(1); else if (want <= 2) ROUTE(2); else if (want <= 4) ROUTE(4); else if (want <= 8) ROUTE(8); else ROUTE(16);
#undef ROUTE
    if (mass) in_stream_order(route_mass<T>, dim3(a.k, splits), 256, 0, s)(a, (long long)d.batch, (const T*)dense, part_mass);
    in_stream_order(route_totals<T>, a.k, 128, 0, s)(ctas, splits, a.k, part_load, part_mass, load, (T*)mass);
    count_launch(mass ? 3 : 2);
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
    const int ctas = route_ctas(d);
    if (d.dtype == SIMNETS_F64)
        in_stream_order(route_gradient<double>, ctas, kRouteThreads, 0, s)(a, (const double*)scores, (const double*)prior, index, (const double*)weights, (const double*)grad, (double*)dscores);
    else
        in_stream_order(route_gradient<float>, ctas, kRouteThreads, 0, s)(a, (const float*)scores, (const float*)prior, index, (const float*)weights, (const float*)grad, (float*)dscores);
    count_launch();
    return cudaGetLastError();
}

}  // namespace simnets

// The norm of a list of gradients, and the gradients scaled so that it is at most a limit.
//
//     norm = sqrt(sum of g^2) over all tensors, or max |g|;   out = g * (limit / norm where norm > limit, else 1)
//
// The partial results of a grid of CTAs are combined in a fixed order, and the host never learns the norm.  Bound by memory: g is read twice and
// written once, the second time from the end, so that what was read last comes from L2.  A list that one wave of CTAs takes (up to 19 MB) is two launches,
// and every CTA of the second combines the partial results again; beyond, one CTA does so in a launch between, which lets the last one
// have as many CTAs as there is work (2.6e8 values: 295 us with a CTA for 16 KB, 310 with 64 a multiprocessor, 324 with 8, a plain copy 318).
//
// Sums are in 64 bits: squares of float32 are exact there and neither overflow nor vanish.  Squares of float64 can do both, so there are three sums of
// them, of g, of g * 2^-600 and of g * 2^600, of which the one that holds numbers is taken.  The product g * scale is rounded once, from 64 bits.
#include "kernels.cuh"

namespace simnets {
namespace {

constexpr int kThreads = 256, kItemBytes = 16 * 1024;       // a CTA takes 16 KB of one tensor at a time
constexpr int kMostTensors = 1088, kFew = 24;                // of a launch: their table is the kernel's argument

struct Partial { double mid, big, small; };
__host__ __device__ constexpr double up600() { return 0x1p600; }
__host__ __device__ constexpr double down600() { return 0x1p-600; }

// Tensors of one type.  Items are counted from 16-byte boundaries: `skip` values of the first one are in front of the tensor.
template <int N>
struct Table {
    const void* in[N];
    void* out[N];
    long long values[N];
    int first[N + 1];                                       // items in front of tensor i
    int tensors;
};

__device__ __forceinline__ double larger_or_nan(double a, double b) { return a > b || a != a ? a : b; }

template <typename T> struct Four;
template <> struct Four<float> { using type = float4; };
template <> struct Four<double> { using type = double2; };
template <typename T>
struct Vector {
    static constexpr int kWidth = 16 / sizeof(T);
    T v[kWidth];
};

// an item of a tensor: the values from `begin` on, which may be below 0, and there may be fewer than an item has
template <typename T>
struct Item {
    const T* in;
    T* out;
    long long begin, values;
    bool aligned;                                           // the 16-byte pieces of `in` from `begin` on are pieces of `out` as well
    template <int N>
    __device__ __forceinline__ Item(const Table<N>& t, int item) {
        int lo = 0, hi = t.tensors - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (t.first[mid] <= item) lo = mid; else hi = mid - 1;
        }
        in = static_cast<const T*>(t.in[lo]);
        out = static_cast<T*>(t.out[lo]);
        values = t.values[lo];
        const int skip = int(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
        begin = (long long)(item - t.first[lo]) * (kItemBytes / sizeof(T)) - skip;
        aligned = (reinterpret_cast<uintptr_t>(in) - reinterpret_cast<uintptr_t>(out)) % 16 == 0;
    }
    __device__ __forceinline__ Vector<T> load(long long at) const {
        Vector<T> x;
        if (at >= 0 && at + Vector<T>::kWidth <= values) {
            const typename Four<T>::type w = *reinterpret_cast<const typename Four<T>::type*>(in + at);
            memcpy(x.v, &w, 16);                            // (an array that is not in registers lies at a multiple of its values' size only)
        } else {
#pragma unroll
            for (int i = 0; i < Vector<T>::kWidth; ++i) x.v[i] = at + i >= 0 && at + i < values ? in[at + i] : T(0);
        }
        return x;
    }
    __device__ __forceinline__ void store(long long at, const Vector<T>& x) const {
        if (aligned && at >= 0 && at + Vector<T>::kWidth <= values) {
            typename Four<T>::type w;
            memcpy(&w, x.v, 16);
            *reinterpret_cast<typename Four<T>::type*>(out + at) = w;
        } else {
#pragma unroll
            for (int i = 0; i < Vector<T>::kWidth; ++i)
                if (at + i >= 0 && at + i < values) out[at + i] = x.v[i];
        }
    }
};

// what one value adds to a sum of squares or a largest magnitude
template <bool MAX, typename T>
__device__ __forceinline__ void take(Partial& p, T g) {
    const double x = double(g);
    if (MAX) {
        p.mid = larger_or_nan(fabs(x), p.mid);
    } else {
        p.mid = fma(x, x, p.mid);
        if (sizeof(T) == 8) {
            const double b = x * down600(), s = x * up600();
            p.big = fma(b, b, p.big);
            p.small = fma(s, s, p.small);
        }
    }
}
template <bool MAX>
__device__ __forceinline__ void join(Partial& p, const Partial& o) {
    if (MAX) {
        p.mid = larger_or_nan(o.mid, p.mid);
    } else {
        p.mid += o.mid;
        p.big += o.big;
        p.small += o.small;
    }
}

// the sum over the CTA, in all of its threads; `room`: one place a warp
template <bool MAX>
__device__ __forceinline__ Partial over_cta(Partial p, Partial* room) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const Partial o = {__shfl_xor_sync(0xffffffffu, p.mid, d), __shfl_xor_sync(0xffffffffu, p.big, d), __shfl_xor_sync(0xffffffffu, p.small, d)};
        join<MAX>(p, o);
    }
    if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = p;
    __syncthreads();
    p = room[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) join<MAX>(p, room[w]);
    return p;
}

template <bool MAX, typename T, int N>
__global__ void __launch_bounds__(kThreads) norm_partials(const __grid_constant__ Table<N> t, Partial* partials) {
    stream_order();
    __shared__ Partial room[kThreads / 32];
    constexpr int kWidth = Vector<T>::kWidth, kSteps = kItemBytes / 16 / kThreads;
    Partial p = {0.0, 0.0, 0.0};
    for (int item = blockIdx.x; item < t.first[t.tensors]; item += gridDim.x) {
        const Item<T> it(t, item);
        Vector<T> x[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) x[s] = it.load(it.begin + (long long)(s * kThreads + threadIdx.x) * kWidth);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int i = 0; i < kWidth; ++i) take<MAX>(p, x[s].v[i]);
    }
    p = over_cta<MAX>(p, room);
    if (threadIdx.x == 0) {
        // (A finite sum of float32 squares other than 0 is between 2^-298 and 2^319.  `big` is taken where all sums together are above 2^1000, of which that
        // is nothing, and `small` where they are below 2^-900, which it is not: both are 0.  Only an infinity counts in `big`.)
        if (!MAX && sizeof(T) == 4) p.big = p.mid == double(CUDART_INF) ? p.mid : 0.0;
        partials[blockIdx.x] = p;
    }
}

// the norm, in all threads of the CTA, rounded to the type that it is returned in
template <bool MAX>
__device__ __forceinline__ double norm_of(const Partial* partials, int count, bool f64, Partial* room) {
    Partial p = {0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < count; i += kThreads) join<MAX>(p, partials[i]);
    p = over_cta<MAX>(p, room);
    double norm = p.mid;
    if (!MAX) {
        // (2^-900 and 2^1000: far from where squares that matter to the sum are rounded to fewer bits or added up to infinity)
        norm = p.mid > 0x1p1000 ? sqrt(p.big) * up600() : p.mid < 0x1p-900 ? sqrt(p.small) * down600() : sqrt(p.mid);
    }
    return f64 ? norm : double(float(norm));
}

__device__ __forceinline__ void write_norm(void* norm, bool f64, double v) {
    if (f64) *static_cast<double*>(norm) = v;
    else *static_cast<float*>(norm) = float(v);
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_finish(const Partial* partials, int count, bool f64, void* norm) {
    stream_order();
    __shared__ Partial room[kThreads / 32];
    const double v = norm_of<MAX>(partials, count, f64, room);
    if (threadIdx.x == 0) write_norm(norm, f64, v);
}

// ALONE: combines the partial results itself; else `norm` is there already.  in_place: every tensor is its own destination, and nothing is to be done
// where the norm is within the limit.
template <bool ALONE, bool MAX, typename T, int N>
__global__ void __launch_bounds__(kThreads) scale_tensors(const __grid_constant__ Table<N> t, const Partial* partials, int count, bool f64, double limit, bool in_place, void* norm,
                                                          bool writes_norm) {
    stream_order();
    constexpr int kWidth = Vector<T>::kWidth, kSteps = kItemBytes / 16 / kThreads;
    double v;
    if (ALONE) {
        __shared__ Partial room[kThreads / 32];
        v = norm_of<MAX>(partials, count, f64, room);
        if (writes_norm && blockIdx.x == 0 && threadIdx.x == 0) write_norm(norm, f64, v);
    } else {
        v = f64 ? *static_cast<const double*>(norm) : double(*static_cast<const float*>(norm));
    }
    // (a norm that is no number, or infinite, changes nothing)
    const bool scaled = v > limit && v < double(CUDART_INF);
    if (!scaled && in_place) return;
    const double scale = scaled ? limit / v : 1.0;
    for (int item = t.first[t.tensors] - 1 - int(blockIdx.x); item >= 0; item -= gridDim.x) {
        const Item<T> it(t, item);
        Vector<T> x[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) x[s] = it.load(it.begin + (long long)(s * kThreads + threadIdx.x) * kWidth);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (scaled) {
#pragma unroll
                for (int i = 0; i < kWidth; ++i) x[s].v[i] = T(double(x[s].v[i]) * scale);
            }
            it.store(it.begin + (long long)(s * kThreads + threadIdx.x) * kWidth, x[s]);
        }
    }
}

// Calls of one list of tensors: those of one type, a table full at a time.
struct Call {
    int tensors;
    const int *dtypes;
    const long long* values;
    const void* const* in;
    void* const* out;
};

long long items_of(const void* in, long long values, int size) {
    const long long skip = (long long)(reinterpret_cast<uintptr_t>(in) % 16) / size;
    return values > 0 ? (skip + values + kItemBytes / size - 1) / (kItemBytes / size) : 0;
}
int grid_of(long long items, int a_multiprocessor) { return int(std::min<long long>(items, (long long)a_multiprocessor * device_sm_count())); }

// body(dtype, table) for every launch
template <int N, class Body>
cudaError_t each_table(const Call& c, Body body) {
    Table<N> t;
    for (int dtype : {SIMNETS_F32, SIMNETS_F64}) {
        t.tensors = 0;
        t.first[0] = 0;
        for (int i = 0; i <= c.tensors; ++i) {
            const int size = dtype == SIMNETS_F64 ? 8 : 4;
            const bool mine = i < c.tensors && (c.dtypes ? c.dtypes[i] : SIMNETS_F32) == dtype && c.values[i] > 0;
            const long long items = mine ? items_of(c.in[i], c.values[i], size) : 0;
            if (t.tensors > 0 && (i == c.tensors || (mine && t.tensors == N))) {
                const cudaError_t e = body(dtype, t);
                if (e != cudaSuccess) return e;
                t.tensors = 0;
            }
            if (!mine) continue;
            t.in[t.tensors] = c.in[i];
            t.out[t.tensors] = c.out ? c.out[i] : nullptr;
            t.values[t.tensors] = c.values[i];
            t.first[t.tensors + 1] = t.first[t.tensors] + int(items);
            ++t.tensors;
        }
    }
    return cudaSuccess;
}

template <bool MAX, int N>
cudaError_t run(const Call& c, bool f64, bool in_place, double limit, void* norm, Partial* partials, cudaStream_t s) {
    int count = 0;
    cudaError_t e = each_table<N>(c, [&](int dtype, const Table<N>& t) {
        const int grid = grid_of(t.first[t.tensors], 8);
        if (dtype == SIMNETS_F64) in_stream_order(norm_partials<MAX, double, N>, grid, kThreads, 0, s)(t, partials + count);
        else in_stream_order(norm_partials<MAX, float, N>, grid, kThreads, 0, s)(t, partials + count);
        count_launch();
        count += grid;
        return cudaGetLastError();
    });
    if (e != cudaSuccess) return e;
    const bool alone = c.out && count > 0 && count < 8 * device_sm_count();
    if (!alone) {
        in_stream_order(norm_finish<MAX>, 1, kThreads, 0, s)(partials, count, f64, norm);
        count_launch();
        e = cudaGetLastError();
        if (e != cudaSuccess || !c.out || count == 0) return e;
    }
    bool first = true;
    return each_table<N>(c, [&](int dtype, const Table<N>& t) {
        // In place most calls have nothing to scale: fewer CTAs that come and go.  (2.6e8 values below / above the limit, norm included, us: 8 CTAs a multiprocessor
        // 157 / 526, 64 162 / 494, 256 177 / 479, as many as items 190 / 473; 5e7: 36 / 93, 40 / 91, 42 / 90, 42 / 90.)
        const int grid = grid_of(t.first[t.tensors], in_place ? 64 : 1 << 20);
        auto launch = [&](auto kernel) { in_stream_order(kernel, grid, kThreads, 0, s)(t, partials, count, f64, limit, in_place, norm, first); };
        if (alone) launch(dtype == SIMNETS_F64 ? scale_tensors<true, MAX, double, N> : scale_tensors<true, MAX, float, N>);
        else launch(dtype == SIMNETS_F64 ? scale_tensors<false, MAX, double, N> : scale_tensors<false, MAX, float, N>);
        count_launch();
        first = false;
        return cudaGetLastError();
    });
}

}  // namespace

// (a launch a type and table, each of at most 8 CTAs a multiprocessor)
size_t gradient_norm_workspace_bytes(int tensors) {
    return sizeof(Partial) * 8 * device_sm_count() * (2 + size_t(tensors <= kFew ? 0 : tensors) / kMostTensors);
}

cudaError_t launch_gradient_norm(int order, int tensors, const int* dtypes, const long long* values, const void* const* in, void* const* out, double limit, void* norm,
                                 bool norm_f64, void* ws, cudaStream_t s) {
    const Call c = {tensors, dtypes, values, in, out};
    bool in_place = out != nullptr;
    for (int i = 0; in_place && i < tensors; ++i) in_place = out[i] == in[i] || values[i] == 0;
    Partial* partials = static_cast<Partial*>(ws);
    if (tensors <= kFew) return order == 0 ? run<true, kFew>(c, norm_f64, in_place, limit, norm, partials, s) : run<false, kFew>(c, norm_f64, in_place, limit, norm, partials, s);
    return order == 0 ? run<true, kMostTensors>(c, norm_f64, in_place, limit, norm, partials, s) : run<false, kMostTensors>(c, norm_f64, in_place, limit, norm, partials, s);
}

}  // namespace simnets

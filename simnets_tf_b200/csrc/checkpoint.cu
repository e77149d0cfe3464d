// 8-bit checkpoints of activations: what a layer keeps of its input for the backward pass.
//
// Per group of G consecutive values the lowest finite one (base) and a step of 1 / 252 of the range; per value the byte
// rint((x - base) / step), or 253, 254, 255 for -infinity, infinity, NaN.  Activations of these networks are log-likelihoods that enter
// exponentials: what counts is their absolute error, which is at most step / 2 here, wherever the range lies (an 8-bit float
// is off by 2 % of a value, which is 1 nat at -50); with step 0 it is below 252 of the type's smallest normal number.
//
// A program may pack and compare elsewhere, so the bytes are defined to the bit: with x / 2 - base / 2 and 2 / step rounded to the type and
// their product exact in front of rint (one fused multiply-add onto 1.5 * 2^23 or 2^52, whose last bits are the integer).  The halves keep
// the range of values of either sign finite.  A range below 252 of the type's smallest normal number has step 0: all bytes 0.
#include "checkpoint.cuh"
#include "kernels.cuh"

namespace simnets {
namespace {

__device__ __forceinline__ float least(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double least(double a, double b) { return a < b ? a : b; }        // (of numbers: no NaN comes this far that counts)
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double most(double a, double b) { return a > b ? a : b; }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < CUDART_INF_F; }
__device__ __forceinline__ bool finite(double v) { return fabs(v) < CUDART_INF; }

constexpr int kPackThreads = 256;

// The group's step and 2 / step from its extremes (hi < lo: it has no finite value, and both become 0).
template <typename T>
__device__ __forceinline__ void group_steps(T& lo, T hi, T& step, T& per) {
    if (lo > hi) lo = hi = T(0);
    step = (hi * T(0.5) - lo * T(0.5)) / T(126);
    if (step < Limits<T>::tiny()) step = T(0);
    per = step > T(0) ? T(2) / step : T(0);
}
template <typename T>
__device__ __forceinline__ uint32_t packed(T v, T half, T per) {
    return finite(v) ? Limits<T>::nearest(Limits<T>::halves(v, half), per) : v != v ? 255u : v < T(0) ? 253u : 254u;
}

// Any address and length: a warp takes a group, a lane every 32nd value of it.  Groups first .. last.
template <typename T, int G>
__device__ __forceinline__ void pack_groups(long long n, long long first, long long last, long long step_groups, const T* __restrict__ x, unsigned char* __restrict__ codes,
                                            T* __restrict__ ranges) {
    const int lane = threadIdx.x & 31;
    for (long long g = first; g < last; g += step_groups) {
        const long long at = g * G + lane;
        T v[G / 32], lo = Limits<T>::inf(), hi = -Limits<T>::inf(), step, per;
#pragma unroll
        for (int i = 0; i < G / 32; ++i) {
            v[i] = at + 32 * i < n ? x[at + 32 * i] : Limits<T>::inf() - Limits<T>::inf();      // (beyond the end: NaN)
            if (finite(v[i])) { lo = least(lo, v[i]); hi = most(hi, v[i]); }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            lo = least(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = most(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        group_steps(lo, hi, step, per);
        const T half = lo * T(0.5);
#pragma unroll
        for (int i = 0; i < G / 32; ++i)
            if (at + 32 * i < n) codes[at + 32 * i] = (unsigned char)packed(v[i], half, per);
        if (lane == 0) { ranges[2 * g] = lo; ranges[2 * g + 1] = step; }
    }
}

// extremes over LANES neighbouring lanes
template <int LANES, typename T>
__device__ __forceinline__ void extremes(T& lo, T& hi) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        lo = least(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = most(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    }
}
template <>
__device__ __forceinline__ void extremes<32, float>(float& lo, float& hi) {
    asm volatile("redux.sync.min.f32 %0, %0, 0xffffffff;" : "+f"(lo));
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(hi));
}

// A lane's 16 bytes: V values, of which a group holds G / V lanes of one row of 32 or several whole rows.
template <typename T, int G>
struct Rows {
    static constexpr int V = 16 / int(sizeof(T)), kRow = 32 * V, kLanes = G / V < 32 ? G / V : 32, kRows = G > kRow ? G / kRow : 1, kUnit = kRow * kRows;
    static constexpr int kUnits = 4 / kRows < 1 ? 1 : 4 / kRows;         // units in flight: four 16-byte loads a lane
};
template <typename T> struct alignas(16) Sixteen { T v[16 / sizeof(T)]; };

// Aligned tensors.  Bound: HBM, 5.06 bytes a value (537 MB of float32 read, 142 MB written: 104 us).  What stands between a load and its
// stores is a chain of a reduction over lanes and two divisions, so that the units in flight are worked on together (one branch for all of them:
// with one per unit 124 us for groups of 128, 138 for groups of 32, float64 311 and 440).
template <typename T, int G>
__global__ void __launch_bounds__(kPackThreads) checkpoint_pack(long long n, bool aligned, const T* __restrict__ x, unsigned char* __restrict__ codes, T* __restrict__ ranges) {
    stream_order();
    using R = Rows<T, G>;
    constexpr int U = R::kUnits;
    const int lane = threadIdx.x & 31;
    const long long warp = (long long)blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5), warps = (long long)gridDim.x * (kPackThreads / 32);
    const long long steps = aligned ? n / (R::kUnit * U) : 0;            // (of U whole units; the rest is a few groups)
    for (long long u = warp; u < steps; u += warps) {
        const long long at = u * (R::kUnit * U) + lane * R::V;
        Sixteen<T> v[U][R::kRows];
        T lo[U], hi[U], step[U], per[U];
        bool fine = true;
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int r = 0; r < R::kRows; ++r) {
                const float4 q = __ldcs(reinterpret_cast<const float4*>(x + at + j * R::kUnit + r * R::kRow));
                v[j][r] = *reinterpret_cast<const Sixteen<T>*>(&q);
            }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            lo[j] = hi[j] = v[j][0].v[0];
#pragma unroll
            for (int r = 0; r < R::kRows; ++r)
#pragma unroll
                for (int i = 0; i < R::V; ++i) {
                    lo[j] = least(lo[j], v[j][r].v[i]);
                    hi[j] = most(hi[j], v[j][r].v[i]);
                    fine = fine && finite(v[j][r].v[i]);
                }
        }
        fine = __all_sync(0xffffffffu, fine);
        if (!fine) {                                                     // extremes of the finite ones only
#pragma unroll
            for (int j = 0; j < U; ++j) {
                lo[j] = Limits<T>::inf(); hi[j] = -lo[j];
#pragma unroll
                for (int r = 0; r < R::kRows; ++r)
#pragma unroll
                    for (int i = 0; i < R::V; ++i)
                        if (finite(v[j][r].v[i])) { lo[j] = least(lo[j], v[j][r].v[i]); hi[j] = most(hi[j], v[j][r].v[i]); }
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) extremes<R::kLanes>(lo[j], hi[j]);
        if constexpr (sizeof(T) == 8 && U == 2) {
            // (divisions of float64 are some thirty instructions each: a lane makes those of one unit, and its group's lanes share them.  Groups of
            // 128, 134 million values: 231 -> 215 us; with four units of one row the shuffles are already the bound: groups of 32 375 -> 504)
            T my_lo = lo[0], my_hi = hi[0], my_step, my_per;
#pragma unroll
            for (int j = 1; j < U; ++j)
                if (lane % U == j) { my_lo = lo[j]; my_hi = hi[j]; }
            group_steps(my_lo, my_hi, my_step, my_per);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                lo[j] = __shfl_sync(0xffffffffu, my_lo, lane / U * U + j);
                step[j] = __shfl_sync(0xffffffffu, my_step, lane / U * U + j);
                per[j] = __shfl_sync(0xffffffffu, my_per, lane / U * U + j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < U; ++j) group_steps(lo[j], hi[j], step[j], per[j]);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const T half = lo[j] * T(0.5);
#pragma unroll
            for (int r = 0; r < R::kRows; ++r) {
                uint32_t c[R::V];
#pragma unroll
                for (int i = 0; i < R::V; ++i) c[i] = fine ? Limits<T>::nearest(Limits<T>::halves(v[j][r].v[i], half), per[j]) : packed(v[j][r].v[i], half, per[j]);
                unsigned char* to = codes + at + j * R::kUnit + r * R::kRow;
                if constexpr (R::V == 4) *reinterpret_cast<uint32_t*>(to) = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
                else *reinterpret_cast<unsigned short*>(to) = (unsigned short)__byte_perm(c[0], c[1], 0x0040);
            }
            if (lane % R::kLanes == 0) {
                T* to = ranges + 2 * ((at + j * R::kUnit) / G);
                to[0] = lo[j]; to[1] = step[j];
            }
        }
    }
    pack_groups<T, G>(n, steps * (R::kUnit * U / G) + warp, (n + G - 1) / G, warps, x, codes, ranges);
}

// The n values of a checkpoint of groups of 2^shift.  Bound: HBM; eight loads of four bytes in flight a thread: 118 us for 134 million
// float32 (5.75 TB/s; with four 125, with one value a thread 165).
template <typename T>
__global__ void __launch_bounds__(kPackThreads) checkpoint_unpack(long long n, int shift, bool aligned, const unsigned char* __restrict__ codes,
                                                                  const T* __restrict__ ranges, T* __restrict__ x) {
    stream_order();
    constexpr int V = 16 / int(sizeof(T)), U = 8;
    const long long thread = (long long)blockIdx.x * kPackThreads + threadIdx.x, threads = (long long)gridDim.x * kPackThreads;
    const long long quads = aligned ? n / V : 0;
    for (long long q0 = (long long)blockIdx.x * (U * kPackThreads) + threadIdx.x; q0 < quads; q0 += U * threads) {
        uint32_t c[U];
        T base[U], step[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const long long q = q0 + j * kPackThreads;
            c[j] = 0; base[j] = step[j] = T(0);
            if (q >= quads) continue;
            if constexpr (V == 4) c[j] = __ldcs(reinterpret_cast<const uint32_t*>(codes) + q);
            else c[j] = __ldcs(reinterpret_cast<const unsigned short*>(codes) + q);
            const T* r = ranges + 2 * ((q * V) >> shift);
            base[j] = __ldg(r); step[j] = __ldg(r + 1);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const long long q = q0 + j * kPackThreads;
            if (q >= quads) continue;
            Sixteen<T> v;
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = unpacked<T>((c[j] >> (8 * i)) & 255u, base[j], step[j]);
            __stcs(reinterpret_cast<float4*>(x) + q, *reinterpret_cast<const float4*>(&v));
        }
    }
    for (long long i = quads * V + thread; i < n; i += threads) {
        const long long g = i >> shift;
        x[i] = unpacked<T>(codes[i], ranges[2 * g], ranges[2 * g + 1]);
    }
}

int pack_grid(long long units) { return int(std::max<long long>(1, std::min<long long>(units, 8LL * device_sm_count()))); }
bool lies_on(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename T>
cudaError_t pack(long long n, int group, const void* x, void* codes, void* ranges, cudaStream_t s) {
    const bool aligned = lies_on(x, 16) && lies_on(codes, 16 / sizeof(T));
    const int grid = pack_grid((n + 2048) / 2048);
#define PACK(G) in_stream_order(checkpoint_pack<T, G>, grid, kPackThreads, 0, s)(n, aligned, (const T*)x, (unsigned char*)codes, (T*)ranges)
    if (group == 32) PACK(32); else if (group == 64) PACK(64); else if (group == 128) PACK(128); else PACK(256);
#undef PACK
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t unpack(long long n, int group, const void* codes, const void* ranges, void* x, cudaStream_t s) {
    int shift = 5;
    while ((1 << shift) < group) ++shift;
    const bool aligned = lies_on(x, 16) && lies_on(codes, 16 / sizeof(T));
    in_stream_order(checkpoint_unpack<T>, pack_grid((n + 2048) / 2048), kPackThreads, 0, s)(n, shift, aligned, (const unsigned char*)codes, (const T*)ranges, (T*)x);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_checkpoint_pack(bool f64, long long n, int group, const void* x, void* codes, void* ranges, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    return f64 ? pack<double>(n, group, x, codes, ranges, s) : pack<float>(n, group, x, codes, ranges, s);
}
cudaError_t launch_checkpoint_unpack(bool f64, long long n, int group, const void* codes, const void* ranges, void* x, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    return f64 ? unpack<double>(n, group, codes, ranges, x, s) : unpack<float>(n, group, codes, ranges, x, s);
}

}  // namespace simnets

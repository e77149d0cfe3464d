// 8-bit checkpoints of activations: what a layer keeps of its input for the backward pass.
//
// Per group of G consecutive values the lowest finite one (base) and a step of 1 / 252 of the range; per value the byte
// rint((x - base) / step), or 253, 254, 255 for -infinity, infinity, NaN.  Activations of these networks are log-likelihoods that enter
// exponentials: what counts is their absolute error, which is at most step / 2 here, wherever the range lies (an 8-bit float
// is off by 2 % of a value, which is 1 nat at -50).
//
// A program may pack and compare elsewhere, so the bytes are defined to the bit: with x / 2 - base / 2 and 2 / step rounded to the type and
// their product exact in front of rint (one fused multiply-add onto 1.5 * 2^23 or 2^52, whose last bits are the integer).  The halves keep
// the range of values of either sign finite.  A range below 252 of the type's smallest normal number has step 0: all bytes 0.
#include "checkpoint.cuh"
#include "kernels.cuh"

namespace simnets {
namespace {

__device__ __forceinline__ float least(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double least(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < CUDART_INF_F; }
__device__ __forceinline__ bool finite(double v) { return fabs(v) < CUDART_INF; }

constexpr int kPackThreads = 256;

// one warp per group of 32 PER values
template <typename T, int PER>
__global__ void __launch_bounds__(kPackThreads) checkpoint_pack(long long n, const T* __restrict__ x, unsigned char* __restrict__ codes, T* __restrict__ ranges) {
    stream_order();
    const int lane = threadIdx.x & 31;
    const long long groups = (n + 32 * PER - 1) / (32 * PER), step_groups = (long long)gridDim.x * (kPackThreads / 32);
    for (long long g = (long long)blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5); g < groups; g += step_groups) {
        const long long at = g * 32 * PER + lane;
        T v[PER], lo = Limits<T>::inf(), hi = -Limits<T>::inf();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            v[i] = at + 32 * i < n ? x[at + 32 * i] : Limits<T>::inf() - Limits<T>::inf();      // (beyond the end: NaN)
            if (finite(v[i])) { lo = least(lo, v[i]); hi = most(hi, v[i]); }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            lo = least(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = most(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        if (lo > hi) lo = hi = T(0);                                        // (no finite value in the group)
        T step = (hi * T(0.5) - lo * T(0.5)) / T(126);
        if (step < Limits<T>::tiny()) step = T(0);
        const T per = step > T(0) ? T(2) / step : T(0), half = lo * T(0.5);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t c = finite(v[i]) ? Limits<T>::nearest(v[i] * T(0.5) - half, per) : v[i] != v[i] ? 255u : v[i] < T(0) ? 253u : 254u;
            if (at + 32 * i < n) codes[at + 32 * i] = (unsigned char)c;
        }
        if (lane == 0) { ranges[2 * g] = lo; ranges[2 * g + 1] = step; }
    }
}

// values first .. first + n of a checkpoint of groups of 2^shift
template <typename T>
__global__ void __launch_bounds__(kPackThreads) checkpoint_unpack(long long first, long long n, int shift, const unsigned char* __restrict__ codes,
                                                                  const T* __restrict__ ranges, T* __restrict__ x) {
    stream_order();
    for (long long i = (long long)blockIdx.x * kPackThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kPackThreads) {
        const long long g = (first + i) >> shift;
        x[i] = unpacked<T>(codes[first + i], ranges[2 * g], ranges[2 * g + 1]);
    }
}

int pack_grid(long long units) { return int(std::max<long long>(1, std::min<long long>(units, 8LL * device_sm_count()))); }

template <typename T>
cudaError_t pack(long long n, int group, const void* x, void* codes, void* ranges, cudaStream_t s) {
    const int grid = pack_grid((n + 8LL * group - 1) / (8LL * group));
#define PACK(PER) in_stream_order(checkpoint_pack<T, PER>, grid, kPackThreads, 0, s)(n, (const T*)x, (unsigned char*)codes, (T*)ranges)
    if (group == 32) PACK(1); else if (group == 64) PACK(2); else if (group == 128) PACK(4); else PACK(8);
#undef PACK
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t unpack(long long first, long long n, int group, const void* codes, const void* ranges, void* x, cudaStream_t s) {
    int shift = 5;
    while ((1 << shift) < group) ++shift;
    in_stream_order(checkpoint_unpack<T>, pack_grid((n + kPackThreads - 1) / kPackThreads), kPackThreads, 0, s)(first, n, shift, (const unsigned char*)codes, (const T*)ranges, (T*)x);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_checkpoint_pack(bool f64, long long n, int group, const void* x, void* codes, void* ranges, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    return f64 ? pack<double>(n, group, x, codes, ranges, s) : pack<float>(n, group, x, codes, ranges, s);
}
cudaError_t launch_checkpoint_unpack(bool f64, long long first, long long n, int group, const void* codes, const void* ranges, void* x, cudaStream_t s) {
    if (n == 0) return cudaSuccess;
    return f64 ? unpack<double>(first, n, group, codes, ranges, x, s) : unpack<float>(first, n, group, codes, ranges, x, s);
}

}  // namespace simnets

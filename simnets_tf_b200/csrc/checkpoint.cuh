// What a byte of an 8-bit checkpoint stands for (see checkpoint.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include <math_constants.h>

namespace simnets {
namespace {

template <typename T> struct Limits;
template <> struct Limits<float> {
    static __device__ __forceinline__ float inf() { return CUDART_INF_F; }
    static __device__ __forceinline__ float tiny() { return 1.17549435e-38f; }
    static __device__ __forceinline__ float most() { return 3.402823466e38f; }
    static __device__ __forceinline__ float halves(float v, float half) { return __fmaf_rn(v, 0.5f, -half); }        // v / 2 - base / 2
    static __device__ __forceinline__ uint32_t nearest(float a, float b) { return __float_as_uint(__fmaf_rn(a, b, 12582912.f)) & 255u; }
    static __device__ __forceinline__ float at(float code, float step, float base) { return fminf(__fmaf_rn(code, step, base), most()); }
};
template <> struct Limits<double> {
    static __device__ __forceinline__ double inf() { return CUDART_INF; }
    static __device__ __forceinline__ double tiny() { return 2.2250738585072014e-308; }
    static __device__ __forceinline__ double most() { return 1.7976931348623157e308; }
    static __device__ __forceinline__ double halves(double v, double half) { return __fma_rn(v, 0.5, -half); }
    static __device__ __forceinline__ uint32_t nearest(double a, double b) { return uint32_t(__double_as_longlong(__fma_rn(a, b, 6755399441055744.0))) & 255u; }
    static __device__ __forceinline__ double at(double code, double step, double base) { return fmin(__fma_rn(code, step, base), most()); }
};

template <typename T>
__device__ __forceinline__ T unpacked(uint32_t c, T base, T step) {
    const T v = Limits<T>::at(T(int(c)), step, base);
    return c < 253u ? v : c == 253u ? -Limits<T>::inf() : c == 254u ? Limits<T>::inf() : Limits<T>::inf() - Limits<T>::inf();
}

}  // namespace
}  // namespace simnets

// Both gradients of a MEX layer at an 8-bit checkpoint of its input, in one pass over the bytes and dy (float32, disjoint blocks of up to
// 128 taps that cover the input).  With x the values that the bytes stand for, a = eps log2(e),
//
//     Ex[j,k] = 2^(a (x - mx_j)),   Eo[m,k] = 2^(a (o - mo_m)),   S[j,m] = sum_k Ex Eo,   Q[j,m] = dy / S,
//     dx[j,k] = Ex sum_m Q Eo,      doff[m,k] = Eo sum_j Q Ex.
//
// The extrema and y drop out: the weights of a patch are a softmax, which no shift changes.  So nothing but the bytes and their
// ranges is read of the forward pass, and neither x nor y nor anything of their size is written.
//
// Bound: the three products, 6 M K operations a position, on the tensor cores (64 taps under 128 instances: 49 k operations for 450 bytes).
// A CTA takes 128 positions of one region: Ex and, 64 or 128 instances at a time, Q lie in shared memory as three bfloat16 planes whose sum
// is the value to the bit (8 + 8 + 8 bits), in core matrices of 8 x 16 bytes.  Such a core matrix is the same whichever of
// its two axes is summed over, so that Ex serves the first and the third product, Q the second and the third and Eo the first and the second without
// a second copy; TF32 operands of that kind have no such layout (4-byte elements are transposed under a swizzle only), and their two planes
// take 16 bytes a value instead of 6.  Six of the nine plane products are taken, small ones first: what an accumulator truncates is
// 2^-24 of what it holds, which then are the largest products' K / 16 steps only.  Accumulators are emptied into FP32 registers or, the
// offsets' sums, into the CTA's own partial sums after every 128 positions.
//
// Offsets whose spread is beyond what the factors hold raise the status word in the prepass; the kernel then leaves at once and the
// kernels behind it, gated by that word, evaluate term by term.
#include "checkpoint.cuh"
#include "tc.cuh"

namespace simnets {
namespace {

constexpr int kFuseThreads = 512, kFuseColumns = 256;

__device__ __forceinline__ void umma_bf16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u) : "memory");
}
// D = F32, A = B = BF16, M = 128, N = nt; `across`: the operand's sum runs over the core matrices' rows, not along their 16 bytes
__host__ __device__ constexpr uint32_t bf16_idesc(int nt, bool a_across, bool b_across) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(a_across) << 15) | (uint32_t(b_across) << 16) | (uint32_t(nt >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}

// A [rows][cols] operand in three planes of [rows / 8][cols / 8] core matrices (8 rows x 8 columns, 16 bytes a row).
template <int ROWS, int COLS>
struct Planes {
    static constexpr uint32_t kPlane = ROWS * COLS * 2, kBytes = 3 * kPlane, kRowGroup = COLS / 8 * 128;
    static __device__ __forceinline__ uint32_t at(int row, int col) { return uint32_t(row >> 3) * kRowGroup + uint32_t(col >> 3) * 128 + uint32_t(row & 7) * 16 + uint32_t(col & 7) * 2; }
    // operand whose rows are the matrix's, summed over 16 columns from step on
    static __device__ __forceinline__ uint64_t along(uint32_t base, int plane, int step) { return umma_desc(base + plane * kPlane + step * 256, 128, kRowGroup); }
    // operand whose rows are the matrix's columns, summed over 16 rows from step on
    static __device__ __forceinline__ uint64_t across(uint32_t base, int plane, int step) { return umma_desc(base + plane * kPlane + step * 2 * kRowGroup, kRowGroup, 128); }
};

// the plane products that are taken, small ones first
__device__ __forceinline__ constexpr int plane_a(int i) { return i == 0 ? 1 : i == 1 ? 0 : i == 2 ? 2 : i == 3 ? 0 : i == 4 ? 1 : 0; }
__device__ __forceinline__ constexpr int plane_b(int i) { return i == 0 ? 1 : i == 1 ? 2 : i == 2 ? 0 : i == 3 ? 1 : 0; }

// two values as three words of two bfloat16 each: the top, middle and last 8 bits
struct Split2 { uint32_t hi, mid, lo; };
__device__ __forceinline__ Split2 split_bf16(float a, float b) {
    Split2 s;
    s.hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
    b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    s.mid = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
    b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    s.lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    return s;
}

// C values of one row from column `col` on (4: half a core row) into the planes
template <class P, int C>
__device__ __forceinline__ void store_row(unsigned char* base, int row, int col, const float (&v)[C]) {
    if constexpr (C == 4) {
        const Split2 s0 = split_bf16(v[0], v[1]), s1 = split_bf16(v[2], v[3]);
        unsigned char* d = base + P::at(row, col);
        *reinterpret_cast<uint2*>(d) = make_uint2(s0.hi, s1.hi);
        *reinterpret_cast<uint2*>(d + P::kPlane) = make_uint2(s0.mid, s1.mid);
        *reinterpret_cast<uint2*>(d + 2 * P::kPlane) = make_uint2(s0.lo, s1.lo);
    } else {
#pragma unroll
        for (int c = 0; c < C; c += 8) {
            const Split2 s0 = split_bf16(v[c], v[c + 1]), s1 = split_bf16(v[c + 2], v[c + 3]), s2 = split_bf16(v[c + 4], v[c + 5]), s3 = split_bf16(v[c + 6], v[c + 7]);
            unsigned char* d = base + P::at(row, col + c);
            *reinterpret_cast<uint4*>(d) = make_uint4(s0.hi, s1.hi, s2.hi, s3.hi);
            *reinterpret_cast<uint4*>(d + P::kPlane) = make_uint4(s0.mid, s1.mid, s2.mid, s3.mid);
            *reinterpret_cast<uint4*>(d + 2 * P::kPlane) = make_uint4(s0.lo, s1.lo, s2.lo, s3.lo);
        }
    }
}

// N consecutive tensor-memory columns of this thread's lane
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[N]) {
    uint32_t r[N];
    if constexpr (N == 32) {
        tmem_ld32(taddr, r);
    } else if constexpr (N == 16) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                       "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    } else if constexpr (N == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    } else {
        static_assert(N == 4);
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}

__host__ __device__ constexpr int fuse_taps(int k) { return k <= 16 ? 16 : k <= 32 ? 32 : k <= 64 ? 64 : 128; }
__host__ __device__ constexpr int fuse_instances(int kp) { return kp <= 64 ? 128 : 64; }        // instances a step: what shared memory holds

// Eo of one row of offsets (blockIdx.x = region * padded instances + instance): plain in eo[R][M][KP], split in the tiles of the main kernel;
// zeros for what is not there.  128 threads.
__global__ void __launch_bounds__(128) fuse_prepare(MexGeo g, int KP, int MC, int Mp, const float* __restrict__ off, float* __restrict__ eo, unsigned char* __restrict__ tiles,
                                                    int* __restrict__ flag) {
    stream_order();
    __shared__ float red[2][4];
    const int r = blockIdx.x / Mp, m = blockIdx.x % Mp, k = threadIdx.x, lane = k & 31, warp = k >> 5;
    const bool in = m < g.M && k < g.K;
    const float v = in ? off[((size_t)r * g.M + m) * g.K + k] : 0.f;
    float hi = in ? v : -CUDART_INF_F, lo = in ? v : CUDART_INF_F;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) { hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d)); lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d)); }
    if (lane == 0) { red[0][warp] = hi; red[1][warp] = lo; }
    __syncthreads();
    hi = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    lo = fminf(fminf(red[1][0], red[1][1]), fminf(red[1][2], red[1][3]));
    const float eps = float(g.eps);
    if (in && (!(fabsf(v) < CUDART_INF_F) || !(fabsf(eps) * (hi - lo) <= kSafeSpread))) flag[0] = 1;
    const float e = in ? ex2_ftz(eps * 1.4426950408889634f * (v - (eps > 0.f ? hi : lo))) : 0.f;
    if (k >= KP) return;
    if (m < g.M) eo[((size_t)r * g.M + m) * KP + k] = e;
    const int row = m % MC;
    unsigned char* d = tiles + ((size_t)r * (Mp / MC) + m / MC) * (3 * MC * KP * 2) + (row >> 3) * (KP / 8 * 128) + (k >> 3) * 128 + (row & 7) * 16 + (k & 7) * 2;
    const Split2 s = split_bf16(e, 0.f);
    *reinterpret_cast<unsigned short*>(d) = (unsigned short)s.hi;
    *reinterpret_cast<unsigned short*>(d + MC * KP * 2) = (unsigned short)s.mid;
    *reinterpret_cast<unsigned short*>(d + 2 * MC * KP * 2) = (unsigned short)s.lo;
}

struct FuseArgs {
    const unsigned char* codes;
    const float2* ranges;
    const unsigned char* tiles;
    const float* dy;
    float* dx;              // may be null
    float* part;            // [CTA][Mp][KP], may be null
    int* flag;
    int shift;              // log2 of the group
    int tiles_m;            // steps of instances
    long long tiles_j;      // tiles of positions of a region
};

template <int KP>
__global__ void __launch_bounds__(kFuseThreads, 1) mex_gradients_at_checkpoint(MexGeo g, FuseArgs a) {
    stream_order();
    constexpr int MC = fuse_instances(KP), KR = KP / 4, MR = MC / 4;
    constexpr bool kByTaps = KP > 64;                    // the offsets' sums with the taps as rows (128 of them), else with the instances
    using X = Planes<128, KP>;
    using Q = Planes<128, MC>;
    using E = Planes<MC, KP>;
    extern __shared__ __align__(1024) unsigned char sm[];
    __shared__ TcShared sh;
    __shared__ float red[4][128];
    __shared__ int tap_off[KP];
    if (a.flag[0]) return;
    unsigned char *const sx = sm, *const sq = sm + X::kBytes, *const se = sq + Q::kBytes;
    const int p = threadIdx.x & 127, part4 = threadIdx.x >> 7;                          // position (tensor-memory lane) and its quarter of the columns
    const uint32_t lane_base = uint32_t((threadIdx.x >> 5) & 3) << 21;                   // (32 lanes a warp, lane number in bits 16 and up)
    const int r = int(blockIdx.x) % g.R, slot = int(blockIdx.x) / g.R, slots = int(gridDim.x) / g.R;
    const int Mp = a.tiles_m * MC;
    for (int k = threadIdx.x; k < KP; k += kFuseThreads) {
        const Tap t = tap_of<false>(g, k < g.K ? k : 0);
        tap_off[k] = (t.c * g.H + t.h) * g.W + t.w;
    }
    const uint32_t tmem = tc_begin(sh, kFuseColumns);                                   // (its barrier also publishes tap_off)
    const uint32_t tS = tmem, tT = tmem + MC, tU = tT + KP;
    const float eps = float(g.eps), a2 = eps * 1.4426950408889634f;
    const long long P = (long long)g.B * g.rs;
    const uint32_t xb = smem_u32(sx), qb = smem_u32(sq), eb = smem_u32(se);
    bool ok = true;
    uint32_t phase = 0;                                                                  // of both barriers

    auto load_offsets = [&](int mt) {
        const unsigned char* src = a.tiles + ((size_t)r * a.tiles_m + mt) * E::kBytes;
        for (int i = threadIdx.x; i < int(E::kBytes / 16); i += kFuseThreads) cp_async16(reinterpret_cast<float*>(se + i * 16), reinterpret_cast<const float*>(src + i * 16), 16);
    };
    if (a.tiles_m == 1) load_offsets(0);

    for (long long jt = slot; jt < a.tiles_j && ok; jt += slots) {
        const Column col = column_of(g, r, jt * 128 + p, P, nullptr);
        const bool live = col.base >= 0;
        const long long xi = (((long long)col.n * g.C + col.c0) * g.H + col.h0) * g.W + col.w0;
        // this thread's taps: part4 * KR .. + KR
        float ex[KR], tsum[KR];
        {
            uint32_t code[KR];
            float mx = eps > 0.f ? -CUDART_INF_F : CUDART_INF_F;
#pragma unroll
            for (int i = 0; i < KR; ++i) code[i] = live && part4 * KR + i < g.K ? a.codes[xi + tap_off[part4 * KR + i]] : 0u;
#pragma unroll
            for (int i = 0; i < KR; ++i) {
                const bool in = live && part4 * KR + i < g.K;
                const float2 range = in ? __ldg(a.ranges + ((xi + tap_off[part4 * KR + i]) >> a.shift)) : make_float2(0.f, 0.f);
                ex[i] = unpacked<float>(code[i], range.x, range.y);
                if (in) mx = eps > 0.f ? fmaxf(mx, ex[i]) : fminf(mx, ex[i]);
            }
            red[part4][p] = mx;
            __syncthreads();
            mx = eps > 0.f ? fmaxf(fmaxf(red[0][p], red[1][p]), fmaxf(red[2][p], red[3][p])) : fminf(fminf(red[0][p], red[1][p]), fminf(red[2][p], red[3][p]));
#pragma unroll
            for (int i = 0; i < KR; ++i) {
                ex[i] = live && part4 * KR + i < g.K ? ex2_ftz(a2 * (ex[i] - mx)) : 0.f;
                tsum[i] = 0.f;
            }
        }
        store_row<X>(sx, p, part4 * KR, ex);
        const float* dyp = a.dy + (live ? col.gbase : 0);
        for (int mt = 0; mt < a.tiles_m; ++mt) {                                          // (`ok` is one value for all threads behind every barrier)
            if (a.tiles_m > 1) load_offsets(mt);
            cp_async_wait_all();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            ok = __syncthreads_and(ok);
            if (threadIdx.x == 0 && ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 6; ++i)
#pragma unroll
                    for (int s = 0; s < KP / 16; ++s) umma_bf16(tS, X::along(xb, plane_a(i), s), E::along(eb, plane_b(i), s), bf16_idesc(MC, false, false), (i | s) != 0);
                umma_commit(&sh.bar_free[0]);
            }
            // this thread's instances: m0 .. + MR
            const int m0 = mt * MC + part4 * MR;
            float q[MR];
#pragma unroll
            for (int i = 0; i < MR; ++i) q[i] = live && m0 + i < g.M ? __ldcs(dyp + (long long)(m0 + i) * g.Ng) : 0.f;
            if (ok) ok = mbar_wait(&sh.bar_free[0], phase);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            {
                float s[MR];
                tmem_ld<MR>(tS + lane_base + part4 * MR, s);
#pragma unroll
                for (int i = 0; i < MR; ++i) q[i] = live && m0 + i < g.M ? __fdividef(q[i], s[i]) : 0.f;
            }
            store_row<Q>(sq, p, part4 * MR, q);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            ok = __syncthreads_and(ok);
            if (threadIdx.x == 0 && ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (a.dx)
#pragma unroll
                    for (int i = 0; i < 6; ++i)
#pragma unroll
                        for (int s = 0; s < MC / 16; ++s) umma_bf16(tT, Q::along(qb, plane_a(i), s), E::across(eb, plane_b(i), s), bf16_idesc(KP, false, true), (i | s) != 0);
                if (a.part)
#pragma unroll
                    for (int i = 0; i < 6; ++i)
#pragma unroll
                        for (int s = 0; s < 8; ++s) {
                            if (kByTaps) umma_bf16(tU, X::across(xb, plane_a(i), s), Q::across(qb, plane_b(i), s), bf16_idesc(MC, true, true), (i | s) != 0);
                            else umma_bf16(tU, Q::across(qb, plane_a(i), s), X::across(xb, plane_b(i), s), bf16_idesc(KP, true, true), (i | s) != 0);
                        }
                umma_commit(&sh.bar_free[1]);
            }
            if (ok) ok = mbar_wait(&sh.bar_free[1], phase);
            phase ^= 1u;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (a.dx) {
                float t[KR];
                tmem_ld<KR>(tT + lane_base + part4 * KR, t);
#pragma unroll
                for (int i = 0; i < KR; ++i) tsum[i] += t[i];
            }
            if (a.part) {
                const bool first = jt == slot;
                if constexpr (kByTaps) {                                                 // row = tap p, columns = instances
                    float u[MR];
                    tmem_ld<MR>(tU + lane_base + part4 * MR, u);
                    float* d = a.part + ((size_t)blockIdx.x * Mp + mt * MC + part4 * MR) * KP + p;
#pragma unroll
                    for (int i = 0; i < MR; ++i) d[i * KP] = first ? u[i] : d[i * KP] + u[i];
                } else {                                                                 // row = instance p, columns = taps
                    float u[KR];
                    tmem_ld<KR>(tU + lane_base + part4 * KR, u);
                    float4* d = reinterpret_cast<float4*>(a.part + ((size_t)blockIdx.x * Mp + mt * MC + p) * KP + part4 * KR);
#pragma unroll
                    for (int i = 0; i < KR / 4; ++i) {
                        const float4 old = first ? make_float4(0.f, 0.f, 0.f, 0.f) : d[i];
                        d[i] = make_float4(old.x + u[4 * i], old.y + u[4 * i + 1], old.z + u[4 * i + 2], old.w + u[4 * i + 3]);
                    }
                }
            }
        }
        if (a.dx && live)
#pragma unroll
            for (int i = 0; i < KR; ++i)
                if (part4 * KR + i < g.K) a.dx[xi + tap_off[part4 * KR + i]] = ex[i] * tsum[i];
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        ok = __syncthreads_and(ok);                                                      // (and Ex may be written anew)
    }
    if (!ok && threadIdx.x == 0) atomicExch(&a.flag[0], 1);                              // a wait expired: the kernels behind redo the call
    cp_async_wait_all();
    tc_end(tmem, kFuseColumns);
}

// doff of one row (blockIdx.x = region * M + instance) from the CTAs' sums, in their order.  128 threads.
__device__ __forceinline__ float row_sum(float v, float (&red)[4]) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
// what a raw row's normalisation does to its gradient: d - softmax(row) sum(d)
__device__ __forceinline__ float raw_gradient(const float* __restrict__ row, int K, float d, float (&red)[4]) {
    const int k = threadIdx.x;
    float hi = k < K ? row[k] : -CUDART_INF_F;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
    __syncthreads();
    if ((k & 31) == 0) red[k >> 5] = hi;
    __syncthreads();
    hi = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float e = k < K ? expf(row[k] - hi) : 0.f;
    const float sum = row_sum(e, red), total = row_sum(d, red);
    return d - e / sum * total;
}
__global__ void __launch_bounds__(128) fuse_offsets_sum(MexGeo g, int KP, int Mp, int ctas, int normalized, int accumulate, const float* __restrict__ off,
                                                        const float* __restrict__ eo, const float* __restrict__ part, float* __restrict__ doff, const int* __restrict__ flag) {
    stream_order();
    if (flag[0]) return;
    __shared__ float red[4];
    const int r = blockIdx.x / g.M, m = blockIdx.x % g.M, k = threadIdx.x;
    float d = 0.f;
    if (k < g.K) {
        const float* s = part + ((size_t)r * Mp + m) * KP + k;
        const size_t step = (size_t)g.R * Mp * KP;
        float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
        int c = r;
        for (; c + 3 * g.R < ctas; c += 4 * g.R, s += 4 * step) { s0 += s[0]; s1 += s[step]; s2 += s[2 * step]; s3 += s[3 * step]; }
        for (; c < ctas; c += g.R, s += step) s0 += s[0];
        d = eo[((size_t)r * g.M + m) * KP + k] * ((s0 + s1) + (s2 + s3));
    }
    const size_t row = ((size_t)r * g.M + m) * g.K;
    if (normalized) d = raw_gradient(off + row, g.K, d, red);
    if (k < g.K) doff[row + k] = accumulate ? doff[row + k] + d : d;
}

// ---- term by term, for offsets that no factorisation takes (gated by the status word) -----------------------------------------------
// a lane has the taps lane + 32 i
struct Taps4 { float v[4]; };
__device__ __forceinline__ Taps4 checkpoint_patch(const MexGeo& g, const FuseArgs& a, long long xi) {
    Taps4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = (threadIdx.x & 31) + 32 * i;
        t.v[i] = 0.f;
        if (k >= g.K) continue;
        const Tap tap = tap_of<false>(g, k);
        const long long at = xi + ((long long)tap.c * g.H + tap.h) * g.W + tap.w;
        const float2 range = a.ranges[at >> a.shift];
        t.v[i] = unpacked<float>(a.codes[at], range.x, range.y);
    }
    return t;
}
// softmax over the taps of eps (x + o)
__device__ __forceinline__ Taps4 patch_weights(const MexGeo& g, const Taps4& x, const float* __restrict__ row) {
    Taps4 t;
    const float eps = float(g.eps);
    float hi = -CUDART_INF_F, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = (threadIdx.x & 31) + 32 * i;
        t.v[i] = k < g.K ? eps * (x.v[i] + row[k]) : -CUDART_INF_F;
        hi = fmaxf(hi, t.v[i]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        t.v[i] = (threadIdx.x & 31) + 32 * i < g.K ? expf(t.v[i] - hi) : 0.f;
        sum += t.v[i];
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float inv = 1.f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) t.v[i] *= inv;
    return t;
}

// a warp per position (of all regions)
__global__ void __launch_bounds__(256) fuse_redo_dx(MexGeo g, FuseArgs a, const float* __restrict__ off) {
    stream_order();
    if (!a.flag[0]) return;
    const long long P = (long long)g.B * g.N;
    for (long long j = blockIdx.x * 8LL + (threadIdx.x >> 5); j < P; j += gridDim.x * 8LL) {
        const int n = int(j / g.N), pos = int(j - (long long)n * g.N), w = pos % g.Wo, h = pos / g.Wo % g.Ho, c = pos / (g.Wo * g.Ho), r = mex_region_of(g, c, h, w);
        const long long xi = (((long long)n * g.C + c * g.sc) * g.H + h * g.sh) * g.W + w * g.sw, at = mex_dy_base(g, n, pos);
        const Taps4 x = checkpoint_patch(g, a, xi);
        double sum[4] = {0, 0, 0, 0};
        for (int m = 0; m < g.M; ++m) {
            const Taps4 p = patch_weights(g, x, off + ((size_t)r * g.M + m) * g.K);
            const float v = a.dy[at + (long long)m * g.Ng];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += v * p.v[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = (threadIdx.x & 31) + 32 * i;
            if (k >= g.K) continue;
            const Tap tap = tap_of<false>(g, k);
            a.dx[xi + ((long long)tap.c * g.H + tap.h) * g.W + tap.w] = float(sum[i]);
        }
    }
}

// a CTA per row of offsets, its warps over the positions
__global__ void __launch_bounds__(256) fuse_redo_doff(MexGeo g, FuseArgs a, int normalized, int accumulate, const float* __restrict__ off, float* __restrict__ doff) {
    stream_order();
    if (!a.flag[0]) return;
    __shared__ double sums[8][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long P = (long long)g.B * g.rs;
    for (int row = blockIdx.x; row < g.R * g.M; row += gridDim.x) {
        const int r = row / g.M, m = row % g.M;
        double sum[4] = {0, 0, 0, 0};
        for (long long j = warp; j < P; j += 8) {
            const Column col = column_of(g, r, j, P, nullptr);
            if (col.base < 0) continue;
            const long long xi = (((long long)col.n * g.C + col.c0) * g.H + col.h0) * g.W + col.w0;
            const Taps4 p = patch_weights(g, checkpoint_patch(g, a, xi), off + (size_t)row * g.K);
            const float v = a.dy[col.gbase + (long long)m * g.Ng];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += v * p.v[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][lane + 32 * i] = sum[i];
        __syncthreads();
        float d = 0.f;
        if (threadIdx.x < 128) {
            double t = 0;
            for (int w = 0; w < 8; ++w) t += sums[w][threadIdx.x];
            if (int(threadIdx.x) < g.K) d = float(t);
        }
        if (normalized) {
            // (all warps take part in the barriers; the last four hold nothing)
            const int k = threadIdx.x;
            __shared__ float e_s[128], d_s[128];
            if (k < 128) { e_s[k] = k < g.K ? off[(size_t)row * g.K + k] : -CUDART_INF_F; d_s[k] = d; }
            __syncthreads();
            float hi = -CUDART_INF_F, se = 0.f, sd = 0.f;
            for (int i = 0; i < g.K; ++i) hi = fmaxf(hi, e_s[i]);
            for (int i = 0; i < g.K; ++i) { se += expf(e_s[i] - hi); sd += d_s[i]; }
            if (k < g.K) d -= expf(e_s[k] - hi) / se * sd;
        }
        if (int(threadIdx.x) < g.K) {
            float* to = doff + (size_t)row * g.K + threadIdx.x;
            *to = accumulate ? *to + d : d;
        }
        __syncthreads();
    }
}

struct FuseWs { int* flag; float *eo, *part; unsigned char* tiles; size_t bytes; };

struct FuseSizes { int KP, MC, Mp, slots; };
FuseSizes fuse_sizes(const MexGeo& g) {
    FuseSizes z;
    z.KP = fuse_taps(g.K);
    z.MC = fuse_instances(z.KP);
    z.Mp = (g.M + z.MC - 1) / z.MC * z.MC;
    const long long tiles = ((long long)g.B * g.rs + 127) / 128;
    z.slots = int(std::max<long long>(1, std::min<long long>(tiles, device_sm_count() / g.R)));
    return z;
}
FuseWs fuse_carve(const MexGeo& g, void* base) {
    const FuseSizes z = fuse_sizes(g);
    FuseWs w;
    char* p = static_cast<char*>(base);
    size_t off = 0;
    auto take = [&](size_t bytes) { char* r = p ? p + off : nullptr; off += align256(bytes); return r; };
    w.flag = reinterpret_cast<int*>(take(256));
    w.eo = reinterpret_cast<float*>(take(sizeof(float) * (size_t)g.R * g.M * z.KP));
    w.tiles = reinterpret_cast<unsigned char*>(take((size_t)g.R * z.Mp * z.KP * 6));
    w.part = reinterpret_cast<float*>(take(sizeof(float) * (size_t)z.slots * g.R * z.Mp * z.KP));
    w.bytes = off;
    return w;
}

template <int KP>
cudaError_t launch_fused(const MexGeo& g, const FuseArgs& a, int ctas, cudaStream_t s) {
    constexpr int MC = fuse_instances(KP), smem = Planes<128, KP>::kBytes + Planes<128, MC>::kBytes + Planes<MC, KP>::kBytes;
    static SmemLimit limit;
    const cudaError_t e = limit.raise(mex_gradients_at_checkpoint<KP>, smem);
    if (e != cudaSuccess) return e;
    in_stream_order(mex_gradients_at_checkpoint<KP>, ctas, kFuseThreads, smem, s)(g, a);
    return cudaSuccess;
}

}  // namespace

// Blocks that cover the input once, in few regions (a CTA works for one).
bool mex_checkpoint_shape(const MexGeo& g, bool f64, uint32_t flags) {
    if (f64 || !g.finite || g.B == 0 || g.K > 128 || (flags & (SIMNETS_FLAG_FORCE_DIRECT | SIMNETS_FLAG_MEX_EXACT | SIMNETS_FLAG_MEX_NO_TENSORCORE))) return false;
    const bool cover = g.sc == g.bc && g.sh == g.bh && g.sw == g.bw && g.pc == 0 && g.ph == 0 && g.pw == 0 && g.Co * g.bc == g.C && g.Ho * g.bh == g.H && g.Wo * g.bw == g.W;
    return cover && g.R <= 16 && g.M <= 8192 && (long long)g.C * g.H * g.W < (1LL << 31) && (long long)g.B * g.rs < (1LL << 38);
}
size_t mex_checkpoint_bytes(const MexGeo& g) { return fuse_carve(g, nullptr).bytes; }

cudaError_t launch_mex_checkpoint(const MexGeo& g, int group, const void* codes, const void* ranges, const float* off, const float* dy, float* dx, float* doff,
                                  bool accumulate, bool normalized, void* ws, cudaStream_t s) {
    const FuseSizes z = fuse_sizes(g);
    const FuseWs w = fuse_carve(g, ws);
    FuseArgs a;
    a.codes = static_cast<const unsigned char*>(codes);
    a.ranges = static_cast<const float2*>(ranges);
    a.tiles = w.tiles;
    a.dy = dy; a.dx = dx; a.part = doff ? w.part : nullptr;
    a.flag = w.flag;
    a.shift = 5;
    while ((1 << a.shift) < group) ++a.shift;
    a.tiles_m = z.Mp / z.MC;
    a.tiles_j = ((long long)g.B * g.rs + 127) / 128;
    cudaError_t e = launch_zero_words(w.flag, 2, s);
    if (e != cudaSuccess) return e;
    in_stream_order(fuse_prepare, g.R * z.Mp, 128, 0, s)(g, z.KP, z.MC, z.Mp, off, w.eo, w.tiles, w.flag);
    const int ctas = z.slots * g.R;
    e = z.KP == 16 ? launch_fused<16>(g, a, ctas, s) : z.KP == 32 ? launch_fused<32>(g, a, ctas, s) : z.KP == 64 ? launch_fused<64>(g, a, ctas, s) : launch_fused<128>(g, a, ctas, s);
    if (e != cudaSuccess) return e;
    count_launch(2);
    if (doff) {
        in_stream_order(fuse_offsets_sum, g.R * g.M, 128, 0, s)(g, z.KP, z.Mp, ctas, int(normalized), int(accumulate), off, w.eo, w.part, doff, w.flag);
        in_stream_order(fuse_redo_doff, std::min(g.R * g.M, 4 * device_sm_count()), 256, 0, s)(g, a, int(normalized), int(accumulate), off, doff);
        count_launch(2);
    }
    if (dx) {
        in_stream_order(fuse_redo_dx, 4 * device_sm_count(), 256, 0, s)(g, a, off);
        count_launch();
    }
    return cudaGetLastError();
}

}  // namespace simnets

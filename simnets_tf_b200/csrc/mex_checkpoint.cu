// Both gradients of a MEX layer at an 8-bit checkpoint of its input, in one pass over the bytes and dy (float32, disjoint blocks of up to
// 128 taps that cover the input).  With x the values that the bytes stand for, a = eps log2(e),
//
//     Ex[j,k] = 2^(a (x - mx_j)),   Eo[m,k] = 2^(a (o - mo_m)),   S[j,m] = sum_k Ex Eo,   Q[j,m] = dy / S,
//     dx[j,k] = Ex sum_m Q Eo,      doff[m,k] = Eo sum_j Q Ex.
//
// The extrema and y drop out: the weights of a patch are a softmax, which no shift changes.  So nothing but the bytes and their
// ranges is read of the forward pass, and neither x nor y is written.  Beside the results there are the offsets' sums of every CTA, 148 M K floats (in whole
// tiles) where positions fill the GPU: 4.8 MB for 64 taps under 128 instances, 155 MB for 128 under 2048, as much as y over 128 positions a CTA.
//
// Bound: the three products, 6 M K operations a position, on the tensor cores (64 taps under 128 instances: 49 k operations for 450 bytes).
// A CTA takes 128 positions of one region: Ex and, 64 or 128 instances at a time, Q lie in shared memory as three bfloat16 planes whose sum
// is the value to the bit (8 + 8 + 8 bits), in core matrices of 8 x 16 bytes.  Such a core matrix is the same whichever of
// its two axes is summed over, so that Ex serves the first and the third product, Q the second and the third and Eo the first and the second without
// a second copy; TF32 operands of that kind have no such layout (4-byte elements are transposed under a swizzle only), and their two planes
// take 16 bytes a value instead of 6.  Six of the nine plane products are taken, small ones first: what an accumulator truncates is
// 2^-24 of what it holds, which then are the largest products' K / 16 steps only.  An instruction with 64 columns waits for its 128 rows (50
// cycles instead of 32), so that the second and third product take the planes of their narrow operand side by side, as up to 192 columns
// (96 cycles for three).  Accumulators are emptied into FP32 after every 128 positions (after 512:
// 4 us less of the 252 below, and the offsets' gradient 1.5e-6 of its norm off instead of 3.7e-7).
//
// Sixteen warps work on the values and one issues the products: a tile's bytes are read and exponentiated while the second product of the tile
// in front runs, the offsets' sums are added to the CTA's while the first one runs.  512 x 64 x 32 x 32 under 128 instances, pooled: 252 to 268 us by card
// (all phases in turn, descriptors made anew for every instruction: 519; the FP32 kernels of the other entry points 1267; the floor of the
// products 95); 32 x 256 x 32 x 32 under 256 instances over 4x2x2 blocks 224 to 228 us (499; 1463; bytes 88).  Where the rest goes: a tile is a chain of
// Ex, S, Q, sums, next Ex, the operands of one tile fill shared memory, and 96 registers a thread are what 17 warps have; warps wait for loads 3.6 of
// 9 cycles, the tensor pipe is busy 27 %.  Half of the warps for the taps and half for the instances were slower (266, 280).
//
// Offsets whose spread is beyond what the factors hold are found in the prepass; the kernel then leaves at once and the one behind it, which
// else adds up the partial sums, evaluates term by term.  Gradients that are infinite, or so large that a quotient or a sum of quotients is no float
// any more (S is as small as e^-60): infinity has no bfloat16 planes that add up to it, so that the results they enter come out as no numbers, and
// the kernel behind evaluates those term by term, and only those.  Term by term a call of 64 x 64 x 32 x 32 under 128 instances takes 7.5 ms instead of 64 us
// (the op's forward pass and gradients at such offsets 6.9), one infinite dy in it 3.6.
//
// Factors below 2^-126 are 0: a tap whose weight is below e^-27 (1.4e-12, where x lies 87 nats under the patch's largest and the offsets' spread is the
// most that the factors take) may have a gradient of 0.
#include "checkpoint.cuh"
#include "ws.cuh"
#include <cmath>

namespace simnets {
namespace {

constexpr int kFuseWorkers = 512, kFuseThreads = kFuseWorkers + 32, kFuseColumns = 512;

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

// A [rows][cols] operand as [rows / 8][3 planes][cols / 8] core matrices (8 rows x 8 columns, 16 bytes a row): the planes are columns side by side.
template <int ROWS, int COLS>
struct Planes {
    static constexpr uint32_t kPlane = COLS / 8 * 128, kRowGroup = 3 * kPlane, kBytes = ROWS / 8 * kRowGroup;
    static __host__ __device__ __forceinline__ constexpr uint32_t at(int row, int col) { return uint32_t(row >> 3) * kRowGroup + uint32_t(col >> 3) * 128 + uint32_t(row & 7) * 16 + uint32_t(col & 7) * 2; }
    // operand whose rows are the matrix's, summed over 16 columns of a plane from step on, from its descriptor at (0, 0)
    static __device__ __forceinline__ uint64_t along(uint32_t base) { return umma_desc(base, 128, kRowGroup); }
    static __host__ __device__ constexpr uint32_t along_at(int plane, int step) { return (plane * kPlane + step * 256) >> 4; }
    // operand whose rows are the matrix's columns from `plane` on, summed over 16 rows from step on
    static __device__ __forceinline__ uint64_t across(uint32_t base) { return umma_desc(base, kRowGroup, 128); }
    static __host__ __device__ constexpr uint32_t across_at(int plane, int step) { return (plane * kPlane + step * 2 * kRowGroup) >> 4; }
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

// a sum of squares of the values' top parts, two at once: infinity or NaN where one of them is no number or above 2^64
__device__ __forceinline__ void add_squares(uint32_t& sum, uint32_t tops) { asm("fma.rn.bf16x2 %0, %1, %1, %0;" : "+r"(sum) : "r"(tops)); }

// C values of one row from column `col` on (4: half a core row) into the planes; `squares`: see add_squares
template <class P, int C>
__device__ __forceinline__ void store_row(unsigned char* base, int row, int col, const float (&v)[C], uint32_t& squares) {
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
            add_squares(squares, s0.hi); add_squares(squares, s1.hi); add_squares(squares, s2.hi); add_squares(squares, s3.hi);
            *reinterpret_cast<uint4*>(d) = make_uint4(s0.hi, s1.hi, s2.hi, s3.hi);
            *reinterpret_cast<uint4*>(d + P::kPlane) = make_uint4(s0.mid, s1.mid, s2.mid, s3.mid);
            *reinterpret_cast<uint4*>(d + 2 * P::kPlane) = make_uint4(s0.lo, s1.lo, s2.lo, s3.lo);
        }
    }
}

template <class P, int C>
__device__ __forceinline__ void store_row(unsigned char* base, int row, int col, const float (&v)[C]) {
    uint32_t squares = 0;
    store_row<P, C>(base, row, col, v, squares);
}

// N consecutive tensor-memory columns of this thread's lane; there once tmem_wait() is through
template <int N>
__device__ __forceinline__ void tmem_request(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 16) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                       "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
    } else if constexpr (N == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
    } else {
        static_assert(N == 4);
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(taddr) : "memory");
    }
}
// (the registers pass through it, so that nothing reads them earlier)
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

__host__ __device__ constexpr int fuse_taps(int k) { return k <= 16 ? 16 : k <= 32 ? 32 : k <= 64 ? 64 : 128; }
__host__ __device__ constexpr int fuse_instances(int kp) { return kp <= 64 ? 128 : 64; }        // instances a step: what shared memory holds

// Eo of one row of offsets (blockIdx.x = region * padded instances + instance): plain in eo[R][M][KP], split in the tiles of the main kernel.
// Taps that are not there are zeros, instances that are not there ones (S must not be 0).  128 threads.
__global__ void __launch_bounds__(128) fuse_prepare(MexGeo g, int KP, int MC, int Mp, const float* __restrict__ off, float* __restrict__ eo, unsigned char* __restrict__ tiles,
                                                    int* __restrict__ status) {
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
    // (the extremes leave a NaN out)
    const int unsafe = __syncthreads_or(in && (!(fabsf(v) < CUDART_INF_F) || !(fabsf(eps) * (hi - lo) <= kSafeSpread)));
    if (k == 0) status[2 + blockIdx.x] = unsafe;
    if (k < 3 && blockIdx.x == 0) status[k < 2 ? k : 2 + gridDim.x] = 0;
    const float e = in ? ex2_ftz(eps * 1.4426950408889634f * (v - (eps > 0.f ? hi : lo))) : m < g.M ? 0.f : 1.f;
    if (k >= KP) return;
    if (m < g.M) eo[((size_t)r * g.M + m) * KP + k] = e;
    const int row = m % MC;
    unsigned char* d = tiles + ((size_t)r * (Mp / MC) + m / MC) * (3 * MC * KP * 2) + (row >> 3) * (3 * KP / 8 * 128) + (k >> 3) * 128 + (row & 7) * 16 + (k & 7) * 2;
    const Split2 s = split_bf16(e, 0.f);
    *reinterpret_cast<unsigned short*>(d) = (unsigned short)s.hi;
    *reinterpret_cast<unsigned short*>(d + KP / 8 * 128) = (unsigned short)s.mid;
    *reinterpret_cast<unsigned short*>(d + 2 * (KP / 8 * 128)) = (unsigned short)s.lo;
}

struct FuseArgs {
    const unsigned char* codes;
    const float2* ranges;
    const unsigned char* tiles;
    const float* dy;
    float* dx;              // may be null
    float* part;            // [CTA][step] of what part_at() lays out, may be null
    int* status;            // the two words of a MEX workspace; then, per row of offsets, whether its spread is beyond what the factors hold; then
                            // whether a quotient was beyond kMostQuotient
    int rows;               // R Mp of those
    int shift;              // log2 of the group
    int tiles_m;            // steps of instances
    int resident;           // all of them lie in shared memory
    int expire;             // test hook: the first product is not taken, and waits are short
    long long tiles_j;      // tiles of positions of a region
};

// Whether the products have not been, or cannot be, taken (all threads of a CTA ask).
__device__ __forceinline__ bool term_by_term(const FuseArgs& a) {
    int any = 0;
    for (int i = threadIdx.x; i <= a.rows; i += blockDim.x) any |= a.status[1 + i];
    return __syncthreads_or(any) != 0;
}

// some tens of microseconds instead of two seconds
__device__ __forceinline__ bool mbar_wait_briefly(uint64_t* bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
    for (int i = 0; i < 64; ++i) {
        if (mbar_try(addr, parity)) return true;
        __nanosleep(256);
    }
    return false;
}

// Place of (instance of a step, tap) in the partial sums of the step, neighbouring lanes side by side: a lane has four taps of an instance at
// once, or, where the taps are the rows, a tap of an instance.
__host__ __device__ constexpr int part_at(int KP, int MC, int m, int k) { return KP > 64 ? m * KP + k : ((k >> 2) * MC + m) * 4 + (k & 3); }

// barriers of a CTA; all but the first two complete once a step (a tile of positions, 64 or 128 instances)
struct FuseShared {
    uint64_t operands;      // workers: Ex (and, where it is not kept, Eo) of the step are there; with Eo kept and S twice, once a tile
    uint64_t sums[2];       // products: S is there (by place in tensor memory)
    uint64_t quotients;     // workers: Q is there, S has been read
    uint64_t taps;          // products: the sums over the instances are there
    uint64_t instances;     // products: the sums over the positions are there, and Ex and Q may be written anew
    uint64_t drained;       // products, after a wait that ran out: none is under way any more
    uint32_t tmem;
    volatile int failed;
    volatile int beyond;    // a quotient was beyond kMostQuotient
};

// Quotients up to here give finite sums: over 8192 instances 2^105, over the positions of any tensor that fits the memory (2^35 values) 2^127.
constexpr float kMostQuotient = 0x1p92f;

// An operand: its descriptor and where its planes and steps lie from there.  (The products are issued by one thread; what it computes between two of
// them is what the tensor cores wait for: an addition to the address field here, 100 cycles an instruction with descriptors made anew.)
template <class P, bool ACROSS>
struct Operand {
    uint64_t desc;
    __device__ __forceinline__ explicit Operand(uint32_t base) : desc(ACROSS ? P::across(base) : P::along(base)) {}
    __device__ __forceinline__ uint64_t operator()(int plane, int step) const { return desc + (ACROSS ? P::across_at(plane, step) : P::along_at(plane, step)); }
    static constexpr bool kAcross = ACROSS;
};
__device__ __forceinline__ bool elected() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

// D[128 x N] (+)= sum over STEPS x 16 of A B with B's planes side by side: (2,0), (1,0) + (1,1), (0,0) + (0,1) + (0,2), the sums of B's plane j in
// the j-th N columns.  a(plane, step), b(plane, step): operands.  (A first step that starts some columns and adds to others is two instructions.)
template <int N, int STEPS, class A, class B>
__device__ __forceinline__ void issue_side_by_side(uint32_t tmem, A a, B b) {
    constexpr uint32_t one = bf16_idesc(N, A::kAcross, B::kAcross), two = bf16_idesc(2 * N, A::kAcross, B::kAcross), three = bf16_idesc(3 * N, A::kAcross, B::kAcross);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) umma_bf16(tmem, a(2, s), b(0, s), one, s != 0);
    umma_bf16(tmem, a(1, 0), b(0, 0), one, 1);
    umma_bf16(tmem + N, a(1, 0), b(1, 0), one, 0);
#pragma unroll
    for (int s = 1; s < STEPS; ++s) umma_bf16(tmem, a(1, s), b(0, s), two, 1);
    umma_bf16(tmem, a(0, 0), b(0, 0), two, 1);
    umma_bf16(tmem + 2 * N, a(0, 0), b(2, 0), one, 0);
#pragma unroll
    for (int s = 1; s < STEPS; ++s) umma_bf16(tmem, a(0, s), b(0, s), three, 1);
}
// the same one plane product after the other, all into the same N columns
template <int N, int STEPS, class A, class B>
__device__ __forceinline__ void issue_in_turn(uint32_t tmem, A a, B b) {
#pragma unroll
    for (int i = 0; i < 6; ++i)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) umma_bf16(tmem, a(plane_a(i), s), b(plane_b(i), s), bf16_idesc(N, A::kAcross, B::kAcross), (i | s) != 0);
}

// sum of BLOCKS blocks of columns, STEP apart
template <int N, int BLOCKS, int STEP>
__device__ __forceinline__ void tmem_sum(uint32_t taddr, float (&v)[N]) {
    uint32_t r[BLOCKS][N];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) tmem_request<N>(taddr + b * STEP, r[b]);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) tmem_wait<N>(r[b]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = __uint_as_float(r[0][i]);
#pragma unroll
        for (int b = 1; b < BLOCKS; ++b) v[i] += __uint_as_float(r[b][i]);
    }
}
__device__ __forceinline__ float reciprocal(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }

template <int KP>
struct Fuse {
    static constexpr int MC = fuse_instances(KP), KR = KP / 4, MR = MC / 4;     // a worker's taps and instances
    static constexpr bool kByTaps = KP > 64;             // the offsets' sums with the taps as rows (128 of them), else with the instances
    using X = Planes<128, KP>;
    using Q = Planes<128, MC>;
    using E = Planes<MC, KP>;
    // tensor memory: S (where there is room twice, so that the next step's is made while this one's quotients are), the sums over the instances
    // (128 taps: one block of columns, three do not fit), the offsets' sums
    static constexpr bool kTwice = KP <= 32;
    static constexpr int kTapBlocks = KP > 64 ? 1 : 3, kT = kTwice ? 2 * MC : MC, kU = kT + kTapBlocks * KP;
    static constexpr int kUBlock = kByTaps ? MC : KP;
    static_assert(kU + 3 * kUBlock <= kFuseColumns);
};

template <int KP>
__global__ void __launch_bounds__(kFuseThreads, 1) mex_gradients_at_checkpoint(MexGeo g, FuseArgs a) {
    stream_order();
    using F = Fuse<KP>;
    using X = typename F::X;
    using Q = typename F::Q;
    using E = typename F::E;
    constexpr int MC = F::MC, KR = F::KR, MR = F::MR;
    extern __shared__ __align__(1024) unsigned char sm[];
    __shared__ FuseShared sh;
    __shared__ float red[2][4][128];
    __shared__ longlong2 place_s[2][128];
    __shared__ __align__(16) int tap_off[KP];
    if (term_by_term(a)) return;
    unsigned char *const sx = sm, *const sq = sm + X::kBytes, *const se = sq + Q::kBytes;
    const int warp = threadIdx.x >> 5;
    const int r = int(blockIdx.x) % g.R, slot = int(blockIdx.x) / g.R, slots = int(gridDim.x) / g.R;
    for (int k = threadIdx.x; k < KP; k += kFuseThreads) {
        const Tap t = tap_of<false>(g, k < g.K ? k : 0);
        tap_off[k] = (t.c * g.H + t.h) * g.W + t.w;
    }
    if (threadIdx.x == 0) {
        mbar_init(&sh.operands, kFuseWorkers / 32); mbar_init(&sh.quotients, kFuseWorkers / 32);
        mbar_init(&sh.sums[0], 1); mbar_init(&sh.sums[1], 1); mbar_init(&sh.taps, 1); mbar_init(&sh.instances, 1); mbar_init(&sh.drained, 1);
        sh.failed = sh.beyond = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kFuseWorkers / 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(uint32_t(kFuseColumns)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sh.tmem;
    const uint32_t tS = tmem, tT = tmem + F::kT, tU = tmem + F::kU;
    const uint32_t xb = smem_u32(sx), qb = smem_u32(sq), eb = smem_u32(se);
    const bool ahead = F::kTwice && a.resident;
    uint32_t phase = 0;                                                                  // of the barriers that complete once a step
    // A wait that runs out sets `failed`; from then on nobody waits and no product is issued, and all leave by the ordinary way.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!sh.failed && !(a.expire ? mbar_wait_briefly(bar, parity) : mbar_wait(bar, parity))) sh.failed = 1;
        __syncwarp();                                                                    // (what follows is done by whole warps)
    };
    // (one arrival a warp: those of 512 threads follow one another)
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
    };

    if (warp == kFuseWorkers / 32) {
        const Operand<X, false> x_along(xb);
        const Operand<X, true> x_across(xb);
        const Operand<Q, false> q_along(qb);
        const Operand<Q, true> q_across(qb);
        auto issue_sums = [&](int mt) {
            const Operand<E, false> e_along(eb + (a.resident ? mt * E::kBytes : 0u));
            const int to = ahead ? mt & 1 : 0;
            if (!sh.failed && !a.expire && elected()) {
                issue_in_turn<MC, KP / 16>(tS + to * MC, x_along, e_along);
                umma_commit(&sh.sums[to]);
            }
            __syncwarp();
        };
        uint32_t there = 0;
        for (long long jt = slot; jt < a.tiles_j; jt += slots)
            for (int mt = 0; mt < a.tiles_m; ++mt, phase ^= 1u) {
                if (!ahead || mt == 0) {
                    wait(&sh.operands, there);
                    there ^= 1u;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    issue_sums(mt);
                    if (ahead && a.tiles_m > 1) issue_sums(1);
                }
                wait(&sh.quotients, phase);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const Operand<E, true> e_across(eb + (a.resident ? mt * E::kBytes : 0u));
                if (!sh.failed && elected()) {
                    if (a.dx) {
                        if constexpr (F::kTapBlocks == 3) issue_side_by_side<KP, MC / 16>(tT, q_along, e_across);
                        else issue_in_turn<KP, MC / 16>(tT, q_along, e_across);
                    }
                    umma_commit(&sh.taps);
                    if (a.part) {
                        if constexpr (F::kByTaps) issue_side_by_side<MC, 8>(tU, x_across, q_across);
                        else issue_side_by_side<KP, 8>(tU, q_across, x_across);
                    }
                    umma_commit(&sh.instances);
                }
                __syncwarp();
                if (ahead && mt + 2 < a.tiles_m) issue_sums(mt + 2);                     // (into the place of the S that has been read)
            }
        if (sh.failed) {                                                                 // tensor memory must not be freed under a product
            if (elected()) umma_commit(&sh.drained);
            __syncwarp();
            mbar_wait(&sh.drained, 0);
        }
    } else {
        const int p = threadIdx.x & 127, part4 = threadIdx.x >> 7;                      // position (tensor-memory lane) and its quarter of the columns
        const uint32_t lane_base = uint32_t(warp & 3) << 21;                             // (32 lanes a warp, lane number in bits 16 and up)
        const int Mp = a.tiles_m * MC, k0 = part4 * KR;
        const float eps = float(g.eps), a2 = eps * 1.4426950408889634f;
        const long long P = (long long)g.B * g.rs;
        auto load_offsets = [&](int mt, unsigned char* to) {
            const unsigned char* src = a.tiles + ((size_t)r * a.tiles_m + mt) * E::kBytes;
            for (int i = threadIdx.x; i < int(E::kBytes / 16); i += kFuseWorkers) cp_async16(reinterpret_cast<float*>(to + i * 16), reinterpret_cast<const float*>(src + i * 16), 16);
        };
        // Where the positions of a tile lie, by the first quarter of the workers: first tap in the input (-1: a position that is not there), first
        // instance in dy.  Their bytes are asked for by the way, a tap a worker: a line has several positions.
        int turn = 0;
        auto find_places = [&](long long jt) {
            if (part4 != 0) return;
            const Column col = column_of(g, r, jt * 128 + p, P, nullptr);
            longlong2 at = make_longlong2(-1, 0);
            if (col.base >= 0) {
                at = make_longlong2((((long long)col.n * g.C + col.c0) * g.H + col.h0) * g.W + col.w0, col.gbase);
#pragma unroll
                for (int k = 0; k < KP; k += 16) {
                    const long long idx = at.x + tap_off[k + (p & 15)];
                    asm volatile("prefetch.global.L1 [%0];" ::"l"(a.codes + idx));
                    asm volatile("prefetch.global.L1 [%0];" ::"l"(a.ranges + (idx >> a.shift)));
                }
            }
            place_s[turn][p] = at;
        };
        // Ex of this worker's taps (k0 .. + KR) of its position of the tile that find_places() was called for.  Taps that are not there read the first
        // one's value and count 0; a position that is not there has a 1 in its first tap, so that its S is no 0.
        struct Place { long long x, dy; bool live; };
        auto decode = [&](float (&ex)[KR]) {
            constexpr int H = KR < 16 ? KR : 16;
            asm volatile("bar.sync 1, %0;" ::"n"(kFuseWorkers) : "memory");
            const longlong2 found = place_s[turn][p];
            const Place at = {found.x < 0 ? 0 : found.x, found.y, found.x >= 0};
            const unsigned char* const codes = a.codes + at.x;
            const float2* const ranges = a.ranges + (at.x >> a.shift);
            const int rest = int(at.x) & ((1 << a.shift) - 1);
            float mx = eps > 0.f ? -CUDART_INF_F : CUDART_INF_F;
#pragma unroll
            for (int i0 = 0; i0 < KR; i0 += H) {
                uint32_t code[H], top = 0;
                float2 range[H];
#pragma unroll
                for (int i = 0; i < H; i += 4) {
                    const int4 t4 = *reinterpret_cast<const int4*>(tap_off + k0 + i0 + i);
                    const int tap[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        code[i + u] = __ldg(codes + tap[u]);
                        range[i + u] = __ldg(ranges + ((unsigned(rest) + unsigned(tap[u])) >> a.shift));
                    }
                }
#pragma unroll
                for (int i = 0; i < H; ++i) top = max(top, code[i]);
                if (__any_sync(0xffffffffu, top > 252u)) {
#pragma unroll
                    for (int i = 0; i < H; ++i) ex[i0 + i] = unpacked<float>(code[i], range[i].x, range[i].y);
                } else {
#pragma unroll
                    for (int i = 0; i < H; ++i) ex[i0 + i] = Limits<float>::at(float(code[i]), range[i].y, range[i].x);
                }
#pragma unroll
                for (int i = 0; i < H; ++i) mx = eps > 0.f ? fmaxf(mx, ex[i0 + i]) : fminf(mx, ex[i0 + i]);
            }
            red[turn][part4][p] = mx;                                                    // (two turns: nobody still reads this one's)
            asm volatile("bar.sync 1, %0;" ::"n"(kFuseWorkers) : "memory");
            const float m0 = red[turn][0][p], m1 = red[turn][1][p], m2 = red[turn][2][p], m3 = red[turn][3][p];
            turn ^= 1;
            mx = eps > 0.f ? fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) : fminf(fminf(m0, m1), fminf(m2, m3));
#pragma unroll
            for (int i = 0; i < KR; ++i) ex[i] = ex2_ftz(a2 * (ex[i] - mx));
            if (k0 + KR > g.K)
#pragma unroll
                for (int i = 0; i < KR; ++i) ex[i] = k0 + i < g.K ? ex[i] : 0.f;
            if (!at.live)
#pragma unroll
                for (int i = 0; i < KR; ++i) ex[i] = k0 + i == 0 ? 1.f : 0.f;
            return at;
        };
        // dy of this worker's instances (a quarter of a step's) of its position
        float q[MR];
        auto load_dy = [&](const Place& at, int mt) {
            const int m0 = mt * MC + part4 * MR;
            const float* from = a.dy + at.dy + (long long)m0 * g.Ng;
            if (m0 + MR <= g.M)
#pragma unroll
                for (int i = 0; i < MR; ++i, from += g.Ng) q[i] = at.live ? __ldcs(from) : 0.f;
            else
#pragma unroll
                for (int i = 0; i < MR; ++i, from += g.Ng) q[i] = at.live && m0 + i < g.M ? __ldcs(from) : 0.f;
        };
        // the offsets' sums of a step onto the CTA's
        auto add_offsets = [&](int mt, bool first) {
            if (!a.part) return;
            float* const to = a.part + ((size_t)blockIdx.x * Mp + mt * MC) * KP;
            if constexpr (F::kByTaps) {                                                  // row = tap p, columns = instances
                float* const d = to + part4 * MR * KP + p;
#pragma unroll
                for (int i0 = 0; i0 < MR; i0 += 8) {
                    float old[8], u[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) old[i] = first ? 0.f : d[(i0 + i) * KP];
                    tmem_sum<8, 3, MC>(tU + lane_base + part4 * MR + i0, u);
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[(i0 + i) * KP] = old[i] + u[i];
                }
            } else {                                                                     // row = instance p, columns = taps
                constexpr int H = KR < 8 ? KR : 8;
                float4* const d = reinterpret_cast<float4*>(to) + (k0 / 4) * MC + p;
#pragma unroll
                for (int i0 = 0; i0 < KR; i0 += H) {
                    float4 old[H / 4];
                    float u[H];
#pragma unroll
                    for (int i = 0; i < H / 4; ++i) old[i] = first ? make_float4(0.f, 0.f, 0.f, 0.f) : d[(i0 / 4 + i) * MC];
                    tmem_sum<H, 3, KP>(tU + lane_base + k0 + i0, u);
#pragma unroll
                    for (int i = 0; i < H / 4; ++i)
                        d[(i0 / 4 + i) * MC] = make_float4(old[i].x + u[4 * i], old[i].y + u[4 * i + 1], old[i].z + u[4 * i + 2], old[i].w + u[4 * i + 3]);
                }
            }
        };

        if (a.resident) for (int mt = 0; mt < a.tiles_m; ++mt) load_offsets(mt, se + mt * E::kBytes);
        float ex[KR];
        find_places(slot);
        Place at = decode(ex);
        if (ahead) load_dy(at, 0);
        uint32_t sum_phase[2] = {0, 0};
        bool due = false;                                                                // the offsets' sums of the step before are to be added
        for (long long jt = slot; jt < a.tiles_j; jt += slots) {
            store_row<X>(sx, p, k0, ex);
            float tsum[KR];
#pragma unroll
            for (int i = 0; i < KR; ++i) tsum[i] = 0.f;
            const bool last_tile = jt + slots >= a.tiles_j, first = jt == slot;
            Place next = at;
            for (int mt = 0; mt < a.tiles_m; ++mt, phase ^= 1u) {
                if (!a.resident) load_offsets(mt, se);
                if (!ahead || mt == 0) {
                    cp_async_wait_all();
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    arrive(&sh.operands);
                }
                // (while the first product runs)
                if (!ahead) load_dy(at, mt);
                if (due) add_offsets(mt == 0 ? a.tiles_m - 1 : mt - 1, mt == 0 ? jt - slots == slot : first);
                due = true;
                const bool last = mt + 1 == a.tiles_m;
                if (last && !last_tile) find_places(jt + slots);
                const int from = ahead ? mt & 1 : 0;
                wait(&sh.sums[from], from ? sum_phase[1] : sum_phase[0]);
                if (from) sum_phase[1] ^= 1u; else sum_phase[0] ^= 1u;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t squares = 0;
#pragma unroll
                for (int i0 = 0; i0 < MR; i0 += 16) {
                    float s[16];
                    tmem_sum<16, 1, 0>(tS + from * MC + lane_base + part4 * MR + i0, s);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = q[i0 + i] * reciprocal(s[i]);
                    store_row<Q>(sq, p, part4 * MR + i0, s, squares);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                arrive(&sh.quotients);
                if ((squares & 0x7f80u) == 0x7f80u || (squares & 0x7f800000u) == 0x7f800000u)            // a NaN or a quotient above 2^64
                    for (int m = part4 * MR; m < (part4 + 1) * MR; ++m)
                        if (fabsf(__uint_as_float(uint32_t(*reinterpret_cast<const unsigned short*>(sq + Q::at(p, m))) << 16)) >= kMostQuotient) sh.beyond = 1;
                // (while the second product runs)
                if (last && !last_tile) next = decode(ex);
                if (ahead && !(last && last_tile)) load_dy(last ? next : at, last ? 0 : mt + 1);
                wait(&sh.taps, phase);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (a.dx) {
                    constexpr int H = KR < 16 ? KR : 16;
#pragma unroll
                    for (int i0 = 0; i0 < KR; i0 += H) {
                        float t[H];
                        tmem_sum<H, F::kTapBlocks, KP>(tT + lane_base + k0 + i0, t);
#pragma unroll
                        for (int i = 0; i < H; ++i) tsum[i0 + i] += t[i];
                    }
                    if (last && at.live) {                                               // (while the third runs) Ex from its planes, which add up to it
                        float* const dx = a.dx + at.x;
#pragma unroll
                        for (int i = 0; i < KR; i += 4) {
                            const int4 tap = *reinterpret_cast<const int4*>(tap_off + k0 + i);
                            uint2 w[3];
#pragma unroll
                            for (int b = 0; b < 3; ++b) w[b] = *reinterpret_cast<const uint2*>(sx + X::at(p, k0 + i) + b * X::kPlane);
                            auto low = [](uint32_t v) { return __uint_as_float(v << 16); };
                            auto high = [](uint32_t v) { return __uint_as_float(v & 0xffff0000u); };
                            const float e0 = (low(w[0].x) + low(w[1].x)) + low(w[2].x), e1 = (high(w[0].x) + high(w[1].x)) + high(w[2].x);
                            const float e2 = (low(w[0].y) + low(w[1].y)) + low(w[2].y), e3 = (high(w[0].y) + high(w[1].y)) + high(w[2].y);
                            if (k0 + i < g.K) dx[tap.x] = e0 * tsum[i];
                            if (k0 + i + 1 < g.K) dx[tap.y] = e1 * tsum[i + 1];
                            if (k0 + i + 2 < g.K) dx[tap.z] = e2 * tsum[i + 2];
                            if (k0 + i + 3 < g.K) dx[tap.w] = e3 * tsum[i + 3];
                        }
                    }
                }
                wait(&sh.instances, phase);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            at = next;
        }
        if (due) add_offsets(a.tiles_m - 1, a.tiles_j - slot <= slots);
        cp_async_wait_all();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kFuseWorkers / 32)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(kFuseColumns)) : "memory");
    if (sh.failed && threadIdx.x == 0) atomicExch(&a.status[1], 1);                      // a wait ran out: the kernel behind redoes the call
    if (sh.beyond && threadIdx.x == 0) atomicExch(&a.status[2 + a.rows], 1);             // the kernel behind redoes what is no number
}

// ---- the offsets' gradient from the CTAs' sums, or, for offsets that no factorisation takes, everything term by term ------------------
struct FinishArgs {
    const float *off, *eo;
    float* doff;            // may be null
    int KP, MC, Mp, ctas;
    int normalized, accumulate;
};
constexpr int kFinishThreads = 256;

// doff of one row from d, its gradient with respect to the row as the op sees it (thread k has tap k): of a raw row d - softmax(row) sum(d).
// All threads of the CTA call it; `work`: three arrays of 128.
__device__ __forceinline__ void finish_row(const MexGeo& g, const FinishArgs& f, int row, float d, float (*work)[128]) {
    const int k = threadIdx.x;
    const float* o = f.off + (size_t)row * g.K;
    if (f.normalized) {
        __syncthreads();
        if (k < 128) { work[0][k] = k < g.K ? o[k] : -CUDART_INF_F; work[1][k] = k < g.K ? d : 0.f; }
        __syncthreads();
        if (k < 32) {
            float hi = fmaxf(fmaxf(work[0][k], work[0][k + 32]), fmaxf(work[0][k + 64], work[0][k + 96]));
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
            float e = 0.f, t = 0.f;
#pragma unroll
            for (int i = 0; i < 128; i += 32) { e += expf(work[0][k + i] - hi); t += work[1][k + i]; }
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) { e += __shfl_xor_sync(0xffffffffu, e, s); t += __shfl_xor_sync(0xffffffffu, t, s); }
            if (k == 0) { work[2][0] = hi; work[2][1] = e; work[2][2] = t; }
        }
        __syncthreads();
        if (k < g.K) d -= expf(work[0][k] - work[2][0]) / work[2][1] * work[2][2];
    }
    if (k < g.K) {
        float* to = f.doff + (size_t)row * g.K + k;
        *to = f.accumulate ? *to + d : d;
    }
}

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

// dx: a warp per position of any region; `some`: only of the patches whose dx is no number
__device__ __forceinline__ void redo_dx(const MexGeo& g, const FuseArgs& a, const float* __restrict__ off, bool some) {
    constexpr int W = kFinishThreads / 32;
    const long long P = (long long)g.B * g.N;
    for (long long j = (long long)blockIdx.x * W + (threadIdx.x >> 5); j < P; j += (long long)gridDim.x * W) {
        const int n = int(j / g.N), pos = int(j - (long long)n * g.N), w = pos % g.Wo, h = pos / g.Wo % g.Ho, c = pos / (g.Wo * g.Ho), r = mex_region_of(g, c, h, w);
        const long long xi = (((long long)n * g.C + c * g.sc) * g.H + h * g.sh) * g.W + w * g.sw, at = mex_dy_base(g, n, pos);
        if (some) {
            bool bad = false;
            for (int k = threadIdx.x & 31; k < g.K; k += 32) {
                const Tap tap = tap_of<false>(g, k);
                bad = bad || !(fabsf(a.dx[xi + ((long long)tap.c * g.H + tap.h) * g.W + tap.w]) < CUDART_INF_F);
            }
            if (!__any_sync(0xffffffffu, bad)) continue;
        }
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

// doff of one row by a whole CTA, its warps over the positions; thread k has tap k's
__device__ __forceinline__ double redo_row(const MexGeo& g, const FuseArgs& a, const float* __restrict__ off, int row, double (*sums)[128]) {
    constexpr int W = kFinishThreads / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = row / g.M, m = row % g.M;
    const long long P = (long long)g.B * g.rs;
    double sum[4] = {0, 0, 0, 0};
    for (long long j = warp; j < P; j += W) {
        const Column col = column_of(g, r, j, P, nullptr);
        if (col.base < 0) continue;
        const long long xi = (((long long)col.n * g.C + col.c0) * g.H + col.h0) * g.W + col.w0;
        const Taps4 p = patch_weights(g, checkpoint_patch(g, a, xi), off + (size_t)row * g.K);
        const float v = a.dy[col.gbase + (long long)m * g.Ng];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += v * p.v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[warp][lane + 32 * i] = sum[i];
    __syncthreads();
    double t = 0;
    if (threadIdx.x < 128)
        for (int w = 0; w < W; ++w) t += sums[w][threadIdx.x];
    return t;
}

__global__ void __launch_bounds__(kFinishThreads, 4) fuse_finish(MexGeo g, FuseArgs a, FinishArgs f) {
    stream_order();
    __shared__ double sums[kFinishThreads / 32][128];
    __shared__ float work[3][128];
    const bool redo = term_by_term(a);
    if (blockIdx.x == 0) {
        int unsafe = 0;
        for (int i = threadIdx.x; i < a.rows; i += kFinishThreads) unsafe |= a.status[2 + i];
        unsafe = __syncthreads_or(unsafe);
        if (threadIdx.x == 0) a.status[0] = unsafe != 0;
    }
    const bool some = !redo && a.status[2 + a.rows] != 0;
    if (a.dx && (redo || some)) redo_dx(g, a, f.off, some);
    if (!f.doff) return;
    // the CTAs' sums in their order, in two halves
    float* const half_sum = reinterpret_cast<float*>(sums);
    const int k = threadIdx.x & 127, half = threadIdx.x >> 7;
    for (int row = blockIdx.x; row < g.R * g.M; row += gridDim.x) {
        float d = 0.f;
        if (!redo) {
            const int r = row / g.M, m = row % g.M;
            float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
            if (k < g.K) {
                const size_t step = (size_t)g.R * f.Mp * f.KP;
                const int slots = f.ctas / g.R, from = half * ((slots + 1) / 2), to = half ? slots : (slots + 1) / 2;
                const float* s = a.part + ((size_t)r * f.Mp + m / f.MC * f.MC) * f.KP + part_at(f.KP, f.MC, m % f.MC, k) + from * step;
                int c = from;
                for (; c + 3 < to; c += 4, s += 4 * step) { s0 += s[0]; s1 += s[step]; s2 += s[2 * step]; s3 += s[3 * step]; }
                for (; c < to; ++c, s += step) s0 += s[0];
            }
            const float mine = (s0 + s1) + (s2 + s3);
            __syncthreads();
            if (half) half_sum[k] = mine;
            __syncthreads();
            if (threadIdx.x < 128 && k < g.K) d = f.eo[((size_t)r * g.M + m) * f.KP + k] * (mine + half_sum[k]);
        }
        if (redo || (some && __syncthreads_or(!(fabsf(d) < CUDART_INF_F)))) d = float(redo_row(g, a, f.off, row, sums));
        finish_row(g, f, row, d, work);
    }
}

struct FuseWs { int* status; float *eo, *part; unsigned char* tiles; size_t bytes; };

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
    w.status = reinterpret_cast<int*>(take(sizeof(int) * (3 + (size_t)g.R * z.Mp)));
    w.eo = reinterpret_cast<float*>(take(sizeof(float) * (size_t)g.R * g.M * z.KP));
    w.tiles = reinterpret_cast<unsigned char*>(take((size_t)g.R * z.Mp * z.KP * 6));
    w.part = reinterpret_cast<float*>(take(sizeof(float) * (size_t)z.slots * g.R * z.Mp * z.KP));
    w.bytes = off;
    return w;
}

constexpr int kFuseShared = 217 * 1024;     // (of 227 KB; the barriers, the extremes, the places and the tap offsets are some 9)

// steps of instances whose Eo stays in shared memory beside Ex and Q
int fuse_resident(int KP) {
    const int MC = fuse_instances(KP);
    return (kFuseShared - 128 * (KP + MC) * 6) / (MC * KP * 6);
}

template <int KP>
cudaError_t launch_fused(const MexGeo& g, const FuseArgs& a, int ctas, cudaStream_t s) {
    static SmemLimit limit;
    const cudaError_t e = limit.raise(mex_gradients_at_checkpoint<KP>, kFuseShared);
    if (e != cudaSuccess) return e;
    using F = Fuse<KP>;
    const size_t smem = F::X::kBytes + F::Q::kBytes + (size_t)F::E::kBytes * (a.resident ? a.tiles_m : 1);
    in_stream_order(mex_gradients_at_checkpoint<KP>, ctas, kFuseThreads, smem, s)(g, a);
    return cudaSuccess;
}

}  // namespace

// Blocks that cover the input once, in few regions (a CTA works for one).
bool mex_checkpoint_shape(const MexGeo& g, bool f64, uint32_t flags) {
    // (a larger epsilon times log2 e is no float any more)
    if (f64 || !g.finite || std::fabs(g.eps) > 1e30 || g.B == 0 || g.K > 128 || (flags & (SIMNETS_FLAG_FORCE_DIRECT | SIMNETS_FLAG_MEX_EXACT | SIMNETS_FLAG_MEX_NO_TENSORCORE))) return false;
    const bool cover = g.sc == g.bc && g.sh == g.bh && g.sw == g.bw && g.pc == 0 && g.ph == 0 && g.pw == 0 && g.Co * g.bc == g.C && g.Ho * g.bh == g.H && g.Wo * g.bw == g.W;
    return cover && g.R <= 16 && g.M <= 8192 && (long long)g.C * g.H * g.W < (1LL << 31) && (long long)g.B * g.rs < (1LL << 38);
}
size_t mex_checkpoint_bytes(const MexGeo& g) { return fuse_carve(g, nullptr).bytes; }

cudaError_t launch_mex_checkpoint(const MexGeo& g, int group, const void* codes, const void* ranges, const float* off, const float* dy, float* dx, float* doff,
                                  bool accumulate, bool normalized, bool expire, void* ws, cudaStream_t s) {
    const FuseSizes z = fuse_sizes(g);
    const FuseWs w = fuse_carve(g, ws);
    FuseArgs a;
    a.codes = static_cast<const unsigned char*>(codes);
    a.ranges = static_cast<const float2*>(ranges);
    a.tiles = w.tiles;
    a.dy = dy; a.dx = dx; a.part = doff ? w.part : nullptr;
    a.status = w.status;
    a.rows = g.R * z.Mp;
    a.expire = expire;
    a.shift = 5;
    while ((1 << a.shift) < group) ++a.shift;
    a.tiles_m = z.Mp / z.MC;
    a.resident = a.tiles_m <= fuse_resident(z.KP);
    a.tiles_j = ((long long)g.B * g.rs + 127) / 128;
    in_stream_order(fuse_prepare, g.R * z.Mp, 128, 0, s)(g, z.KP, z.MC, z.Mp, off, w.eo, w.tiles, w.status);
    const int ctas = z.slots * g.R;
    const cudaError_t e = z.KP == 16 ? launch_fused<16>(g, a, ctas, s) : z.KP == 32 ? launch_fused<32>(g, a, ctas, s) : z.KP == 64 ? launch_fused<64>(g, a, ctas, s) : launch_fused<128>(g, a, ctas, s);
    if (e != cudaSuccess) return e;
    const FinishArgs f = {off, w.eo, doff, z.KP, z.MC, z.Mp, ctas, int(normalized), int(accumulate)};
    in_stream_order(fuse_finish, std::min(std::max(g.R * g.M, device_sm_count()), 4 * device_sm_count()), kFinishThreads, 0, s)(g, a, f);
    count_launch(3);
    return cudaGetLastError();
}

}  // namespace simnets

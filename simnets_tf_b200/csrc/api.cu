// C ABI of the library (include/simnets_b200.h): validates descriptors, picks a kernel family and
// enqueues it on the caller's stream.  No entry point here allocates, frees or synchronises.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <limits>
#include "simnets_b200.h"
#include "host_dims.hpp"
#include "kernels.cuh"

namespace simnets {
static std::atomic<uint64_t> g_launches{0};
void count_launch(int n) { g_launches.fetch_add(uint64_t(n), std::memory_order_relaxed); }
int device_sm_count() {
    static std::atomic<int> sms[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    int n = sms[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        sms[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}
}  // namespace simnets

using namespace simnets;

namespace {
inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }
inline int from_cuda(cudaError_t e) { return e == cudaSuccess ? SIMNETS_OK : int(e); }

// The MEX gradients that have a place to go (an empty batch may come without tensors of its size).
int mex_gradients(const MexGeo& g, const simnets_mex_desc* d, const void* x, const void* off, const void* y, const void* dy, void* dx, void* doff,
                  void* ws, size_t ws_bytes, void* products, size_t products_bytes, cudaStream_t s) {
    const bool f64 = d->dtype == SIMNETS_F64, acc = (d->flags & SIMNETS_FLAG_ACCUMULATE) != 0;
    const bool alone = mex_gradients_by_gemm(g, f64, d->flags), gemm = alone || mex_use_gemm(g, f64, d->flags), tiled = !gemm && mex_use_tiled(g, f64, d->flags);
    if ((d->flags & SIMNETS_FLAG_MEX_NORMALIZED_OFFSETS) && g.B > 0 && !gemm && !tiled) return SIMNETS_E_UNSUPPORTED;
    if (gemm || tiled) {
        if (!ws || ws_bytes < (gemm ? mex_gemm_workspace_bytes(g, f64) : mex_workspace_bytes(g, f64, d->flags))) return SIMNETS_E_WORKSPACE;
        const size_t need = dx ? mex_products_bytes(g, f64, d->flags) : 0;
        if (need > 0 && (!products || products_bytes < need)) return SIMNETS_E_WORKSPACE;
    }
    const uint32_t unprimed = ~uint32_t(alone ? SIMNETS_FLAG_MEX_WORKSPACE_PRIMED | SIMNETS_FLAG_MEX_MAXIMA_GIVEN : 0);
    if (gemm) return from_cuda(launch_mex_bwd_gemm(g, f64, x, off, y, dy, dx, doff, acc, ws, products, d->flags & unprimed, s));
    if (tiled) {
        const float *xf = (const float*)x, *of = (const float*)off, *yf = (const float*)y, *dyf = (const float*)dy;
        if (dx && doff) return from_cuda(launch_mex_backward_tiled(g, xf, of, yf, dyf, (float*)dx, (float*)doff, acc, ws, products, d->flags, s));
        return from_cuda(dx ? launch_mex_dx_tiled(g, xf, of, yf, dyf, (float*)dx, ws, products, d->flags, s)
                            : launch_mex_doff_tiled(g, xf, of, yf, dyf, (float*)doff, acc, ws, d->flags, s));
    }
    cudaError_t e = dx ? launch_mex_dx_direct(g, f64, x, off, y, dy, dx, s) : cudaSuccess;
    if (e == cudaSuccess && doff) e = launch_mex_doff_direct(g, f64, x, off, y, dy, doff, acc, s);
    return from_cuda(e);
}

// the same with the products at the end of one workspace
int mex_gradients_in(const MexGeo& g, const simnets_mex_desc* d, const void* x, const void* off, const void* y, const void* dy, void* dx, void* doff,
                     void* ws, size_t ws_bytes, cudaStream_t s) {
    const bool f64 = d->dtype == SIMNETS_F64;
    const size_t kept = mex_use_gemm(g, f64, d->flags) ? mex_gemm_workspace_bytes(g, f64) : mex_workspace_bytes(g, f64, d->flags);
    const bool more = ws && ws_bytes > kept;
    return mex_gradients(g, d, x, off, y, dy, dx, doff, ws, ws_bytes, more ? static_cast<char*>(ws) + kept : nullptr, more ? ws_bytes - kept : 0, s);
}

// ---- 8-bit checkpoints and routing
int checkpoint_check(int32_t dtype, int64_t count, int32_t group) {
    if (dtype != SIMNETS_F32 && dtype != SIMNETS_F64) return SIMNETS_E_DTYPE;
    return count < 0 || (group != 32 && group != 64 && group != 128 && group != 256) ? SIMNETS_E_DESC : SIMNETS_OK;
}

// Sums in FP32: the tensor-core kernels truncate what they add, and here y goes through them as well (a 64-tap layer of 128 instances over
// 524288 positions: gradients 1.2e-5 of their norm off, with FP32 sums 1.3e-6).
uint32_t checkpoint_route(const MexGeo& g, const simnets_mex_desc& d) {
    const bool f64 = d.dtype == SIMNETS_F64;
    if (d.flags & SIMNETS_FLAG_MEX_CHECKPOINT_TENSORCORE) return 0u;
    return mex_use_gemm(g, f64, d.flags) || mex_gradients_by_gemm(g, f64, d.flags) ? 0u : uint32_t(SIMNETS_FLAG_MEX_NO_TENSORCORE);
}

// the values of the checkpoint, y again from them, the layer's workspace, the products of overlapping blocks
struct MexCheckpointWs { void *x, *y, *layer, *products; size_t layer_bytes, products_bytes, bytes; };
MexCheckpointWs mex_checkpoint_carve(const MexGeo& g, const simnets_mex_desc& d, void* base) {
    MexCheckpointWs w;
    const size_t size = d.dtype == SIMNETS_F64 ? 8 : 4;
    size_t off = 0;
    auto take = [&](size_t bytes) { void* p = base ? static_cast<char*>(base) + off : nullptr; off += (bytes + 255) & ~size_t(255); return p; };
    simnets_mex_desc f = d, q = d;
    f.flags = (f.flags | checkpoint_route(g, d)) & ~uint32_t(SIMNETS_FLAG_MEX_DY_POOLED2);
    q.flags |= checkpoint_route(g, d);
    w.x = take(size * g.B * g.C * g.H * g.W);
    w.y = take(size * g.B * g.M * g.N);
    w.layer_bytes = std::max<size_t>(std::max(simnets_mex_forward_workspace_bytes(&f), simnets_mex_forward_workspace_bytes(&q)), 256);
    w.layer = take(w.layer_bytes);
    w.products_bytes = simnets_mex_products_bytes(&q);
    w.products = take(w.products_bytes);
    w.bytes = off;
    return w;
}

size_t sim_checkpoint_values(const SimGeo& g, const simnets_sim_desc& d) {
    return ((d.dtype == SIMNETS_F64 ? 8 : 4) * (size_t)g.B * g.C * g.H * g.W + 255) & ~size_t(255);
}

int route_check(const simnets_route_desc* d) {
    if (!d) return SIMNETS_E_NULL;
    if (d->dtype != SIMNETS_F32 && d->dtype != SIMNETS_F64) return SIMNETS_E_DTYPE;
    if (d->batch < 0 || d->positions < 0 || d->components < 1 || d->top_k < 1 || d->groups < 1 || d->top_groups < 1 || d->reserved != 0) return SIMNETS_E_DESC;
    if (d->components % d->groups || d->top_groups > d->groups || d->top_k > (long long)d->top_groups * (d->components / d->groups)) return SIMNETS_E_DESC;
    // (a normal number of the weights' type, so that it and its reciprocal are numbers there)
    const bool f64 = d->dtype == SIMNETS_F64;
    const double most = f64 ? std::numeric_limits<double>::max() : std::numeric_limits<float>::max(), least = f64 ? std::numeric_limits<double>::min() : std::numeric_limits<float>::min();
    if (!(std::fabs(d->scale) >= least && std::fabs(d->scale) <= most)) return SIMNETS_E_DESC;
    const bool all = d->top_groups == d->groups;        // (then there is no choice of groups)
    if (d->components > 4096 || d->top_k > 16 || (!all && (d->groups > 64 || d->top_groups > 16))) return SIMNETS_E_UNSUPPORTED;
    // (a load is counted in 32 bits by every CTA)
    return d->batch > 0 && d->positions > ((1LL << 40) / d->batch) ? SIMNETS_E_UNSUPPORTED : SIMNETS_OK;
}

// ---- log probabilities, norms of gradients
int likelihood_check(const simnets_likelihood_desc* d) {
    if (!d) return SIMNETS_E_NULL;
    if (d->dtype != SIMNETS_F32 && d->dtype != SIMNETS_F64) return SIMNETS_E_DTYPE;
    if (d->classes < 1 || d->batch < 0 || d->positions < 0 || d->top_k < 0 || d->top_k > d->classes || d->stride_batch < 0 || d->stride_class < 0 || d->stride_position < 0)
        return SIMNETS_E_DESC;
    // (classes are counted in 32 bits, CTAs of positions as well: eight positions each at least, or 4096 classes)
    if (d->top_k > 16 || d->classes > (1 << 30) || (d->batch > 0 && d->positions > std::min(1LL << 33, (1LL << 43) / d->classes) / d->batch)) return SIMNETS_E_UNSUPPORTED;
    return SIMNETS_OK;
}

// whether a place cannot hold values of the type, or whole numbers and workspaces of 64 bits
bool misplaced(const void* p, int32_t dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == SIMNETS_F64 ? 8 : 4) != 0; }
bool misplaced64(const void* p) { return reinterpret_cast<uintptr_t>(p) % 8 != 0; }

int gradients_check(int32_t order, int32_t tensors, const int32_t* dtypes, const int64_t* counts, const void* const* in, const void* norm, const void* ws, size_t ws_bytes) {
    if ((order != 0 && order != 2) || tensors < 0) return SIMNETS_E_DESC;
    if (!norm || (tensors > 0 && (!counts || !in))) return SIMNETS_E_NULL;
    long long total = 0;
    bool f64 = false;
    for (int i = 0; i < tensors; ++i) {
        if (dtypes && dtypes[i] != SIMNETS_F32 && dtypes[i] != SIMNETS_F64) return SIMNETS_E_DTYPE;
        if (counts[i] < 0) return SIMNETS_E_DESC;
        if (counts[i] > 0 && !in[i]) return SIMNETS_E_NULL;
        if (counts[i] > 0 && misplaced(in[i], dtypes ? dtypes[i] : SIMNETS_F32)) return SIMNETS_E_UNSUPPORTED;
        if (counts[i] > (1LL << 40) - total) return SIMNETS_E_UNSUPPORTED;          // (pieces of 16 KB are counted in 32 bits)
        total += counts[i];
        f64 = f64 || (dtypes && dtypes[i] == SIMNETS_F64);
    }
    if (misplaced(norm, f64 ? SIMNETS_F64 : SIMNETS_F32) || misplaced64(ws)) return SIMNETS_E_UNSUPPORTED;
    return !ws || ws_bytes < gradient_norm_workspace_bytes(tensors) ? SIMNETS_E_WORKSPACE : SIMNETS_OK;
}

int gradients(int32_t order, double limit, int32_t tensors, const int32_t* dtypes, const int64_t* counts, const void* const* in, void* const* out, void* norm, void* ws,
              void* stream) {
    bool f64 = false;
    for (int i = 0; dtypes && i < tensors; ++i) f64 = f64 || dtypes[i] == SIMNETS_F64;
    return from_cuda(launch_gradient_norm(order, tensors, dtypes, reinterpret_cast<const long long*>(counts), in, out, limit, norm, f64, ws, as_stream(stream)));
}
}  // namespace

extern "C" {

int simnets_abi_version(void) { return 1; }
uint64_t simnets_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }

const char* simnets_status_string(int status) {
    switch (status) {
    case SIMNETS_OK: return "ok";
    case SIMNETS_E_NULL: return "a required pointer is NULL";
    case SIMNETS_E_DESC: return "invalid descriptor (fails the operator's attribute / shape validation)";
    case SIMNETS_E_DTYPE: return "dtype must be float32 (0) or float64 (1)";
    case SIMNETS_E_WORKSPACE: return "workspace missing or smaller than the *_workspace_bytes query";
    case SIMNETS_E_UNSUPPORTED: return "valid descriptor outside the supported index range";
    case SIMNETS_E_TOO_LARGE: return "problem exceeds the fixed capacity of this entry point";
    default: break;
    }
    if (status > 0) return cudaGetErrorString(static_cast<cudaError_t>(status));
    return "unknown status";
}

/* ------------------------------------------------------------- Similarity */
int simnets_similarity_output_dims(const simnets_sim_desc* d, int32_t* out_h, int32_t* out_w) {
    SimGeo g;
    const int rc = sim_geometry(d, &g);
    if (rc) return rc;
    if (!out_h || !out_w) return SIMNETS_E_NULL;
    *out_h = g.oh; *out_w = g.ow;
    return SIMNETS_OK;
}

size_t simnets_similarity_workspace_bytes(const simnets_sim_desc* d) {
    SimGeo g;
    if (sim_geometry(d, &g)) return 0;
    return sim_workspace_bytes(g, d->dtype == SIMNETS_F64, d->flags);
}

int simnets_similarity_forward(const simnets_sim_desc* d, const void* x, const void* t, const void* w, void* y,
                               void* ws, size_t ws_bytes, void* stream) {
    SimGeo g;
    const int rc = sim_geometry(d, &g);
    if (rc) return rc;
    if (!t || !w || (g.B > 0 && (!x || !y))) return SIMNETS_E_NULL;   // batch-sized tensors may be NULL when batch == 0
    const bool f64 = d->dtype == SIMNETS_F64;
    if (sim_use_tiled(g, f64, d->flags)) {
        if (!ws || ws_bytes < sim_workspace_bytes(g, f64, d->flags)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_sim_fwd_tiled(g, (const float*)x, (const float*)t, (const float*)w, (float*)y, ws, d->flags, as_stream(stream)));
    }
    return from_cuda(launch_sim_fwd_direct(g, f64, x, t, w, y, as_stream(stream)));
}

int simnets_similarity_forward_extrema(const simnets_sim_desc* d, const void* x, const void* t, const void* w, void* y, void* ch_max, void* ch_min,
                                       void* ws, size_t ws_bytes, void* stream) {
    SimGeo g;
    const int rc = sim_geometry(d, &g);
    if (rc) return rc;
    if (d->dtype != SIMNETS_F32) return SIMNETS_E_UNSUPPORTED;
    if (!t || !w || (g.B > 0 && (!x || !y))) return SIMNETS_E_NULL;
    if (g.B == 0) return SIMNETS_OK;
    if (sim_use_tiled(g, false, d->flags)) {
        if (!ws || ws_bytes < sim_workspace_bytes(g, false, d->flags)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_sim_fwd_tiled(g, (const float*)x, (const float*)t, (const float*)w, (float*)y, ws, d->flags, as_stream(stream),
                                              (float*)ch_max, (float*)ch_min));
    }
    const cudaError_t e = launch_sim_fwd_direct(g, false, x, t, w, y, as_stream(stream));
    if (e != cudaSuccess) return from_cuda(e);
    return from_cuda(launch_sim_extrema(g, (const float*)y, (float*)ch_max, (float*)ch_min, as_stream(stream)));
}

void* simnets_mex_workspace_maxima(const simnets_mex_desc* d, void* workspace) {
    MexGeo g;
    if (!d || !workspace || mex_geometry(d, nullptr, &g)) return nullptr;
    if (d->dtype == SIMNETS_F32 && mex_use_gemm(g, false, d->flags)) return mex_gemm_maxima(g, false, workspace);
    if (!mex_use_tiled(g, d->dtype == SIMNETS_F64, d->flags)) return nullptr;
    return mex_workspace_maxima(g, workspace, d->flags);
}

int simnets_similarity_input_grad(const simnets_sim_desc* d, const void* x, const void* t, const void* w, const void* dy,
                                  void* dx, void* ws, size_t ws_bytes, void* stream) {
    SimGeo g;
    const int rc = sim_geometry(d, &g);
    if (rc) return rc;
    if (!t || !w || (g.B > 0 && (!x || !dy || !dx))) return SIMNETS_E_NULL;
    const bool f64 = d->dtype == SIMNETS_F64;
    if (sim_use_tiled(g, f64, d->flags)) {
        if (!ws || ws_bytes < sim_workspace_bytes(g, f64, d->flags)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_sim_dx_tiled(g, (const float*)x, (const float*)t, (const float*)w, (const float*)dy, (float*)dx, ws, as_stream(stream)));
    }
    return from_cuda(launch_sim_dx_direct(g, f64, x, t, w, dy, dx, as_stream(stream)));
}

int simnets_similarity_params_grad(const simnets_sim_desc* d, const void* x, const void* t, const void* w, const void* dy,
                                   void* dt, void* dw, void* ws, size_t ws_bytes, void* stream) {
    SimGeo g;
    const int rc = sim_geometry(d, &g);
    if (rc) return rc;
    if (!t || !w || !dt || !dw || (g.B > 0 && (!x || !dy))) return SIMNETS_E_NULL;
    const bool f64 = d->dtype == SIMNETS_F64;
    const bool acc = (d->flags & SIMNETS_FLAG_ACCUMULATE) != 0;
    if (sim_use_tiled(g, f64, d->flags)) {
        if (!ws || ws_bytes < sim_workspace_bytes(g, f64, d->flags)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_sim_dparams_tiled(g, (const float*)x, (const float*)t, (const float*)w, (const float*)dy,
                                                  (float*)dt, (float*)dw, acc, ws, as_stream(stream)));
    }
    return from_cuda(launch_sim_dparams_direct(g, f64, x, t, w, dy, dt, dw, acc, as_stream(stream)));
}

/* -------------------------------------------------------------------- MEX */
int simnets_mex_dims(const simnets_mex_desc* d, simnets_mex_geometry* out) {
    if (!out) return SIMNETS_E_NULL;
    return mex_geometry(d, out, nullptr);
}

int get_mex_offsets_nregions(int n_input_dim, const int* input_dim, int n_padding, const int* padding, int n_strides,
                             const int* strides, int num_instances, int blocks_round_down, int use_unshared_regions,
                             int n_blocks, const int* blocks, int n_shared, const int* shared, int n_unshared,
                             const int* unshared) {
    if (!input_dim || !padding || !strides || !blocks || !shared || !unshared) return -1;
    if (n_input_dim != 3 || n_blocks != 3) return -1;
    if (n_shared < 1 || n_unshared < 1) return -1;
    simnets_mex_desc d = {};
    d.dtype = SIMNETS_F32;
    d.batch = 1; d.channels = input_dim[0]; d.height = input_dim[1]; d.width = input_dim[2];
    d.num_instances = num_instances;
    auto three = [](int n, const int* v, int32_t* dst) {
        if (n == 1) { dst[0] = dst[1] = dst[2] = v[0]; return true; }          // broadcast
        if (n == 2) { dst[0] = -1; dst[1] = v[0]; dst[2] = v[1]; return true; } // as ExpandDimSpec prepends -1
        if (n == 3) { dst[0] = v[0]; dst[1] = v[1]; dst[2] = v[2]; return true; }
        return false;
    };
    if (!three(n_padding, padding, d.padding) || !three(n_strides, strides, d.strides)) return -1;
    for (int a = 0; a < 3; ++a) d.blocks[a] = blocks[a];
    d.epsilon = 1.0f;
    d.blocks_round_down = blocks_round_down > 0;
    d.use_unshared_regions = use_unshared_regions > 0;
    // A region list that is not three long stands for its first entry applied to height and width, as
    // MexDimensionsData::CalculateDimensions reads it (src/kernels/mex_kernel_common.cpp:86-93, 113-120); the op itself
    // accepts one or three entries only (mex_kernel_common.cpp:51-54), this helper any length, like the reference's.
    auto region = [](int n, const int* v, int32_t* dst, int32_t* n_dst) {
        if (n == 3) { dst[0] = v[0]; dst[1] = v[1]; dst[2] = v[2]; *n_dst = 3; }
        else { dst[0] = v[0]; *n_dst = 1; }
    };
    region(n_shared, shared, d.shared_offset_region, &d.n_shared_offset_region);
    region(n_unshared, unshared, d.unshared_offset_region, &d.n_unshared_offset_region);
    simnets_mex_geometry g;
    if (mex_geometry(&d, &g, nullptr)) return -1;
    return g.num_regions;
}

size_t simnets_mex_forward_workspace_bytes(const simnets_mex_desc* d) {
    MexGeo g;
    if (mex_geometry(d, nullptr, &g)) return 0;
    const bool f64 = d->dtype == SIMNETS_F64;
    // (room for either family: a caller may size a workspace once and pass other flags later)
    const bool gemm = mex_use_gemm(g, f64, d->flags) || mex_gradients_by_gemm(g, f64, d->flags);
    return std::max(mex_workspace_bytes(g, f64, d->flags), gemm ? mex_gemm_workspace_bytes(g, f64) : size_t(256));
}

size_t simnets_mex_products_bytes(const simnets_mex_desc* d) {
    MexGeo g;
    return mex_geometry(d, nullptr, &g) ? 0 : mex_products_bytes(g, d->dtype == SIMNETS_F64, d->flags);
}

size_t simnets_mex_workspace_bytes(const simnets_mex_desc* d) {
    MexGeo g;
    if (mex_geometry(d, nullptr, &g)) return 0;
    const bool f64 = d->dtype == SIMNETS_F64;
    return simnets_mex_forward_workspace_bytes(d) +
           std::max(mex_products_bytes(g, f64, d->flags), mex_products_bytes(g, f64, d->flags | SIMNETS_FLAG_MEX_NO_SMALL_TILES));
}

int simnets_mex_forward(const simnets_mex_desc* d, const void* x, const void* off, void* y, void* ws, size_t ws_bytes, void* stream) {
    MexGeo g;
    const int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if (!off || (g.B > 0 && (!x || !y))) return SIMNETS_E_NULL;
    const bool f64 = d->dtype == SIMNETS_F64;
    if ((d->flags & SIMNETS_FLAG_MEX_NORMALIZED_OFFSETS) && g.B > 0 && !mex_use_gemm(g, f64, d->flags) && !mex_use_tiled(g, f64, d->flags)) return SIMNETS_E_UNSUPPORTED;
    if (mex_use_gemm(g, f64, d->flags)) {
        if (!ws || ws_bytes < mex_gemm_workspace_bytes(g, f64)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_mex_fwd_gemm(g, f64, x, off, y, ws, d->flags, as_stream(stream)));
    }
    if (mex_use_tiled(g, f64, d->flags)) {
        if (!ws || ws_bytes < mex_workspace_bytes(g, f64, d->flags)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_mex_fwd_tiled(g, (const float*)x, (const float*)off, (float*)y, ws, d->flags, as_stream(stream)));
    }
    return from_cuda(launch_mex_fwd_direct(g, f64, x, off, y, as_stream(stream)));
}

size_t simnets_softmax_cross_entropy_workspace_bytes(int32_t batch) { return softmax_xent_workspace_bytes(batch < 0 ? 0 : batch); }

int simnets_softmax_cross_entropy(int32_t batch, int32_t classes, float scale, const float* logits, const int64_t* labels, float* loss,
                                  float* dlogits, void* ws, size_t ws_bytes, void* stream) {
    if (batch < 0 || classes < 1) return SIMNETS_E_DESC;
    if (!loss || (batch > 0 && (!logits || !labels))) return SIMNETS_E_NULL;
    if (!ws || ws_bytes < softmax_xent_workspace_bytes(batch)) return SIMNETS_E_WORKSPACE;
    return from_cuda(launch_softmax_xent(batch, classes, scale, logits, reinterpret_cast<const long long*>(labels), loss, dlogits, ws,
                                         as_stream(stream)));
}

int simnets_mex_forward_pool2x2(const simnets_mex_desc* d, const void* x, const void* off, void* y, void* y_pooled, void* ws, size_t ws_bytes,
                                void* stream) {
    MexGeo g;
    const int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if (d->dtype != SIMNETS_F32 || g.Ho % 2 || g.Wo % 2) return SIMNETS_E_UNSUPPORTED;
    if (!off || (g.B > 0 && (!x || !y || !y_pooled))) return SIMNETS_E_NULL;
    if (g.B == 0) return SIMNETS_OK;
    if (mex_use_gemm(g, false, d->flags)) {
        if (!ws || ws_bytes < mex_gemm_workspace_bytes(g, false)) return SIMNETS_E_WORKSPACE;
        const cudaError_t e = launch_mex_fwd_gemm(g, false, x, off, y, ws, d->flags, as_stream(stream));
        if (e != cudaSuccess) return from_cuda(e);
        return from_cuda(launch_sum_pool2((long long)g.B * g.M * g.Co, g.Ho, g.Wo, (const float*)y, (float*)y_pooled, as_stream(stream)));
    }
    if (mex_use_tiled(g, false, d->flags)) {
        if (!ws || ws_bytes < mex_workspace_bytes(g, false, d->flags)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_mex_fwd_tiled(g, (const float*)x, (const float*)off, (float*)y, ws, d->flags, as_stream(stream), (float*)y_pooled));
    }
    if (d->flags & SIMNETS_FLAG_MEX_NORMALIZED_OFFSETS) return SIMNETS_E_UNSUPPORTED;
    const cudaError_t e = launch_mex_fwd_direct(g, false, x, off, y, as_stream(stream));
    if (e != cudaSuccess) return from_cuda(e);
    return from_cuda(launch_sum_pool2((long long)g.B * g.M * g.Co, g.Ho, g.Wo, (const float*)y, (float*)y_pooled, as_stream(stream)));
}

int simnets_similarity_workspace_status(const void* ws, void* stream, int32_t* host_out) {
    if (!ws || !host_out) return SIMNETS_E_NULL;
    return from_cuda(cudaMemcpyAsync(host_out, ws, 2 * sizeof(int32_t), cudaMemcpyDeviceToHost, as_stream(stream)));
}

int simnets_mex_workspace_status(const void* ws, void* stream, int32_t* host_out) {
    if (!ws || !host_out) return SIMNETS_E_NULL;
    return from_cuda(cudaMemcpyAsync(host_out, ws, 2 * sizeof(int32_t), cudaMemcpyDeviceToHost, as_stream(stream)));
}

int simnets_mex_forward_static_scratch(const simnets_mex_desc* d, const void* x, const void* off, void* y, void* stream) {
    MexGeo g;
    const int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if (!off || (g.B > 0 && (!x || !y))) return SIMNETS_E_NULL;
    if (d->flags & SIMNETS_FLAG_MEX_NORMALIZED_OFFSETS) return SIMNETS_E_UNSUPPORTED;
    const bool f64 = d->dtype == SIMNETS_F64;
    if (!mex_use_tiled(g, f64, d->flags))        // these shapes run on kernels that need no scratch at all
        return from_cuda(launch_mex_fwd_direct(g, f64, x, off, y, as_stream(stream)));
    return launch_mex_fwd_static(g, (const float*)x, (const float*)off, (float*)y, d->flags, as_stream(stream));
}

int simnets_mex_gradients(const simnets_mex_desc* d, const void* x, const void* off, const void* y, const void* dy, void* dx, void* doff,
                          void* ws, size_t ws_bytes, void* products, size_t products_bytes, void* stream) {
    MexGeo g;
    const int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if (!off || (g.B > 0 && (!x || !y || !dy || (!dx && !doff)))) return SIMNETS_E_NULL;
    return mex_gradients(g, d, x, off, y, dy, dx, doff, ws, ws_bytes, products, products_bytes, as_stream(stream));
}

int simnets_mex_input_grad(const simnets_mex_desc* d, const void* x, const void* off, const void* y, const void* dy, void* dx,
                           void* ws, size_t ws_bytes, void* stream) {
    MexGeo g;
    const int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if (!off || (g.B > 0 && (!x || !y || !dy || !dx))) return SIMNETS_E_NULL;
    return mex_gradients_in(g, d, x, off, y, dy, dx, nullptr, ws, ws_bytes, as_stream(stream));
}

int simnets_mex_offsets_grad(const simnets_mex_desc* d, const void* x, const void* off, const void* y, const void* dy,
                             void* doff, void* ws, size_t ws_bytes, void* stream) {
    MexGeo g;
    const int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if (!off || !doff || (g.B > 0 && (!x || !y || !dy))) return SIMNETS_E_NULL;
    return mex_gradients_in(g, d, x, off, y, dy, nullptr, doff, ws, ws_bytes, as_stream(stream));
}

int simnets_mex_backward(const simnets_mex_desc* d, const void* x, const void* off, const void* y, const void* dy,
                         void* dx, void* doff, void* ws, size_t ws_bytes, void* stream) {
    MexGeo g;
    const int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if (!off || !doff || (g.B > 0 && (!x || !y || !dy || !dx))) return SIMNETS_E_NULL;
    return mex_gradients_in(g, d, x, off, y, dy, dx, doff, ws, ws_bytes, as_stream(stream));
}

int simnets_normalize_offsets_forward(int64_t rows, int32_t k, const void* off, void* out, void* stream) {
    if (rows < 0 || k < 0) return SIMNETS_E_DESC;
    if (rows > 0 && k > 0 && (!off || !out)) return SIMNETS_E_NULL;
    return from_cuda(launch_normalize_offsets_fwd(rows, k, (const float*)off, (float*)out, as_stream(stream)));
}

int simnets_normalize_offsets_backward(int64_t rows, int32_t k, const void* off, const void* dout, void* doff, void* stream) {
    if (rows < 0 || k < 0) return SIMNETS_E_DESC;
    if (rows > 0 && k > 0 && (!off || !dout || !doff)) return SIMNETS_E_NULL;
    return from_cuda(launch_normalize_offsets_bwd(rows, k, (const float*)off, (const float*)dout, (float*)doff, as_stream(stream)));
}

size_t simnets_mixture_workspace_bytes(const simnets_sim_desc* d) {
    SimGeo g;
    if (sim_geometry(d, &g) || !mixture_shape(g, d->dtype == SIMNETS_F64, d->flags)) return 0;
    return mixture_workspace_bytes(g);
}

int simnets_mixture_statistics(const simnets_sim_desc* d, const void* x, const void* means, const void* covs, void* stats, void* ws, size_t ws_bytes, void* stream) {
    SimGeo g;
    const int rc = sim_geometry(d, &g);
    if (rc) return rc;
    if (!mixture_shape(g, d->dtype == SIMNETS_F64, d->flags)) return SIMNETS_E_UNSUPPORTED;
    if (!x || !means || !covs || !stats) return SIMNETS_E_NULL;
    if (!ws || ws_bytes < mixture_workspace_bytes(g)) return SIMNETS_E_WORKSPACE;
    return from_cuda(launch_mixture_statistics(g, (const float*)x, (const float*)means, (const float*)covs, (float*)stats, ws, as_stream(stream)));
}

int simnets_mixture_parameters(int32_t k, int32_t taps, float min_var, const float* stats, const float* means, float* new_means, float* new_covs, void* stream) {
    if (k < 1 || taps < 1 || (long long)k * taps > (1LL << 30)) return SIMNETS_E_DESC;
    if (!stats || !means || !new_means || !new_covs) return SIMNETS_E_NULL;
    return from_cuda(launch_mixture_parameters(k, taps, min_var, stats, means, new_means, new_covs, as_stream(stream)));
}

int64_t simnets_checkpoint_groups(int64_t count, int32_t group) { return count < 0 || group < 1 ? 0 : (count + group - 1) / group; }

int simnets_checkpoint_pack(int32_t dtype, int64_t count, int32_t group, const void* x, void* codes, void* ranges, void* stream) {
    const int rc = checkpoint_check(dtype, count, group);
    if (rc) return rc;
    if (count > 0 && (!x || !codes || !ranges)) return SIMNETS_E_NULL;
    return from_cuda(launch_checkpoint_pack(dtype == SIMNETS_F64, count, group, x, codes, ranges, as_stream(stream)));
}

int simnets_checkpoint_unpack(int32_t dtype, int64_t count, int32_t group, const void* codes, const void* ranges, void* x, void* stream) {
    const int rc = checkpoint_check(dtype, count, group);
    if (rc) return rc;
    if (count > 0 && (!x || !codes || !ranges)) return SIMNETS_E_NULL;
    return from_cuda(launch_checkpoint_unpack(dtype == SIMNETS_F64, count, group, codes, ranges, x, as_stream(stream)));
}

size_t simnets_mex_checkpoint_workspace_bytes(const simnets_mex_desc* d) {
    MexGeo g;
    if (mex_geometry(d, nullptr, &g)) return 0;
    return mex_checkpoint_shape(g, d->dtype == SIMNETS_F64, d->flags) ? mex_checkpoint_bytes(g) : mex_checkpoint_carve(g, *d, nullptr).bytes;
}

int simnets_mex_checkpoint_one_pass(const simnets_mex_desc* d) {
    MexGeo g;
    return d && !mex_geometry(d, nullptr, &g) && mex_checkpoint_shape(g, d->dtype == SIMNETS_F64, d->flags);
}

int simnets_mex_checkpoint_gradients(const simnets_mex_desc* d, int32_t group, const void* codes, const void* ranges, const void* off, const void* dy, void* dx,
                                     void* doff, void* ws, size_t ws_bytes, void* stream) {
    MexGeo g;
    int rc = mex_geometry(d, nullptr, &g);
    if (rc) return rc;
    if ((rc = checkpoint_check(d->dtype, 1, group))) return rc;
    if (d->flags & (SIMNETS_FLAG_MEX_WORKSPACE_PRIMED | SIMNETS_FLAG_MEX_MAXIMA_GIVEN)) return SIMNETS_E_UNSUPPORTED;
    if (!off || (g.B > 0 && (!codes || !ranges || !dy || (!dx && !doff)))) return SIMNETS_E_NULL;
    if (g.B == 0) return mex_gradients(g, d, nullptr, off, nullptr, nullptr, nullptr, doff, ws, ws_bytes, nullptr, 0, as_stream(stream));
    if (mex_checkpoint_shape(g, d->dtype == SIMNETS_F64, d->flags)) {
        if (reinterpret_cast<uintptr_t>(ranges) % 8) return SIMNETS_E_UNSUPPORTED;          // (read as pairs)
        if (!ws || ws_bytes < mex_checkpoint_bytes(g)) return SIMNETS_E_WORKSPACE;
        return from_cuda(launch_mex_checkpoint(g, group, codes, ranges, (const float*)off, (const float*)dy, (float*)dx, (float*)doff, (d->flags & SIMNETS_FLAG_ACCUMULATE) != 0,
                                               (d->flags & SIMNETS_FLAG_MEX_NORMALIZED_OFFSETS) != 0, (d->flags & SIMNETS_FLAG_MEX_TEST_EXPIRE_WAIT) != 0, ws, as_stream(stream)));
    }
    const MexCheckpointWs w = mex_checkpoint_carve(g, *d, ws);
    if (!ws || ws_bytes < w.bytes) return SIMNETS_E_WORKSPACE;
    const cudaError_t e = launch_checkpoint_unpack(d->dtype == SIMNETS_F64, (long long)g.B * g.C * g.H * g.W, group, codes, ranges, w.x, as_stream(stream));
    if (e != cudaSuccess) return from_cuda(e);
    simnets_mex_desc f = *d;
    const uint32_t route = checkpoint_route(g, *d);
    f.flags = (d->flags | route) & ~uint32_t(SIMNETS_FLAG_MEX_DY_POOLED2 | SIMNETS_FLAG_ACCUMULATE);
    rc = simnets_mex_forward(&f, w.x, off, w.y, w.layer, w.layer_bytes, stream);
    if (rc) return rc;
    f.flags = d->flags | route | SIMNETS_FLAG_MEX_WORKSPACE_PRIMED;
    return mex_gradients(g, &f, w.x, off, w.y, dy, dx, doff, w.layer, w.layer_bytes, w.products, w.products_bytes, as_stream(stream));
}

size_t simnets_similarity_checkpoint_workspace_bytes(const simnets_sim_desc* d) {
    SimGeo g;
    return sim_geometry(d, &g) ? 0 : sim_checkpoint_values(g, *d) + std::max<size_t>(sim_workspace_bytes(g, d->dtype == SIMNETS_F64, d->flags), 256);
}

int simnets_similarity_checkpoint_gradients(const simnets_sim_desc* d, int32_t group, const void* codes, const void* ranges, const void* t, const void* w,
                                            const void* dy, void* dx, void* dt, void* dw, void* ws, size_t ws_bytes, void* stream) {
    SimGeo g;
    int rc = sim_geometry(d, &g);
    if (rc) return rc;
    if ((rc = checkpoint_check(d->dtype, 1, group))) return rc;
    if (!t || !w || (dt == nullptr) != (dw == nullptr) || (!dx && !dt && g.B > 0) || (g.B > 0 && (!codes || !ranges || !dy))) return SIMNETS_E_NULL;
    if (!ws || ws_bytes < simnets_similarity_checkpoint_workspace_bytes(d)) return SIMNETS_E_WORKSPACE;
    const cudaError_t e = launch_checkpoint_unpack(d->dtype == SIMNETS_F64, (long long)g.B * g.C * g.H * g.W, group, codes, ranges, ws, as_stream(stream));
    if (e != cudaSuccess) return from_cuda(e);
    const size_t values = sim_checkpoint_values(g, *d);
    void* rest = static_cast<char*>(ws) + values;
    if (dx && g.B > 0 && (rc = simnets_similarity_input_grad(d, ws, t, w, dy, dx, rest, ws_bytes - values, stream))) return rc;
    return dt ? simnets_similarity_params_grad(d, ws, t, w, dy, dt, dw, rest, ws_bytes - values, stream) : SIMNETS_OK;
}

size_t simnets_route_workspace_bytes(const simnets_route_desc* d) { return route_check(d) ? 0 : std::max<size_t>(route_workspace_bytes(*d), 256); }

int simnets_route(const simnets_route_desc* d, const void* scores, const void* prior, const void* bias, int32_t* index, void* weights, void* dense, int64_t* load,
                  void* mass, void* ws, size_t ws_bytes, void* stream) {
    const int rc = route_check(d);
    if (rc) return rc;
    if (!load || (d->batch > 0 && d->positions > 0 && ((mass && !dense) || !scores || (!index && !weights && !dense)))) return SIMNETS_E_NULL;
    if (!ws || ws_bytes < route_workspace_bytes(*d)) return SIMNETS_E_WORKSPACE;
    return from_cuda(launch_route(*d, scores, prior, bias, index, weights, dense, reinterpret_cast<long long*>(load), mass, ws, as_stream(stream)));
}

int simnets_route_gradient(const simnets_route_desc* d, const void* scores, const void* prior, const int32_t* index, const void* weights, const void* grad,
                           void* dscores, void* stream) {
    const int rc = route_check(d);
    if (rc) return rc;
    if (d->batch > 0 && d->positions > 0 && ((d->sigmoid && !scores) || !index || !weights || !grad || !dscores)) return SIMNETS_E_NULL;
    return from_cuda(launch_route_gradient(*d, scores, prior, index, weights, grad, dscores, as_stream(stream)));
}

size_t simnets_log_probabilities_workspace_bytes(const simnets_likelihood_desc* d) { return likelihood_check(d) ? 0 : log_probabilities_workspace_bytes(*d); }

int simnets_log_probabilities(const simnets_likelihood_desc* d, const void* logits, const int64_t* labels, void* label, void* entropy, int32_t* top_index, void* top,
                              void* stats, void* ws, size_t ws_bytes, void* stream) {
    const int rc = likelihood_check(d);
    if (rc) return rc;
    if (d->batch == 0 || d->positions == 0) return SIMNETS_OK;
    if (!logits || (label && !labels) || (top == nullptr) != (top_index == nullptr)) return SIMNETS_E_NULL;
    if ((d->top_k > 0) != (top != nullptr)) return SIMNETS_E_DESC;
    for (const void* p : {logits, (const void*)label, (const void*)entropy, (const void*)top, (const void*)stats})
        if (misplaced(p, d->dtype)) return SIMNETS_E_UNSUPPORTED;
    if (misplaced64(labels) || misplaced(top_index, SIMNETS_F32) || misplaced64(ws)) return SIMNETS_E_UNSUPPORTED;
    if (const size_t need = log_probabilities_workspace_bytes(*d); need > 0 && (!ws || ws_bytes < need)) return SIMNETS_E_WORKSPACE;
    return from_cuda(launch_log_probabilities(*d, logits, reinterpret_cast<const long long*>(labels), label, entropy, top_index, top, stats, ws, as_stream(stream)));
}

int simnets_log_probabilities_gradient(const simnets_likelihood_desc* d, const void* logits, const int64_t* labels, const void* stats, const int32_t* top_index,
                                       const void* g_label, const void* g_entropy, const void* g_top, void* dlogits, void* stream) {
    const int rc = likelihood_check(d);
    if (rc) return rc;
    if (d->batch == 0 || d->positions == 0) return SIMNETS_OK;
    if (!logits || !stats || !dlogits || (g_label && !labels) || (g_top && !top_index)) return SIMNETS_E_NULL;
    if ((d->top_k > 0) != (g_top != nullptr)) return SIMNETS_E_DESC;
    for (const void* p : {logits, stats, g_label, g_entropy, g_top, (const void*)dlogits})
        if (misplaced(p, d->dtype)) return SIMNETS_E_UNSUPPORTED;
    if (misplaced64(labels) || misplaced(top_index, SIMNETS_F32)) return SIMNETS_E_UNSUPPORTED;
    return from_cuda(launch_log_probabilities_gradient(*d, logits, reinterpret_cast<const long long*>(labels), stats, top_index, g_label, g_entropy, g_top, dlogits,
                                                       as_stream(stream)));
}

size_t simnets_gradient_norm_workspace_bytes(int32_t tensors) { return tensors < 0 ? 0 : gradient_norm_workspace_bytes(tensors); }

int simnets_gradient_norm(int32_t order, int32_t tensors, const int32_t* dtypes, const int64_t* counts, const void* const* in, void* norm, void* ws, size_t ws_bytes,
                          void* stream) {
    const int rc = gradients_check(order, tensors, dtypes, counts, in, norm, ws, ws_bytes);
    return rc ? rc : gradients(order, 0.0, tensors, dtypes, counts, in, nullptr, norm, ws, stream);
}

int simnets_clip_gradients(int32_t order, double max_norm, int32_t tensors, const int32_t* dtypes, const int64_t* counts, const void* const* in, void* const* out, void* norm,
                           void* ws, size_t ws_bytes, void* stream) {
    if (!(max_norm >= 0)) return SIMNETS_E_DESC;
    if (tensors > 0 && !out) return SIMNETS_E_NULL;
    const int rc = gradients_check(order, tensors, dtypes, counts, in, norm, ws, ws_bytes);
    if (rc) return rc;
    for (int i = 0; i < tensors; ++i) {
        if (counts[i] > 0 && !out[i]) return SIMNETS_E_NULL;
        if (counts[i] > 0 && misplaced(out[i], dtypes ? dtypes[i] : SIMNETS_F32)) return SIMNETS_E_UNSUPPORTED;
    }
    return gradients(order, max_norm, tensors, dtypes, counts, in, out, norm, ws, stream);
}

int64_t simnets_fp32_fma_probe(int32_t packed, int32_t iters, void* scratch, void* stream) {
    if (iters < 1 || !scratch) return SIMNETS_E_DESC;
    const int blocks = device_sm_count() * 2;                       // two CTAs of 1024 threads fill an SM
    const cudaError_t e = launch_fp32_probe(packed != 0, blocks, iters, (float*)scratch, as_stream(stream));
    if (e != cudaSuccess) return -int64_t(e) - 1000;
    return int64_t(blocks) * 1024 * 16 * iters;
}

int simnets_sum_pool2x2_forward(int64_t planes, int32_t height, int32_t width, const void* x, void* y, void* stream) {
    if (planes < 0 || height < 0 || width < 0) return SIMNETS_E_DESC;
    if (height % 2 || width % 2) return SIMNETS_E_UNSUPPORTED;
    if (planes > 0 && height > 0 && width > 0 && (!x || !y)) return SIMNETS_E_NULL;
    return from_cuda(launch_sum_pool2(planes, height, width, (const float*)x, (float*)y, as_stream(stream)));
}

}  // extern "C"

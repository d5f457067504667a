// C ABI of the norms before and after a block, with its gate and residual scale.
#include <algorithm>

#include "block_norm.cuh"
#include "common.cuh"
#include "host.cuh"

using namespace bissd;

static bool dtype_ok(int t) { return t >= BISSD_F32 && t <= BISSD_F16; }
static bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static int block_norm_sizes(const bissd_block_norm_args *a) {
    if (!a) return BISSD_ERR_NULL;
    for (const int64_t n : {a->rows, a->stride_x, a->stride_residual, a->stride_gate, a->stride_dr, a->stride_dnormed})
        if (n < 0 || n > 0x3fffffff) return BISSD_ERR_SHAPE;     // rows and strides are 32-bit in the kernels, offsets 64
    if (a->rows <= 0 || a->width <= 0 || a->width > bnorm::kMaxWidth || a->gate_rows < 0 || (a->gate_rows > 0 && a->rows % a->gate_rows))
        return BISSD_ERR_SHAPE;
    if (!dtype_ok(a->dtype) || (a->r_dtype != a->dtype && a->r_dtype != BISSD_F32) || (a->w_dtype != a->dtype && a->w_dtype != BISSD_F32))
        return BISSD_ERR_DTYPE;
    if (a->gate_act < BISSD_GATE_NONE || a->gate_act > BISSD_GATE_SILU) return BISSD_ERR_SHAPE;
    return BISSD_OK;
}
static int block_norm_check(const bissd_block_norm_args *a, bool backward) {
    if (!a || !a->x || !a->residual) return BISSD_ERR_NULL;
    if (!backward && (!a->r || (a->pre_weight && !a->normed))) return BISSD_ERR_NULL;
    if (backward && !a->rstd && (a->post_weight || a->dnormed)) return BISSD_ERR_NULL;
    if (backward && a->dnormed && !a->pre_weight) return BISSD_ERR_NULL;
    return block_norm_sizes(a);
}
// Rows side by side in a block: up to 256 threads.  A row of more than 512 is two blocks' in the backward pass.
static int block_norm_pair(const bnorm::Params &p, bool backward) { return backward && p.threads_row > 512 ? 2 : 1; }
static int block_norm_threads(const bnorm::Params &p, bool backward) {
    return p.threads_row * std::max(1, 256 / p.threads_row) / block_norm_pair(p, backward);
}
// Channels that lie aligned together in every row: 8 (16 bytes of the narrower type), 2, or 0 where not even pairs do.
static int block_norm_vec(const bissd_block_norm_args *a) {
    const size_t es = a->dtype == BISSD_F32 ? 4 : 2, rs = a->r_dtype == BISSD_F32 ? 4 : 2;
    auto fits = [&](int n) {
        bool ok = a->width % n == 0;
        for (const void *p : {a->x, a->gate, (const void *)a->normed, a->dnormed, (const void *)a->dx, (const void *)a->dgate})
            ok = ok && reinterpret_cast<uintptr_t>(p) % (n == 8 ? 16 : 2 * es) == 0;
        for (const void *p : {a->residual, (const void *)a->r, a->dr, (const void *)a->dresidual})
            ok = ok && reinterpret_cast<uintptr_t>(p) % (n == 8 ? 16 : 2 * rs) == 0;
        for (const int64_t s : {a->stride_x, a->stride_residual, a->stride_gate, a->stride_dr, a->stride_dnormed}) ok = ok && s % n == 0;
        return ok;
    };
    return fits(8) ? 8 : fits(2) ? 2 : 0;
}
static long long block_norm_entries(const bnorm::Params &p) { return p.gate && p.gate_rows > 0 ? p.rows / p.gate_rows : 1; }
static bnorm::Params block_norm_params(const bissd_block_norm_args *a) {
    bnorm::Params p{};
    p.rows = (int)a->rows;
    p.gate_rows = a->gate_rows == 1 ? 0 : (int)a->gate_rows;          // a gate row for each row
    p.D = a->width;
    const int threads = ceil_div(a->width, bnorm::kCh), whole = threads > 512 ? 64 : 32;   // of a row: whole warps, also in two blocks
    p.threads_row = ceil_div(threads, whole) * whole;
    p.w_dtype = a->w_dtype; p.act = a->gate_act;
    p.scale = a->scale; p.eps = a->eps;
    p.sx = (int)a->stride_x; p.sres = (int)a->stride_residual; p.sgate = (int)a->stride_gate; p.sdr = (int)a->stride_dr; p.sdu = (int)a->stride_dnormed;
    p.x = a->x; p.res = a->residual; p.gate = a->gate; p.scale_v = a->scale_vector; p.w2 = a->post_weight; p.w1 = a->pre_weight;
    p.r = a->r; p.u = a->pre_weight ? a->normed : nullptr; p.rstd = a->rstd;
    p.dr = a->dr; p.du = a->dnormed; p.dx = a->dx; p.dres = a->dresidual; p.dgate = a->gate ? a->dgate : nullptr;
    return p;
}
constexpr int kFwd = 3, kBwd = 2;                                // blocks of 256 threads an SM: what the registers allow
constexpr int kFwdWide = 2, kBwdWide = 1;                        // of up to 512 (and one of 1024)
// Blocks (or pairs) to an entry: those that are resident, shared by the entries, and no more than there are rows.
static int block_norm_blocks(const bnorm::Params &p, bool backward) {
    const int threads = block_norm_threads(p, backward);
    const int resident = threads <= 256 ? (backward ? kBwd : kFwd) : backward ? kBwdWide : threads <= 512 ? kFwdWide : 1;
    const long long entries = block_norm_entries(p), per = std::max(1, threads / p.threads_row);
    const long long want = std::max<long long>(1, 148LL * resident / block_norm_pair(p, backward) / entries);
    return (int)std::min<long long>(want, (p.rows / entries + per - 1) / per);
}

// Bytes of the rows that a block copies ahead.
template <class T> static size_t block_norm_ring(int pieces, int threads, bool backward) {
    const int rows = threads <= 256   ? bnorm::Ahead<T, 256, 1>::rows
                     : backward       ? bnorm::Ahead<T, 512, kBwdWide>::rows
                     : threads <= 512 ? bnorm::Ahead<T, 512, kFwdWide>::rows
                                      : bnorm::Ahead<T, 1024, 1>::rows;
    return (size_t)rows * pieces * 16 * threads;
}
typedef void (*BlockNormKernel)(bnorm::Params);
template <class T, class R, int VEC> static BlockNormKernel block_norm_kernel(int threads, int pair, bool backward) {
    if (backward)
        return pair > 1        ? bnorm::block_norm_bwd<T, R, VEC, true, 512, kBwdWide>
               : threads > 256 ? bnorm::block_norm_bwd<T, R, VEC, false, 512, kBwdWide>
                               : bnorm::block_norm_bwd<T, R, VEC, false, 256, kBwd>;
    return threads > 512   ? bnorm::block_norm_fwd<T, R, VEC, false, 1024, 1>
           : threads > 256 ? bnorm::block_norm_fwd<T, R, VEC, false, 512, kFwdWide>
                           : bnorm::block_norm_fwd<T, R, VEC, false, 256, kFwd>;
}
template <class T, class R> static BlockNormKernel block_norm_pick(int vec, int threads, int pair, bool backward) {
    return vec == 8   ? block_norm_kernel<T, R, 8>(threads, pair, backward)
           : vec == 2 ? block_norm_kernel<T, R, 2>(threads, pair, backward)
                      : block_norm_kernel<T, R, 0>(threads, pair, backward);
}
template <class T, class R> static int block_norm_forward_impl(const bissd_block_norm_args *a, cudaStream_t s) {
    bnorm::Params p = block_norm_params(a);
    const int threads = block_norm_threads(p, false);
    const int vec = block_norm_vec(a);
    p.blocks = block_norm_blocks(p, false);
    const long long grid = block_norm_entries(p) * p.blocks;
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    const int pieces = (int)(sizeof(T) * (a->gate && p.gate_rows == 0 ? 2 : 1) + sizeof(R)) / 2;
    const size_t smem = vec ? block_norm_ring<T>(pieces, threads, false) : 0;
    const auto kernel = block_norm_pick<T, R>(vec, threads, 1, false);
    BISSD_ALLOW(kernel, smem + 512);                             // the limit is on static memory too
    BISSD_LAUNCH("block_norm_fwd", launch_pdl(kernel, (int)grid, threads, smem, s, p));
    return BISSD_OK;
}
template <class T, class R> static int block_norm_backward_impl(const bissd_block_norm_args *a, float *part, cudaStream_t s) {
    bnorm::Params p = block_norm_params(a);
    const int threads = block_norm_threads(p, true), pair = block_norm_pair(p, true), per = std::max(1, threads / p.threads_row);
    const int vec = block_norm_vec(a);
    const long long entries = block_norm_entries(p);
    p.blocks = block_norm_blocks(p, true);
    if (entries * p.blocks > 0x3fffffffLL || (entries + 3) * ceil_div(p.D, 32) > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    p.part = part;
    const int pieces = (int)(sizeof(T) * (1 + (a->gate && p.gate_rows == 0) + (a->dnormed != nullptr)) + sizeof(R) * (1 + (a->dr != nullptr))) / 2;
    const size_t rows = (size_t)(per - 1) * p.threads_row * bnorm::kCh * sizeof(float);
    const size_t smem = std::max(rows, vec ? block_norm_ring<T>(pieces, threads, true) : 0);
    const auto kernel = block_norm_pick<T, R>(vec, threads, pair, true);
    BISSD_ALLOW(kernel, smem + 512);                             // the limit is on static memory too
    BISSD_LAUNCH("block_norm_bwd", launch_cluster(kernel, (int)(entries * p.blocks) * pair, threads, smem, s, pair, p));
    bnorm::SumParams q{};
    q.part = part; q.D = p.D; q.blocks = p.blocks; q.entries = (int)entries; q.w_dtype = p.w_dtype; q.g_dtype = a->dtype;
    q.dpre = a->dnormed ? a->dpre : nullptr; q.dpost = a->post_weight ? a->dpost : nullptr;
    q.dscale = a->scale_vector ? a->dscale : nullptr; q.dgate = p.gate_rows > 0 ? p.dgate : nullptr;
    if (q.dpre || q.dpost || q.dscale || q.dgate)
        BISSD_LAUNCH("block_norm_sums", launch_pdl(bnorm::block_norm_sums, (int)((3 + (q.dgate ? entries : 0)) * ceil_div(p.D, 32)),
                                                   dim3(32, 8), 0, s, q));
    return BISSD_OK;
}
template <class F> static int by_types(const bissd_block_norm_args *a, F f) {
    if (a->dtype == BISSD_F32) return f(float(), float());
    if (a->dtype == BISSD_BF16) return a->r_dtype == BISSD_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
    return a->r_dtype == BISSD_F32 ? f(__half(), float()) : f(__half(), __half());
}

extern "C" {

int bissd_block_norm_workspace_bytes(const bissd_block_norm_args *a, size_t *bwd_bytes) {
    const int rc = block_norm_sizes(a);
    if (rc != BISSD_OK) return rc;
    const bnorm::Params p = block_norm_params(a);
    if (bwd_bytes) *bwd_bytes = align256((size_t)block_norm_entries(p) * block_norm_blocks(p, true) * 4 * p.D * sizeof(float));
    return BISSD_OK;
}

int bissd_block_norm_forward(const bissd_block_norm_args *a, void *stream) {
    int rc = block_norm_check(a, false);
    if (rc == BISSD_OK) rc = check_device();
    if (rc != BISSD_OK) return rc;
    return by_types(a, [&](auto t, auto r) { return block_norm_forward_impl<decltype(t), decltype(r)>(a, static_cast<cudaStream_t>(stream)); });
}

int bissd_block_norm_backward(const bissd_block_norm_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    int rc = block_norm_check(a, true);
    size_t need = 0;
    if (rc == BISSD_OK) rc = bissd_block_norm_workspace_bytes(a, &need);
    if (rc != BISSD_OK) return rc;
    if (!workspace || workspace_bytes < need) return BISSD_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return BISSD_ERR_ALIGN;
    rc = check_device();
    if (rc != BISSD_OK) return rc;
    return by_types(a, [&](auto t, auto r) {
        return block_norm_backward_impl<decltype(t), decltype(r)>(a, static_cast<float *>(workspace), static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"

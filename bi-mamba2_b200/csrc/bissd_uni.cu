// C ABI of what a decoder built from this library's layers needs: causal linear attention with a decay for each head, its
// single-token form, and the norms around a residual block.
#include <algorithm>
#include <cmath>

#include "block_norm.cuh"
#include "common.cuh"
#include "host.cuh"
#include "uni_plan.cuh"
#include "uni_step.cuh"
#include "uni_walk.cuh"

using namespace bissd;

static bool dtype_ok(int t) { return t >= BISSD_F32 && t <= BISSD_F16; }
static size_t dtype_size(int t) { return t == BISSD_F32 ? 4 : 2; }
template <class F> static int by_dtype(int t, F f) {
    if (t == BISSD_F32) return f(float());
    if (t == BISSD_BF16) return f(__nv_bfloat16());
    return f(__half());
}
static View view(const bissd_tensor &t) { return View{t.ptr, (long long)t.stride_batch, (long long)t.stride_seq, (long long)t.stride_head}; }
static bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// ---- one token ---------------------------------------------------------------------------------------------------
static int step_check(const bissd_decay_step_args *a) {
    if (!a || !a->q.ptr || !a->k.ptr || !a->v.ptr || !a->g.ptr || !a->o.ptr || !a->state) return BISSD_ERR_NULL;
    if (a->batch <= 0 || a->nheads <= 0 || a->nkheads <= 0 || a->nheads % a->nkheads || a->kdim <= 0 || a->kdim > 256 || a->vdim <= 0 ||
        a->vdim > 256 || a->nslots <= 0 || (!a->slots && a->nslots < a->batch))
        return BISSD_ERR_SHAPE;
    if (a->slot_stride < (int64_t)a->nheads * a->kdim * a->vdim) return BISSD_ERR_SHAPE;
    if ((long long)a->batch * a->nheads * ceil_div(a->vdim, uni::kStepColumns) > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    if (!dtype_ok(a->dtype) || !dtype_ok(a->g_dtype)) return BISSD_ERR_DTYPE;
    if (reinterpret_cast<uintptr_t>(a->state) % 4) return BISSD_ERR_ALIGN;
    return BISSD_OK;
}
static int step_launch(const bissd_decay_step_args *a, cudaStream_t s) {
    uni::StepParams p;
    p.q = view(a->q); p.k = view(a->k); p.v = view(a->v); p.g = view(a->g);
    if (a->g_per_head) { p.g.sb = 0; p.g.sh = 1; }
    p.o = MutView{a->o.ptr, (long long)a->o.stride_batch, 0, (long long)a->o.stride_head};
    p.state = a->state; p.slot_stride = a->slot_stride; p.slots = a->slots;
    p.batch = a->batch; p.H = a->nheads; p.hk = a->nkheads; p.N = a->kdim; p.P = a->vdim; p.nslots = a->nslots; p.g_dtype = a->g_dtype;
    p.column_blocks = ceil_div(a->vdim, uni::kStepColumns);
    p.scale = a->scale;
    const int grid = a->batch * a->nheads * p.column_blocks;
    const bool quads = a->vdim % 4 == 0 && a->slot_stride % 4 == 0 && aligned16(a->state);
    return by_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        const auto kernel = !quads ? uni::decay_step<T, 1, 32>
                                   : (p.N <= 64 ? uni::decay_step<T, 4, 2> : (p.N <= 128 ? uni::decay_step<T, 4, 4> : uni::decay_step<T, 4, 8>));
        BISSD_LAUNCH("decay_step", launch_pdl(kernel, grid, uni::kStepThreads, 0, s, p));
        return BISSD_OK;
    });
}

// ---- the norms around a block --------------------------------------------------------------------------------------
static int block_norm_check(const bissd_block_norm_args *a, bool backward) {
    if (!a || !a->x || !a->residual) return BISSD_ERR_NULL;
    if (!backward && (!a->r || (a->pre_weight && !a->normed))) return BISSD_ERR_NULL;
    if (backward && !a->rstd && (a->post_weight || a->dnormed)) return BISSD_ERR_NULL;
    if (backward && a->dnormed && !a->pre_weight) return BISSD_ERR_NULL;
    if (a->rows <= 0 || a->width <= 0 || a->width > bnorm::kMaxWidth || a->gate_rows < 0 || (a->gate_rows > 0 && a->rows % a->gate_rows))
        return BISSD_ERR_SHAPE;
    if (!dtype_ok(a->dtype) || (a->r_dtype != a->dtype && a->r_dtype != BISSD_F32) || (a->w_dtype != a->dtype && a->w_dtype != BISSD_F32))
        return BISSD_ERR_DTYPE;
    if (a->gate_act < BISSD_GATE_NONE || a->gate_act > BISSD_GATE_SILU) return BISSD_ERR_SHAPE;
    return BISSD_OK;
}
static bnorm::Params block_norm_params(const bissd_block_norm_args *a) {
    bnorm::Params p{};
    p.rows = a->rows;
    p.gate_rows = a->gate_rows == 1 ? 0 : a->gate_rows;          // a gate row for each row
    p.D = a->width;
    p.threads_row = ceil_div(ceil_div(a->width, bnorm::kCh), 32) * 32;
    p.w_dtype = a->w_dtype; p.act = a->gate_act;
    p.scale = a->scale; p.eps = a->eps;
    p.sx = a->stride_x; p.sres = a->stride_residual; p.sgate = a->stride_gate; p.sdr = a->stride_dr; p.sdu = a->stride_dnormed;
    p.x = a->x; p.res = a->residual; p.gate = a->gate; p.scale_v = a->scale_vector; p.w2 = a->post_weight; p.w1 = a->pre_weight;
    p.r = a->r; p.u = a->pre_weight ? a->normed : nullptr; p.rstd = a->rstd;
    p.dr = a->dr; p.du = a->dnormed; p.dx = a->dx; p.dres = a->dresidual; p.dgate = a->gate ? a->dgate : nullptr;
    return p;
}
// 16-byte pieces: every row starts at a multiple of 16 bytes
static bool block_norm_vec(const bissd_block_norm_args *a) {
    bool ok = a->width % 8 == 0;
    for (const void *p : {a->x, a->residual, a->gate, (const void *)a->r, (const void *)a->normed, a->dr, a->dnormed, (const void *)a->dx,
                          (const void *)a->dresidual, (const void *)a->dgate})
        ok = ok && aligned16(p);
    for (const int64_t s : {a->stride_x, a->stride_residual, a->stride_gate, a->stride_dr, a->stride_dnormed}) ok = ok && s % 8 == 0;
    return ok;
}
// Rows side by side in a block: up to 256 threads.
static int block_norm_threads(const bnorm::Params &p) { return p.threads_row * std::max(1, 256 / p.threads_row); }
// Blocks of the backward pass to an entry (rows that share a gate row whose gradient is wanted; else all rows): as many as are
// resident at two blocks of 256 threads an SM, shared by the entries, and no more than there are rows.
static void block_norm_split(const bnorm::Params &p, long long *entries, int *blocks) {
    *entries = p.gate_rows > 0 && p.dgate ? p.rows / p.gate_rows : 1;
    const long long rows = p.rows / *entries, per = block_norm_threads(p) / p.threads_row;
    const long long want = std::max<long long>(1, 148LL * std::max(1, 512 / block_norm_threads(p)) / *entries);
    *blocks = (int)std::min<long long>(want, (rows + per - 1) / per);
}

template <class T, class R> static int block_norm_forward_impl(const bissd_block_norm_args *a, cudaStream_t s) {
    const bnorm::Params p = block_norm_params(a);
    const int threads = block_norm_threads(p), per = threads / p.threads_row;
    const bool vec = block_norm_vec(a), big = threads > 512;
    const auto kernel = big ? (vec ? bnorm::block_norm_fwd<T, R, true, 1024> : bnorm::block_norm_fwd<T, R, false, 1024>)
                            : (vec ? bnorm::block_norm_fwd<T, R, true, 512> : bnorm::block_norm_fwd<T, R, false, 512>);
    const long long rows = (a->rows + per - 1) / per;
    const int grid = (int)std::min<long long>(rows, (long long)sm_count() * resident_blocks(kernel, threads, 0));
    BISSD_LAUNCH("block_norm_fwd", launch_pdl(kernel, grid, threads, 0, s, p));
    return BISSD_OK;
}
template <class T, class R> static int block_norm_backward_impl(const bissd_block_norm_args *a, float *part, cudaStream_t s) {
    bnorm::Params p = block_norm_params(a);
    const int threads = block_norm_threads(p), per = threads / p.threads_row;
    const bool vec = block_norm_vec(a), big = threads > 512;
    long long entries;
    block_norm_split(p, &entries, &p.blocks);
    if (entries * p.blocks > 0x7fffffffLL || (entries + 3) * ceil_div(p.D, 32) > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    p.part = part;
    const auto kernel = big ? (vec ? bnorm::block_norm_bwd<T, R, true, 1024> : bnorm::block_norm_bwd<T, R, false, 1024>)
                            : (vec ? bnorm::block_norm_bwd<T, R, true, 512> : bnorm::block_norm_bwd<T, R, false, 512>);
    const size_t smem = (size_t)(per - 1) * p.threads_row * bnorm::kCh * sizeof(float);
    BISSD_LAUNCH("block_norm_bwd", launch_pdl(kernel, (int)(entries * p.blocks), threads, smem, s, p));
    bnorm::SumParams q{};
    q.part = part; q.D = p.D; q.blocks = p.blocks; q.entries = (int)entries; q.w_dtype = p.w_dtype; q.g_dtype = a->dtype;
    q.dpre = a->dnormed ? a->dpre : nullptr; q.dpost = a->post_weight ? a->dpost : nullptr;
    q.dscale = a->scale_vector ? a->dscale : nullptr; q.dgate = p.gate_rows > 0 ? p.dgate : nullptr;
    if (q.dpre || q.dpost || q.dscale || q.dgate)
        BISSD_LAUNCH("block_norm_sums", launch_pdl(bnorm::block_norm_sums, (int)((3 + (q.dgate ? entries : 0)) * ceil_div(p.D, 32)),
                                                   dim3(32, 8), 0, s, q));
    return BISSD_OK;
}

// ---- the decay attention ---------------------------------------------------------------------------------------------
namespace {

struct Bump {                                                    // the workspace's arrays, one after another
    char *base;
    size_t used = 256;                                           // the status word's header
    template <class T> T *take(size_t n) {
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += align256(n * sizeof(T));
        return p;
    }
};

struct Sizes {
    int sequences, H, hk, N, P, lanes_n, lanes_p;                // lanes that share a column when S's rows are kdim, vdim
    long long tokens;
};

int power_lanes(int rows) {                                      // 32 rows a thread at most
    int l = 1;
    while (l * 32 < rows) l *= 2;
    return l;
}

int decay_check(const bissd_decay_args *a, bool backward) {
    if (!a) return BISSD_ERR_NULL;
    if (a->batch <= 0 || a->seqlen <= 0 || a->nheads <= 0 || a->nkheads <= 0 || a->nheads % a->nkheads || a->kdim <= 0 || a->kdim > 256 ||
        a->vdim <= 0 || a->vdim > 256 || a->nseq < 0 || (a->nseq > 0 && a->batch != 1))
        return BISSD_ERR_SHAPE;
    if (!dtype_ok(a->dtype) || !dtype_ok(a->g_dtype)) return BISSD_ERR_DTYPE;
    if ((long long)a->batch * a->seqlen > 0x7fffffffLL / 256) return BISSD_ERR_SHAPE;
    (void)backward;
    return BISSD_OK;
}
int decay_pointers(const bissd_decay_args *a, bool backward) {
    if (!a->q.ptr || !a->k.ptr || !a->v.ptr || !a->g.ptr || (a->nseq > 0 && !a->cu_seqlens)) return BISSD_ERR_NULL;
    if (!backward && !a->o) return BISSD_ERR_NULL;
    if (backward && (!a->dout.ptr || !a->dq || !a->dk || !a->dv)) return BISSD_ERR_NULL;
    return BISSD_OK;
}
Sizes sizes_of(const bissd_decay_args *a) {
    Sizes z;
    z.sequences = a->nseq > 0 ? a->nseq : a->batch;
    z.H = a->nheads; z.hk = a->nkheads; z.N = a->kdim; z.P = a->vdim;
    z.lanes_n = power_lanes(a->kdim); z.lanes_p = power_lanes(a->vdim);
    z.tokens = (long long)a->batch * a->seqlen;
    return z;
}

uni::Plan plan_of(const bissd_decay_args *a, int seg, Bump &ws, uni::PlanOut *out) {
    uni::Plan p{};
    p.packed = a->nseq > 0; p.L = a->seqlen; p.seg = seg;
    p.per_seq = ceil_div(a->seqlen, seg);
    p.most = p.packed ? p.per_seq + a->nseq : p.per_seq * a->batch;
    if (p.packed) {
        out->seg = seg; out->most = p.most;
        out->table = ws.take<int4>(p.most);
        out->first = ws.take<int>(a->nseq + 1);
        out->bounds = ws.take<int>(a->nseq + 1);
        p.table = out->table; p.first = out->first;
    }
    return p;
}

// Tokens to a segment on CUDA cores: long rows in as many as fill the SMs four times over, none under 256 tokens (what two more walks
// without outputs cost then); packed sequences in segments of 256.
int walk_segment(const bissd_decay_args *a, const Sizes &z) {
    if (a->nseq > 0) return 256;
    const long long blocks = (long long)a->batch * z.H * ceil_div(z.P * z.lanes_n, uni::kWalkThreads);
    const long long parts = std::max<long long>(1, 4 * 148 / blocks);
    return std::max(256, ceil_div((int)((a->seqlen + parts - 1) / parts), 256) * 256);
}

int launch_walk(int dtype, const uni::WalkParams &w, cudaStream_t s) {
    const int ipt = w.I <= 16 ? 16 : 32, cols = uni::kWalkThreads / w.lanes;
    const size_t smem = uni::walk_smem(w.lanes, ipt);
    const long long grid = (long long)w.plan.most * w.H * ceil_div(w.J, cols);
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    return by_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const auto kernel = ipt == 16 ? uni::decay_walk<T, 16> : uni::decay_walk<T, 32>;
        BISSD_ALLOW(kernel, smem);
        BISSD_LAUNCH(w.y ? "decay_walk" : "decay_walk_states", launch_pdl(kernel, (int)grid, uni::kWalkThreads, smem, s, w));
        return BISSD_OK;
    });
}
int launch_chain(const uni::ChainParams &c, cudaStream_t s) {
    const long long grid = (long long)c.nseq * c.H * ceil_div(c.per, 256);
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    BISSD_LAUNCH("decay_chain", launch_pdl(uni::decay_chain, (int)grid, 256, 0, s, c));
    return BISSD_OK;
}
int launch_plan(const bissd_decay_args *a, const uni::PlanOut &x, const uni::PlanOut *y, cudaStream_t s) {
    if (a->nseq == 0) return BISSD_OK;
    BISSD_LAUNCH("decay_plan", launch_pdl(uni::decay_plan, y ? 2 : 1, 1024, 0, s, a->cu_seqlens, (int)a->nseq, (int)a->seqlen, x, y ? *y : x));
    return BISSD_OK;
}
int launch_gaps(const bissd_decay_args *a, int dtype, void *out, int row, const int *bounds, cudaStream_t s) {
    if (a->nseq == 0 || !out) return BISSD_OK;
    return by_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        BISSD_LAUNCH("decay_gaps", launch_pdl(uni::decay_gaps<T>, 32, 256, 0, s, static_cast<T *>(out), (long long)row, row, (int)a->seqlen,
                                              bounds, (int)a->nseq));
        return BISSD_OK;
    });
}

struct Walks {                                                   // what the launches on CUDA cores share
    const bissd_decay_args *a;
    Sizes z;
    uni::Plan plan;
    uni::Vector q, k, v, dout;
    View g;
};
Walks walks_of(const bissd_decay_args *a, const uni::Plan &plan) {
    Walks w{a, sizes_of(a), plan, {view(a->q), 1}, {view(a->k), 1}, {view(a->v), 0}, {view(a->dout), 0}, view(a->g)};
    if (a->g_per_head) { w.g.sb = w.g.sl = 0; w.g.sh = 1; }
    return w;
}
// Rows of S from `av` (kdim where of_q), columns from `bv`.
uni::WalkParams walk_params(const Walks &w, const uni::Vector &av, const uni::Vector &bv, const uni::Vector &rv, bool reverse) {
    uni::WalkParams p{};
    p.plan = w.plan; p.H = w.z.H; p.hk = w.z.hk; p.reverse = reverse;
    const bool rows_k = av.of_q;                                 // S as stored, or its two sides exchanged
    p.I = rows_k ? w.z.N : w.z.P; p.J = rows_k ? w.z.P : w.z.N;
    p.lanes = rows_k ? w.z.lanes_n : w.z.lanes_p;
    p.si = rows_k ? w.z.P : 1; p.sj = rows_k ? 1 : w.z.P;
    p.a = av; p.b = bv; p.r = rv; p.g = w.g; p.g_dtype = w.a->g_dtype;
    p.a_scale = p.y_scale = 1.f;
    return p;
}

struct WalkSpace {                                               // the workspace of a pass on CUDA cores
    uni::Plan plan;
    uni::PlanOut table{};
    float *states, *decay;
    float *dstates, *ddecay, *final_, *dqh, *dkh, *flow, *dg_tokens;   // backward
};
WalkSpace walk_space(const bissd_decay_args *a, Bump &ws, bool backward) {
    const Sizes z = sizes_of(a);
    WalkSpace s{};
    s.plan = plan_of(a, walk_segment(a, z), ws, &s.table);
    const size_t states = (size_t)s.plan.most * z.H * z.N * z.P, decays = (size_t)s.plan.most * z.H;
    if (backward || s.plan.packed || s.plan.per_seq > 1) {
        s.states = ws.take<float>(states);
        s.decay = ws.take<float>(decays);
    }
    if (backward) {
        s.dstates = ws.take<float>(states);
        s.ddecay = ws.take<float>(decays);
        s.final_ = ws.take<float>((size_t)z.sequences * z.H * z.N * z.P);
        s.dqh = ws.take<float>((size_t)z.tokens * z.H * z.N);
        s.dkh = ws.take<float>((size_t)z.tokens * z.H * z.N);
        s.flow = ws.take<float>((size_t)z.tokens * z.H);
        if (a->g_per_head) s.dg_tokens = ws.take<float>((size_t)z.tokens * z.H);
    }
    return s;
}
uni::ChainParams chain_params(const Walks &w, bool reverse, const float *start, float *states, const float *decay, float *end) {
    uni::ChainParams c{};
    c.plan = w.plan; c.H = w.z.H; c.per = w.z.N * w.z.P; c.reverse = reverse; c.nseq = w.z.sequences;
    c.start = start; c.states = states; c.decay = decay; c.end = end; c.g = w.g; c.g_dtype = w.a->g_dtype;
    return c;
}

#define BISSD_DO(...)                       \
    do {                                    \
        const int rc_ = (__VA_ARGS__);      \
        if (rc_ != BISSD_OK) return rc_;    \
    } while (0)

int walk_forward(const bissd_decay_args *a, Bump &ws, cudaStream_t s) {
    const WalkSpace sp = walk_space(a, ws, false);
    const Walks w = walks_of(a, sp.plan);
    int *status = reinterpret_cast<int *>(ws.base);
    BISSD_DO(launch_plan(a, sp.table, nullptr, s));
    BISSD_DO(launch_gaps(a, a->dtype, a->o, w.z.H * w.z.P, sp.table.bounds, s));
    uni::WalkParams p = walk_params(w, w.k, w.v, w.q, false);
    p.status = status;
    if (sp.states) {                                             // each segment's own sum, then what enters each
        p.fin = sp.states; p.decay = sp.decay;
        BISSD_DO(launch_walk(a->dtype, p, s));
        BISSD_DO(launch_chain(chain_params(w, false, a->initial_state, sp.states, sp.decay, a->final_state), s));
        p.init = sp.states; p.fin = nullptr; p.decay = nullptr;
    } else {
        p.init = a->initial_state; p.fin = a->final_state;
    }
    p.y = a->o; p.y_dtype = a->dtype; p.y_scale = a->scale;
    p.y_batch = (long long)a->seqlen * w.z.H * w.z.P;
    return launch_walk(a->dtype, p, s);
}

int walk_backward(const bissd_decay_args *a, Bump &ws, cudaStream_t s) {
    const WalkSpace sp = walk_space(a, ws, true);
    const Walks w = walks_of(a, sp.plan);
    const Sizes &z = w.z;
    BISSD_DO(launch_plan(a, sp.table, nullptr, s));
    BISSD_DO(launch_gaps(a, a->dtype, a->dv, z.H * z.P, sp.table.bounds, s));
    if (a->dg && !a->g_per_head) BISSD_DO(launch_gaps(a, a->g_dtype, a->dg, z.H, sp.table.bounds, s));
    BISSD_DO(launch_gaps(a, BISSD_F32, sp.dg_tokens, z.H, sp.table.bounds, s));
    BISSD_DO(launch_gaps(a, BISSD_F32, sp.dqh, z.H * z.N, sp.table.bounds, s));
    BISSD_DO(launch_gaps(a, BISSD_F32, sp.dkh, z.H * z.N, sp.table.bounds, s));
    // states that enter the segments from the left, gradients that enter them from the right
    uni::WalkParams p = walk_params(w, w.k, w.v, w.q, false);
    p.status = reinterpret_cast<int *>(ws.base);
    p.fin = sp.states; p.decay = sp.decay;
    BISSD_DO(launch_walk(a->dtype, p, s));
    BISSD_DO(launch_chain(chain_params(w, false, a->initial_state, sp.states, sp.decay, a->dfinal_state ? sp.final_ : nullptr), s));
    p = walk_params(w, w.q, w.dout, w.k, true);
    p.a_scale = a->scale; p.fin = sp.dstates; p.decay = sp.ddecay;
    BISSD_DO(launch_walk(a->dtype, p, s));
    BISSD_DO(launch_chain(chain_params(w, true, a->dfinal_state, sp.dstates, sp.ddecay, a->dinitial_state), s));
    // dv, and for each head dk and dq
    p.fin = nullptr; p.decay = nullptr; p.init = sp.dstates;
    p.y = a->dv; p.y_dtype = a->dtype; p.y_batch = (long long)a->seqlen * z.H * z.P;
    BISSD_DO(launch_walk(a->dtype, p, s));
    p = walk_params(w, w.dout, w.q, w.v, true);
    p.a_scale = a->scale; p.init = sp.dstates;
    p.y = sp.dkh; p.y_dtype = BISSD_F32; p.y_batch = (long long)a->seqlen * z.H * z.N;
    BISSD_DO(launch_walk(a->dtype, p, s));
    p = walk_params(w, w.v, w.k, w.dout, false);
    p.y_scale = a->scale; p.init = sp.states;
    p.y = sp.dqh; p.y_dtype = BISSD_F32; p.y_batch = (long long)a->seqlen * z.H * z.N;
    BISSD_DO(launch_walk(a->dtype, p, s));
    uni::FinishParams f{};
    f.L = a->seqlen; f.H = z.H; f.hk = z.hk; f.N = z.N; f.tokens = z.tokens; f.q = w.q.v; f.k = w.k.v;
    f.dqh = sp.dqh; f.dkh = sp.dkh; f.dq = a->dq; f.dk = a->dk; f.flow = sp.flow;
    const long long grid = (z.tokens * z.hk + 7) / 8;
    if (grid > 0x7fffffffLL || (long long)sp.plan.most * z.H > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    BISSD_DO(by_dtype(a->dtype, [&](auto t) -> int {
        BISSD_LAUNCH("decay_finish", launch_pdl(uni::decay_finish<decltype(t)>, (int)grid, 256, 0, s, f));
        return BISSD_OK;
    }));
    if (!a->dg) return BISSD_OK;
    uni::DecayGradParams d{};
    d.plan = sp.plan; d.H = z.H; d.per = z.N * z.P; d.g_dtype = a->g_dtype; d.L = a->seqlen;
    d.out_dtype = a->g_per_head ? BISSD_F32 : a->g_dtype;
    d.flow = sp.flow; d.enter = sp.states; d.denter = sp.dstates; d.final_ = sp.final_; d.dfinal = a->dfinal_state; d.g = w.g;
    d.dg = a->g_per_head ? sp.dg_tokens : a->dg;
    BISSD_LAUNCH("decay_dg", launch_pdl(uni::decay_dg, sp.plan.most * z.H, 256, 0, s, d));
    if (a->g_per_head)
        BISSD_LAUNCH("decay_dg_heads", launch_pdl(uni::decay_dg_heads, z.H, 1024, 0, s, (const float *)sp.dg_tokens, z.tokens, z.H, a->dg, (int)a->g_dtype));
    return BISSD_OK;
}

}  // namespace

extern "C" {

int bissd_decay_workspace_bytes(const bissd_decay_args *a, size_t *fwd_bytes, size_t *bwd_bytes) {
    const int rc = decay_check(a, false);
    if (rc != BISSD_OK) return rc;
    if (fwd_bytes) {
        Bump b{nullptr};
        walk_space(a, b, false);
        *fwd_bytes = b.used;
    }
    if (bwd_bytes) {
        Bump b{nullptr};
        walk_space(a, b, true);
        *bwd_bytes = b.used;
    }
    return BISSD_OK;
}

int bissd_decay_forward(const bissd_decay_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    BISSD_DO(bissd_decay_workspace_bytes(a, &need, nullptr));
    BISSD_DO(decay_pointers(a, false));
    if (!workspace || workspace_bytes < need) return BISSD_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return BISSD_ERR_ALIGN;
    BISSD_DO(check_device());
    Bump b{static_cast<char *>(workspace)};
    return walk_forward(a, b, static_cast<cudaStream_t>(stream));
}

int bissd_decay_backward(const bissd_decay_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    BISSD_DO(bissd_decay_workspace_bytes(a, nullptr, &need));
    BISSD_DO(decay_pointers(a, true));
    if (!workspace || workspace_bytes < need) return BISSD_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return BISSD_ERR_ALIGN;
    BISSD_DO(check_device());
    Bump b{static_cast<char *>(workspace)};
    return walk_backward(a, b, static_cast<cudaStream_t>(stream));
}

int bissd_decay_step(const bissd_decay_step_args *a, void *stream) {
    BISSD_DO(step_check(a));
    BISSD_DO(check_device());
    return step_launch(a, static_cast<cudaStream_t>(stream));
}

int bissd_block_norm_workspace_bytes(const bissd_block_norm_args *a, size_t *bwd_bytes) {
    BISSD_DO(block_norm_check(a, false) == BISSD_ERR_NULL ? (a ? BISSD_OK : BISSD_ERR_NULL) : block_norm_check(a, false));
    long long entries;
    int blocks;
    const bnorm::Params p = block_norm_params(a);
    block_norm_split(p, &entries, &blocks);
    if (bwd_bytes) *bwd_bytes = align256((size_t)entries * blocks * 4 * p.D * sizeof(float));
    return BISSD_OK;
}

int bissd_block_norm_forward(const bissd_block_norm_args *a, void *stream) {
    BISSD_DO(block_norm_check(a, false));
    BISSD_DO(check_device());
    const auto s = static_cast<cudaStream_t>(stream);
    return by_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        return a->r_dtype == a->dtype ? block_norm_forward_impl<T, T>(a, s) : block_norm_forward_impl<T, float>(a, s);
    });
}

int bissd_block_norm_backward(const bissd_block_norm_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    BISSD_DO(block_norm_check(a, true));
    size_t need = 0;
    BISSD_DO(bissd_block_norm_workspace_bytes(a, &need));
    if (!workspace || workspace_bytes < need) return BISSD_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return BISSD_ERR_ALIGN;
    BISSD_DO(check_device());
    const auto s = static_cast<cudaStream_t>(stream);
    return by_dtype(a->dtype, [&](auto t) -> int {
        using T = decltype(t);
        float *part = static_cast<float *>(workspace);
        return a->r_dtype == a->dtype ? block_norm_backward_impl<T, T>(a, part, s) : block_norm_backward_impl<T, float>(a, part, s);
    });
}

}  // extern "C"

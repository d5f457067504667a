// C ABI of the causal linear attention with a decay for each head and of its single-token form.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "host.cuh"
#include "uni_plan.cuh"
#include "uni_step.cuh"
#include "uni_tc.cuh"
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

constexpr int kSms = 148;                                        // of the GPU this is written for

struct Sizes {
    int sequences, H, hk, N, P, lanes_n, lanes_p;                // lanes that share a column when S's rows are kdim, vdim
    long long tokens;
};

// Lanes that share a column of `rows` rows: enough for 32 rows a thread at most, and as many as leave no thread of a block without
// a column, down to four rows a thread (a walk is a chain of tokens: us for 253 tokens of 4 heads of 16 x 32 fp32, one lane a column
// 126, four 56).
int walk_lanes(int rows, int columns) {
    int l = 1;
    while (l * 32 < rows) l *= 2;
    while (l < 32 && l * 4 < rows && uni::kWalkThreads / l > columns) l *= 2;
    return l;
}
int walk_rows(int rows, int lanes) {                             // rows a thread
    int n = 4;
    while (n * lanes < rows) n *= 2;
    return n;
}

int decay_check(const bissd_decay_args *a) {
    if (!a) return BISSD_ERR_NULL;
    if (a->batch <= 0 || a->seqlen <= 0 || a->nheads <= 0 || a->nkheads <= 0 || a->nheads % a->nkheads || a->kdim <= 0 || a->kdim > 256 ||
        a->vdim <= 0 || a->vdim > 256 || a->nseq < 0 || (a->nseq > 0 && a->batch != 1))
        return BISSD_ERR_SHAPE;
    if (!dtype_ok(a->dtype) || !dtype_ok(a->g_dtype)) return BISSD_ERR_DTYPE;
    if ((long long)a->batch * a->seqlen > 0x7fffffffLL / 256) return BISSD_ERR_SHAPE;
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
    z.lanes_n = walk_lanes(a->kdim, a->vdim); z.lanes_p = walk_lanes(a->vdim, a->kdim);
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

// Tokens to a segment on CUDA cores: rows in as many as fill the SMs four times over, but a token takes 0.2 us in a block, twice, and a
// segment 0.25 in the chain: none under the root of 0.6 tokens, or under 32, and rows of up to 96 in one (two launches fewer).  With 64
// at least and one up to 192, us: 4 heads of 16 x 32 fp32, 192 tokens 26.5 for 11.7, 253 17.5 for 12.1; 24 of 112 x 128, 128
// tokens 46 for 51, 400 148 for 103.  The same for packed sequences: 2048 tokens of 8, 8 heads of 64 x 64, in segments of 256 171, in
// these 113.
int walk_segment(const bissd_decay_args *a, const Sizes &z) {
    const long long blocks = (long long)a->batch * z.H * ceil_div(z.P * z.lanes_n, uni::kWalkThreads);
    const long long parts = std::max<long long>(1, 4 * kSms / blocks);
    const int least = std::max(32, (int)std::sqrt(0.6 * a->seqlen)), seg = std::max(least, (int)((a->seqlen + parts - 1) / parts));
    return a->seqlen <= 96 || parts == 1 ? a->seqlen : ceil_div(seg, 16) * 16;
}

template <class T, int Y> auto walk_kernel(int ipt) {
    return ipt == 4 ? uni::decay_walk<T, 4, Y> : ipt == 8 ? uni::decay_walk<T, 8, Y> : ipt == 16 ? uni::decay_walk<T, 16, Y> : uni::decay_walk<T, 32, Y>;
}
int launch_walk(int dtype, const uni::WalkParams &w, cudaStream_t s) {
    const int ipt = walk_rows(w.I, w.lanes), cols = uni::kWalkThreads / w.lanes;
    const size_t smem = uni::walk_smem(w.lanes, ipt);
    const long long grid = (long long)w.plan.most * w.H * ceil_div(w.J, cols);
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    return by_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const auto kernel = !w.y ? walk_kernel<T, uni::kStates>(ipt) : w.others ? walk_kernel<T, uni::kOthers>(ipt) : walk_kernel<T, uni::kOutputs>(ipt);
        BISSD_ALLOW(kernel, smem);
        BISSD_LAUNCH(w.y ? "decay_walk" : "decay_walk_states", launch_pdl(kernel, (int)grid, uni::kWalkThreads, smem, s, w));
        return BISSD_OK;
    });
}
// out: a forward pass's, or dv; dk and dq NULL in a forward pass.
int launch_walks_again(uni::WalkParams out, const uni::WalkParams *dk, const uni::WalkParams *dq, cudaStream_t s) {
    uni::WalkParams w[3] = {out, dk ? *dk : out, dq ? *dq : out};
    size_t smem = 0;
    long long blocks[3] = {}, all = 0;
    for (int i = 0; i < (dk ? 3 : 1); ++i) {
        w[i].lanes = 1;
        while (w[i].lanes * uni::kAgainRows < w[i].I) w[i].lanes *= 2;
        smem = std::max(smem, uni::walk_smem(w[i].lanes, uni::kAgainRows));
        all += blocks[i] = (long long)w[i].plan.most * w[i].H * ceil_div(w[i].J, uni::kWalkThreads / w[i].lanes);
    }
    if (all > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    BISSD_ALLOW(uni::decay_walks_again<__half>, smem);
    BISSD_LAUNCH("decay_walks_again", launch_pdl(uni::decay_walks_again<__half>, (int)std::min<long long>(all, 4 * kSms), uni::kWalkThreads, smem, s, w[0], w[1], w[2],
                                                 (int)blocks[0], (int)blocks[1], (int)all));
    return BISSD_OK;
}
int launch_chain(const uni::ChainParams &c, cudaStream_t s) {
    const bool quads = c.per % 4 == 0 && aligned16(c.start) && aligned16(c.states) && aligned16(c.end);
    const long long grid = (long long)c.nseq * c.H * ceil_div(c.per, quads ? 1024 : 256);
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    BISSD_LAUNCH("decay_chain", launch_pdl(quads ? uni::decay_chain<4> : uni::decay_chain<1>, (int)grid, 256, 0, s, c));
    return BISSD_OK;
}
// What packed sequences leave over: rows of outputs that belong to none of them, and the states of those without a token.
struct Rest {
    uni::RestParams p{};
    void rows(void *out, int dtype, long long elems) {
        if (!out) return;
        p.out[p.outs] = static_cast<char *>(out);
        p.bytes[p.outs++] = elems * (long long)dtype_size(dtype);
    }
    // The tables of segments, and what they leave over.
    int launch(const bissd_decay_args *a, const uni::PlanOut &x, const uni::PlanOut *y, cudaStream_t s) {
        if (a->nseq == 0) return BISSD_OK;
        p.L = a->seqlen; p.nseq = a->nseq;
        p.per = (long long)a->nheads * a->kdim * a->vdim;
        const int tables = y ? 2 : 1, others = a->nseq <= uni::kNear ? kSms : 0;
        BISSD_LAUNCH("decay_plan", launch_pdl(uni::decay_plan, tables + others, 1024, 0, s, a->cu_seqlens, (int)a->nseq, (int)a->seqlen, x, y ? *y : x,
                                              tables, p));
        if (!others) BISSD_LAUNCH("decay_rest", launch_pdl(uni::decay_rest, kSms, 1024, 0, s, p, (const int *)x.bounds));
        return BISSD_OK;
    }
};

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
    float *dstates, *ddecay, *final_, *dqh, *dkh, *into, *from, *dg_tokens;   // backward
};
void gradient_space(const Sizes &z, Bump &ws, WalkSpace &s) {    // of walk_gradients
    s.final_ = ws.take<float>((size_t)z.sequences * z.H * z.N * z.P);
    s.dqh = ws.take<float>((size_t)z.tokens * z.H * z.N);
    s.dkh = ws.take<float>((size_t)z.tokens * z.H * z.N);
    s.into = ws.take<float>((size_t)z.tokens * z.H);
    s.from = ws.take<float>((size_t)z.tokens * z.H);
}
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
        gradient_space(z, ws, s);
        if (a->g_per_head) s.dg_tokens = ws.take<float>((size_t)z.tokens * z.H);
    }
    return s;
}
uni::ChainParams chain_params(const Walks &w, bool reverse, const float *start, float *states, const float *decay, float *end) {
    uni::ChainParams c{};
    c.plan = w.plan; c.H = w.z.H; c.per = w.z.N * w.z.P; c.reverse = reverse; c.nseq = w.z.sequences;
    c.start = start; c.states = states; c.decay = decay; c.end = end; c.first_decay = reverse; c.g = w.g; c.g_dtype = w.a->g_dtype;
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
    Rest rest;
    rest.rows(a->o, a->dtype, w.z.H * w.z.P);
    BISSD_DO(rest.launch(a, sp.table, nullptr, s));
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

// dv, and for each head dk and dq without the tokens' own pairs, and from these dq, dk and dg; given the states that enter the segments from
// the left and the gradients that enter them from the right (NULL: zeros).
int walk_gradients(const Walks &w, const WalkSpace &sp, const float *states, const float *dstates, const int *bounds, float *dinitial, const int *again,
                   cudaStream_t s) {
    const bissd_decay_args *a = w.a;
    const Sizes &z = w.z;
    uni::WalkParams dv = walk_params(w, w.q, w.dout, w.k, true), dk = walk_params(w, w.dout, w.q, w.v, true), dq = walk_params(w, w.v, w.k, w.dout, false);
    dv.a_scale = dk.a_scale = dq.y_scale = a->scale;
    dv.init = dk.init = dstates;
    dq.init = states;
    dv.again = dk.again = dq.again = again;
    dv.y = a->dv; dv.y_dtype = a->dtype; dv.y_batch = (long long)a->seqlen * z.H * z.P;
    dk.y = sp.dkh; dq.y = sp.dqh;
    dk.others = dq.others = 1;
    dk.y_dtype = dq.y_dtype = BISSD_F32;
    dk.y_batch = dq.y_batch = (long long)a->seqlen * z.H * z.N;
    dv.fin = dinitial; dv.first_decay = dinitial != nullptr;
    dq.fin = a->dg && a->dfinal_state ? sp.final_ : nullptr;
    if (again) {
        BISSD_DO(launch_walks_again(dv, &dk, &dq, s));
    } else {
        for (const uni::WalkParams *p : {&dv, &dk, &dq}) BISSD_DO(launch_walk(a->dtype, *p, s));
    }
    uni::FinishParams f{};
    f.L = a->seqlen; f.H = z.H; f.hk = z.hk; f.N = z.N; f.P = z.P; f.tokens = z.tokens; f.scale = a->scale;
    f.q = w.q.v; f.k = w.k.v; f.v = w.v.v; f.dout = w.dout.v; f.bounds = bounds; f.nseq = a->nseq;
    f.dqh = sp.dqh; f.dkh = sp.dkh; f.dq = a->dq; f.dk = a->dk; f.again = again;
    if (a->dg) { f.into = sp.into; f.from = sp.from; }
    const long long all = (z.tokens * (z.hk + (a->dg ? z.H : 0)) + 7) / 8, grid = again ? std::min<long long>(all, kSms) : all;
    if (grid > 0x7fffffffLL || (long long)w.plan.most * z.H > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    BISSD_DO(by_dtype(a->dtype, [&](auto t) -> int {
        BISSD_LAUNCH("decay_finish", launch_pdl(uni::decay_finish<decltype(t)>, (int)grid, 256, 0, s, f));
        return BISSD_OK;
    }));
    if (!a->dg) return BISSD_OK;
    uni::DecayGradParams d{};
    d.plan = w.plan; d.H = z.H; d.per = z.N * z.P; d.g_dtype = a->g_dtype; d.L = a->seqlen;
    d.out_dtype = a->g_per_head ? BISSD_F32 : a->g_dtype;
    d.into = sp.into; d.from = sp.from; d.enter = states; d.denter = dstates; d.final_ = sp.final_; d.dfinal = a->dfinal_state; d.g = w.g;
    d.dg = a->g_per_head ? sp.dg_tokens : a->dg; d.again = again;
    BISSD_LAUNCH("decay_dg", launch_pdl(uni::decay_dg, w.plan.most * z.H, 256, 0, s, d));
    return BISSD_OK;
}
int launch_dg_heads(const bissd_decay_args *a, const float *dg_tokens, const int *bounds, cudaStream_t s) {
    BISSD_LAUNCH("decay_dg_heads", launch_pdl(uni::decay_dg_heads, (int)a->nheads, 1024, 0, s, dg_tokens, (long long)a->batch * a->seqlen, (int)a->nheads, a->dg,
                                              (int)a->g_dtype, bounds, (int)a->nseq));
    return BISSD_OK;
}

int walk_backward(const bissd_decay_args *a, Bump &ws, cudaStream_t s) {
    const WalkSpace sp = walk_space(a, ws, true);
    const Walks w = walks_of(a, sp.plan);
    const Sizes &z = w.z;
    Rest rest;
    rest.rows(a->dv, a->dtype, z.H * z.P);
    if (!a->g_per_head) rest.rows(a->dg, a->g_dtype, z.H);
    BISSD_DO(rest.launch(a, sp.table, nullptr, s));
    // states that enter the segments from the left, gradients that enter them from the right
    uni::WalkParams p = walk_params(w, w.k, w.v, w.q, false);
    p.status = reinterpret_cast<int *>(ws.base);
    p.fin = sp.states; p.decay = sp.decay;
    BISSD_DO(launch_walk(a->dtype, p, s));
    BISSD_DO(launch_chain(chain_params(w, false, a->initial_state, sp.states, sp.decay, nullptr), s));
    p = walk_params(w, w.q, w.dout, w.k, true);
    p.a_scale = a->scale; p.fin = sp.dstates; p.decay = sp.ddecay;
    BISSD_DO(launch_walk(a->dtype, p, s));
    BISSD_DO(launch_chain(chain_params(w, true, a->dfinal_state, sp.dstates, sp.ddecay, a->dinitial_state), s));
    BISSD_DO(walk_gradients(w, sp, sp.states, sp.dstates, sp.table.bounds, nullptr, nullptr, s));
    return a->dg && a->g_per_head ? launch_dg_heads(a, sp.dg_tokens, sp.table.bounds, s) : BISSD_OK;
}

using tc::make_map2;
using tc::make_map4;

// ---- on the tensor cores ----------------------------------------------------------------------------------------------

// 16-bit types with head sizes and rows that 16-byte loads fit, a positive scale (it is added to the decays' logarithms).
bool tc_sizes(const bissd_decay_args *a) {
    return a->dtype != BISSD_F32 && a->kdim % 8 == 0 && a->kdim <= 128 && a->vdim % 8 == 0 && a->scale > 0.f && std::isfinite(a->scale);
}
bool tc_tensor(const bissd_tensor &t, long long batch, long long seq, long long heads) {
    auto fits = [](long long stride, long long n) { return n == 1 || (stride > 0 && stride % 8 == 0 && stride < (1LL << 38)); };
    return aligned16(t.ptr) && fits(t.stride_batch, batch) && fits(t.stride_seq, seq) && fits(t.stride_head, heads);
}
bool tc_inputs(const bissd_decay_args *a) {
    return tc_sizes(a) && tc_tensor(a->q, a->batch, a->seqlen, a->nkheads) && tc_tensor(a->k, a->batch, a->seqlen, a->nkheads) &&
           tc_tensor(a->v, a->batch, a->seqlen, a->nheads);
}
bool tc_forward_ok(const bissd_decay_args *a) { return tc_inputs(a) && aligned16(a->o); }

struct TcSpace {
    int NT, PB;
    uni::Plan seg, chunk;
    uni::PlanOut seg_table{}, chunk_table{};
    bool split;                                                  // sequences in several segments, or packed
    uni::Again again{};                                          // fp16
    float *dg_tokens;                                            // backward, one decay for each head
    size_t kept;                                                 // bytes of the workspace that what is done again does not write over
    uint16_t *tiles;                                              // states as 16-bit tiles
    float *states, *decay;
};

// Tokens to a segment of the walk over the chunks, a block for each (segment, head, 64 columns), two blocks an SM.  A walk in pieces
// needs each piece's own sum first and a chain over them, so it pays where rows are long and heads few; packed sequences are taken
// to be up to three times as long as their mean.  us, measured: a step of the walk 2.2, of one for exact states 2.6, a block's start 6, a
// chain 6 (3 rows of 8 chunks, 32 blocks each: 62 in two pieces, 22 in one; 512 chunks of 32 heads: 277 in 9 pieces, 1130 in one by
// these figures).
int tc_segment(const bissd_decay_args *a, int PB) {
    const int chunks = ceil_div(a->seqlen, unitc::kQ);
    const double heads = (double)a->nheads * PB, work = (double)a->batch * chunks * heads / (2 * kSms);
    const int longest = a->nseq > 0 ? std::min(chunks, ceil_div(3 * chunks, a->nseq)) : chunks;
    int best = chunks;
    double least = std::max<double>(longest, work) * 2.2 + 6;
    for (int parts = 2; parts <= std::min(longest / 4, 128); ++parts) {
        const int steps = ceil_div(longest, parts);
        const double segments = ((double)a->batch * ceil_div(chunks, steps) + a->nseq) * heads, rounds = std::ceil(segments / (2 * kSms));
        const double time = rounds * (steps * (2.2 + 2.6) + 2 * 6) + 6 + segments * a->kdim * unitc::kP * 12 / 5e6;   // a chain moves 12 bytes a value
        if (time < least) {
            least = time;
            best = steps;
        }
    }
    return best * unitc::kQ;
}
size_t tc_tile_values(const bissd_decay_args *a, const TcSpace &t) { return (size_t)t.chunk.most * a->nheads * t.PB * t.NT * unitc::kP; }
TcSpace tc_space(const bissd_decay_args *a, Bump &ws, bool backward) {
    TcSpace t{};
    t.NT = a->kdim <= 64 ? 64 : 128;
    t.PB = ceil_div(a->vdim, unitc::kP);
    t.chunk = plan_of(a, unitc::kQ, ws, &t.chunk_table);
    t.seg = plan_of(a, tc_segment(a, t.PB), ws, &t.seg_table);
    t.split = t.seg.per_seq > 1;
    if (a->dtype == BISSD_F16) {
        t.again.H = a->nheads; t.again.seg = t.seg; t.again.per_segment = a->nheads * t.PB;
        t.again.flags = ws.take<int>(1 + (size_t)(a->nseq > 0 ? a->nseq : a->batch) * a->nheads);
        t.again.bad = ws.take<int>((size_t)t.seg.most * t.again.per_segment);
    }
    if (backward && a->g_per_head) t.dg_tokens = ws.take<float>((size_t)a->batch * a->seqlen * a->nheads);
    t.kept = ws.used;
    t.tiles = a->saved ? static_cast<uint16_t *>(a->saved) : ws.take<uint16_t>(tc_tile_values(a, t));
    if (t.split && !(a->saved && backward)) {
        t.states = ws.take<float>((size_t)t.seg.most * a->nheads * a->kdim * a->vdim);
        t.decay = ws.take<float>((size_t)t.seg.most * a->nheads);
    }
    return t;
}
unitc::Heads tc_heads(const bissd_decay_args *a, int PB) {
    unitc::Heads h{};
    h.H = a->nheads; h.hk = a->nkheads; h.N = a->kdim; h.P = a->vdim; h.PB = PB;
    h.g = view(a->g); h.g_dtype = a->g_dtype;
    if (a->g_per_head) { h.g.sb = h.g.sl = 0; h.g.sh = 1; }
    h.log_scale = std::log2(a->scale);
    return h;
}
bool tc_map(CUtensorMap *m, const bissd_decay_args *a, const bissd_tensor &t, int inner, int heads) {
    auto bytes = [](long long stride, int n) { return n == 1 ? 16ULL : (unsigned long long)stride * 2; };
    return make_map4(m, a->dtype, t.ptr, {(unsigned long long)inner, (unsigned long long)heads, (unsigned long long)a->seqlen, (unsigned long long)a->batch},
                     {bytes(t.stride_head, heads), bytes(t.stride_seq, a->seqlen), bytes(t.stride_batch, a->batch)}, {64, 1, unitc::kQ, 1});
}

template <class T> auto states_kernel(int NT, bool exact) {
    return NT == 64 ? (exact ? unitc::decay_states<T, 64, true> : unitc::decay_states<T, 64, false>)
                    : (exact ? unitc::decay_states<T, 128, true> : unitc::decay_states<T, 128, false>);
}
template <class T> auto chunks_kernel(int NT) { return NT == 64 ? unitc::decay_chunks<T, 64> : unitc::decay_chunks<T, 128>; }
template <class T> auto grads_kernel(int NT, bool dg) {
    return NT == 64 ? (dg ? unitc::decay_grads<T, 64, true> : unitc::decay_grads<T, 64, false>)
                    : (dg ? unitc::decay_grads<T, 128, true> : unitc::decay_grads<T, 128, false>);
}
// The states that enter the chunks (or the gradients, backwards), as 16-bit tiles; those that enter and leave the sequences in fp32.
int tc_states(const bissd_decay_args *a, TcSpace &t, const CUtensorMap &rows, const CUtensorMap &cols, const CUtensorMap &tiles, bool reverse,
              const float *start, float *end, float *states, float *decay, int *status, bool clear, bool first, cudaStream_t s) {
    unitc::StatesParams p{};
    p.h = tc_heads(a, t.PB);
    p.seg = t.seg; p.chunk = t.chunk; p.reverse = reverse; p.status = status;
    p.clear = clear;
    p.again = first ? t.again.flags : nullptr;
    const long long grid = (long long)t.seg.most * a->nheads * t.PB;
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    if (end) t.again.bads = t.again.flags ? (int)grid : 0;
    auto launch = [&](const char *name, bool exact) -> int {
        const auto kernel = a->dtype == BISSD_BF16 ? states_kernel<__nv_bfloat16>(t.NT, exact) : states_kernel<__half>(t.NT, exact);
        const size_t smem = unitc::states_smem(t.NT, exact);
        p.bad = exact ? t.again.bad : nullptr;
        BISSD_ALLOW(kernel, smem);
        BISSD_LAUNCH(name, launch_pdl(kernel, (int)grid, unitc::kStatesThreads, smem, s, p, rows, cols, tiles));
        p.clear = 0;
        p.again = nullptr;
        return BISSD_OK;
    };
    if (t.split) {
        p.fin = states; p.decay = decay;
        BISSD_DO(launch("decay_states_own", end != nullptr));
        uni::ChainParams c{};
        c.plan = t.seg; c.H = a->nheads; c.per = a->kdim * a->vdim; c.reverse = reverse; c.nseq = a->nseq > 0 ? a->nseq : a->batch;
        c.start = start; c.states = states; c.decay = decay; c.end = end;
        BISSD_DO(launch_chain(c, s));
        p.init = states; p.fin = p.decay = nullptr;
    } else {
        p.init = start; p.fin = end; p.by_seq = 1;
    }
    p.tiles = 1;
    return launch("decay_states", !t.split && end != nullptr);
}
bool tc_tile_map(CUtensorMap *m, const bissd_decay_args *a, const TcSpace &t, const uint16_t *tiles) {
    return make_map2(m, a->dtype, tiles, unitc::kP, (unsigned long long)t.chunk.most * a->nheads * t.PB * t.NT, unitc::kP, t.NT);
}

// Sequences as they are walked again on CUDA cores: one segment each.
Walks again_walks(const bissd_decay_args *a, const TcSpace &t) {
    uni::Plan p{};
    p.packed = a->nseq > 0; p.L = p.seg = a->seqlen; p.per_seq = 1;
    p.most = a->nseq > 0 ? a->nseq : a->batch;
    p.bounds = t.chunk_table.bounds;
    return walks_of(a, p);
}

constexpr double kChunkStart = 2.0;                              // a block's start and the product q.k, in tiles of v

int tc_forward(const bissd_decay_args *a, Bump &ws, cudaStream_t s) {
    TcSpace t = tc_space(a, ws, false);
    int *status = reinterpret_cast<int *>(ws.base);
    if ((long long)t.chunk.most * a->nheads * t.PB * t.NT > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    CUtensorMap q, k, v, tiles;
    if (!tc_map(&q, a, a->q, a->kdim, a->nkheads) || !tc_map(&k, a, a->k, a->kdim, a->nkheads) || !tc_map(&v, a, a->v, a->vdim, a->nheads) ||
        !tc_tile_map(&tiles, a, t, t.tiles))
        return note_cuda(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    Rest rest;
    rest.p.status = status;
    rest.rows(a->o, a->dtype, a->nheads * a->vdim);
    rest.p.start = a->initial_state;
    rest.p.end = t.split ? nullptr : a->final_state;             // the chain sees to them otherwise
    BISSD_DO(rest.launch(a, t.chunk_table, &t.seg_table, s));
    BISSD_DO(tc_states(a, t, k, v, tiles, false, a->initial_state, a->final_state, t.states, t.decay, status, a->nseq == 0, true, s));
    unitc::ChunksParams p{};
    p.h = tc_heads(a, t.PB);
    p.chunk = t.chunk; p.o = a->o; p.status = status; p.again = t.again;
    // blocks a (chunk, head of q): as many as fill two blocks an SM, in the fewest rounds
    const int tiles_v = a->nheads / a->nkheads * t.PB;
    const long long items = (long long)t.chunk.most * a->nkheads, slots = 2 * kSms;
    double best = 0;
    for (int parts = 1; parts <= tiles_v; ++parts) {
        const int vpc = ceil_div(tiles_v, parts);
        const double time = (double)((items * ceil_div(tiles_v, vpc) + slots - 1) / slots) * (kChunkStart + vpc);
        if (parts == 1 || time < best) {
            best = time;
            p.vpc = vpc;
        }
    }
    p.parts = ceil_div(tiles_v, p.vpc);
    const auto kernel = a->dtype == BISSD_BF16 ? chunks_kernel<__nv_bfloat16>(t.NT) : chunks_kernel<__half>(t.NT);
    const size_t smem = unitc::chunks_smem(t.NT);
    const long long grid = (long long)t.chunk.most * a->nkheads * p.parts;
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    BISSD_ALLOW(kernel, smem);
    BISSD_LAUNCH("decay_chunks", launch_pdl(kernel, (int)grid, 256, smem, s, p, q, k, v, tiles));
    if (!t.again.flags) return BISSD_OK;
    const Walks w = again_walks(a, t);
    uni::WalkParams f = walk_params(w, w.k, w.v, w.q, false);
    f.again = t.again.flags;
    f.init = a->initial_state; f.fin = a->final_state;
    f.y = a->o; f.y_dtype = a->dtype; f.y_scale = a->scale;
    f.y_batch = (long long)a->seqlen * w.z.H * w.z.P;
    return launch_walks_again(f, nullptr, nullptr, s);
}

struct TcGradSpace {
    TcSpace t;
    uint16_t *grads;                                                 // tiles of the states' gradients
    float *gstates, *gdecay;
    int vpc, parts;
    float *part;
};
TcGradSpace tc_grad_space(const bissd_decay_args *a, Bump &ws) {
    TcGradSpace g{};
    g.t = tc_space(a, ws, true);
    const long long tokens = (long long)a->batch * a->seqlen;
    g.grads = ws.take<uint16_t>(tc_tile_values(a, g.t));
    if (g.t.split) {
        g.gstates = ws.take<float>((size_t)g.t.seg.most * a->nheads * a->kdim * a->vdim);
        g.gdecay = ws.take<float>((size_t)g.t.seg.most * a->nheads);
    }
    // Heads that share q and k are walked by one block, or by several: what takes the fewest rounds of one block an SM, a block's start
    // being worth 1.5 tiles (of 6 us), and the parts of dq and dk 16 bytes a value at 5 TB/s.
    const int R = a->nheads / a->nkheads;
    const long long items = (long long)g.t.chunk.most * a->nkheads;
    double best = 0;
    for (int parts = 1; parts <= R; ++parts) {
        const int heads = ceil_div(R, parts), real = ceil_div(R, heads);
        const double rounds = (double)((items * real + kSms - 1) / kSms), sums = real > 1 ? 16.0 * real * tokens * a->nkheads * a->kdim / 30e6 : 0;
        const double time = rounds * (heads * g.t.PB + 1.5) + sums;
        if (parts == 1 || time < best) {
            best = time;
            g.vpc = heads * g.t.PB;
            g.parts = real;
        }
    }
    if (g.parts > 1) g.part = ws.take<float>((size_t)2 * g.parts * tokens * a->nkheads * a->kdim);
    return g;
}
bool tc_backward_ok(const bissd_decay_args *a) {
    return tc_inputs(a) && tc_tensor(a->dout, a->batch, a->seqlen, a->nheads) && aligned16(a->dq) && aligned16(a->dk) && aligned16(a->dv);
}

int tc_backward(const bissd_decay_args *a, Bump &ws, cudaStream_t s) {
    TcGradSpace g = tc_grad_space(a, ws);
    TcSpace &t = g.t;
    int *status = reinterpret_cast<int *>(ws.base);
    if ((long long)t.chunk.most * a->nheads * t.PB * t.NT > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    CUtensorMap q, k, v, dout, tiles, grads;
    if (!tc_map(&q, a, a->q, a->kdim, a->nkheads) || !tc_map(&k, a, a->k, a->kdim, a->nkheads) || !tc_map(&v, a, a->v, a->vdim, a->nheads) ||
        !tc_map(&dout, a, a->dout, a->vdim, a->nheads) || !tc_tile_map(&tiles, a, t, t.tiles) || !tc_tile_map(&grads, a, t, g.grads))
        return note_cuda(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    Rest rest;
    rest.p.status = status;
    rest.rows(a->dv, a->dtype, a->nheads * a->vdim);
    rest.rows(a->dq, a->dtype, a->nkheads * a->kdim);
    rest.rows(a->dk, a->dtype, a->nkheads * a->kdim);
    if (!a->g_per_head) rest.rows(a->dg, a->g_dtype, a->nheads);
    rest.p.start = a->dfinal_state;
    rest.p.end = t.split ? nullptr : a->dinitial_state;
    rest.p.parts = g.part; rest.p.n_parts = g.part ? 2 * g.parts : 0; rest.p.part_row = (long long)a->nkheads * a->kdim;
    BISSD_DO(rest.launch(a, t.chunk_table, &t.seg_table, s));
    if (!a->saved) BISSD_DO(tc_states(a, t, k, v, tiles, false, a->initial_state, nullptr, t.states, t.decay, status, a->nseq == 0, true, s));
    BISSD_DO(tc_states(a, t, q, dout, grads, true, a->dfinal_state, a->dinitial_state, g.gstates, g.gdecay, status, a->saved && a->nseq == 0,
                       a->saved != nullptr, s));
    unitc::GradsParams p{};
    p.h = tc_heads(a, t.PB);
    p.chunk = t.chunk; p.vpc = g.vpc; p.parts = g.parts;
    p.dq = a->dq; p.dk = a->dk; p.dv = a->dv;
    p.part = g.part; p.tokens = (long long)a->batch * a->seqlen;
    p.dg = a->dg ? (a->g_per_head ? t.dg_tokens : a->dg) : nullptr;
    p.dg_dtype = a->g_per_head ? BISSD_F32 : a->g_dtype;
    p.status = status; p.again = t.again;
    const bool dg = p.dg != nullptr;
    const auto kernel = a->dtype == BISSD_BF16 ? grads_kernel<__nv_bfloat16>(t.NT, dg) : grads_kernel<__half>(t.NT, dg);
    const size_t smem = unitc::grads_smem(t.NT);
    const long long grid = (long long)t.chunk.most * a->nkheads * p.parts;
    if (grid > 0x7fffffffLL) return BISSD_ERR_SHAPE;
    BISSD_ALLOW(kernel, smem);
    BISSD_LAUNCH("decay_grads", launch_pdl(kernel, (int)grid, 512, smem, s, p, q, k, v, dout, tiles, grads));
    if (g.parts > 1) {
        const long long each = p.tokens * a->nkheads * a->kdim;
        const int blocks = (int)((2 * each / 4 + 255) / 256);
        const int rc = by_dtype(a->dtype, [&](auto x) -> int {
            using T = decltype(x);
            if constexpr (sizeof(T) == 2)
                BISSD_LAUNCH("decay_sum_parts", launch_pdl(unitc::decay_sum_parts<T>, blocks, 256, 0, s, (const float *)g.part, g.parts, each,
                                                           static_cast<T *>(a->dq), static_cast<T *>(a->dk)));
            return BISSD_OK;
        });
        if (rc != BISSD_OK) return rc;
    }
    if (t.again.flags) {
        Bump over{ws.base, t.kept};
        const Walks w = again_walks(a, t);
        WalkSpace sp{};
        gradient_space(w.z, over, sp);
        sp.dg_tokens = t.dg_tokens;
        BISSD_DO(walk_gradients(w, sp, a->initial_state, a->dfinal_state, t.chunk_table.bounds, a->dinitial_state, t.again.flags, s));
    }
    return a->dg && a->g_per_head ? launch_dg_heads(a, t.dg_tokens, t.chunk_table.bounds, s) : BISSD_OK;
}

}  // namespace

extern "C" {

int bissd_decay_saved_bytes(const bissd_decay_args *a, size_t *bytes) {
    const int rc = decay_check(a);
    if (rc != BISSD_OK) return rc;
    if (!bytes) return BISSD_ERR_NULL;
    *bytes = 0;
    if (tc_sizes(a)) {                                           // the states that enter the chunks
        Bump b{nullptr};
        *bytes = align256(tc_tile_values(a, tc_space(a, b, false)) * sizeof(uint16_t));
    }
    return BISSD_OK;
}

int bissd_decay_workspace_bytes(const bissd_decay_args *a, size_t *fwd_bytes, size_t *bwd_bytes) {
    const int rc = decay_check(a);
    if (rc != BISSD_OK) return rc;
    if (fwd_bytes) {
        Bump b{nullptr}, c{nullptr};                              // which of the two runs is known at the call
        walk_space(a, b, false);
        if (tc_sizes(a)) tc_space(a, c, false);
        *fwd_bytes = std::max(b.used, c.used);
    }
    if (bwd_bytes) {
        Bump b{nullptr}, c{nullptr};
        walk_space(a, b, true);
        if (tc_sizes(a)) {
            const size_t kept = tc_grad_space(a, c).t.kept;
            if (a->dtype == BISSD_F16) {
                Bump over{nullptr, kept};
                WalkSpace sp{};
                gradient_space(sizes_of(a), over, sp);
                c.used = std::max(c.used, over.used);
            }
        }
        *bwd_bytes = std::max(b.used, c.used);
    }
    return BISSD_OK;
}

int bissd_decay_forward(const bissd_decay_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    BISSD_DO(bissd_decay_workspace_bytes(a, &need, nullptr));
    BISSD_DO(decay_pointers(a, false));
    // The backward pass of these inputs would read `saved`, and the CUDA cores, for such an o, do not write it.
    if (a->saved && tc_inputs(a) && !tc_forward_ok(a)) return BISSD_ERR_ALIGN;
    if (!workspace || workspace_bytes < need) return BISSD_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 256 || reinterpret_cast<uintptr_t>(a->saved) % 256) return BISSD_ERR_ALIGN;
    BISSD_DO(check_device());
    Bump b{static_cast<char *>(workspace)};
    const auto s = static_cast<cudaStream_t>(stream);
    return tc_forward_ok(a) ? tc_forward(a, b, s) : walk_forward(a, b, s);
}

int bissd_decay_backward(const bissd_decay_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    BISSD_DO(bissd_decay_workspace_bytes(a, nullptr, &need));
    BISSD_DO(decay_pointers(a, true));
    if (!workspace || workspace_bytes < need) return BISSD_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 256 || reinterpret_cast<uintptr_t>(a->saved) % 256) return BISSD_ERR_ALIGN;
    BISSD_DO(check_device());
    Bump b{static_cast<char *>(workspace)};
    const auto s = static_cast<cudaStream_t>(stream);
    return tc_backward_ok(a) ? tc_backward(a, b, s) : walk_backward(a, b, s);
}

int bissd_decay_step(const bissd_decay_step_args *a, void *stream) {
    BISSD_DO(step_check(a));
    BISSD_DO(check_device());
    return step_launch(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

// Host path of the causal decay attention, its single-token form and the norms around a block: argument checks, allocation, the
// library calls and the autograd nodes.  One call from Python each; whatever is wrong with the arguments is raised from here.
#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <stdexcept>

#include "../../include/bissd.h"
#include "torch_errors.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// Text without streams: a compiler newer than PyTorch's may link parts of its own stream library in, which do not mix.
std::string text(const char *s) { return s; }
std::string text(const std::string &s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(int v) { return std::to_string(v); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(at::IntArrayRef v) {
    std::string s = "(";
    for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
    return s + ")";
}
template <class... Args> [[noreturn]] void bad(const Args &...args) {
    throw std::invalid_argument((text(args) + ...));             // ValueError in Python
}
bool given(const OptTensor &t) { return t && t->defined(); }
Tensor value(const OptTensor &t) { return given(t) ? *t : Tensor(); }
int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return BISSD_F32;
        case at::kBFloat16: return BISSD_BF16;
        case at::kHalf: return BISSD_F16;
        default: return -1;
    }
}
void *ptr(const Tensor &t) { return t.defined() ? const_cast<void *>(t.const_data_ptr()) : nullptr; }

// Memory that the kernels may take the address of, on one device.
void on_device(const char *who, const char *name, const Tensor &t, c10::Device dev) {
    const auto ks = t.key_set();
    if (!t.is_cuda()) throw std::runtime_error(std::string(who) + ": " + name + " must be on a CUDA device (no CPU implementation is shipped)");
    if (t.device() != dev) bad(who, ": ", name, " is on ", t.device().str(), ", q on ", dev.str());
    if (t.layout() != at::kStrided || ks.has(c10::DispatchKey::Python) || ks.has(c10::DispatchKey::FuncTorchBatched) ||
        ks.has(c10::DispatchKey::FuncTorchGradWrapper) || ks.has(c10::DispatchKey::Functionalize) || t.is_conj() || t.is_neg() || t._is_zerotensor())
        bad(who, ": ", name, " must be a plain dense tensor");
}
// A tangent would be dropped: nothing here looks at it.
void refuse_tangents(const char *who, std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts)
        if (t->defined() && t->_fw_grad(0).defined())
            throw std::runtime_error(std::string(who) + ": an input carries a forward-mode tangent, for which no derivative is defined");
}
bool wants_grad(std::initializer_list<const Tensor *> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// A leaf whose gradient an eager graph still alive also leads to keeps that graph's stream: PyTorch's engine then waits across streams in
// the middle of a captured backward pass, which spoils the capture and can end the process.  Refused before anything is recorded.
void refuse_mixed_capture(const char *who, std::initializer_list<const Tensor *> ts) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    for (const Tensor *t : ts) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        if (!node) continue;
        const auto stream = node->stream();
        if (stream && *stream != c10::cuda::getCurrentCUDAStream(t->device().index()).unwrap())
            throw std::runtime_error(std::string(who) + ": captured with gradients while an eager graph of the same leaves is alive on another "
                                     "stream; release that graph first");
    }
}
// As the kernels read it in place: unit inner stride and, for 16-bit tensors, 16-byte aligned rows that do not repeat; else a copy.
Tensor in_place(const Tensor &t) {
    if (!t.defined()) return t;
    const auto st = t.strides();
    bool ok = st.back() == 1 || t.size(-1) == 1;
    if (ok && t.element_size() == 2 && t.dim() > 1) {
        ok = reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
        for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && st[i] % 8 == 0 && (st[i] != 0 || t.size(i) == 1);
    }
    // a dimension of one element may have any stride, also one that no descriptor holds
    for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && st[i] >= 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);       // contiguous() would leave an odd address as it is
}
Tensor contiguous(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
void once(const char *who) {
    if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(who) + ": the gradients cannot be differentiated again (create_graph)");
}
struct Scratch {                                                 // from the caching allocator, on the current stream
    c10::DataPtr p;
    explicit Scratch(size_t bytes) : p(c10::cuda::CUDACachingAllocator::get()->allocate(std::max<size_t>(bytes, 256))) {}
};

// ---- decay attention ---------------------------------------------------------------------------------------------------
constexpr const char *kAttention = "decay_attention";

struct Config {
    double scale;
    int64_t nseq;
    bool check_status;
};
bissd_tensor tensor4(const Tensor &t) { return bissd_tensor{ptr(t), t.stride(0), t.stride(1), t.stride(2)}; }
bissd_tensor tensor3(const Tensor &t) { return bissd_tensor{ptr(t), t.stride(0), t.stride(1), t.dim() > 2 ? t.stride(2) : 0}; }

bissd_decay_args decay_args(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, const Tensor &initial, const Tensor &cu,
                            const Config &cfg) {
    bissd_decay_args a{};
    a.batch = (int)q.size(0); a.seqlen = (int)q.size(1); a.nheads = (int)v.size(2); a.nkheads = (int)q.size(2);
    a.kdim = (int)q.size(3); a.vdim = (int)v.size(3); a.nseq = (int)cfg.nseq;
    a.dtype = dtype_code(q.scalar_type()); a.g_dtype = dtype_code(g.scalar_type()); a.g_per_head = g.dim() == 1;
    a.scale = (float)cfg.scale;
    a.q = tensor4(q); a.k = tensor4(k); a.v = tensor4(v);
    a.g = g.dim() == 1 ? bissd_tensor{ptr(g), 0, 0, 1} : tensor3(g);
    a.cu_seqlens = static_cast<const int32_t *>(ptr(cu));
    a.initial_state = static_cast<const float *>(ptr(initial));
    return a;
}
at::DimVector state_shape(const Tensor &q, const Tensor &v, const Config &cfg) {
    return {cfg.nseq > 0 ? cfg.nseq : q.size(0), v.size(2), q.size(3), v.size(3)};
}

struct Attention {
    Tensor out, final_, saved;
};
Attention attention_forward(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &g_, const Tensor &initial_, const Tensor &cu,
                            const Config &cfg, bool finals, bool keep) {
    const Tensor q = in_place(q_), k = in_place(k_), v = in_place(v_), initial = contiguous(initial_);
    const Tensor g = g_.dim() == 1 ? g_.contiguous() : g_;
    Attention r;
    r.out = at::empty(v.sizes(), v.options());
    const auto shape = state_shape(q, v, cfg);
    if (q.size(0) * q.size(1) == 0) {                            // no token: the states stay
        if (finals) r.final_ = initial.defined() ? initial.clone() : at::zeros(shape, v.options().dtype(at::kFloat));
        return r;
    }
    if (finals) r.final_ = at::empty(shape, v.options().dtype(at::kFloat));
    bissd_decay_args a = decay_args(q, k, v, g, initial, cu, cfg);
    a.o = ptr(r.out);
    a.final_state = static_cast<float *>(ptr(r.final_));
    size_t bytes = 0;
    if (keep) {
        bissd_check(bissd_decay_saved_bytes(&a, &bytes));
        if (bytes) r.saved = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
        a.saved = ptr(r.saved);
    }
    bissd_check(bissd_decay_workspace_bytes(&a, &bytes, nullptr));
    const Scratch ws(bytes);
    const auto stream = c10::cuda::getCurrentCUDAStream(q.device().index());
    bissd_check(bissd_decay_forward(&a, ws.p.get(), bytes, stream.stream()));
    bissd_check_device_status(cfg.check_status, ws.p.get(), stream.stream());
    return r;
}

struct AttentionFn : public torch::autograd::Function<AttentionFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g,
                                 const OptTensor &initial, const OptTensor &cu, double scale, int64_t nseq, bool finals, bool check_status) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Config cfg{scale, nseq, check_status};
        Attention r = attention_forward(q, k, v, g, value(initial), value(cu), cfg, finals, true);
        ctx->save_for_backward({q, k, v, g, value(initial), value(cu), r.saved});
        auto &s = ctx->saved_data;
        s["scale"] = scale; s["nseq"] = nseq; s["check_status"] = check_status;
        ctx->set_materialize_grads(false);
        if (finals) return {r.out, r.final_};
        return {r.out};
    }
    static variable_list backward(AutogradContext *ctx, variable_list go) {
        once(kAttention);
        const variable_list saved = ctx->get_saved_variables();
        auto &sd = ctx->saved_data;
        const Config cfg{sd["scale"].toDouble(), sd["nseq"].toInt(), sd["check_status"].toBool()};
        const c10::cuda::CUDAGuard guard(saved[0].device());
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor q = in_place(saved[0]), k = in_place(saved[1]), v = in_place(saved[2]), cu = saved[5];
        const Tensor g = saved[3].dim() == 1 ? saved[3].contiguous() : saved[3], initial = contiguous(saved[4]);
        const Tensor none, dfinal = go.size() > 1 ? contiguous(go[1]) : none;
        const Tensor dout = go[0].defined() ? in_place(go[0].scalar_type() == v.scalar_type() ? go[0] : go[0].to(v.scalar_type()))
                                            : at::zeros(v.sizes(), v.options());
        const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
        Tensor dg, dinitial;
        if (ctx->needs_input_grad(3)) dg = at::empty(g.sizes(), g.options());
        if (initial.defined()) dinitial = at::empty(initial.sizes(), initial.options());
        if (q.size(0) * q.size(1) == 0) {
            if (dg.defined()) dg.zero_();
            if (dinitial.defined()) dfinal.defined() ? dinitial.copy_(dfinal) : dinitial.zero_();
            return {dq, dk, dv, dg, dinitial, none, none, none, none, none};
        }
        bissd_decay_args a = decay_args(q, k, v, g, initial, cu, cfg);
        a.saved = ptr(saved[6]);
        a.dout = tensor4(dout);
        a.dq = ptr(dq); a.dk = ptr(dk); a.dv = ptr(dv); a.dg = ptr(dg);
        a.dfinal_state = static_cast<const float *>(ptr(dfinal));
        a.dinitial_state = static_cast<float *>(ptr(dinitial));
        size_t bytes = 0;
        bissd_check(bissd_decay_workspace_bytes(&a, nullptr, &bytes));
        const Scratch ws(bytes);
        const auto stream = c10::cuda::getCurrentCUDAStream(q.device().index());
        bissd_check(bissd_decay_backward(&a, ws.p.get(), bytes, stream.stream()));
        bissd_check_device_status(cfg.check_status, ws.p.get(), stream.stream());
        return {dq, dk, dv, dg, dinitial, none, none, none, none, none};
    }
};

// Sizes and types shared by the two forms: `lead` dimensions before the heads.
void check_qkvg(const char *who, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, int lead) {
    if (q.dim() != lead + 2 || v.dim() != lead + 2) bad(who, ": q and v must have ", lead + 2, " dimensions, not ", q.dim(), " and ", v.dim());
    if (k.sizes() != q.sizes()) bad(who, ": k must have q's shape ", q.sizes(), ", not ", k.sizes());
    const int64_t hk = q.size(lead), n = q.size(lead + 1), h = v.size(lead), p = v.size(lead + 1);
    for (int i = 0; i < lead; ++i)
        if (v.size(i) != q.size(i)) bad(who, ": v's batch and sequence must be q's, not ", v.sizes(), " beside ", q.sizes());
    if (hk < 1 || h < 1 || h % hk) bad(who, ": v's heads (", h, ") must be a multiple of q's (", hk, ")");
    if (n < 1 || n > 256 || p < 1 || p > 256) bad(who, ": head sizes must be 1 to 256, not ", n, " and ", p);
    if (dtype_code(q.scalar_type()) < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
        bad(who, ": q, k and v must be of one type, float32, bfloat16 or float16");
    if (g.dim() == 1 ? g.size(0) != h : (g.dim() != lead + 1 || g.sizes().slice(0, lead) != q.sizes().slice(0, lead) || g.size(lead) != h))
        bad(who, ": g must be (heads) or one value for each token and head, not ", g.sizes());
    if (dtype_code(g.scalar_type()) < 0 || (g.scalar_type() != at::kFloat && g.scalar_type() != q.scalar_type()))
        bad(who, ": g must be float32 or of q's type");
}

py::object decay_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &g, std::optional<double> scale,
                           const OptTensor &initial, bool finals, const OptTensor &cu_, bool check_status) {
    check_qkvg(kAttention, q, k, v, g, 2);
    int64_t nseq = 0;
    if (given(cu_)) {
        if (cu_->dim() != 1 || cu_->size(0) < 2 || (cu_->scalar_type() != at::kInt && cu_->scalar_type() != at::kLong))
            bad(kAttention, ": cu_seqlens must be int32 or int64 of one dimension, with at least two values");
        if (q.size(0) != 1) bad(kAttention, ": packed sequences are one row, not a batch of ", q.size(0));
        nseq = cu_->size(0) - 1;
    }
    if (q.size(0) * q.size(1) > 0x7fffffffLL / 256) bad(kAttention, ": more than ", int64_t(0x7fffffffLL / 256), " tokens");
    const Config cfg{scale ? *scale : 1.0 / std::sqrt((double)q.size(3)), nseq, check_status};
    if (given(initial)) {
        if (initial->scalar_type() != at::kFloat || initial->sizes() != at::IntArrayRef(state_shape(q, v, cfg)))
            bad(kAttention, ": initial_state must be float32 ", at::IntArrayRef(state_shape(q, v, cfg)), ", not ", initial->scalar_type(), " ",
                initial->sizes());
    }
    const Tensor init = value(initial);
    refuse_tangents(kAttention, {&q, &k, &v, &g, &init});
    const auto dev = q.device();
    on_device(kAttention, "q", q, dev);
    on_device(kAttention, "k", k, dev);
    on_device(kAttention, "v", v, dev);
    on_device(kAttention, "g", g, dev);
    if (given(initial)) on_device(kAttention, "initial_state", *initial, dev);
    if (given(cu_)) on_device(kAttention, "cu_seqlens", *cu_, dev);
    const c10::cuda::CUDAGuard guard(dev);
    Tensor cu = value(cu_);
    const bool grad = wants_grad({&q, &k, &v, &g, &init});
    if (grad) refuse_mixed_capture(kAttention, {&q, &k, &v, &g, &init});
    variable_list r;
    {
        py::gil_scoped_release nogil;
        if (cu.defined()) cu = (cu.scalar_type() == at::kLong ? cu.clamp(0, q.size(1)).to(at::kInt) : cu).contiguous();   // what lies outside would wrap
        if (grad) {
            r = AttentionFn::apply(q, k, v, g, initial, cu.defined() ? OptTensor(cu) : OptTensor(), cfg.scale, nseq, finals, check_status);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            Attention o = attention_forward(q, k, v, g, init, cu, cfg, finals, false);
            r = finals ? variable_list{o.out, o.final_} : variable_list{o.out};
        }
    }
    if (finals) return py::make_tuple(r[0], r[1]);
    return py::cast(r[0]);
}

// ---- one token ---------------------------------------------------------------------------------------------------------
Tensor decay_step(const Tensor &state, const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &g_, std::optional<double> scale,
                  const OptTensor &slots_) {
    constexpr const char *who = "decay_attention_step";
    check_qkvg(who, q_, k_, v_, g_, 1);
    const int64_t b = q_.size(0), hk = q_.size(1), n = q_.size(2), h = v_.size(1), p = v_.size(2);
    if (state.dim() != 4 || state.scalar_type() != at::kFloat || state.size(1) != h || state.size(2) != n || state.size(3) != p)
        bad(who, ": state must be float32 (slots, ", h, ", ", n, ", ", p, "), not ", state.scalar_type(), " ", state.sizes());
    if (state.stride(3) != 1 || state.stride(2) != p || state.stride(1) != n * p || (state.size(0) > 1 && state.stride(0) < h * n * p))
        bad(who, ": each slot of state must be contiguous: it is updated in place");
    if (!given(slots_) && state.size(0) < b) bad(who, ": ", b, " requests and only ", state.size(0), " states");
    if (given(slots_) && (slots_->dim() != 1 || slots_->size(0) != b || (slots_->scalar_type() != at::kInt && slots_->scalar_type() != at::kLong)))
        bad(who, ": slots must be int32 or int64 (", b, ")");
    refuse_tangents(who, {&state, &q_, &k_, &v_, &g_});
    if (wants_grad({&state, &q_, &k_, &v_, &g_})) throw std::runtime_error(std::string(who) + ": no gradient is defined; call it under torch.no_grad()");
    if (state.size(0) == 0 && b > 0) bad(who, ": no state");
    if (state.size(0) > 0x7fffffffLL || b > 0x7fffffffLL / (h * 8)) bad(who, ": too many requests or states");
    const auto dev = q_.device();
    on_device(who, "q", q_, dev);
    on_device(who, "k", k_, dev);
    on_device(who, "v", v_, dev);
    on_device(who, "g", g_, dev);
    on_device(who, "state", state, dev);
    if (given(slots_)) on_device(who, "slots", *slots_, dev);
    const c10::cuda::CUDAGuard guard(dev);
    py::gil_scoped_release nogil;
    at::AutoDispatchBelowADInplaceOrView below;
    auto rows = [](const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); };
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_), out = at::empty({b, h, p}, v.options());
    const Tensor g = g_.dim() == 1 ? g_.contiguous() : g_;
    if (b == 0) return out;
    Tensor slots = value(slots_);
    if (slots.defined()) slots = slots.scalar_type() == at::kInt ? slots.contiguous() : slots.clamp(-1, state.size(0)).to(at::kInt).contiguous();
    bissd_decay_step_args a{};
    a.batch = (int)b; a.nheads = (int)h; a.nkheads = (int)hk; a.kdim = (int)n; a.vdim = (int)p;
    a.dtype = dtype_code(q.scalar_type()); a.g_dtype = dtype_code(g.scalar_type()); a.g_per_head = g.dim() == 1;
    a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)n));
    auto t2 = [](const Tensor &t) { return bissd_tensor{ptr(t), t.stride(0), 0, t.stride(1)}; };
    a.q = t2(q); a.k = t2(k); a.v = t2(v); a.o = t2(out);
    a.g = g.dim() == 1 ? bissd_tensor{ptr(g), 0, 0, 1} : t2(g);
    a.state = static_cast<float *>(ptr(state));
    a.slot_stride = state.size(0) > 1 ? state.stride(0) : h * n * p;
    a.nslots = (int)state.size(0);
    a.slots = static_cast<const int32_t *>(ptr(slots));
    bissd_check(bissd_decay_step(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return out;
}

// ---- the norms around a block --------------------------------------------------------------------------------------------
constexpr const char *kNorm = "block_norm";

struct NormConfig {
    double scale, eps;
    int64_t act, gate_rows;
};
// Rows of `width` channels a fixed stride apart; a copy where they are not.
struct Rows {
    Tensor t;
    void *p = nullptr;
    int64_t n = 0, stride = 0;
};
Rows rows_of(const Tensor &t, int64_t width) {
    Rows r;
    if (!t.defined()) return r;
    r.t = t;
    r.n = t.numel() / width;
    if (t.is_contiguous()) {
        r.stride = width;
    } else {
        r.t = t.reshape({-1, width});
        const bool repeats = r.n > 1 && r.t.stride(0) < width;
        const bool far = r.t.stride(0) > 0x3fffffff;             // the kernels' strides have 32 bits
        if ((width > 1 && r.t.stride(1) != 1) || repeats || (far && r.n > 1)) r.t = r.t.contiguous();
        r.stride = r.n > 1 ? r.t.stride(0) : width;
    }
    r.p = ptr(r.t);
    return r;
}
bissd_block_norm_args norm_args(const Rows &x, const Rows &res, const Rows &gate, int64_t width, const Tensor &scale, const Tensor &post,
                                const Tensor &pre, const NormConfig &c) {
    bissd_block_norm_args a{};
    a.rows = x.n; a.width = (int)width; a.gate_rows = gate.p ? c.gate_rows : 0;
    a.dtype = dtype_code(x.t.scalar_type()); a.r_dtype = dtype_code(res.t.scalar_type());
    a.w_dtype = a.dtype;
    for (const Tensor *w : {&scale, &post, &pre})
        if (w->defined()) a.w_dtype = dtype_code(w->scalar_type());
    a.gate_act = (int)c.act; a.scale = (float)c.scale; a.eps = (float)c.eps;
    a.x = x.p; a.residual = res.p; a.gate = gate.p; a.scale_vector = ptr(scale); a.post_weight = ptr(post); a.pre_weight = ptr(pre);
    a.stride_x = x.stride; a.stride_residual = res.stride; a.stride_gate = gate.stride;
    return a;
}
struct Normed {
    Tensor r, u, rstd;
};
Normed norm_forward(const Tensor &x_, const Tensor &res_, const Tensor &gate_, const Tensor &scale_, const Tensor &post_, const Tensor &pre_,
                    const NormConfig &c, bool keep) {
    Normed o;
    o.r = at::empty(res_.sizes(), res_.options());
    if (pre_.defined()) o.u = at::empty(x_.sizes(), x_.options());
    if (x_.numel() == 0) return o;
    const int64_t d = x_.size(-1);
    const Rows x = rows_of(x_, d), res = rows_of(res_, d), gate = rows_of(gate_, d);
    const Tensor scale = contiguous(scale_), post = contiguous(post_), pre = contiguous(pre_);
    bissd_block_norm_args a = norm_args(x, res, gate, d, scale, post, pre, c);
    if (keep) o.rstd = at::empty({2, x.n}, x_.options().dtype(at::kFloat));
    a.r = ptr(o.r); a.normed = ptr(o.u); a.rstd = static_cast<float *>(ptr(o.rstd));
    bissd_check(bissd_block_norm_forward(&a, c10::cuda::getCurrentCUDAStream(x_.device().index()).stream()));
    return o;
}

struct NormFn : public torch::autograd::Function<NormFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &res, const OptTensor &gate, const OptTensor &scale,
                                 const OptTensor &post, const OptTensor &pre, double scale_number, double eps, int64_t act, int64_t gate_rows) {
        at::AutoDispatchBelowADInplaceOrView below;
        const NormConfig c{scale_number, eps, act, gate_rows};
        Normed o = norm_forward(x, res, value(gate), value(scale), value(post), value(pre), c, true);
        ctx->save_for_backward({x, res, value(gate), value(scale), value(post), value(pre), o.rstd});
        auto &s = ctx->saved_data;
        s["scale"] = scale_number; s["eps"] = eps; s["act"] = act; s["gate_rows"] = gate_rows;
        ctx->set_materialize_grads(false);
        if (o.u.defined()) return {o.r, o.u};
        return {o.r};
    }
    static variable_list backward(AutogradContext *ctx, variable_list go) {
        once(kNorm);
        const variable_list v = ctx->get_saved_variables();
        auto &s = ctx->saved_data;
        const NormConfig c{s["scale"].toDouble(), s["eps"].toDouble(), s["act"].toInt(), s["gate_rows"].toInt()};
        const c10::cuda::CUDAGuard guard(v[0].device());
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor none;
        Tensor d_[6];                                            // of what is given and wanted; edges count what is given
        for (int i = 0, edge = 0; i < 6; ++i)
            if (v[i].defined() && ctx->needs_input_grad(edge++)) d_[i] = at::empty(v[i].sizes(), v[i].options());
        const Tensor &dx = d_[0], &dres = d_[1], &dgate = d_[2], &dscale = d_[3], &dpost = d_[4], &dpre = d_[5];
        if (v[0].numel() == 0) {
            for (const Tensor *t : {&dgate, &dscale, &dpost, &dpre})
                if (t->defined()) t->zero_();
        } else {
            const int64_t d = v[0].size(-1);
            auto typed = [&](const Tensor &t, const Tensor &like) { return !t.defined() || t.scalar_type() == like.scalar_type() ? t : t.to(like.scalar_type()); };
            const Rows x = rows_of(v[0], d), res = rows_of(v[1], d), gate = rows_of(v[2], d);
            const Tensor scale = contiguous(v[3]), post = contiguous(v[4]), pre = contiguous(v[5]);
            const Rows dr = rows_of(typed(go[0], v[1]), d), du = go.size() > 1 ? rows_of(typed(go[1], v[0]), d) : Rows();
            if (dpre.defined() && !du.p) dpre.zero_();
            bissd_block_norm_args a = norm_args(x, res, gate, d, scale, post, pre, c);
            a.rstd = static_cast<float *>(ptr(v[6]));
            a.dr = dr.p; a.dnormed = du.p;
            a.stride_dr = dr.stride; a.stride_dnormed = du.stride;
            a.dx = ptr(dx); a.dresidual = ptr(dres); a.dgate = ptr(dgate); a.dscale = ptr(dscale); a.dpost = ptr(dpost); a.dpre = ptr(dpre);
            size_t bytes = 0;
            bissd_check(bissd_block_norm_workspace_bytes(&a, &bytes));
            const Scratch ws(bytes);
            bissd_check(bissd_block_norm_backward(&a, ws.p.get(), bytes, c10::cuda::getCurrentCUDAStream(v[0].device().index()).stream()));
        }
        return {dx, dres, dgate, dscale, dpost, dpre, none, none, none, none};
    }
};

py::object block_norm(const Tensor &x, const Tensor &residual, const OptTensor &gate_, const OptTensor &scale_, double scale_number,
                      const OptTensor &post_, const OptTensor &pre_, int64_t act, double eps) {
    const Tensor gate = value(gate_), scale = value(scale_), post = value(post_), pre = value(pre_);
    if (x.dim() < 1 || residual.sizes() != x.sizes()) bad(kNorm, ": residual must have x's shape ", x.sizes(), ", not ", residual.sizes());
    const int64_t d = x.size(-1);
    if (d < 1 || d > 8192) bad(kNorm, ": width must be 1 to 8192, not ", d);
    const auto st = x.scalar_type();
    if (dtype_code(st) < 0) bad(kNorm, ": x must be float32, bfloat16 or float16");
    if (x.numel() / d > 0x3fffffff) bad(kNorm, ": more than ", int64_t(0x3fffffff), " rows");
    if (residual.scalar_type() != st && residual.scalar_type() != at::kFloat) bad(kNorm, ": residual must be float32 or of x's type");
    at::ScalarType wt = at::kFloat;
    bool first = true;
    for (const Tensor *w : {&scale, &post, &pre}) {
        if (!w->defined()) continue;
        if (w->dim() != 1 || w->size(0) != d) bad(kNorm, ": weights and a scale vector must be (", d, "), not ", w->sizes());
        if (w->scalar_type() != st && w->scalar_type() != at::kFloat) bad(kNorm, ": weights must be float32 or of x's type");
        if (!first && w->scalar_type() != wt) bad(kNorm, ": weights and a scale vector must be of one type");
        wt = w->scalar_type();
        first = false;
    }
    int64_t gate_rows = 0;
    if (gate.defined()) {
        if (gate.scalar_type() != st) bad(kNorm, ": gate must be of x's type");
        bool row = gate.dim() == x.dim() && gate.dim() >= 2 && gate.size(-1) == d && (gate.size(0) == x.size(0) || gate.size(0) == 1);
        for (int64_t i = 1; row && i + 1 < gate.dim(); ++i) row = gate.size(i) == 1;
        if (gate.sizes() != x.sizes()) {
            if (!row) bad(kNorm, ": gate must have x's shape or one row for each entry of the first dimension, not ", gate.sizes());
            gate_rows = gate.size(0) > 0 && x.numel() > 0 ? x.numel() / d / gate.size(0) : 1;
        }
    }
    refuse_tangents(kNorm, {&x, &residual, &gate, &scale, &post, &pre});
    const auto dev = x.device();
    on_device(kNorm, "x", x, dev);
    on_device(kNorm, "residual", residual, dev);
    const Tensor *opt[] = {&gate, &scale, &post, &pre};
    const char *names[] = {"gate", "scale", "post_weight", "pre_weight"};
    for (int i = 0; i < 4; ++i)
        if (opt[i]->defined()) on_device(kNorm, names[i], *opt[i], dev);
    const c10::cuda::CUDAGuard guard(dev);
    const bool grad = wants_grad({&x, &residual, &gate, &scale, &post, &pre});
    if (grad) refuse_mixed_capture(kNorm, {&x, &residual, &gate, &scale, &post, &pre});
    variable_list r;
    {
        py::gil_scoped_release nogil;
        if (grad) {
            r = NormFn::apply(x, residual, gate_, scale_, post_, pre_, scale_number, eps, act, gate_rows);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            Normed o = norm_forward(x, residual, gate, scale, post, pre, NormConfig{scale_number, eps, act, gate_rows}, false);
            r = o.u.defined() ? variable_list{o.r, o.u} : variable_list{o.r};
        }
    }
    if (r.size() > 1) return py::make_tuple(r[0], r[1]);
    return py::cast(r[0]);
}

}  // namespace

void bind_uni(py::module_ &m) {
    m.def("decay_attention", &decay_attention);
    m.def("decay_step", &decay_step);
    m.def("block_norm", &block_norm);
}

// block_ext.cpp — the tensor side of ops_block: argument checks, outputs, scratch and autograd nodes around the C entry points of cdae.h.
//
// Why native: the kernels of one call take 10..50 us at the sizes of a training step, while the same dispatch in Python took 160..250 us for a forward
// and a backward (measured: norms of 8192 x 384 rows 230 us of host time around 60 us of kernels; clipping 390 tensors 545 us around 225 us).
// A node's backward runs on autograd's own thread without the interpreter.  Nothing is kept between calls.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "cdae.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

namespace {

struct Refused : std::runtime_error { using std::runtime_error::runtime_error; };
#define REFUSE(ok, ...) do { if (!(ok)) throw Refused(c10::str(__VA_ARGS__)); } while (0)
void check(int rc) { if (rc != 0) throw Refused(cdae_last_error()); }

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return 0;
        case at::kHalf: return 1;
        case at::kFloat: return 2;
        default: return -1;
    }
}
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
Tensor scratch(size_t bytes, const Tensor& like) { return at::empty({(int64_t)(bytes ? bytes : 1)}, like.options().dtype(at::kByte).requires_grad(false)); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor fresh(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, at::TensorOptions().dtype(like.dtype()).device(like.device())); }

// (a tensor whose values lie negated in memory, until someone asks for them)
Tensor as_written(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// A tensor [..., C] as rows whose values lie side by side, at a pitch of at least a row: as it lies, or a dense copy
struct Rows { Tensor t; long pitch; };
Rows rows_of(const Tensor& as_given, int64_t C) {
    const Tensor t = as_written(as_given);
    if (!t.defined()) return {t, 0};
    const int64_t d = t.dim();
    bool ok = C == 1 || t.stride(d - 1) == 1;
    int64_t pitch = C, count = 1;                              // pitch and number of the rows seen so far, innermost dimension first
    bool first = true;
    for (int64_t i = d - 2; ok && i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (first) { pitch = t.stride(i); first = false; ok = pitch >= C; }
        else ok = t.stride(i) == pitch * count;
        count *= t.size(i);
    }
    if (ok || t.numel() == 0) return {t, (long)pitch};
    return {t.contiguous(), (long)C};
}
Tensor side_by_side(const Tensor& as_given) {
    const Tensor t = as_written(as_given);
    return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// forward-mode derivatives: a tangent would be lost without a word
void no_tangent(const char* who, const Tensor& t) { REFUSE(!t.defined() || !t._fw_grad(0).defined(), who, ": there are no forward-mode derivatives"); }

bool has_values(const Tensor& t) { return t.layout() == at::kStrided && !t.is_nested() && t.has_storage(); }      // (a sparse or nested tensor's do not lie in rows)

void same_device(const char* who, const Tensor& x, std::initializer_list<Tensor> others) {
    REFUSE(x.is_cuda(), who, ": tensors on an MI355X device required; there is no CPU form");
    REFUSE(has_values(x), who, ": dense tensors required");
    no_tangent(who, x);
    for (const Tensor& t : others) {
        REFUSE(!t.defined() || has_values(t), who, ": dense tensors required");
        REFUSE(!t.defined() || t.device() == x.device(), who, ": all tensors on one device (", x.device().str(), ")");
        no_tangent(who, t);
    }
}
bool wanted(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts) if (t.defined() && t.requires_grad()) return true;
    return false;
}
bool capturing(at::Device dev) {
    const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return st && hipStreamIsCapturing(st, &status) == hipSuccess && status != hipStreamCaptureStatusNone;      // (the default stream is never captured)
}
// A leaf's gradient is summed on the stream on which its first live graph was made.  If that is the default stream and this forward is being captured, the
// captured backward would have the default stream wait on the capture, which HIP does not allow, and the error surfaces on autograd's thread, where it
// ends the process: refused here, before anything is launched.
void capturable(const char* who, const Tensor& x, std::initializer_list<Tensor> leaves) {
    if (!capturing(x.device())) return;
    for (const Tensor& t : leaves) {
        if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
        const auto sum = torch::autograd::impl::try_get_grad_accumulator(t);
        if (!sum) continue;
        const std::optional<c10::Stream> on = sum->stream();
        REFUSE(!on || on->id() != 0, who, ": captured while an eager graph over the same leaf, made on the default stream, is alive; free its results first");
    }
}
// first derivatives only: with create_graph the gradients lead to a node that says so
variable_list once(variable_list&& g) {
    if (!at::GradMode::is_enabled()) return std::move(g);
    variable_list have;
    for (const Tensor& t : g) if (t.defined()) have.push_back(t.detach().requires_grad_());
    auto node = std::make_shared<torch::autograd::DelayedError>("ops_block: the operators have first derivatives only", (int64_t)have.size());
    have = (*node)(std::move(have));
    size_t k = 0;
    for (Tensor& t : g) if (t.defined()) t = have[k++];
    return std::move(g);
}

// ----------------------------------------------------------------------------- linear layer with activation and residual
int act_of(const std::string& a) {
    static const std::pair<const char*, int> known[] = {{"none", 0}, {"silu", 1}, {"relu", 3}, {"gelu", 5}, {"gelu_tanh", 6}};
    for (const auto& k : known) if (a == k.first) return k.second;
    throw Refused("linear_act: act is one of none, silu, relu, gelu, gelu_tanh");
}

bool as_it_lies(const Rows& r) {
    return r.t.size(-1) % 8 == 0 && r.pitch % 8 == 0 && r.pitch <= 1L << 22 && reinterpret_cast<uintptr_t>(r.t.const_data_ptr()) % 16 == 0;
}
size_t linear_scratch(int op, const Rows& x, const Rows& w, int64_t M) {
    return cdae_lin16_workspace_bytes(op | (as_it_lies(x) && as_it_lies(w) ? CDAE_LIN16_ALIGNED : 0), (int)M, (int)w.t.size(0), (int)w.t.size(1));
}

Tensor linear_forward(const Rows& x, const Rows& w, const Tensor& b, const Tensor& res_, int act, Tensor* z, const Tensor& x_as_given) {
    const int64_t K = w.t.size(1), N = w.t.size(0), M = x.t.numel() / K;
    std::vector<int64_t> shape(x_as_given.sizes().begin(), x_as_given.sizes().end());
    shape.back() = N;
    Tensor y = fresh(shape, x.t);
    if (z) *z = at::empty({M, N}, x.t.options().dtype(at::kHalf).requires_grad(false));
    if (!M) return y;
    const Tensor bias = side_by_side(b);
    const Rows res = rows_of(res_, N);
    const size_t need = linear_scratch(CDAE_LIN16_FWD, x, w, M);
    const Tensor ws = scratch(need, x.t);
    check(cdae_lin16_fwd(ptr(x.t), x.pitch, ptr(w.t), w.pitch, ptr(bias), ptr(res.t), res.pitch, mptr(y), N, z ? mptr(*z) : nullptr, N, (int)M, (int)N, (int)K, act,
                         type_of(x.t), mptr(ws), need, stream_of(x.t)));
    return y;
}

Tensor of(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// (an absent tensor is no input of the node: the edges are those of the present ones, in order)
struct LinearAct : torch::autograd::Function<LinearAct> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const std::optional<Tensor>& b, const std::optional<Tensor>& res, int64_t act) {
        const Rows x = rows_of(x_, w_.size(1)), w = rows_of(w_, w_.size(1));
        Tensor z;
        // By the tensors alone: ctx->needs_input_grad asks the backward that is running, if one is, so that a forward recomputed inside a backward over
        // some of the inputs would keep nothing for a later one over others.
        const bool products = x_.requires_grad() || w_.requires_grad() || (b && b->requires_grad());
        Tensor y = linear_forward(x, w, of(b), of(res), (int)act, products && act ? &z : nullptr, x_);
        if (products) ctx->save_for_backward({x.t, w.t, z});
        ctx->saved_data["act"] = act;
        ctx->saved_data["bias"] = b.has_value();
        ctx->saved_data["res"] = res.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor& dy_ = grads[0];
        no_tangent("linear_act", dy_);
        variable_list g(5);
        const bool bias = ctx->saved_data["bias"].toBool(), res = ctx->saved_data["res"].toBool();
        const bool want_b = bias && ctx->needs_input_grad(2);
        if (res && ctx->needs_input_grad(bias ? 3 : 2)) g[3] = dy_;
        if (!ctx->needs_input_grad(0) && !ctx->needs_input_grad(1) && !want_b) return once(std::move(g));
        const variable_list saved = ctx->get_saved_variables();
        REFUSE(saved.size() == 3, "linear_act: the forward kept nothing for this backward");
        const Tensor &xt = saved[0], &wt = saved[1], &z = saved[2];
        const int64_t K = wt.size(1), N = wt.size(0), M = xt.numel() / K;
        c10::DeviceGuard on(xt.device());
        if (ctx->needs_input_grad(0)) g[0] = fresh(xt.sizes(), xt);
        if (ctx->needs_input_grad(1)) g[1] = fresh({N, K}, xt);
        if (want_b) g[2] = fresh({N}, xt);
        if (!M) {
            for (int i : {1, 2}) if (g[i].defined()) g[i].zero_();          // (no rows: the sums over them are zero)
            return once(std::move(g));
        }
        const Rows x = rows_of(xt, K), w = rows_of(wt, K), dy = rows_of(dy_, N);
        const Tensor zd = z.defined() ? z.contiguous() : z;                  // (a hook on saved tensors may hand them back in another layout)
        const size_t need = linear_scratch(CDAE_LIN16_BWD, x, w, M);
        const Tensor ws = scratch(need, xt);
        check(cdae_lin16_bwd(ptr(dy.t), dy.pitch, ptr(x.t), x.pitch, ptr(w.t), w.pitch, ptr(zd), N, mptr(g[0]), K, mptr(g[1]), K, mptr(g[2]), (int)M, (int)N, (int)K,
                             (int)ctx->saved_data["act"].toInt(), type_of(xt), mptr(ws), need, stream_of(xt)));
        return once(std::move(g));
    }
};

Tensor linear_act(const Tensor& x, const Tensor& w, const std::optional<Tensor>& b_, const std::optional<Tensor>& res_, const std::string& act_) {
    const Tensor b = of(b_), res = of(res_);
    same_device("linear_act", x, {w, b, res});
    const int act = act_of(act_);
    REFUSE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "linear_act: bf16 or fp16 rows (got ", x.scalar_type(), "; ops.linear takes fp32)");
    REFUSE(x.dim() >= 1 && w.dim() == 2 && w.size(0) >= 1 && w.size(1) >= 1 && x.size(-1) == w.size(1), "linear_act: rows [..., K] and a weight [N, K] (got ", x.sizes(),
           " and ", w.sizes(), ")");
    const int64_t N = w.size(0), K = w.size(1);
    const auto same = [&](const Tensor& t) { return !t.defined() || t.scalar_type() == x.scalar_type(); };
    REFUSE(same(w) && same(b) && same(res), "linear_act: x, w, b and res of one type");
    REFUSE(!b.defined() || (b.dim() == 1 && b.size(0) == N), "linear_act: a bias [", N, "]");
    if (res.defined()) {
        bool ok = res.dim() == x.dim() && res.size(-1) == N;
        for (int64_t i = 0; ok && i + 1 < x.dim(); ++i) ok = res.size(i) == x.size(i);
        REFUSE(ok, "linear_act: a residual of the result's shape (nothing is broadcast)");
    }
    REFUSE(x.numel() / K <= (1LL << 30) && N <= (1LL << 22) && K <= (1LL << 22), "linear_act: at most 2^30 rows and 2^22 features");
    c10::DeviceGuard on(x.device());
    if (wanted({x, w, b, res})) {
        capturable("linear_act", x, {x, w, b, res});
        return LinearAct::apply(x, w, maybe(b), maybe(res), (int64_t)act);
    }
    return linear_forward(rows_of(x, K), rows_of(w, K), b, res, act, nullptr, x);
}

// ----------------------------------------------------------------------------- the norms around a block
struct NormCfg { int64_t B, T, C; double alpha, eps; bool layer, post, pre; };
enum { T_X, T_F, T_GATE, T_SCALE, T_SHIFT, T_W1, T_B1, T_W2, T_B2, T_COUNT };

cdae_resnorm norm_args(const Tensor* t, const long* pitch, const NormCfg& c) {
    cdae_resnorm p{};
    p.B = (int)c.B; p.T = (int)c.T; p.C = (int)c.C; p.dt = type_of(t[T_X]); p.layer = c.layer; p.post = c.post; p.pre = c.pre;
    p.alpha = (float)c.alpha; p.eps = (float)c.eps;
    for (int i : {T_GATE, T_SCALE, T_SHIFT}) if (t[i].defined() && t[i].scalar_type() == at::kFloat) p.vec32 = 1;
    for (int i : {T_W1, T_B1, T_W2, T_B2}) if (t[i].defined() && t[i].scalar_type() == at::kFloat) p.w32 = 1;
    p.x = ptr(t[T_X]); p.ld_x = pitch[0];
    p.f = ptr(t[T_F]); p.ld_f = pitch[1];
    const auto vec = [&](int i, const void*& v, long& ld, int& shared) {
        if (!t[i].defined()) return;
        v = ptr(t[i]); ld = (long)t[i].stride(0); shared = t[i].dim() == 1;
    };
    vec(T_GATE, p.gate, p.ld_gate, p.shared_gate);
    vec(T_SCALE, p.scale, p.ld_scale, p.shared_scale);
    vec(T_SHIFT, p.shift, p.ld_shift, p.shared_shift);
    p.w1 = ptr(t[T_W1]); p.b1 = ptr(t[T_B1]); p.w2 = ptr(t[T_W2]); p.b2 = ptr(t[T_B2]);
    return p;
}

// r (where there is a block output) and u (where there is a pre norm); t[] leaves as the rows and vectors that the backward reads
variable_list norm_forward(Tensor* t, const NormCfg& c) {
    const std::vector<int64_t> shape(t[T_X].sizes().begin(), t[T_X].sizes().end());
    const Rows x = rows_of(t[T_X], c.C), f = rows_of(t[T_F], c.C);
    t[T_X] = x.t; t[T_F] = f.t;
    for (int i = T_GATE; i < T_COUNT; ++i) t[i] = side_by_side(t[i]);
    const Tensor r = f.t.defined() ? fresh(shape, x.t) : Tensor(), u = c.pre ? fresh(shape, x.t) : Tensor();
    if (c.B * c.T) {
        const long pitch[2] = {x.pitch, f.pitch};
        cdae_resnorm p = norm_args(t, pitch, c);
        p.r = mptr(r); p.u = mptr(u);
        check(cdae_resnorm_fwd(&p, stream_of(x.t)));
    }
    variable_list out;
    if (r.defined()) out.push_back(r);
    if (u.defined()) out.push_back(u);
    return out;
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    using Opt = std::optional<Tensor>;
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Opt& f, const Opt& gate, const Opt& scale, const Opt& shift, const Opt& w1, const Opt& b1,
                                 const Opt& w2, const Opt& b2, const NormCfg& c) {
        Tensor t[T_COUNT] = {x, of(f), of(gate), of(scale), of(shift), of(w1), of(b1), of(w2), of(b2)};
        variable_list out = norm_forward(t, c);
        ctx->save_for_backward(variable_list(t, t + T_COUNT));
        ctx->set_materialize_grads(false);
        ctx->saved_data["n"] = std::vector<int64_t>{c.B, c.T, c.C, c.layer, c.post, c.pre};
        ctx->saved_data["s"] = std::vector<double>{c.alpha, c.eps};
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list g(T_COUNT + 1);
        variable_list t = ctx->get_saved_variables();
        const std::vector<int64_t> n = ctx->saved_data["n"].toIntVector();
        const std::vector<double> s = ctx->saved_data["s"].toDoubleVector();
        const NormCfg c{n[0], n[1], n[2], s[0], s[1], n[3] != 0, n[4] != 0, n[5] != 0};
        const bool has_f = t[T_F].defined();
        const Tensor dr_ = has_f ? grads[0] : Tensor(), du_ = c.pre ? grads[has_f ? 1 : 0] : Tensor();
        if (!dr_.defined() && !du_.defined()) return g;
        no_tangent("residual_norm", dr_);
        no_tangent("residual_norm", du_);
        const bool none = c.B * c.T == 0;
        c10::DeviceGuard on(t[T_X].device());
        bool want[T_COUNT];
        for (size_t i = 0, edge = 0; i < T_COUNT; ++i) want[i] = t[i].defined() && ctx->needs_input_grad(edge++);
        for (int i = 0; i < T_COUNT; ++i) if (want[i]) g[i] = fresh(t[i].sizes(), t[i]);     // (each with memory of its own: one that is kept keeps no other)
        if (none) for (int i = T_GATE; i < T_COUNT; ++i) if (g[i].defined()) g[i].zero_();
        if (none) return once(std::move(g));
        const Rows x = rows_of(t[T_X], c.C), f = rows_of(t[T_F], c.C), dr = rows_of(dr_, c.C), du = rows_of(du_, c.C);
        const long pitch[2] = {x.pitch, f.pitch};
        t[T_X] = x.t; t[T_F] = f.t;                                           // (a hook on saved tensors may hand them back in another layout)
        for (int i = T_GATE; i < T_COUNT; ++i) t[i] = side_by_side(t[i]);
        cdae_resnorm p = norm_args(t.data(), pitch, c);
        p.dr = ptr(dr.t); p.ld_dr = dr.pitch;
        p.du = ptr(du.t); p.ld_du = du.pitch;
        p.dx = mptr(g[T_X]); p.df = mptr(g[T_F]); p.dgate = mptr(g[T_GATE]); p.dscale = mptr(g[T_SCALE]); p.dshift = mptr(g[T_SHIFT]);
        p.dw1 = mptr(g[T_W1]); p.db1 = mptr(g[T_B1]); p.dw2 = mptr(g[T_W2]); p.db2 = mptr(g[T_B2]);
        p.ws_bytes = std::any_of(want + T_GATE, want + T_COUNT, [](bool w) { return w; }) ? cdae_resnorm_workspace_bytes(p.B, p.T, p.C) : 256;
        const Tensor ws = scratch(p.ws_bytes, x.t);
        p.ws = (float*)mptr(ws);
        check(cdae_resnorm_bwd(&p, stream_of(x.t)));
        return once(std::move(g));
    }
};

py::tuple residual_norm(const Tensor& x, const std::optional<Tensor>& f_, const std::optional<Tensor>& gate, const std::optional<Tensor>& scale,
                        const std::optional<Tensor>& shift, bool post, const std::optional<Tensor>& w1, const std::optional<Tensor>& b1, bool pre,
                        const std::optional<Tensor>& w2, const std::optional<Tensor>& b2, double alpha, const std::string& kind, double eps) {
    const char* who = "residual_norm";
    const Tensor f = of(f_);
    const Tensor vec[3] = {of(gate), of(scale), of(shift)}, w[4] = {of(w1), of(b1), of(w2), of(b2)};
    same_device(who, x, {f, vec[0], vec[1], vec[2], w[0], w[1], w[2], w[3]});
    REFUSE(kind == "layer" || kind == "rms", who, ": kind is \"layer\" or \"rms\"");
    REFUSE(type_of(x) >= 0, who, ": bf16, fp16 or fp32 rows (got ", x.scalar_type(), ")");
    REFUSE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 8192, who, ": rows of 1 to 8192 features");
    const int64_t C = x.size(-1), M = x.numel() / C;
    REFUSE(M <= (1LL << 30), who, ": at most 2^30 rows");
    REFUSE(std::isfinite((float)alpha) && std::isfinite((float)eps) && eps >= 0, who, ": alpha finite, eps finite and not negative");
    REFUSE(!f.defined() || (f.sizes() == x.sizes() && f.scalar_type() == x.scalar_type()), who, ": f of x's shape and type");
    REFUSE(f.defined() || pre, who, ": without f there is only the pre norm to compute");
    REFUSE(f.defined() || (!vec[0].defined() && !post), who, ": a gate and a post norm belong to f");
    REFUSE(pre || (!vec[1].defined() && !vec[2].defined()), who, ": scale and shift belong to the pre norm");
    const auto type_ok = [&](const Tensor& t) { return t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat; };
    const Tensor* one = nullptr;
    for (const Tensor& t : w) {
        if (!t.defined()) continue;
        REFUSE(t.dim() == 1 && t.size(0) == C && type_ok(t), who, ": weights and biases [", C, "] in the rows' type or fp32");
        REFUSE(!one || one->scalar_type() == t.scalar_type(), who, ": weights and biases of one type");
        one = &t;
    }
    one = nullptr;
    int64_t B = -1;
    for (const Tensor& t : vec) {
        if (!t.defined()) continue;
        REFUSE((t.dim() == 1 || t.dim() == 2) && t.size(-1) == C && type_ok(t), who, ": gate, scale and shift [", C, "] or [B, ", C, "] in the rows' type or fp32");
        REFUSE(!one || one->scalar_type() == t.scalar_type(), who, ": gate, scale and shift of one type");
        one = &t;
        if (t.dim() == 1) continue;
        const int64_t b = t.size(0);
        REFUSE(x.dim() > 2 ? b == x.size(0) : b == M || (b >= 1 && M % b == 0), who, ": gate, scale and shift have a row for each sample of x (got ", t.sizes(), " beside ",
               x.sizes(), ")");
        REFUSE(B < 0 || B == b, who, ": gate, scale and shift for the same samples");
        B = b;
    }
    if (B < 0) B = 1;
    const NormCfg c{B, B ? M / B : 0, C, alpha, eps, kind == "layer", post, pre};
    c10::DeviceGuard on(x.device());
    variable_list out;
    if (wanted({x, f, vec[0], vec[1], vec[2], w[0], w[1], w[2], w[3]})) {
        REFUSE(B < (1LL << 22), who, ": with gradients fewer than 2^22 samples");
        capturable(who, x, {x, f, vec[0], vec[1], vec[2], w[0], w[1], w[2], w[3]});
        out = ResidualNorm::apply(x, maybe(f), maybe(vec[0]), maybe(vec[1]), maybe(vec[2]), maybe(w[0]), maybe(w[1]), maybe(w[2]), maybe(w[3]), c);
    } else {
        Tensor t[T_COUNT] = {x, f, vec[0], vec[1], vec[2], w[0], w[1], w[2], w[3]};
        out = norm_forward(t, c);
    }
    const Tensor r = f.defined() ? out[0] : x;
    return py::make_tuple(r, pre ? py::cast(out.back()) : py::object(py::none()));
}

// ----------------------------------------------------------------------------- the global norm of many gradients
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

struct List {
    std::vector<Tensor> t;
    std::vector<const void*> p;
    std::vector<long> n;
    std::vector<int> ty;
    at::Device dev{at::kCUDA, 0};
    List(const char* who, const py::handle& list) {
        for (py::handle h : list) {
            REFUSE(THPVariable_Check(h.ptr()), who, ": a list of tensors");
            const Tensor& x = THPVariable_Unpack(h.ptr());
            REFUSE(x.is_cuda() && has_values(x) && type_of(x) >= 0, who, ": dense bf16, fp16 or fp32 tensors on an MI355X device; there is no CPU form");
            REFUSE(t.empty() || x.device() == t[0].device(), who, ": tensors of one device");
            no_tangent(who, x);
            t.push_back(x);
        }
        dev = t.empty() ? at::Device(at::kCUDA, c10::hip::current_device()) : t[0].device();
    }
    void read_dense() {
        for (Tensor& x : t) {
            if (x.is_neg()) x = x.detach().resolve_neg();
            if (!dense(x)) x = x.detach().contiguous();
        }
    }
    void arrays() {
        p.clear(); n.clear(); ty.clear();
        for (const Tensor& x : t) { p.push_back(x.const_data_ptr()); n.push_back((long)x.numel()); ty.push_back(type_of(x)); }
    }
};
void numbers(const char* who, double scale, double max_norm) {
    REFUSE(std::isfinite(scale), who, ": scale must be finite");
    REFUSE(max_norm >= 0, who, ": max_norm must be a number >= 0");
}

Tensor norm_and_factor(List& l, double scale, double max_norm) {
    c10::DeviceGuard on(l.dev);
    l.arrays();
    Tensor out = at::empty({2}, at::TensorOptions().dtype(at::kFloat).device(l.dev));
    const size_t need = cdae_grad_workspace_bytes();
    const Tensor ws = scratch(need, out);
    check(cdae_grad_norm(l.p.data(), l.n.data(), l.ty.data(), (int)l.t.size(), scale, max_norm, (float*)mptr(out), mptr(ws), need, stream_of(out)));
    return out;
}
Tensor grad_factor(const char* who, const py::object& grads, double scale, double max_norm) {
    numbers(who, scale, max_norm);
    List l(who, grads);
    l.read_dense();
    return norm_and_factor(l, scale, max_norm);
}

Tensor clip_grad_norm(const py::object& grads, double max_norm, double scale, const py::object& out, bool error_if_nonfinite) {
    const char* who = "clip_grad_norm_";
    numbers(who, scale, max_norm);
    at::NoGradGuard no_grad;
    List src(who, grads);
    c10::DeviceGuard on(src.dev);
    REFUSE(!error_if_nonfinite || !capturing(src.dev), who, ": error_if_nonfinite waits for the device and cannot be captured");
    std::vector<std::pair<Tensor, Tensor>> later;              // (tensor with gaps or negated, dense copy): written back at the end
    List dst = out.is_none() ? src : List(who, out);
    REFUSE(dst.t.size() == src.t.size(), who, ": an output for every gradient");
    for (size_t i = 0; i < src.t.size(); ++i) {
        Tensor &a = src.t[i], &b = dst.t[i];
        if (out.is_none()) {
            if (dense(a) && !a.is_neg()) continue;
            for (int64_t d = 0; d < a.dim(); ++d) REFUSE(a.size(d) <= 1 || a.stride(d) != 0, who, ": an expanded tensor cannot be written in place");
            b = as_written(a).contiguous();
            later.emplace_back(a, b);
            a = b;
        } else {
            REFUSE(a.sizes() == b.sizes() && b.device() == src.dev, who, ": outputs of the gradients' shapes, on their device");
            REFUSE(dense(b) && !b.is_neg(), who, ": outputs without gaps, their values as they are");
            if (a.is_neg()) a = a.resolve_neg();
            if (!(a.is_contiguous() && b.is_contiguous()) && !(dense(a) && a.strides() == b.strides())) a = at::empty_strided(b.sizes(), b.strides(), a.options()).copy_(a);
        }
    }
    src.arrays();
    dst.arrays();
    Tensor norm = at::empty({2}, at::TensorOptions().dtype(at::kFloat).device(src.dev));
    if (error_if_nonfinite) {
        const float n = norm_and_factor(src, scale, max_norm)[0].item<float>();
        REFUSE(std::isfinite(n), who, ": the norm of the gradients is not finite (", n, ")");
    }
    const size_t need = cdae_grad_workspace_bytes();
    const Tensor ws = scratch(need, norm);
    check(cdae_grad_clip(src.p.data(), src.n.data(), src.ty.data(), (void* const*)dst.p.data(), dst.ty.data(), (int)src.t.size(), scale, max_norm, (float*)mptr(norm), mptr(ws),
                         need, stream_of(norm)));
    for (const auto& k : later) k.first.copy_(k.second);
    for (const Tensor& t : dst.t) if (!t.is_inference()) torch::autograd::impl::bump_version(t);       // (the kernel wrote them behind autograd's back)
    return norm[0];
}

PyObject* error_class = nullptr;
PyObject* memory_class = nullptr;

}  // namespace

PYBIND11_MODULE(_block_ext, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused& e) {
            PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
        } catch (const c10::OutOfMemoryError& e) {
            PyErr_SetString(memory_class ? memory_class : PyExc_RuntimeError, e.what_without_backtrace());
        }
    });
    m.def("set_errors", [](py::object refused, py::object memory) { error_class = refused.release().ptr(); memory_class = memory.release().ptr(); });
    m.def("linear_act", &linear_act);
    m.def("residual_norm", &residual_norm);
    m.def("grad_norm", [](const py::object& g, double scale) { return grad_factor("grad_norm", g, scale, INFINITY)[0]; });
    m.def("grad_factor", [](const py::object& g, double max_norm, double scale) { return grad_factor("grad_factor", g, scale, max_norm); });
    m.def("clip_grad_norm_", &clip_grad_norm);
}

// torch side of the sequence operators (ops.py documents them): argument checks, the autograd nodes and the calls into
// libnsdecode.so, whose entry points bind() is handed as addresses.  Host code only.  In C++ because a layer calls these
// several times a step: through Python's autograd functions a forward and backward pass of a small attention took 70 to
// 130 us of the host's time, according to where the engine's thread ran.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/custom_class.h>
#include <torch/extension.h>
#include <cmath>
#include <string>
#include "nsdecode.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct NsdError : std::runtime_error { using std::runtime_error::runtime_error; };

struct Entries {
    decltype(&nsd_strerror) strerror;
    decltype(&nsd_attn_fwd_workspace) attn_fwd_workspace;
    decltype(&nsd_attn_fwd) attn_fwd;
    decltype(&nsd_attn_bwd_workspace) attn_bwd_workspace;
    decltype(&nsd_attn_bwd) attn_bwd;
    decltype(&nsd_attn_prefix_workspace) attn_prefix_workspace;
    decltype(&nsd_attn_prefix) attn_prefix;
    decltype(&nsd_attn_step) attn_step;
    decltype(&nsd_add_rmsnorm) add_rmsnorm;
    decltype(&nsd_add_rmsnorm_bwd_workspace) add_rmsnorm_bwd_workspace;
    decltype(&nsd_add_rmsnorm_bwd) add_rmsnorm_bwd;
} lib;

void check(int rc, const char *what)
{
    if (rc) throw NsdError(std::string(what) + " failed: " + lib.strerror(rc) + " (" + std::to_string(rc) + ")");
}
[[noreturn]] void bad_value(const std::string &s) { throw pybind11::value_error(s); }

std::string shape(const Tensor &t)
{
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}
void same_device(const char *name, const Tensor &first, std::initializer_list<const Tensor *> more)
{
    if (!first.is_cuda()) throw NsdError(std::string(name) + " needs device tensors (there is no CPU fall-back)");
    for (const Tensor *t : more)
        if (t->defined() && t->device() != first.device())
            bad_value(std::string(name) + ": tensors on " + first.device().str() + " and " + t->device().str());
}
// the element type's number, the same for all
int same_type(const char *name, const Tensor &first, std::initializer_list<const Tensor *> more)
{
    if (first.scalar_type() != at::kFloat && first.scalar_type() != at::kBFloat16)
        throw pybind11::type_error(std::string(name) + " takes float32 or bfloat16");
    for (const Tensor *t : more)
        if (t->defined() && t->scalar_type() != first.scalar_type())
            throw pybind11::type_error(std::string(name) + ": tensors of different types");
    return first.scalar_type() == at::kBFloat16;
}
// Tangents of forward-mode differentiation would be lost in the calls below, whether or not the tensor also requires a
// gradient.
void no_tangents(const char *name, std::initializer_list<const Tensor *> ts)
{
    for (const Tensor *t : ts)
        if (t->defined() && t->_fw_grad(/*level=*/0).defined()) bad_value(std::string(name) + " has no forward-mode derivative");
}
double scale_or_default(const char *name, std::optional<double> scale, int64_t hd)
{
    const double s = scale ? *scale : 1.0 / std::sqrt((double)hd);
    if (!(s > 0.0) || !((float)s > 0.0f) || !std::isfinite((float)s)) bad_value(std::string(name) + ": scale is a positive number");
    return s;
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor scratch(int64_t bytes, const Tensor &like)
{
    return bytes ? at::empty({bytes}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
bool aligned(const Tensor &t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }

// t, or a copy of it, with consecutive elements in its rows and everything else in steps of 16 bytes, and with the values
// themselves in memory (a view may have a sign that is not applied there yet: the imaginary part of a conjugate)
Tensor in_rows(const Tensor &t)
{
    const int64_t piece = 16 / t.element_size();
    bool ok = t.stride(-1) == 1 && !t.is_neg() && aligned(t);
    for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) == 1 || t.stride(i) % piece == 0);
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
Tensor packed(const Tensor &t)
{
    const Tensor c = t.resolve_neg().contiguous();
    return aligned(c) ? c : c.clone();
}
void strides(int64_t (&s)[3], const Tensor &t, int a, int b, int c)
{
    const int axis[3] = {a, b, c};                              // (the stride of an axis of one element says nothing)
    for (int i = 0; i < 3; ++i) s[i] = t.size(axis[i]) > 1 ? t.stride(axis[i]) : 0;
}

// What a node keeps for its backward pass beside tensors: a number and a truth value of the call, and the way to its
// arguments' own nodes.
struct Kept : torch::CustomClassHolder {
    double number;
    bool flag;
    torch::autograd::edge_list edges;
};
template <class... Args> void keep(AutogradContext *ctx, double number, bool flag, const Args &...args)
{
    auto k = c10::make_intrusive<Kept>();
    k->number = number;
    k->flag = flag;
    k->edges = torch::autograd::collect_next_edges(args...);
    ctx->saved_data["kept"] = at::IValue::make_capsule(std::move(k));
}
const Kept &kept(AutogradContext *ctx) { return *static_cast<const Kept *>(ctx->saved_data["kept"].toCapsule().get()); }

// Gradients computed by these nodes are not differentiable themselves: where a graph of them is asked for, they carry a
// node that raises when it is walked.  It leads on to what they depend on, the operator's arguments and the gradients that
// came in: a walk to one of those that met no node on its way would take them for independent of it, and give zeros.
variable_list once(AutogradContext *ctx, const variable_list &came_in, variable_list grads, const char *name)
{
    if (!at::GradMode::is_enabled()) return grads;
    auto edges = kept(ctx).edges;
    for (auto &e : torch::autograd::collect_next_edges(came_in)) edges.push_back(std::move(e));
    const auto error = std::make_shared<torch::autograd::Error>(std::string(name) + " is differentiable once", std::move(edges));
    for (auto &g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::set_history(g, error);
        }
    return grads;
}

// ---------------------------------------------------------------------- attention of whole sequences
NsdSeqAttn seq_of(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &mask, bool causal, double scale)
{
    NsdSeqAttn p{};
    p.batch = (int)q.size(0); p.len_q = (int)q.size(1); p.heads = (int)q.size(2); p.hd = (int)q.size(3);
    p.len_k = (int)k.size(1); p.kv_heads = (int)k.size(2);
    p.dtype = q.scalar_type() == at::kBFloat16;
    p.causal = causal;
    p.scale = (float)scale;
    strides(p.q_stride, q, 0, 1, 2);
    strides(p.k_stride, k, 0, 1, 2);
    strides(p.v_stride, v, 0, 1, 2);
    p.key_mask = (const uint8_t *)ptr(mask);
    return p;
}

Tensor attn_fwd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &mask, bool causal, double scale, Tensor *lse, Tensor *rest)
{
    const c10::DeviceGuard guard(q.device());
    const auto opt = q.options().requires_grad(false);
    const NsdSeqAttn p = seq_of(q, k, v, mask, causal, scale);
    Tensor out = at::empty(q.sizes(), opt);
    if (lse) {
        *lse = at::empty({q.size(0), k.size(2), q.size(1), q.size(2) / k.size(2)}, opt.dtype(at::kFloat));
        if (p.dtype) *rest = at::empty(q.sizes(), opt.dtype(at::kByte));
    }
    const int64_t n = lib.attn_fwd_workspace(&p);
    const Tensor ws = scratch(n, q);
    check(lib.attn_fwd(ptr(q), ptr(k), ptr(v), &p, ptr(out), lse ? (float *)ptr(*lse) : nullptr, lse ? (uint8_t *)ptr(*rest) : nullptr,
                       ptr(ws), n, stream_of(q)), "nsd_attn_fwd");
    return out;
}

struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q0, const Tensor &k0, const Tensor &v0, const OptTensor &mask0, bool causal, double scale)
    {
        const Tensor mask = mask0 ? *mask0 : Tensor();
        const Tensor q = in_rows(q0), k = in_rows(k0), v = in_rows(v0);
        Tensor lse, rest;
        Tensor out = attn_fwd(q, k, v, mask, causal, scale, &lse, &rest);
        ctx->save_for_backward({q, k, v, mask, out, lse, rest});
        keep(ctx, scale, causal, q0, k0, v0);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &mask = saved[3], &out = saved[4], &lse = saved[5], &rest = saved[6];
        no_tangents("attention's gradient", {&q, &k, &v, &grads[0]});
        variable_list d(6);
        {
            const c10::DeviceGuard guard(q.device());
            const at::AutoGradMode no_grad(false);
            const NsdSeqAttn p = seq_of(q, k, v, mask, kept(ctx).flag, kept(ctx).number);
            const auto opt = q.options().requires_grad(false);
            const Tensor dout = packed(grads[0]);
            d[0] = at::empty(q.sizes(), opt);
            d[1] = at::empty(k.sizes(), opt);
            d[2] = at::empty(k.sizes(), opt);
            const int64_t n = lib.attn_bwd_workspace(&p);
            const Tensor ws = scratch(n, q);
            check(lib.attn_bwd(ptr(q), ptr(k), ptr(v), ptr(out), (const float *)ptr(lse), (const uint8_t *)ptr(rest), ptr(dout), &p,
                               ptr(d[0]), ptr(d[1]), ptr(d[2]), ptr(ws), n, stream_of(q)), "nsd_attn_bwd");
        }
        return once(ctx, grads, std::move(d), "attention");
    }
};

Tensor attention(const Tensor &q, const Tensor &k, const Tensor &v, bool causal, const OptTensor &key_mask, std::optional<double> scale)
{
    if (q.dim() != 4 || k.dim() != 4 || !v.sizes().equals(k.sizes()))
        bad_value("attention takes q [Z, Lq, heads, hd] and k, v [Z, Lk, kv_heads, hd]");
    const int64_t Z = q.size(0), H = q.size(2), D = q.size(3), KVH = k.size(2);
    if (k.size(0) != Z || k.size(3) != D || KVH < 1 || H < 1 || H % KVH)
        bad_value("attention: q " + shape(q) + " does not go with k " + shape(k));
    if (D < 8 || D > 128 || D % 8) bad_value("attention: head dimension " + std::to_string(D) + " is not a multiple of 8 up to 128");
    for (int64_t n : {Z, q.size(1), k.size(1), H})
        if (n > INT32_MAX) bad_value("attention: an axis of more than 2^31 - 1");
    Tensor mask = key_mask ? *key_mask : Tensor();
    no_tangents("attention", {&q, &k, &v});
    const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
    if (grad && Z > 0) {                                        // a shape that only the gradients refuse is refused here
        NsdSeqAttn p = seq_of(q, k, v, Tensor(), causal, 1.0);
        p.len_q = p.len_q > 0 ? p.len_q : 1;                    // (no queries need no scratch either)
        if (!lib.attn_bwd_workspace(&p)) check(NSD_E_SIZE, "nsd_attn_bwd");
    }
    same_device("attention", q, {&k, &v, &mask});
    same_type("attention", q, {&k, &v});
    if (mask.defined()) {
        if ((mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte) || mask.dim() != 2 || mask.size(0) != Z || mask.size(1) != k.size(1))
            bad_value("attention: key_mask is [Z, Lk] of bool or uint8");
        mask = mask.contiguous();
    }
    const double s = scale_or_default("attention", scale, D);
    if (grad)
        return Attention::apply(q, k, v, mask.defined() ? OptTensor(mask) : OptTensor(), causal, s);
    const at::AutoGradMode no_grad(false);
    return attn_fwd(in_rows(q), in_rows(k), in_rows(v), mask, causal, s, nullptr, nullptr);
}

// ---------------------------------------------------------------------- a beam step over shared prefixes
Tensor shared_prefix_attention(const Tensor &q0, const std::vector<std::vector<Tensor>> &prefixes, const Tensor &kgen, const Tensor &vgen,
                               const OptTensor &anc0, int64_t t, int64_t beam, std::optional<double> scale)
{
    const char *name = "shared_prefix_attention";
    const std::string at_ = std::string(name) + ": ";
    const Tensor anc = anc0 ? *anc0 : Tensor();
    if (q0.dim() != 3 || kgen.dim() != 4 || !vgen.sizes().equals(kgen.sizes()))
        bad_value(at_ + "q is [M, heads, hd], kgen and vgen [T, M, kv_heads, hd]");
    const int64_t M = q0.size(0), H = q0.size(1), D = q0.size(2), T = kgen.size(0), KVH = kgen.size(2);
    const int64_t G = KVH > 0 && H % KVH == 0 ? H / KVH : 0;
    if (kgen.size(1) != M || kgen.size(3) != D || !(G == 1 || G == 2 || G == 3 || G == 4 || G == 8))
        bad_value(at_ + "q " + shape(q0) + " does not go with kgen " + shape(kgen));
    if (D < 8 || D > 128 || (D & (D - 1))) bad_value(at_ + "head dimension " + std::to_string(D) + " is not a power of two from 8 to 128");
    if (beam < 1 || beam > NSD_MAX_BEAM || M % beam || t < 0 || t >= T || M > INT32_MAX)
        bad_value(at_ + "beam divides M and is at most 64, and 0 <= t < len(kgen)");
    no_tangents(name, {&q0, &kgen, &vgen});
    for (const auto &p : prefixes)
        if (p.size() >= 2) no_tangents(name, {&p[0], &p[1]});
    same_device(name, q0, {&kgen, &vgen, &anc});
    const int dt = same_type(name, q0, {&kgen, &vgen});
    bool grad = q0.requires_grad() || kgen.requires_grad() || vgen.requires_grad();
    if (!kgen.is_contiguous() || !vgen.is_contiguous() || kgen.is_neg() || vgen.is_neg() || (anc.defined() && !anc.is_contiguous()))
        bad_value(at_ + "the generated cache and its ancestor table are contiguous");
    if (t > 0 && (!anc.defined() || anc.scalar_type() != at::kByte || anc.dim() != 2 || anc.size(0) < t || anc.size(1) != M))
        bad_value(at_ + "anc is uint8 [>= t, M]");
    for (const auto &p : prefixes) {
        if ((p.size() != 2 && p.size() != 3) || p[0].dim() != 4 || !p[1].sizes().equals(p[0].sizes()))
            bad_value(at_ + "a prefix is (k, v) or (k, v, lens), k and v [groups, kv_heads, P, hd]");
        const int64_t n = p[0].size(0);
        if (n < 1 || M % n || p[0].size(1) != KVH || p[0].size(3) != D || p[0].size(2) > INT32_MAX)
            bad_value(at_ + "a prefix " + shape(p[0]) + " does not go with q " + shape(q0));
        same_device(name, q0, {&p[0], &p[1]});
        same_type(name, q0, {&p[0], &p[1]});
        grad = grad || p[0].requires_grad() || p[1].requires_grad();
        if (p.size() == 3) {
            same_device(name, q0, {&p[2]});
            if (p[2].scalar_type() != at::kInt || p[2].dim() != 1 || p[2].size(0) != n) bad_value(at_ + "lens is int32 [groups]");
        }
    }
    if (at::GradMode::is_enabled() && grad) bad_value(at_ + "it has no gradient: call it under torch.no_grad()");
    const double s = scale_or_default(name, scale, D);

    const at::AutoGradMode no_grad(false);
    const c10::DeviceGuard guard(q0.device());
    void *stream = stream_of(q0);
    const Tensor q = packed(q0);
    Tensor out = at::empty(q.sizes(), q.options().requires_grad(false));
    if (M == 0) return out;
    if (!aligned(kgen) || !aligned(vgen)) bad_value(at_ + "the generated cache starts at a multiple of 16 bytes");
    Tensor state;
    float *po = nullptr, *pm = nullptr, *pl = nullptr;
    for (const auto &p : prefixes) {
        const Tensor k = in_rows(p[0]), v = in_rows(p[1]), lens = p.size() == 3 ? p[2].contiguous() : Tensor();
        const bool first = !state.defined();
        if (first) {
            state = at::empty({M * H * (D + 2)}, q.options().dtype(at::kFloat).requires_grad(false));
            po = (float *)state.data_ptr();
            pm = po + M * H * D;
            pl = pm + M * H;
        }
        NsdSeqAttn a{};
        a.batch = (int)k.size(0); a.len_q = (int)(M / k.size(0)); a.len_k = (int)k.size(2);
        a.heads = (int)H; a.kv_heads = (int)KVH; a.hd = (int)D; a.dtype = dt;
        a.scale = (float)s;
        a.q_stride[0] = a.len_q * H * D; a.q_stride[1] = H * D; a.q_stride[2] = D;
        strides(a.k_stride, k, 0, 2, 1);
        strides(a.v_stride, v, 0, 2, 1);
        a.key_len = (const int32_t *)ptr(lens);
        const int64_t n = lib.attn_prefix_workspace(&a);
        const Tensor ws = scratch(n, q);
        check(lib.attn_prefix(ptr(q), ptr(k), ptr(v), &a, !first, po, pm, pl, ptr(ws), n, stream), "nsd_attn_prefix");
    }
    check(lib.attn_step(ptr(q), nullptr, nullptr, ptr(kgen), ptr(vgen), (const uint8_t *)ptr(anc), ptr(out), (int)(M / beam), (int)beam, (int)H,
                        (int)KVH, (int)D, 0, (int)t, (float)s, dt, po, pm, pl, stream), "nsd_attn_step");
    return out;
}

// ---------------------------------------------------------------------- residual add + RMSNorm
// (x_out, h); x_out is x itself where there is no delta
std::pair<Tensor, Tensor> norm_fwd(const Tensor &x, const Tensor &xc, const Tensor &dc, const Tensor &wc, double eps)
{
    const c10::DeviceGuard guard(x.device());
    const auto opt = x.options().requires_grad(false);
    const int64_t hidden = x.size(-1);
    Tensor h = at::empty(x.sizes(), opt), x_out = dc.defined() ? at::empty(x.sizes(), opt) : Tensor();
    check(lib.add_rmsnorm(ptr(xc), ptr(dc), ptr(wc), (float)eps, (int)(x.numel() / hidden), (int)hidden, x.scalar_type() == at::kBFloat16,
                          ptr(x_out), ptr(h), stream_of(x)), "nsd_add_rmsnorm");
    return {x_out.defined() ? x_out : x, h};
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &delta0, const Tensor &w, double eps)
    {
        const Tensor delta = delta0 ? *delta0 : Tensor();
        ctx->set_materialize_grads(false);
        const Tensor xc = packed(x), dc = delta.defined() ? packed(delta) : Tensor(), wc = packed(w);
        auto [x_out, h] = norm_fwd(x, xc, dc, wc, eps);
        ctx->save_for_backward({delta.defined() ? x_out : xc, wc});
        keep(ctx, eps, delta.defined(), x, delta, w);
        return {x_out, h};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1];
        no_tangents("add_rms_norm's gradient", {&x, &w, &grads[0], &grads[1]});
        const bool delta = kept(ctx).flag;
        const bool want_w = ctx->needs_input_grad(delta ? 2 : 1);   // (counts the tensors among the inputs)
        variable_list d(4);
        {
            const c10::DeviceGuard guard(x.device());
            const at::AutoGradMode no_grad(false);
            const int64_t hidden = x.size(-1), rows = x.numel() / hidden;
            const auto opt = x.options().requires_grad(false);
            Tensor dx, dw;
            if (!grads[1].defined()) {                          // h is not used: the sum's gradient passes through
                dx = grads[0];
                if (want_w) dw = at::zeros(w.sizes(), opt);
            } else {
                const Tensor dh = packed(grads[1]), go = grads[0].defined() ? packed(grads[0]) : Tensor();
                dx = at::empty(x.sizes(), opt);
                if (want_w) dw = at::empty(w.sizes(), opt);
                const int64_t n = want_w ? lib.add_rmsnorm_bwd_workspace((int)rows, (int)hidden) : 0;
                const Tensor ws = scratch(n, x);
                check(lib.add_rmsnorm_bwd(ptr(x), ptr(w), ptr(dh), ptr(go), (float)kept(ctx).number, (int)rows, (int)hidden,
                                          x.scalar_type() == at::kBFloat16, ptr(dx), ptr(dw), ptr(ws), n, stream_of(x)), "nsd_add_rmsnorm_bwd");
            }
            if (ctx->needs_input_grad(0)) d[0] = dx;
            if (delta && ctx->needs_input_grad(1)) d[1] = dx;
            d[2] = dw;
        }
        if (!grads[1].defined()) return d;                      // (what only passed through keeps its own history)
        return once(ctx, grads, std::move(d), "add_rms_norm");
    }
};

std::pair<Tensor, Tensor> add_rms_norm(const Tensor &x, const OptTensor &delta0, const Tensor &w, double eps)
{
    const Tensor delta = delta0 ? *delta0 : Tensor();
    if (x.dim() < 1 || w.dim() != 1 || w.size(0) != x.size(-1) || (delta.defined() && !delta.sizes().equals(x.sizes())))
        bad_value("add_rms_norm takes x and delta [..., hidden] and w [hidden]");
    no_tangents("add_rms_norm", {&x, &delta, &w});
    same_device("add_rms_norm", x, {&delta, &w});
    const int dt = same_type("add_rms_norm", x, {&delta, &w}), unit = dt ? 8 : 4;
    const int64_t hidden = x.size(-1);
    if (hidden < 1 || hidden % unit || hidden > INT32_MAX)
        bad_value("add_rms_norm: hidden = " + std::to_string(hidden) + " is not a multiple of " + std::to_string(unit));
    if (x.numel() / hidden > INT32_MAX) bad_value("add_rms_norm: at most 2^31 - 1 rows");
    if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (delta.defined() && delta.requires_grad()))) {
        auto r = AddRmsNorm::apply(x, delta0, w, eps);
        return {r[0], r[1]};
    }
    const at::AutoGradMode no_grad(false);
    return norm_fwd(x, packed(x), delta.defined() ? packed(delta) : Tensor(), packed(w), eps);
}

template <class F> void set(F &f, const std::map<std::string, uintptr_t> &a, const char *name) { f = reinterpret_cast<F>(a.at(name)); }

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    namespace py = pybind11;
    // addresses of the library's entry points, and the class its errors are raised as
    m.def("bind", [](const std::map<std::string, uintptr_t> &a, py::object error) {
        set(lib.strerror, a, "nsd_strerror");
        set(lib.attn_fwd_workspace, a, "nsd_attn_fwd_workspace");
        set(lib.attn_fwd, a, "nsd_attn_fwd");
        set(lib.attn_bwd_workspace, a, "nsd_attn_bwd_workspace");
        set(lib.attn_bwd, a, "nsd_attn_bwd");
        set(lib.attn_prefix_workspace, a, "nsd_attn_prefix_workspace");
        set(lib.attn_prefix, a, "nsd_attn_prefix");
        set(lib.attn_step, a, "nsd_attn_step");
        set(lib.add_rmsnorm, a, "nsd_add_rmsnorm");
        set(lib.add_rmsnorm_bwd_workspace, a, "nsd_add_rmsnorm_bwd_workspace");
        set(lib.add_rmsnorm_bwd, a, "nsd_add_rmsnorm_bwd");
        static PyObject *cls = nullptr;
        Py_XDECREF(cls);
        cls = error.release().ptr();
        static bool once = false;
        if (!once) {
            once = true;
            py::register_exception_translator([](std::exception_ptr e) {
                try {
                    if (e) std::rethrow_exception(e);
                } catch (const NsdError &x) {
                    PyErr_SetString(cls, x.what());
                }
            });
        }
    });
    const auto release = py::call_guard<py::gil_scoped_release>();
    m.def("attention", &attention, release);
    m.def("shared_prefix_attention", &shared_prefix_attention, release);
    m.def("add_rms_norm", &add_rms_norm, release);
}

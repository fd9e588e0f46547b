// Host path of the sequence-model operators: torch autograd nodes over the C
// entries of liblifb (include/lifscan_b200.h), without Python in them.
//
// What bounds a small call is the host: a kernel of 3 us behind 6 to 14 us of calls, and
// in training an autograd engine that alone takes 50 to 90 us a backward.  Measured a
// call, through ctypes and torch.autograd.Function -> through these functions:
//   attention step, 1 token, 4 heads of 64      14.0 ->  6.1 us
//   norm/gate/residual, 1 row of 256            17.2 ->  7.6
//   embedding, 64 tokens                        11.5 ->  6.2
//   norm/gate/residual, training, fp32           164 ->  121  (65536 rows of 256)
//   embedding, training, 65536 tokens of 700     105 ->   70
// They take the calls whose types, shapes, devices and layouts the C entries take as they
// are and return None for all others: the Python functions of the same names then convert
// what can be converted and refuse the rest.
//
// The library is not linked: bind() gets the addresses of its functions, and the
// Python function that turns a status into the package's exception.
#include <atomic>
#include <chrono>

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "lifscan_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entries {
    decltype(&lifb_embed_fwd) embed_fwd;
    decltype(&lifb_embed_bwd) embed_bwd;
    decltype(&lifb_embed_bwd_workspace_bytes) embed_bwd_ws;
    decltype(&lifb_norm_gate_fwd) norm_fwd;
    decltype(&lifb_norm_gate_bwd) norm_bwd;
    decltype(&lifb_norm_gate_bwd_workspace_bytes) norm_bwd_ws;
    decltype(&lifb_leaky_attn_fwd) attn_fwd;
    decltype(&lifb_leaky_attn_bwd) attn_bwd;
    decltype(&lifb_leaky_attn_workspace_bytes) attn_ws;
    decltype(&lifb_leaky_attn_step) attn_step;
    decltype(&lifb_poll_device) poll;
    py::object *check;  // check(status, what) raises; never freed: outlives the interpreter's teardown
} L;

void bind(const std::map<std::string, uint64_t> &at, const py::object &check)
{
    auto set = [&](auto &fn, const char *name) {
        fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(at.at(name));
    };
    set(L.embed_fwd, "lifb_embed_fwd");
    set(L.embed_bwd, "lifb_embed_bwd");
    set(L.embed_bwd_ws, "lifb_embed_bwd_workspace_bytes");
    set(L.norm_fwd, "lifb_norm_gate_fwd");
    set(L.norm_bwd, "lifb_norm_gate_bwd");
    set(L.norm_bwd_ws, "lifb_norm_gate_bwd_workspace_bytes");
    set(L.attn_fwd, "lifb_leaky_attn_fwd");
    set(L.attn_bwd, "lifb_leaky_attn_bwd");
    set(L.attn_ws, "lifb_leaky_attn_workspace_bytes");
    set(L.attn_step, "lifb_leaky_attn_step");
    set(L.poll, "lifb_poll_device");
    if (!L.check) L.check = new py::object();
    *L.check = check;
}

int type_of(const Tensor &t)
{
    switch (t.scalar_type()) {
        case torch::kFloat: return LIFB_F32;
        case torch::kBFloat16: return LIFB_BF16;
        case torch::kHalf: return LIFB_F16;
        default: return -1;
    }
}

void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
void *at(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *at_f32(const Tensor &t) { return static_cast<float *>(at(t)); }
const int32_t *at_i32(const Tensor &t) { return static_cast<const int32_t *>(at(t)); }

// A call's status, in Python's thread
void done(int status, const char *what)
{
    if (status != LIFB_OK) (*L.check)(status, what);
}

// The library's poll of the current device, at most every 20 ms and not while a graph is
// captured
int poll_sometimes()
{
    static std::atomic<int64_t> again[64];  // a device each
    const int64_t now = std::chrono::duration_cast<std::chrono::milliseconds>(
                            std::chrono::steady_clock::now().time_since_epoch())
                            .count();
    auto &due = again[c10::cuda::current_device() & 63];
    if (now < due.load(std::memory_order_relaxed) ||
        c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
        return LIFB_OK;
    due.store(now + 20, std::memory_order_relaxed);
    return L.poll();
}

// Before a forward: one that raises has then changed nothing
void ready(const char *what) { done(poll_sometimes(), what); }

// A call's status in the autograd engine's thread, which carries torch's own form of a
// Python exception to the caller; then the poll
void done_in_backward(int status, const char *what)
{
    if (status == LIFB_OK) status = poll_sometimes();
    if (status == LIFB_OK) return;
    py::gil_scoped_acquire gil;
    try {
        (*L.check)(status, what);
    } catch (py::error_already_set &e) {
        e.restore();
        python_error err;
        err.persist();
        throw std::move(err);
    }
}

// The gradients of a backward that was asked for a graph (create_graph): good as they
// are, and an error for who differentiates them
variable_list once(variable_list out, bool graph, const char *what)
{
    if (!graph) return out;
    for (Tensor &t : out)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    auto node = std::make_shared<torch::autograd::DelayedError>(
        std::string(what) + ": the gradient is not differentiable", (int)out.size());
    return (*node)(std::move(out));
}

bool graph_wanted(const variable_list &grads)
{
    if (torch::GradMode::is_enabled())
        for (const Tensor &t : grads)
            if (t.defined() && t.requires_grad()) return true;
    return false;
}

// Distance of t's rows [..., D] as one list of rows, or -1 where they are not that
int64_t row_stride(const Tensor &t)
{
    const int64_t D = t.size(-1);
    if (D != 1 && t.stride(-1) != 1) return -1;
    int64_t s = -1, next = 0;
    for (int64_t i = t.dim() - 2; i >= 0; i--) {
        const int64_t n = t.size(i), st = t.stride(i);
        if (n == 1) continue;
        if (s < 0)
            s = st;
        else if (st != next)
            return -1;
        next = st * n;
    }
    return s < 0 ? D : s < D ? -1 : s;
}

Tensor bytes(size_t n, const Tensor &like)
{
    return n ? torch::empty({(int64_t)n}, like.options().dtype(torch::kByte)) : Tensor();
}

bool on(const Tensor &t, int64_t dev) { return t.is_cuda() && t.get_device() == dev; }

bool wants_grad(std::initializer_list<const Tensor *> ts)
{
    if (!torch::GradMode::is_enabled()) return false;
    for (const Tensor *t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Whether one of them is a dual tensor: no operator has a forward-mode derivative, and the
// Python functions refuse it
bool has_tangent(std::initializer_list<const Tensor *> ts)
{
    for (const Tensor *t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) return true;
    return false;
}

// ---- embedding

Tensor embed_forward(const Tensor &tokens, const Tensor &weight, double scale)
{
    const c10::cuda::CUDAGuard guard(weight.device());
    ready("embedding");
    auto shape = tokens.sizes().vec();
    shape.push_back(weight.size(1));
    Tensor y = torch::empty(shape, weight.options());
    done(L.embed_fwd(at(tokens), (int)tokens.element_size(), at(weight), at(y), tokens.numel(), weight.size(0),
                     weight.size(1), weight.size(1), (float)scale, type_of(weight), stream_of(weight)),
         "embedding");
    return y;
}

struct EmbedFn : torch::autograd::Function<EmbedFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &tokens, const Tensor &weight, double scale)
    {
        ctx->save_for_backward({tokens});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["V"] = weight.size(0);
        return embed_forward(tokens, weight, scale);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const bool graph = graph_wanted(grads);
        const at::AutoGradMode no_grad(false);
        const Tensor tokens = ctx->get_saved_variables()[0];
        Tensor dy = grads[0];
        const int64_t n = tokens.numel(), V = ctx->saved_data["V"].toInt(), D = dy.size(-1);
        const c10::cuda::CUDAGuard guard(dy.device());
        int64_t row = row_stride(dy);
        if (row < 0) dy = dy.contiguous(), row = D;
        Tensor dw = torch::empty({V, D}, dy.options());
        const size_t nb = L.embed_bwd_ws(n, V, D);
        Tensor ws = bytes(nb, dy);
        done_in_backward(L.embed_bwd(at(tokens), (int)tokens.element_size(), at(dy), at(dw), n, V, D, row,
                                     (float)ctx->saved_data["scale"].toDouble(), type_of(dy), at(ws), nb,
                                     stream_of(dy)),
                         "embedding");
        return once({Tensor(), dw, Tensor()}, graph, "embedding");
    }
};

py::object embedding(const Tensor &tokens, const Tensor &weight, double scale)
{
    const auto tt = tokens.scalar_type();
    if (!weight.is_cuda() || weight.dim() != 2 || !weight.is_contiguous() || type_of(weight) < 0 ||
        !on(tokens, weight.get_device()) || !tokens.is_contiguous() || (tt != torch::kInt && tt != torch::kLong) ||
        has_tangent({&weight}))
        return py::none();
    return py::cast(wants_grad({&weight}) ? EmbedFn::apply(tokens, weight, scale) : embed_forward(tokens, weight, scale));
}

// ---- norms, gate and residual

lifb_norm_gate norm_args(const Tensor &x, const Tensor &h, const Tensor &gate, const Tensor &post, const Tensor &pre,
                         const Tensor &rstd, double scale, double eps, int64_t act)
{
    lifb_norm_gate a{};
    const int64_t D = x.size(-1), gc = gate.defined() ? gate.size(-1) : 0;
    a.x = at(x), a.h = at(h), a.gate = at(gate), a.post = at(post), a.pre = at(pre), a.rstd = at_f32(rstd);
    a.R = x.numel() / D, a.D = D, a.gate_cols = gc;
    a.x_stride = row_stride(x), a.h_stride = h.defined() ? row_stride(h) : 0, a.gate_stride = gc ? row_stride(gate) : 0;
    a.scale = (float)scale, a.eps = (float)eps, a.act = (int)act;
    a.dtype = type_of(x), a.weight_dtype = type_of(post.defined() ? post : pre);
    return a;
}

// x' where there is a block (h), n where there is a norm after it (pre)
variable_list norm_forward(const Tensor &x, const Tensor &h, const Tensor &gate, const Tensor &post, const Tensor &pre,
                           const Tensor &rstd, double scale, double eps, int64_t act)
{
    const c10::cuda::CUDAGuard guard(x.device());
    ready("norm_gate_residual");
    Tensor xo, n;
    if (h.defined()) xo = torch::empty(x.sizes(), x.options());
    if (pre.defined()) n = torch::empty(x.sizes(), x.options());
    const lifb_norm_gate a = norm_args(x, h, gate, post, pre, rstd, scale, eps, act);
    done(L.norm_fwd(&a, at(xo), at(n), stream_of(x)), "norm_gate_residual");
    variable_list out;
    if (xo.defined()) out.push_back(xo);
    if (n.defined()) out.push_back(n);
    return out;
}

struct NormFn : torch::autograd::Function<NormFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &h_, const OptTensor &gate_,
                                 const OptTensor &post_, const OptTensor &pre_, double scale, double eps, int64_t act)
    {
        const Tensor h = h_.value_or(Tensor()), gate = gate_.value_or(Tensor()), post = post_.value_or(Tensor()),
                     pre = pre_.value_or(Tensor());
        Tensor rstd = torch::empty({2, x.numel() / x.size(-1)}, x.options().dtype(torch::kFloat));
        ctx->save_for_backward({x, h, gate, post, pre, rstd});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["act"] = act;
        ctx->set_materialize_grads(false);
        return norm_forward(x, h, gate, post, pre, rstd, scale, eps, act);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const bool graph = graph_wanted(grads);
        const at::AutoGradMode no_grad(false);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &h = s[1], &gate = s[2], &post = s[3], &pre = s[4], &rstd = s[5];
        Tensor dxo = h.defined() ? grads[0] : Tensor(), dn = pre.defined() ? grads.back() : Tensor();
        variable_list out(8);
        if (!dxo.defined() && !dn.defined()) return out;
        const c10::cuda::CUDAGuard guard(x.device());
        const int64_t D = x.size(-1);
        int64_t row_xo = D, row_n = D;
        if (dxo.defined() && (row_xo = row_stride(dxo)) < 0) dxo = dxo.contiguous(), row_xo = D;
        if (dn.defined() && (row_n = row_stride(dn)) < 0) dn = dn.contiguous(), row_n = D;
        int edge = 0;  // absent inputs have none
        for (int i = 0; i < 5; i++)
            if (s[i].defined() && ctx->needs_input_grad(edge++)) out[i] = torch::empty(s[i].sizes(), s[i].options());
        const lifb_norm_gate a = norm_args(x, h, gate, post, pre, rstd, ctx->saved_data["scale"].toDouble(),
                                           ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt());
        const size_t nb = out[3].defined() || out[4].defined() ? L.norm_bwd_ws(a.R, a.D, a.dtype) : 0;
        Tensor ws = bytes(nb, x);
        done_in_backward(L.norm_bwd(&a, at(dxo), row_xo, at(dn), row_n, at(out[0]), at(out[1]), at(out[2]), at(out[3]),
                                    at(out[4]), at(ws), nb, stream_of(x)),
                         "norm_gate_residual");
        return once(std::move(out), graph, "norm_gate_residual");
    }
};

py::object norm_gate(const Tensor &x, const OptTensor &h_, const OptTensor &gate_, const OptTensor &post_,
                     const OptTensor &pre_, double scale, double eps, int64_t act)
{
    const Tensor h = h_.value_or(Tensor()), gate = gate_.value_or(Tensor()), post = post_.value_or(Tensor()),
                 pre = pre_.value_or(Tensor());
    if (!x.is_cuda() || x.dim() < 1 || type_of(x) < 0 || has_tangent({&x, &h, &gate, &post, &pre})) return py::none();
    const int64_t dev = x.get_device(), D = x.size(-1);
    if (D < 1 || row_stride(x) < 0 || D > 8192 || (!post.defined() && !pre.defined()) || h.defined() != post.defined()) return py::none();
    for (const Tensor *t : {&h, &gate})
        if (t->defined()) {
            if (!on(*t, dev) || t->scalar_type() != x.scalar_type() || t->dim() != x.dim()) return py::none();
            const bool row = t == &gate && t->size(-1) == 1;
            for (int64_t i = 0; i < x.dim(); i++)
                if (t->size(i) != x.size(i) && !(row && i == x.dim() - 1)) return py::none();
            if (row_stride(*t) < 0) return py::none();
        }
    auto wd = (post.defined() ? post : pre).scalar_type();
    if (wd != torch::kFloat && wd != x.scalar_type()) return py::none();
    for (const Tensor *t : {&post, &pre})
        if (t->defined() && (!on(*t, dev) || t->dim() != 1 || t->size(0) != D || !t->is_contiguous() || t->scalar_type() != wd))
            return py::none();
    const variable_list out = wants_grad({&x, &h, &gate, &post, &pre})
                                  ? NormFn::apply(x, h_, gate_, post_, pre_, scale, eps, act)
                                  : norm_forward(x, h, gate, post, pre, Tensor(), scale, eps, act);
    if (out.size() == 1) return py::cast(out[0]);
    return py::make_tuple(out[0], out[1]);
}

// ---- leaky attention

lifb_leaky_attn attn_args(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &ld, const Tensor &state,
                          const Tensor &lengths, double scale)
{
    lifb_leaky_attn a{};
    a.q = at(q), a.k = at(k), a.v = at(v), a.log_decay = at_f32(ld), a.state = at_f32(state), a.lengths = at_i32(lengths);
    a.B = q.size(0), a.T = q.size(1), a.H = q.size(2), a.Hk = v.size(2), a.Dk = q.size(3), a.Dv = v.size(3);
    for (int i = 0; i < 3; i++) {
        a.q_strides[i] = q.stride(i);
        a.k_strides[i] = k.stride(i);
        a.v_strides[i] = v.stride(i);
    }
    a.scale = (float)scale, a.dtype = type_of(q);
    return a;
}

// Whether the widths are ones that the tensor-core kernels take: rows of whole 16 bytes
bool tc_widths(const Tensor &q, const Tensor &v)
{
    return q.size(-1) * q.element_size() % 16 == 0 && v.size(-1) * v.element_size() % 16 == 0;
}

// An operand as those kernels read it: address and distances multiples of 16 bytes, in bf16
// (tensor maps) none of 0.  One that is not so is copied: left as it is, it would send the
// whole call, in a backward all three passes, to the fp32 pipe (a bf16 training pass of B 8,
// T 2048, 8 heads of 128 x 128: 153 us; k and v expanded from one head 3492, now 216; the
// gradient of a sum over time 2448, now 185; q at an odd distance 5014, now 191).
Tensor tc_rows(const Tensor &t, bool tc)
{
    const int64_t e = t.element_size();
    bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; i++)
        if (t.size(i) > 1 && (t.stride(i) * e % 16 != 0 || (e == 2 && t.stride(i) == 0))) fits = false;
    return fits || !tc ? t : t.clone(at::MemoryFormat::Contiguous);
}

variable_list attn_forward(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &ld, const Tensor &state,
                           const Tensor &lengths, double scale, bool return_state)
{
    const c10::cuda::CUDAGuard guard(q.device());
    ready("leaky_attention");
    const lifb_leaky_attn a = attn_args(q, k, v, ld, state, lengths, scale);
    variable_list out{torch::empty({a.B, a.T, a.H, a.Dv}, q.options())};
    if (return_state) out.push_back(torch::empty({a.B, a.H, a.Dk, a.Dv}, q.options().dtype(torch::kFloat)));
    const size_t nb = L.attn_ws(&a, 0);
    Tensor ws = bytes(nb, q);
    done(L.attn_fwd(&a, at(out[0]), return_state ? at_f32(out[1]) : nullptr, at(ws), nb, stream_of(q)),
         "leaky_attention");
    return out;
}

struct AttnFn : torch::autograd::Function<AttnFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &ld,
                                 const OptTensor &state_, const OptTensor &lengths_, double scale, bool return_state)
    {
        const Tensor state = state_.value_or(Tensor()), lengths = lengths_.value_or(Tensor());
        ctx->save_for_backward({q, k, v, ld, state, lengths});
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return attn_forward(q, k, v, ld, state, lengths, scale, return_state);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const bool graph = graph_wanted(grads);
        const at::AutoGradMode no_grad(false);
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &ld = s[3], &state = s[4], &lengths = s[5];
        Tensor d_o = grads[0], d_state = grads.size() > 1 ? grads[1] : Tensor();
        variable_list out(8);
        if (!d_o.defined() && !d_state.defined()) return out;
        const c10::cuda::CUDAGuard guard(q.device());
        const lifb_leaky_attn a = attn_args(q, k, v, ld, state, lengths, ctx->saved_data["scale"].toDouble());
        if (!d_o.defined()) d_o = torch::zeros({a.B, a.T, a.H, a.Dv}, q.options());
        if (d_o.stride(3) != 1) d_o = d_o.contiguous();
        d_o = tc_rows(d_o, tc_widths(q, v));
        if (d_state.defined()) d_state = d_state.contiguous();
        out[0] = torch::empty(q.sizes(), q.options());
        out[1] = torch::empty(k.sizes(), k.options());
        out[2] = torch::empty(v.sizes(), v.options());
        if (state.defined() && ctx->needs_input_grad(4)) out[4] = torch::empty(state.sizes(), state.options());
        const int64_t strides[3] = {d_o.stride(0), d_o.stride(1), d_o.stride(2)};
        const size_t nb = L.attn_ws(&a, 1);
        Tensor ws = bytes(nb, q);
        done_in_backward(L.attn_bwd(&a, at(d_o), strides, at_f32(d_state), at(out[0]), at(out[1]), at(out[2]),
                                    at_f32(out[4]), at(ws), nb, stream_of(q)),
                         "leaky_attention");
        return once(std::move(out), graph, "leaky_attention");
    }
};

// q, k, v of `lead` + 2 dimensions that fit one another, dense in the last; the decay
bool attn_fits(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &ld, int lead)
{
    if (!q.is_cuda() || q.dim() != lead + 2 || k.dim() != lead + 2 || v.dim() != lead + 2) return false;
    const int64_t dev = q.get_device(), H = q.size(lead), Hk = v.size(lead), Dk = q.size(lead + 1), Dv = v.size(lead + 1);
    if (!on(k, dev) || !on(v, dev) || !on(ld, dev)) return false;
    for (int i = 0; i < lead; i++)
        if (k.size(i) != q.size(i) || v.size(i) != q.size(i)) return false;
    return k.size(lead) == Hk && k.size(lead + 1) == Dk && Hk > 0 && H % Hk == 0 && Dk > 0 && Dk <= 128 && Dv <= 128 &&
           k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && q.stride(-1) == 1 &&
           k.stride(-1) == 1 && v.stride(-1) == 1 && ld.dim() == 1 && ld.size(0) == H &&
           ld.scalar_type() == torch::kFloat && ld.is_contiguous() && !ld.requires_grad();
}

py::object attention(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &ld, const OptTensor &state_,
                     const OptTensor &lengths_, std::optional<double> scale, bool return_state)
{
    const Tensor state = state_.value_or(Tensor()), lengths = lengths_.value_or(Tensor());
    if (!attn_fits(q_, k_, v_, ld, 2) || (type_of(q_) != LIFB_F32 && type_of(q_) != LIFB_BF16) ||
        has_tangent({&q_, &k_, &v_, &ld, &state}))
        return py::none();
    const int64_t dev = q_.get_device(), B = q_.size(0), H = q_.size(2), Dk = q_.size(3), Dv = v_.size(3);
    if (state.defined() && (!on(state, dev) || state.scalar_type() != torch::kFloat || !state.is_contiguous() ||
                            state.sizes() != at::IntArrayRef({B, H, Dk, Dv})))
        return py::none();
    if (lengths.defined() && (!on(lengths, dev) || lengths.scalar_type() != torch::kInt || !lengths.is_contiguous() ||
                              lengths.dim() != 1 || lengths.size(0) != B))
        return py::none();
    const double sc = scale ? *scale : 1.0 / std::sqrt((double)Dk);
    const bool tc = tc_widths(q_, v_);
    const Tensor q = tc_rows(q_, tc), k = tc_rows(k_, tc), v = tc_rows(v_, tc);
    const variable_list out = wants_grad({&q, &k, &v, &state})
                                  ? AttnFn::apply(q, k, v, ld, state_, lengths_, sc, return_state)
                                  : attn_forward(q, k, v, ld, state, lengths, sc, return_state);
    if (!return_state) return py::cast(out[0]);
    return py::make_tuple(out[0], out[1]);
}

// Slots and heads in the usual order, none over another; other orders are looked at in Python
bool apart(const Tensor &state)
{
    const int64_t n = state.size(0), H = state.size(1), mat = state.size(2) * state.size(3);
    return (H == 1 || state.stride(1) >= mat) && (n == 1 || state.stride(0) >= (H - 1) * state.stride(1) + mat);
}

py::object attention_step(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &ld, const Tensor &state,
                          const OptTensor &slots_, std::optional<double> scale)
{
    const Tensor slots = slots_.value_or(Tensor());
    if (!attn_fits(q, k, v, ld, 1) || type_of(q) < 0 || wants_grad({&q, &k, &v, &state}) ||
        has_tangent({&q, &k, &v, &ld, &state}))
        return py::none();
    const int64_t dev = q.get_device(), B = q.size(0), H = q.size(1), Dk = q.size(2), Dv = v.size(2);
    if (!on(state, dev) || state.dim() != 4 || state.scalar_type() != torch::kFloat || state.size(1) != H ||
        state.size(2) != Dk || state.size(3) != Dv || state.stride(3) != 1 || state.stride(2) != Dv || !apart(state))
        return py::none();
    if (slots.defined() ? !on(slots, dev) || slots.scalar_type() != torch::kInt || !slots.is_contiguous() ||
                              slots.dim() != 1 || slots.size(0) != B
                        : state.size(0) < B)
        return py::none();
    const c10::cuda::CUDAGuard guard(q.device());
    ready("leaky_attention_step");
    if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();  // who has saved it hears of the change
    Tensor o = torch::empty({B, H, Dv}, q.options());
    lifb_leaky_attn_step_args a{};
    a.q = at(q), a.k = at(k), a.v = at(v), a.log_decay = at_f32(ld), a.slots = at_i32(slots);
    a.B = B, a.H = H, a.Hk = v.size(1), a.Dk = Dk, a.Dv = Dv, a.n_slots = state.size(0);
    for (int i = 0; i < 2; i++) {
        a.q_strides[i] = q.stride(i);
        a.k_strides[i] = k.stride(i);
        a.v_strides[i] = v.stride(i);
        a.state_strides[i] = state.stride(i);
    }
    a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)Dk)), a.dtype = type_of(q);
    done(L.attn_step(&a, at(o), at_f32(state), stream_of(q)), "leaky_attention_step");
    return py::cast(o);
}

}  // namespace

PYBIND11_MODULE(lifb_seq, m)
{
    m.def("bind", &bind);
    m.def("embedding", &embedding);
    m.def("norm_gate", &norm_gate);
    m.def("attention", &attention);
    m.def("attention_step", &attention_step);
}

// Autograd nodes of the transformer operators (`kungfu_amd._nodes`).
//
// A node in Python costs a training step of a small model more than its
// kernels: the engine's thread waits for the interpreter, and every
// attribute of a tensor is a call. Here the nodes are C++ over the kernels
// of `_hip`, which come in a capsule (csrc/hip/kernel_api.h). Arguments are
// checked in Python, in kungfu_amd/ops; what these entries take is right in
// shape, type and device, of any strides.
//
// A node runs on the device and stream that its forward ran on, as the
// engine arranges, so the stream's handle is kept from there.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../hip/kernel_api.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::Variable;
using torch::autograd::variable_list;

namespace {

const kf_kernels *K = nullptr;

void check(int code, const char *what)
{
    if (code != 0)
        throw std::runtime_error(std::string(what) + ": " + K->error(code));
}

int type_code(at::ScalarType t)
{
    switch (t) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: throw std::runtime_error("no kernel for this type");
    }
}

uintptr_t ptr(const Tensor &t)
{
    return t.defined() && t.numel() ? (uintptr_t)t.data_ptr() : 0;
}

// An argument that may be missing. A missing one reaches a node as an empty
// optional: it takes no undefined tensors.
typedef std::optional<Tensor> Maybe;

Tensor or_none(const Maybe &t)
{
    return t.has_value() ? *t : Tensor();
}

// Row-major, uninitialised, of t's shape and type whatever its strides.
Tensor dense_like(const Tensor &t)
{
    return at::empty(t.sizes(), t.options());
}

Tensor contiguous(const Tensor &t)
{
    return t.defined() ? t.contiguous() : t;
}

// Strides of the leading dimensions; 0 where the size is 1, whose stride
// is arbitrary and never used.
void row_strides(const Tensor &t, std::vector<long long> &to)
{
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        to.push_back(t.size(i) == 1 ? 0 : (long long)t.stride(i));
}

// t (batch, length, heads, width), or a copy of it, whose rows are dense and
// start at 16 bytes, as the kernels that load 16 bytes at a time need, and
// whose tokens are near enough for 32-bit offsets within a tile.
Tensor rows16(const Tensor &t)
{
    const int64_t each = 16 / t.element_size();
    bool ok = t.stride(-1) == 1 && ptr(t) % 16 == 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        ok = ok && (t.size(i) == 1 || t.stride(i) % each == 0);
    ok = ok && (t.size(1) == 1 || t.stride(1) < 1 << 24);
    if (ok) return t;
    const Tensor c = t.contiguous();
    return ptr(c) % 16 == 0 ? c : c.clone();
}

// Gradients that cannot be differentiated again. Where they are made for
// that, they hang on a node that raises, and the node on all of `from`: what
// they were computed from. Any way through the operator to a leaf then
// raises, instead of adding nothing without a word; ways past it stay open.
variable_list once(variable_list grads, const variable_list &from)
{
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (const auto &g : grads)
        if (g.defined()) in.push_back(g);
    for (const auto &t : from)
        if (t.defined() && t.requires_grad()) in.push_back(t);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "this operator has no second derivative", (int64_t)in.size());
    const variable_list out = (*error)(std::move(in));
    size_t i = 0;
    for (auto &g : grads)
        if (g.defined()) g = out[i++];
    return grads;
}

// Refuses the calls whose results would be wrong without a word: of inputs
// that have a tangent, since there are no forward-mode derivatives, and
// those that a tracer records, since it would see the outputs' allocation
// and not the launch that fills them.
void usable(const char *what, const variable_list &ts)
{
    for (const auto &t : ts)
        if (t.defined() && t._fw_grad(0).defined())
            throw std::runtime_error(
                std::string(what) + " has no forward-mode derivative");
    if (torch::jit::tracer::isTracing() ||
        c10::impl::TorchDispatchModeTLS::get_mode(
            c10::impl::TorchDispatchModeKey::PROXY))
        throw std::runtime_error(std::string(what) + " cannot be traced");
}

bool wants_grad(std::initializer_list<Tensor> ts)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const auto &t : ts)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

// ---- embedding ----

struct EmbedArgs {
    double scale;
    int64_t padding, stream;
    at::ScalarType out;
};

Tensor embed_forward(const Tensor &ids, const Tensor &weight,
                     const EmbedArgs &a)
{
    auto shape = ids.sizes().vec();
    shape.push_back(weight.size(1));
    const Tensor out = at::empty(shape, weight.options().dtype(a.out));
    if (ids.numel() == 0) return out;
    c10::DeviceGuard guard(weight.device());
    check(K->embed_fwd(ids.data_ptr(), ids.scalar_type() == at::kLong,
                       weight.data_ptr(), weight.stride(0),
                       type_code(weight.scalar_type()), out.data_ptr(),
                       type_code(a.out), ids.numel(), weight.size(0),
                       (int)weight.size(1), (float)a.scale,
                       (void *)a.stream),
          "embedding");
    return out;
}

struct Embedding : Function<Embedding> {
    static Tensor forward(AutogradContext *ctx, const Tensor &ids,
                          const Tensor &weight, EmbedArgs a)
    {
        ctx->save_for_backward({ids});
        auto &d = ctx->saved_data;
        d["V"] = weight.size(0);
        d["H"] = weight.size(1);
        d["type"] = (int64_t)weight.scalar_type();
        d["out"] = (int64_t)a.out;
        d["scale"] = a.scale;
        d["padding"] = a.padding;
        d["stream"] = a.stream;
        return embed_forward(ids, weight, a);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        usable("embedding backward", grads);
        // before autograd is off: a checkpoint computes them again here
        const Tensor ids = ctx->get_saved_variables()[0].contiguous();
        at::AutoDispatchBelowADInplaceOrView below;
        auto &d = ctx->saved_data;
        const auto type = (at::ScalarType)d["type"].toInt();
        const auto otype = (at::ScalarType)d["out"].toInt();
        const int64_t V = d["V"].toInt(), H = d["H"].toInt();
        const int64_t N = ids.numel();
        const Tensor dout = grads[0].to(otype).contiguous();
        const Tensor dw = at::empty({V, H}, dout.options().dtype(type));
        c10::DeviceGuard guard(dout.device());
        const Tensor ws = at::empty({(int64_t)K->embed_ws(N, V, (int)H)},
                                    dout.options().dtype(at::kByte));
        check(K->embed_bwd((const void *)ptr(ids),
                           ids.scalar_type() == at::kLong,
                           (const void *)ptr(dout), type_code(otype),
                           dw.data_ptr(), type_code(type), N, V, (int)H,
                           d["padding"].toInt(),
                           (float)d["scale"].toDouble(), ws.data_ptr(),
                           (void *)d["stream"].toInt()),
              "embedding backward");
        // linear in dout, and no function of the weight
        return once({Tensor(), dw, Tensor()}, grads);
    }
};

Tensor embedding(const Tensor &ids, const Tensor &weight, double scale,
                 int64_t padding, at::ScalarType out, int64_t stream)
{
    usable("embedding", {weight});
    const EmbedArgs a = {scale, padding, stream, out};
    if (wants_grad({weight})) return Embedding::apply(ids, weight, a);
    return embed_forward(ids, weight, a);
}

// ---- query/key norm and rotation ----

struct QKArgs {
    int64_t start, stream;
    double eps;
};

void qk_launch(const Tensor &q, const Tensor &k, const Tensor &qw,
               const Tensor &kw, const Tensor &rope, const Tensor &positions,
               const Tensor &oq, const Tensor &ok, const QKArgs &a,
               const Tensor *grads)  // dyq, dyk, dqw, dkw, partial sums
{
    long long pb = 0, ps = 0;
    if (positions.defined()) {
        ps = positions.stride(-1);
        pb = positions.dim() == 2 ? positions.stride(0) : 0;
    }
    const Tensor &w = qw.defined() ? qw : kw;
    std::vector<uintptr_t> ptrs = {ptr(q),  ptr(k),  ptr(qw),   ptr(kw),
                                   ptr(oq), ptr(ok), ptr(rope), ptr(positions)};
    std::vector<long long> dims = {q.size(0) * q.size(1), q.size(1),
                                   q.size(3), q.size(2), k.size(2)};
    row_strides(q, dims);
    row_strides(k, dims);
    dims.push_back(rope.defined() ? rope.size(0) : 0);
    dims.push_back(a.start);
    dims.push_back(pb);
    dims.push_back(ps);
    dims.push_back(positions.defined() &&
                   positions.scalar_type() == at::kLong);
    dims.push_back(w.defined() && w.scalar_type() == at::kFloat);
    if (grads) {
        for (int i = 0; i < 5; ++i) ptrs.push_back(ptr(grads[i]));
        row_strides(grads[0], dims);
        row_strides(grads[1], dims);
    }
    c10::DeviceGuard guard(q.device());
    check(K->qk_norm_rope(ptrs.data(), dims.data(),
                          type_code(q.scalar_type()), (float)a.eps,
                          grads != nullptr, (void *)a.stream),
          "qk_norm_rope");
}

variable_list qk_forward(const Tensor &q, const Tensor &k, const Tensor &qw,
                         const Tensor &kw, const Tensor &rope,
                         const Tensor &positions, const QKArgs &a)
{
    const Tensor oq = dense_like(q), ok = dense_like(k);
    if (oq.numel() || ok.numel())
        qk_launch(q, k, qw, kw, rope, positions, oq, ok, a, nullptr);
    return {oq, ok};
}

Tensor dense_rows(const Tensor &t)
{
    return t.stride(-1) == 1 ? t : t.contiguous();
}

struct QKNormRope : Function<QKNormRope> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q,
                                 const Tensor &k, const Maybe &qw_,
                                 const Maybe &kw_, const Maybe &rope_,
                                 const Maybe &positions_, QKArgs a)
    {
        const Tensor qw = or_none(qw_), kw = or_none(kw_);
        const Tensor rope = or_none(rope_), positions = or_none(positions_);
        ctx->save_for_backward({q, k, qw, kw, rope, positions});
        auto &d = ctx->saved_data;
        d["start"] = a.start;
        d["stream"] = a.stream;
        d["eps"] = a.eps;
        return qk_forward(q, k, qw, kw, rope, positions, a);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        usable("qk_norm_rope backward", grads);
        const auto s = ctx->get_saved_variables();  // with autograd on
        at::AutoDispatchBelowADInplaceOrView below;
        // hooks of kept tensors may give them back in another layout
        const Tensor q = dense_rows(s[0]), k = dense_rows(s[1]);
        const Tensor qw = contiguous(s[2]), kw = contiguous(s[3]);
        auto &d = ctx->saved_data;
        const QKArgs a = {d["start"].toInt(), d["stream"].toInt(),
                          d["eps"].toDouble()};
        const Tensor dq = dense_like(q), dk = dense_like(k);
        Tensor more[5] = {dense_rows(grads[0]), dense_rows(grads[1])};
        if (qw.defined()) more[2] = dense_like(qw);
        if (kw.defined()) more[3] = dense_like(kw);
        if (q.numel() == 0 && k.numel() == 0) {
            for (int i = 2; i < 4; ++i)
                if (more[i].defined()) more[i].zero_();
        } else {
            if (qw.defined() || kw.defined())
                more[4] = at::empty(
                    {(int64_t)K->qk_ws((int)q.size(3),
                                       (int)(q.size(2) + k.size(2)))},
                    q.options().dtype(at::kFloat));
            qk_launch(q, k, qw, kw, contiguous(s[4]), s[5], dq, dk, a, more);
        }
        return once({dq, dk, more[2], more[3], Tensor(), Tensor(), Tensor()},
                    {s[0], s[1], s[2], s[3], grads[0], grads[1]});
    }
};

std::pair<Tensor, Tensor> qk_norm_rope(const Tensor &q, const Tensor &k,
                                       const Maybe &qw, const Maybe &kw,
                                       const Maybe &rope,
                                       const Maybe &positions, int64_t start,
                                       double eps, int64_t stream)
{
    usable("qk_norm_rope",
           {q, k, or_none(qw), or_none(kw), or_none(rope)});
    const QKArgs a = {start, stream, eps};
    const auto out =
        wants_grad({q, k, or_none(qw), or_none(kw)})
            ? QKNormRope::apply(q, k, qw, kw, rope, positions, a)
            : qk_forward(q, k, or_none(qw), or_none(kw), or_none(rope),
                         or_none(positions), a);
    return {out[0], out[1]};
}

// ---- window attention ----

struct AttnArgs {
    int64_t window, sinks, causal, stream;
    double scale;
};

std::vector<long long> attn_dims(const Tensor &q, const Tensor &k,
                                 const AttnArgs &a)
{
    return {q.size(0), q.size(1),
            k.size(1), k.size(2),
            q.size(2) / k.size(2), q.size(3),
            a.window,  a.sinks,
            a.causal};
}

std::vector<long long> attn_strides(const Tensor &q, const Tensor &k,
                                    const Tensor &v)
{
    std::vector<long long> s;
    row_strides(q, s);
    row_strides(k, s);
    row_strides(v, s);
    return s;
}

// The output and, to keep for the backward, each row's log-sum-exp in
// powers of two and what rounding took off the output.
void attn_forward(const Tensor &q, const Tensor &k, const Tensor &v,
                  const Tensor &lengths, const Tensor &starts,
                  const AttnArgs &a, const Tensor &out, const Tensor &lse,
                  const Tensor &rest)
{
    const auto dims = attn_dims(q, k, a);
    const auto strides = attn_strides(q, k, v);
    c10::DeviceGuard guard(q.device());
    const long long size = K->attn_ws(dims.data(), 0);
    Tensor ws;
    if (size > 0) ws = at::empty({(int64_t)size}, q.options().dtype(at::kByte));
    const uintptr_t ptrs[9] = {ptr(q),   ptr(k),    ptr(v),
                               ptr(out), ptr(lse),  ptr(rest),
                               ptr(lengths), ptr(starts), ptr(ws)};
    check(K->attn_fwd(ptrs, dims.data(), strides.data(), (float)a.scale,
                      type_code(q.scalar_type()), (void *)a.stream),
          "window_attention");
}

struct WindowAttention : Function<WindowAttention> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q,
                          const Tensor &k, const Tensor &v,
                          const Maybe &lengths_, const Maybe &starts_,
                          AttnArgs a)
    {
        const Tensor lengths = or_none(lengths_), starts = or_none(starts_);
        const Tensor out = dense_like(q), rest = dense_like(q);
        const Tensor lse = at::empty({q.size(0) * q.size(1) * q.size(2)},
                                     q.options().dtype(at::kFloat));
        attn_forward(q, k, v, lengths, starts, a, out, lse, rest);
        ctx->save_for_backward({q, k, v, lengths, starts, out, lse, rest});
        auto &d = ctx->saved_data;
        d["window"] = a.window;
        d["sinks"] = a.sinks;
        d["causal"] = a.causal;
        d["stream"] = a.stream;
        d["scale"] = a.scale;
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        usable("window_attention backward", grads);
        const auto s = ctx->get_saved_variables();  // with autograd on
        at::AutoDispatchBelowADInplaceOrView below;
        // hooks of kept tensors may give them back in another layout
        const Tensor q = rows16(s[0]), k = rows16(s[1]), v = rows16(s[2]);
        Tensor kept[5];  // lengths, starts, out, lse, rest
        for (int i = 0; i < 5; ++i) kept[i] = contiguous(s[3 + i]);
        auto &d = ctx->saved_data;
        const AttnArgs a = {d["window"].toInt(), d["sinks"].toInt(),
                            d["causal"].toInt(), d["stream"].toInt(),
                            d["scale"].toDouble()};
        const Tensor dout = rows16(grads[0]);
        const Tensor dq = dense_like(q), dk = dense_like(k),
                     dv = dense_like(v);
        const auto dims = attn_dims(q, k, a);
        auto strides = attn_strides(q, k, v);
        row_strides(dout, strides);
        c10::DeviceGuard guard(q.device());
        const Tensor ws =
            at::empty({(int64_t)K->attn_ws(dims.data(), 1)},
                      q.options().dtype(at::kByte));
        const uintptr_t ptrs[13] = {
            ptr(q),       ptr(k),       ptr(v),       ptr(kept[2]),
            ptr(kept[3]), ptr(kept[4]), ptr(kept[0]), ptr(kept[1]),
            ptr(dout),    ptr(dq),      ptr(dk),      ptr(dv),
            ptr(ws)};
        check(K->attn_bwd(ptrs, dims.data(), strides.data(), (float)a.scale,
                          type_code(q.scalar_type()), (void *)a.stream),
              "window_attention backward");
        return once({dq, dk, dv, Tensor(), Tensor(), Tensor()},
                    {s[0], s[1], s[2], grads[0]});
    }
};

Tensor window_attention(const Tensor &q_, const Tensor &k_, const Tensor &v_,
                        const Maybe &lengths, const Maybe &starts,
                        int64_t window, int64_t sinks, bool causal,
                        double scale, int64_t stream)
{
    usable("window_attention", {q_, k_, v_});
    // copies, where there are any, are part of the autograd graph
    const Tensor q = rows16(q_), k = rows16(k_), v = rows16(v_);
    const AttnArgs a = {window, sinks, causal, stream, scale};
    if (wants_grad({q, k, v}))
        return WindowAttention::apply(q, k, v, lengths, starts, a);
    const Tensor out = dense_like(q);
    attn_forward(q, k, v, or_none(lengths), or_none(starts), a, out,
                 Tensor(), Tensor());
    return out;
}

}  // namespace

PYBIND11_MODULE(_nodes, m)
{
    m.doc() = "KungFu-AMD autograd nodes over the gfx950 HIP kernels";
    const py::capsule c = py::module_::import("kungfu_amd._hip")
                              .attr("kernels")
                              .cast<py::capsule>();
    K = (const kf_kernels *)PyCapsule_GetPointer(c.ptr(),
                                                 KF_KERNELS_CAPSULE);
    if (!K) throw py::error_already_set();
    // other threads of the interpreter go on while memory is waited for
    typedef py::call_guard<py::gil_scoped_release> Released;
    m.def("embedding", &embedding, Released());
    m.def("qk_norm_rope", &qk_norm_rope, Released());
    m.def("window_attention", &window_attention, Released());
}

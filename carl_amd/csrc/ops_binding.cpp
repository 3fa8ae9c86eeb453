// ops_binding.cpp - the `carl_amd._ops` Python module: torch tensors to the
// C-ABI of include/carl_amd_ops.h.
//
// Every tensor is checked (type, device, shape, strides) before anything is
// queued, raising TypeError / ValueError like the environment's binding; work
// is queued on torch's current stream, so it is ordered like any torch
// operation; outputs and scratch memory come from torch's allocator.
#include <torch/extension.h>

#include <torch/csrc/autograd/forward_grad.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/carl_amd_ops.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

void check(int rc)
{
    if (rc == CARL_OK) return;
    const std::string msg = carl_last_error();
    if (rc == CARL_ERR_TYPE) throw py::type_error(msg);
    if (rc == CARL_ERR_VALUE) throw py::value_error(msg);
    throw std::runtime_error(msg);
}

// The current stream of device 0, where all tensors are: that device is made
// current too while a call launches (the default stream's handle is null,
// which is any current device's).
class Queue {
    const c10::DeviceGuard guard_{ at::Device(at::kCUDA, 0) };

public:
    operator void*() const { return c10::hip::getCurrentHIPStream(0).stream(); }
};

// The message is made of its parts only where it is thrown.
template <typename... Parts> std::string message(const Parts&... parts)
{
    std::string s;
    (s.append(parts), ...);
    return s;
}

template <typename... Parts> void require(bool ok, const Parts&... parts)
{
    if (!ok) throw py::value_error(message(parts...));
}

template <typename... Parts> void requireType(bool ok, const Parts&... parts)
{
    if (!ok) throw py::type_error(message(parts...));
}

// The check of every tensor of a call.  A forward-mode tangent is refused: the
// results, made without autograd, would lose it.  (Whether there can be one is
// asked once a call: of a step's 210 tensors one by one it took 0.7 us.)
class OnDevice {
    const bool tangents_ = torch::autograd::ForwardADLevel::try_get_by_idx(0) && c10::AutogradState::get_tls_state().get_fw_grad_mode();

public:
    void operator()(const Tensor& t, const char* name) const
    {
        require(t.defined(), name, " must be a tensor");
        require(!tangents_ || !t._fw_grad(0).defined(), name, " has a forward-mode tangent: the operators have no forward-mode derivatives");
        require(t.is_cuda() && t.get_device() == 0, name, " must be on cuda:0");
        require(t.layout() == at::kStrided, name, " must be a dense tensor");
    }
};

int elementType(const Tensor& t, const char* name)
{
    switch (t.scalar_type()) {
    case at::kFloat: return CARL_OP_F32;
    case at::kBFloat16: return CARL_OP_BF16;
    case at::kHalf: return CARL_OP_F16;
    default: throw py::type_error(message(name, " must have dtype float32, bfloat16 or float16"));
    }
}

// ------------------------------------------------------- linear attention

carl_rows rowsOf(const Tensor& t, bool steps = true)
{
    return steps ? carl_rows{ t.data_ptr(), t.stride(0), t.stride(1), t.stride(2) }
                 : carl_rows{ t.data_ptr(), t.stride(0), 0, t.stride(1) };
}

// The checks of q, k, v, log_decay, starts and the memory; the sizes of the call.
carl_attention attentionOf(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& logDecay,
                           const OptTensor& starts, const OptTensor& memory, double scale, bool steps)
{
    const OnDevice onDevice;
    const int dims = steps ? 4 : 3;
    const char* lead = steps ? "[batch, steps, " : "[batch, ";
    for (const auto& [t, name] : { std::pair{ &q, "q" }, { &k, "k" }, { &v, "v" } }) {
        onDevice(*t, name);
        require(t->dim() == dims, name, " must have shape ", lead, "heads, width]");
        require(t->stride(dims - 1) == 1 || t->size(dims - 1) <= 1, name, " must be contiguous in its last dimension");
        requireType(t->scalar_type() == q.scalar_type(), "q, k and v must have the same dtype");
    }
    carl_attention a{};
    a.type = elementType(q, "q");
    a.batch = q.size(0);
    a.steps = steps ? q.size(1) : 1;
    for (const Tensor* t : { &k, &v })
        require(t->size(0) == a.batch && (!steps || t->size(1) == a.steps), "k and v must have q's batch and steps");
    require(q.size(dims - 2) <= 65535, "heads must be in [1, 65535]");
    a.heads = (int32_t)q.size(dims - 2);
    require(k.size(dims - 2) == v.size(dims - 2), "k and v must have the same heads");
    a.kv_heads = (int32_t)std::min<int64_t>(k.size(dims - 2), 65536);
    require(k.size(dims - 1) == q.size(dims - 1), "q and k must have the same width");
    a.key_dim = (int32_t)std::min<int64_t>(q.size(dims - 1), 1 << 20);
    a.value_dim = (int32_t)std::min<int64_t>(v.size(dims - 1), 1 << 20);
    a.scale = (float)scale;
    a.q = rowsOf(q, steps);
    a.k = rowsOf(k, steps);
    a.v = rowsOf(v, steps);
    onDevice(logDecay, "log_decay");
    requireType(logDecay.scalar_type() == at::kFloat, "log_decay must have dtype float32");
    require(logDecay.dim() == 1 && logDecay.size(0) == a.heads, "log_decay must have shape [heads]");
    require(logDecay.is_contiguous(), "log_decay must be contiguous");
    require(!at::GradMode::is_enabled() || !logDecay.requires_grad(), "log_decay has no gradient: detach it");
    a.log_decay = logDecay.data_ptr<float>();
    if (starts) {
        onDevice(*starts, "starts");
        requireType(starts->scalar_type() == at::kBool, "starts must have dtype bool");
        require(starts->dim() == dims - 2 && starts->size(0) == a.batch && (!steps || starts->size(1) == a.steps),
                steps ? "starts must have shape [batch, steps]" : "starts must have shape [batch]");
        a.starts = static_cast<const uint8_t*>(starts->data_ptr());
        a.starts_batch = starts->stride(0);
        a.starts_step = steps ? starts->stride(1) : 0;
    }
    if (memory) {
        const char* name = steps ? "initial_state" : "state";
        onDevice(*memory, name);
        requireType(memory->scalar_type() == at::kFloat, name, " must have dtype float32");
        require(memory->dim() == 4 && memory->size(0) == a.batch && memory->size(1) == a.heads
                    && memory->size(2) == a.key_dim && memory->size(3) == a.value_dim,
                name, " must have shape [batch, heads, key width, value width]");
        require(memory->is_contiguous(), name, " must be contiguous");
    }
    return a;
}

// Rows like q's but of the width of v, in q's order of batch and steps.
Tensor rowsLike(const Tensor& q, int64_t width)
{
    if (q.stride(1) > q.stride(0) && q.size(0) > 1)
        return at::empty({ q.size(1), q.size(0), q.size(2), width }, q.options()).transpose(0, 1);
    return at::empty({ q.size(0), q.size(1), q.size(2), width }, q.options());
}

// For the gradient of t: its order of dimensions, but the last one contiguous
// whatever t's is.  (Of a t that overlaps itself empty_like keeps the order of
// the strides, which may put the last dimension anywhere.)
Tensor gradientLike(const Tensor& t)
{
    Tensor g = at::empty_like(t);
    return g.stride(3) == 1 || g.size(3) <= 1 ? g : rowsLike(t, t.size(3));
}

Tensor workspaceOf(const carl_attention& a, bool backward, const Tensor& like)
{
    int64_t bytes = 0;
    check(carl_linear_attention_workspace(&a, backward, &bytes));
    return bytes ? at::empty({ bytes }, like.options().dtype(at::kByte)) : Tensor();
}

std::tuple<Tensor, Tensor> linearAttentionForward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& logDecay,
                                                  const OptTensor& starts, const OptTensor& initial, double scale)
{
    carl_attention a = attentionOf(q, k, v, logDecay, starts, initial, scale, true);
    Tensor out = rowsLike(q, a.value_dim);
    Tensor last = at::empty({ a.batch, a.heads, a.key_dim, a.value_dim }, logDecay.options());
    a.out = rowsOf(out);
    a.initial_state = initial ? initial->data_ptr<float>() : nullptr;
    a.final_state = last.data_ptr<float>();
    const Tensor work = workspaceOf(a, false, q);
    a.workspace = work.defined() ? work.data_ptr() : nullptr;
    check(carl_linear_attention(&a, Queue()));
    return { out, last };
}

// Autograd's own bookkeeping is worth skipping where nothing asks for it (5 us a call).
bool wantsGradient(std::initializer_list<const Tensor*> tensors)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->requires_grad()) return true;
    return false;
}

struct LinearAttention : torch::autograd::Function<LinearAttention> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                  const Tensor& v, const Tensor& logDecay, const OptTensor& starts,
                                                  const OptTensor& initial, double scale)
    {
        auto [out, last] = linearAttentionForward(q, k, v, logDecay, starts, initial, scale);
        ctx->save_for_backward({ q, k, v, logDecay, starts ? *starts : Tensor(), initial ? *initial : Tensor() });
        ctx->saved_data["scale"] = scale;
        ctx->set_materialize_grads(false);
        return { out, last };
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        if (at::GradMode::is_enabled()) throw std::runtime_error("linear_attention has no second derivative");
        const auto saved = ctx->get_saved_variables();
        const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &logDecay = saved[3];
        const OptTensor starts = saved[4].defined() ? OptTensor(saved[4]) : std::nullopt;
        const OptTensor initial = saved[5].defined() ? OptTensor(saved[5]) : std::nullopt;
        if (!grads[0].defined() && !grads[1].defined()) return { {}, {}, {}, {}, {}, {}, {} };
        carl_attention a = attentionOf(q.detach(), k.detach(), v.detach(), logDecay, starts, initial, ctx->saved_data["scale"].toDouble(), true);
        Tensor dOut = grads[0];
        if (!dOut.defined()) dOut = at::zeros({ a.batch, a.steps, a.heads, a.value_dim }, q.options());
        if (dOut.stride(3) != 1 && dOut.size(3) > 1) dOut = dOut.contiguous();
        const Tensor dLast = grads[1].defined() ? grads[1].contiguous() : Tensor();
        const Tensor dq = gradientLike(q), dk = gradientLike(k), dv = gradientLike(v);
        // edges count the tensors that were given
        const Tensor dFirst = initial && ctx->needs_input_grad(starts ? 5 : 4) ? at::empty_like(*initial) : Tensor();
        a.initial_state = initial ? initial->data_ptr<float>() : nullptr;
        a.d_out = rowsOf(dOut);
        a.d_q = rowsOf(dq);
        a.d_k = rowsOf(dk);
        a.d_v = rowsOf(dv);
        a.d_final_state = dLast.defined() ? dLast.data_ptr<float>() : nullptr;
        a.d_initial_state = dFirst.defined() ? dFirst.data_ptr<float>() : nullptr;
        const Tensor work = workspaceOf(a, true, q);
        a.workspace = work.defined() ? work.data_ptr() : nullptr;
        check(carl_linear_attention_backward(&a, Queue()));
        return { dq, dk, dv, {}, {}, dFirst, {} };
    }
};

std::tuple<Tensor, Tensor> linearAttention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& logDecay,
                                           const OptTensor& starts, const OptTensor& initial, std::optional<double> scale)
{
    const double s = scale ? *scale : q.dim() && q.size(-1) ? 1.0 / std::sqrt((double)q.size(-1)) : 1.0;
    if (!wantsGradient({ &q, &k, &v, initial ? &*initial : &q })) return linearAttentionForward(q, k, v, logDecay, starts, initial, s);
    auto out = LinearAttention::apply(q, k, v, logDecay, starts, initial, s);
    return { out[0], out[1] };
}

Tensor linearAttentionStep(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& logDecay, const Tensor& state,
                           const OptTensor& starts, std::optional<double> scale)
{
    const double s = scale ? *scale : q.dim() && q.size(-1) ? 1.0 / std::sqrt((double)q.size(-1)) : 1.0;
    if (at::GradMode::is_enabled())
        for (const Tensor* t : { &q, &k, &v, &state })
            require(!t->requires_grad(), "linear_attention_step has no gradient: call it under torch.no_grad()");
    carl_attention a = attentionOf(q, k, v, logDecay, starts, state, s, false);
    Tensor out = at::empty({ a.batch, a.heads, a.value_dim }, q.options());
    a.out = rowsOf(out, false);
    state.unsafeGetTensorImpl()->bump_version();        // refuses what may not be changed in place
    check(carl_linear_attention_step(&a, state.data_ptr<float>(), Queue()));
    return out;
}

// ------------------------------------------------- gated feed-forward block

// x as rows of its last dimension, without a copy where its strides allow.
Tensor asRows(const Tensor& x)
{
    const int64_t width = x.size(-1);
    Tensor rows = x.dim() == 2 ? x : x.reshape({ width ? x.numel() / width : 0, width });
    return rows.stride(1) == 1 || width <= 1 ? rows : rows.contiguous();
}

carl_ffn ffnOf(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int64_t activation)
{
    const OnDevice onDevice;
    for (const auto& [t, name] : { std::pair{ &x, "x" }, { &gate, "w_gate" }, { &up, "w_up" }, { &down, "w_down" } }) {
        onDevice(*t, name);
        requireType(t->scalar_type() == x.scalar_type(), "x and the weights must have the same dtype");
    }
    carl_ffn f{};
    f.type = elementType(x, "x");
    require(x.dim() >= 1, "x must have shape [..., width]");
    const int64_t width = x.size(-1);
    require(gate.dim() == 2 && gate.size(1) == width, "w_gate must have shape [inner, width]");
    require(up.sizes() == gate.sizes(), "w_up must have shape [inner, width]");
    require(down.dim() == 2 && down.size(0) == width && down.size(1) == gate.size(0), "w_down must have shape [width, inner]");
    require(width >= 1 && width <= CARL_FFN_MAX_DIM, "width must be in [1, 65536]");
    require(gate.size(0) >= 1 && gate.size(0) <= CARL_FFN_MAX_DIM, "inner must be in [1, 65536]");
    f.rows = x.numel() / width;
    f.width = (int32_t)width;
    f.inner = (int32_t)gate.size(0);
    f.activation = (int32_t)activation;
    return f;
}

Tensor gatedFfnForward(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, int64_t activation)
{
    carl_ffn f = ffnOf(x, gate, up, down, activation);
    const Tensor rows = asRows(x), g = gate.contiguous(), u = up.contiguous(), d = down.contiguous();
    Tensor y = at::empty(x.sizes(), x.options());
    f.x = rows.data_ptr();
    f.x_row = rows.stride(0);
    f.w_gate = g.data_ptr();
    f.w_up = u.data_ptr();
    f.w_down = d.data_ptr();
    f.y = y.data_ptr();
    int64_t bytes = 0;
    check(carl_gated_ffn_workspace(&f, 0, &bytes));
    const Tensor work = at::empty({ bytes }, x.options().dtype(at::kByte));
    f.workspace = work.data_ptr();
    check(carl_gated_ffn(&f, Queue()));
    return y;
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up,
                          const Tensor& down, int64_t activation)
    {
        const Tensor y = gatedFfnForward(x, gate, up, down, activation);
        ctx->save_for_backward({ x, gate, up, down });
        ctx->saved_data["activation"] = activation;
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        if (at::GradMode::is_enabled()) throw std::runtime_error("gated_ffn has no second derivative");
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &gate = saved[1], &up = saved[2], &down = saved[3];
        if (!grads[0].defined()) return { {}, {}, {}, {}, {} };
        carl_ffn f = ffnOf(x, gate, up, down, ctx->saved_data["activation"].toInt());
        const Tensor rows = asRows(x.detach()), dy = asRows(grads[0]);
        const Tensor g = gate.detach().contiguous(), u = up.detach().contiguous(), d = down.detach().contiguous();
        f.x = rows.data_ptr();
        f.x_row = rows.stride(0);
        f.dy = dy.data_ptr();
        f.dy_row = dy.stride(0);
        f.w_gate = g.data_ptr();
        f.w_up = u.data_ptr();
        f.w_down = d.data_ptr();
        const auto wanted = [&](int i, const Tensor& t) {
            return ctx->needs_input_grad(i) ? at::empty(t.sizes(), t.options()) : Tensor();
        };
        const Tensor dx = wanted(0, x), dg = wanted(1, gate), du = wanted(2, up), dd = wanted(3, down);
        f.dx = dx.defined() ? dx.data_ptr() : nullptr;
        f.dw_gate = dg.defined() ? dg.data_ptr() : nullptr;
        f.dw_up = du.defined() ? du.data_ptr() : nullptr;
        f.dw_down = dd.defined() ? dd.data_ptr() : nullptr;
        int64_t bytes = 0;
        check(carl_gated_ffn_workspace(&f, 1, &bytes));
        const Tensor work = at::empty({ bytes }, x.options().dtype(at::kByte));
        f.workspace = work.data_ptr();
        check(carl_gated_ffn_backward(&f, Queue()));
        return { dx, dg, du, dd, {} };
    }
};

Tensor gatedFfn(const Tensor& x, const Tensor& gate, const Tensor& up, const Tensor& down, const std::string& activation)
{
    require(activation == "silu" || activation == "gelu", "activation must be 'silu' or 'gelu'");
    const int64_t which = activation == "silu" ? CARL_SILU : CARL_GELU;
    if (!wantsGradient({ &x, &gate, &up, &down })) return gatedFfnForward(x, gate, up, down, which);
    return GatedFfn::apply(x, gate, up, down, which);
}

// ------------------------------------------------------------------- AdamW

// A sequence of tensors, looked at in place: a step's six lists of a policy's
// tensors would take longer to convert than the step (35 tensors: 20 us).
class TensorList {
    py::object held_;
    std::vector<const Tensor*> items_;

public:
    TensorList(const py::object& sequence, const char* name)
    {
        if (sequence.is_none()) return;
        held_ = py::reinterpret_steal<py::object>(PySequence_Fast(sequence.ptr(), "sequences of tensors expected"));
        if (!held_) throw py::error_already_set();
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(held_.ptr());
        items_.reserve(n);
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject* const item = PySequence_Fast_GET_ITEM(held_.ptr(), i);
            requireType(THPVariable_Check(item), name, " must be tensors");
            items_.push_back(&THPVariable_Unpack(item));
        }
    }
    size_t size() const { return items_.size(); }
    const Tensor& operator[](size_t i) const { return *items_[i]; }
};

void adamwStep(const py::object& paramList, const py::object& gradList, const py::object& firstList, const py::object& secondList,
               const py::object& firstScaleList, const py::object& secondScaleList, int64_t step, double lr, double beta1,
               double beta2, double eps, double weightDecay, const OptTensor& gradScale)
{
    const TensorList params(paramList, "params"), grads(gradList, "grads"), first(firstList, "exp_avg"),
        second(secondList, "exp_avg_sq"), firstScale(firstScaleList, "exp_avg_scale"), secondScale(secondScaleList, "exp_avg_sq_scale");
    const size_t n = params.size();
    require(grads.size() == n && first.size() == n && second.size() == n,
            "params, grads, exp_avg and exp_avg_sq must have the same length");
    const bool eight = n > 0 && first[0].scalar_type() == at::kChar;
    if (eight) require(firstScale.size() == n && secondScale.size() == n, "8-bit moments need exp_avg_scale and exp_avg_sq_scale");
    else require(firstScale.size() == 0 && secondScale.size() == 0, "float32 moments have no scales");
    const OnDevice onDevice;
    std::vector<carl_adamw_tensor> list(n);
    for (size_t i = 0; i < n; i++) {
        const Tensor &p = params[i], &g = grads[i], &m = first[i], &v = second[i];
        onDevice(p, "params");
        onDevice(g, "grads");
        onDevice(m, "exp_avg");
        onDevice(v, "exp_avg_sq");
        require(g.sizes() == p.sizes(), "grads must have their parameters' shapes");
        require(m.numel() == p.numel() && v.numel() == p.numel(), "moments must have their parameters' sizes");
        require(p.is_contiguous(), "params must be contiguous");
        require(g.is_contiguous(), "grads must be contiguous");
        require(m.is_contiguous() && v.is_contiguous(), "moments must be contiguous");
        requireType(m.scalar_type() == (eight ? at::kChar : at::kFloat), "exp_avg must all have dtype float32, or all int8");
        requireType(v.scalar_type() == (eight ? at::kByte : at::kFloat), "exp_avg_sq must have dtype float32, or uint8 with an int8 exp_avg");
        carl_adamw_tensor& t = list[i];
        t = { p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), nullptr, nullptr, p.numel(),
              elementType(p, "params"), elementType(g, "grads") };
        if (eight) {
            const int64_t blocks = (p.numel() + CARL_ADAMW_BLOCK - 1) / CARL_ADAMW_BLOCK;
            for (const Tensor* s : { &firstScale[i], &secondScale[i] }) {
                onDevice(*s, "scales");
                requireType(s->scalar_type() == at::kFloat, "scales must have dtype float32");
                require(s->numel() == blocks && s->is_contiguous(), "scales must be contiguous with one value for each 256 elements");
            }
            t.exp_avg_scale = firstScale[i].data_ptr<float>();
            t.exp_avg_sq_scale = secondScale[i].data_ptr<float>();
        }
    }
    carl_adamw h{ lr, beta1, beta2, eps, weightDecay, step, eight ? 8 : 32, nullptr };
    if (gradScale) {
        onDevice(*gradScale, "grad_scale");
        requireType(gradScale->scalar_type() == at::kFloat, "grad_scale must have dtype float32");
        require(gradScale->numel() == 1, "grad_scale must hold one value");
        h.grad_scale = gradScale->data_ptr<float>();
    }
    // refuses what may not be changed in place
    for (const TensorList* tensors : { &params, &first, &second, &firstScale, &secondScale })
        for (size_t i = 0; i < tensors->size(); i++) (*tensors)[i].unsafeGetTensorImpl()->bump_version();
    check(carl_adamw_step(list.data(), (int)n, &h, Queue()));
}

int64_t momentBlocks(const Tensor& m) { return (m.numel() + CARL_ADAMW_BLOCK - 1) / CARL_ADAMW_BLOCK; }

std::tuple<Tensor, Tensor> decodeMoments(const Tensor& m, const Tensor& ms, const Tensor& v, const Tensor& vs)
{
    const OnDevice onDevice;
    for (const Tensor* t : { &m, &ms, &v, &vs }) {
        onDevice(*t, "moments");
        require(t->is_contiguous(), "moments must be contiguous");
    }
    requireType(m.scalar_type() == at::kChar && v.scalar_type() == at::kByte, "codes must have dtypes int8 and uint8");
    requireType(ms.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat, "scales must have dtype float32");
    require(m.sizes() == v.sizes(), "moments must have the same shape");
    require(ms.numel() == momentBlocks(m) && vs.numel() == momentBlocks(m), "scales must have one value for each 256 elements");
    Tensor mOut = at::empty(m.sizes(), ms.options()), vOut = at::empty(m.sizes(), ms.options());
    check(carl_adamw_decode(m.data_ptr<int8_t>(), ms.data_ptr<float>(), v.data_ptr<uint8_t>(), vs.data_ptr<float>(),
                            m.numel(), mOut.data_ptr<float>(), vOut.data_ptr<float>(), Queue()));
    return { mOut, vOut };
}

std::tuple<Tensor, Tensor, Tensor, Tensor> encodeMoments(const Tensor& m, const Tensor& v)
{
    const OnDevice onDevice;
    for (const Tensor* t : { &m, &v }) {
        onDevice(*t, "moments");
        require(t->is_contiguous(), "moments must be contiguous");
        requireType(t->scalar_type() == at::kFloat, "moments must have dtype float32");
    }
    require(m.sizes() == v.sizes(), "moments must have the same shape");
    Tensor mOut = at::empty(m.sizes(), m.options().dtype(at::kChar)), vOut = at::empty(m.sizes(), m.options().dtype(at::kByte));
    Tensor ms = at::empty({ momentBlocks(m) }, m.options()), vs = at::empty({ momentBlocks(m) }, m.options());
    check(carl_adamw_encode(m.data_ptr<float>(), v.data_ptr<float>(), m.numel(), mOut.data_ptr<int8_t>(),
                            ms.data_ptr<float>(), vOut.data_ptr<uint8_t>(), vs.data_ptr<float>(), Queue()));
    return { mOut, ms, vOut, vs };
}

}  // namespace

PYBIND11_MODULE(_ops, m)
{
    m.doc() = "The learner's operators of the MI355X engine (C-ABI in include/carl_amd_ops.h).";
    m.def("linear_attention", &linearAttention);
    m.def("linear_attention_step", &linearAttentionStep);
    m.def("gated_ffn", &gatedFfn);
    m.def("adamw_step", &adamwStep);
    m.def("decode_moments", &decodeMoments);
    m.def("encode_moments", &encodeMoments);
}

// The policy operators on torch tensors: argument checks, outputs and scratch from torch's allocator
// on the current stream, and the autograd nodes, around the C ABI of include/policy.h.
//
// In C++ because the operators' smallest calls take a few microseconds on the GPU: the same steps in
// Python took 26 us for a forward call and 170 us for one with gradients.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <vector>

#include "policy.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<Tensor>;

#define REQUIRE(ok, ...) TORCH_CHECK(ok, __VA_ARGS__)

bool known_type(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
int32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? POLICY_F32 : POLICY_BF16; }

// A trace sees no call of this module: it would hold the result as a constant.
void check_not_traced() { REQUIRE(!torch::jit::tracer::isTracing(), "the policy operators cannot be traced"); }

// A result without a tangent would say that the derivative is 0.
void check_tangent(const char* name, const Tensor& t)
{
    REQUIRE(!t._fw_grad(0).defined(), name, " carries a tangent: forward-mode derivatives are not supported");
}

void check_heads(const char* name, const Tensor& t, const Tensor& like)
{
    REQUIRE(t.is_cuda(), name, " must be a CUDA tensor. CPU tensors are not supported.");
    REQUIRE(t.dim() == 4, name, " must have shape [batch, tokens, heads, dim]");
    REQUIRE(known_type(t), name, " must be float32 or bfloat16");
    REQUIRE(t.scalar_type() == like.scalar_type(), name, " must have the type of q");
    REQUIRE(t.device() == like.device(), name, " must be on the device of q");
    check_tangent(name, t);
}

// The tensor, or a contiguous copy where its rows are not dense or not 16-byte aligned.
Tensor rows(const Tensor& t)
{
    const auto e = static_cast<int64_t>(t.element_size());
    bool ok = (t.stride(3) == 1 || t.size(3) <= 1) && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) * e % 16 == 0);
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Strides of batch, token and head; the stride of an axis with one entry is never used and may be anything.
void put_strides(int64_t (&s)[3], const Tensor& t)
{
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// autograd's apply takes a missing tensor as an empty optional only
OptionalTensor optional(const Tensor& t) { return t.defined() ? OptionalTensor(t) : std::nullopt; }

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const void* const_data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

Tensor scratch(uint64_t bytes, const Tensor& like)
{
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void check_status(int rc, const char* what)
{
    TORCH_CHECK(rc == POLICY_OK, what, " failed (", rc, "): ", policy_last_error());
}

// What torch.autograd.function.once_differentiable does: a gradient of these gradients is an error.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>("the policy operators can be differentiated once only",
                                                                 static_cast<int64_t>(grads.size()));
    std::vector<size_t> at;
    variable_list some;
    for (size_t i = 0; i < grads.size(); ++i)
        if (grads[i].defined()) {
            at.push_back(i);
            some.push_back(grads[i].requires_grad_(true));  // a leaf of its own: the error node records it
        }
    some = (*error)(std::move(some));
    for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = some[i];
    return grads;
}

// --- cross attention -------------------------------------------------------------

policy_attention attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& key_mask, const Tensor& key_lengths,
                                double scale)
{
    policy_attention a{};
    a.device = q.device().index();
    a.dtype = dtype_of(q);
    a.batch = q.size(0), a.lq = q.size(1), a.lk = k.size(1);
    a.heads = static_cast<int32_t>(q.size(2)), a.kv_heads = static_cast<int32_t>(k.size(2)), a.dim = static_cast<int32_t>(q.size(3));
    a.scale = static_cast<float>(scale);
    a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr();
    put_strides(a.q_strides, q);
    put_strides(a.k_strides, k);
    put_strides(a.v_strides, v);
    a.key_mask = static_cast<const uint8_t*>(const_data(key_mask));
    a.key_mask_stride = key_mask.defined() && key_mask.size(0) > 1 ? key_mask.stride(0) : 0;
    a.key_lengths = static_cast<const int32_t*>(const_data(key_lengths));
    return a;
}

Tensor attend(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& key_mask, const Tensor& key_lengths, double scale,
              Tensor* stats, Tensor* rest)
{
    Tensor out = at::empty(q.sizes(), q.options());
    policy_attention a = attention_args(q, k, v, key_mask, key_lengths, scale);
    a.out = out.data_ptr();
    if (stats) {  // for the backward pass
        *stats = at::empty({q.size(0), q.size(1), q.size(2), 2}, q.options().dtype(at::kFloat));
        a.stats = stats->data_ptr<float>();
        if (a.dtype == POLICY_BF16) *rest = at::empty(q.sizes(), q.options());
        a.out_rest = data(*rest);
    }
    const Tensor ws = scratch(policy_cross_attention_workspace_bytes(&a, 0), q);
    a.workspace = data(ws);
    check_status(policy_cross_attention(&a, stream_of(q)), "policy_cross_attention");
    return out;
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptionalTensor& mask,
                          const OptionalTensor& lengths, double scale)
    {
        const Tensor key_mask = mask.value_or(Tensor()), key_lengths = lengths.value_or(Tensor());
        const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
        Tensor stats, rest;
        Tensor out = attend(q, k, v, key_mask, key_lengths, scale, &stats, &rest);
        ctx->save_for_backward({q, k, v, key_mask, key_lengths, out, stats, rest});
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[5], &stats = s[6], &rest = s[7];
        const Tensor dout = rows(grads[0].detach());
        policy_attention a = attention_args(q, k, v, s[3], s[4], ctx->saved_data["scale"].toDouble());
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(k.sizes(), k.options());
        a.out = out.data_ptr();
        a.stats = stats.data_ptr<float>();
        a.out_rest = data(rest);
        a.dout = dout.const_data_ptr();
        put_strides(a.dout_strides, dout);
        a.dq = dq.data_ptr(), a.dk = dk.data_ptr(), a.dv = dv.data_ptr();
        const Tensor ws = scratch(policy_cross_attention_workspace_bytes(&a, 1), q);
        a.workspace = data(ws);
        check_status(policy_cross_attention_backward(&a, stream_of(q)), "policy_cross_attention_backward");
        return once({dq, dk, dv, Tensor(), Tensor(), Tensor()});
    }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptionalTensor& mask, const OptionalTensor& lengths,
                       const std::optional<double>& scale_)
{
    check_not_traced();
    check_heads("q", q, q);
    check_heads("k", k, q);
    check_heads("v", v, q);
    const int64_t b = q.size(0), h = q.size(2), d = q.size(3), lk = k.size(1), hk = k.size(2);
    REQUIRE(k.sizes() == v.sizes(), "k and v must have the same shape");
    REQUIRE(k.size(0) == b && k.size(3) == d, "k and v must have the batch and the dim of q");
    REQUIRE(hk > 0 && h > 0 && h % hk == 0, "the heads of q must be a positive multiple of those of k");
    REQUIRE(d >= 8 && d <= 128 && d % 8 == 0, "dim must be a multiple of 8 from 8 to 128");
    const double scale = scale_ ? *scale_ : 1.0 / std::sqrt(static_cast<double>(d));
    REQUIRE(scale > 0.0 && std::isfinite(scale), "scale must be positive and finite");
    Tensor key_mask, key_lengths;
    if (mask) {
        REQUIRE(mask->device() == q.device(), "key_mask must be on the device of q");
        REQUIRE(mask->scalar_type() == at::kBool && mask->dim() == 2 && mask->size(0) == b && mask->size(1) == lk,
                "key_mask must be a bool tensor of shape [batch, lk]");
        key_mask = mask->stride(1) == 1 || lk <= 1 ? *mask : mask->contiguous();
    }
    if (lengths) {
        REQUIRE(lengths->device() == q.device(), "key_lengths must be on the device of q");
        REQUIRE(lengths->scalar_type() == at::kInt && lengths->dim() == 1 && lengths->size(0) == b,
                "key_lengths must be an int32 tensor of shape [batch]");
        key_lengths = lengths->is_contiguous() ? *lengths : lengths->contiguous();
    }
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
        return CrossAttention::apply(q, k, v, optional(key_mask), optional(key_lengths), scale);
    at::NoGradGuard no_grad;
    return attend(rows(q), rows(k), rows(v), key_mask, key_lengths, scale, nullptr, nullptr);
}

// --- norms of queries and keys with rotation -------------------------------------

struct Side {
    Tensor x, weight, table, positions;
};

policy_qk_norm norm_args(const Side (&side)[2], double eps)
{
    policy_qk_norm a{};
    const Tensor& q = side[0].x;
    a.device = q.device().index();
    a.dtype = dtype_of(q);
    a.batch = q.size(0);
    a.dim = static_cast<int32_t>(q.size(3));
    a.rotary = side[0].table.defined() ? static_cast<int32_t>(2 * side[0].table.size(2)) : 0;
    a.eps = static_cast<float>(eps);
    for (int i = 0; i < 2; ++i) {
        policy_norm_side& s = a.side[i];
        s.x = side[i].x.const_data_ptr();
        put_strides(s.strides, side[i].x);
        s.tokens = side[i].x.size(1);
        s.heads = static_cast<int32_t>(side[i].x.size(2));
        s.weight = static_cast<const float*>(const_data(side[i].weight));
        s.table = static_cast<const float*>(const_data(side[i].table));
        s.table_rows = side[i].table.defined() ? side[i].table.size(0) : 0;
        s.positions = static_cast<const int32_t*>(const_data(side[i].positions));
    }
    return a;
}

variable_list norm(const Side (&side)[2], double eps)
{
    policy_qk_norm a = norm_args(side, eps);
    variable_list y;
    for (int i = 0; i < 2; ++i) {
        y.push_back(at::empty(side[i].x.sizes(), side[i].x.options()));
        a.side[i].y = y[i].data_ptr();
    }
    check_status(policy_qk_norm_rotary(&a, stream_of(side[0].x)), "policy_qk_norm_rotary");
    return y;
}

struct QkNormRotary : torch::autograd::Function<QkNormRotary> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptionalTensor& q_weight,
                                 const OptionalTensor& k_weight, const OptionalTensor& q_table, const OptionalTensor& k_table,
                                 const OptionalTensor& q_positions, const OptionalTensor& k_positions, double eps)
    {
        const Tensor none;
        const Side side[2] = {{rows(q), q_weight.value_or(none), q_table.value_or(none), q_positions.value_or(none)},
                              {rows(k), k_weight.value_or(none), k_table.value_or(none), k_positions.value_or(none)}};
        ctx->save_for_backward({side[0].x, side[1].x, side[0].weight, side[1].weight, side[0].table, side[1].table, side[0].positions,
                                side[1].positions});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["weights"] = (q_weight && q_weight->requires_grad() ? 1 : 0) + (k_weight && k_weight->requires_grad() ? 2 : 0);
        return norm(side, eps);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list s = ctx->get_saved_variables();
        const Side side[2] = {{s[0], s[2], s[4], s[6]}, {s[1], s[3], s[5], s[7]}};
        const int64_t weights = ctx->saved_data["weights"].toInt();
        policy_qk_norm a = norm_args(side, ctx->saved_data["eps"].toDouble());
        variable_list out(9);
        Tensor dy[2];
        for (int i = 0; i < 2; ++i) {
            dy[i] = rows(grads[i].detach());
            out[i] = at::empty(side[i].x.sizes(), side[i].x.options());
            a.side[i].dy = dy[i].const_data_ptr();
            put_strides(a.side[i].dy_strides, dy[i]);
            a.side[i].dx = out[i].data_ptr();
            if (weights & (1 << i)) {
                out[2 + i] = at::empty({a.dim}, side[i].x.options().dtype(at::kFloat));
                a.side[i].dweight = out[2 + i].data_ptr<float>();
            }
        }
        const Tensor ws = scratch(weights ? policy_qk_norm_workspace_bytes(&a) : 0, side[0].x);
        a.workspace = data(ws);
        check_status(policy_qk_norm_rotary_backward(&a, stream_of(side[0].x)), "policy_qk_norm_rotary_backward");
        return once(std::move(out));
    }
};

// (a conversion that changes nothing still costs a dispatch, a good part of a small call)
Tensor aligned(const Tensor& t)
{
    const Tensor c = t.is_contiguous() ? t : t.contiguous();
    return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0 ? c : c.clone();
}

Tensor check_weight(const char* name, const OptionalTensor& w, const Tensor& x)
{
    if (!w) return Tensor();
    REQUIRE(w->device() == x.device() && (w->scalar_type() == at::kFloat || w->scalar_type() == x.scalar_type()) && w->dim() == 1 &&
                w->size(0) == x.size(3),
            name, " must be a [dim] tensor in float32 or the type of q, on its device");
    check_tangent(name, *w);
    return aligned(w->scalar_type() == at::kFloat ? *w : w->to(at::kFloat));
}

Tensor check_table(const char* name, const OptionalTensor& table, const Tensor& x, bool positions)
{
    if (!table) return Tensor();
    REQUIRE(table->device() == x.device() && table->scalar_type() == at::kFloat && table->dim() == 3 && table->size(1) == 2, name,
            " must be a float32 tensor of shape [rows, 2, rotary_dim / 2] on the device of q");
    REQUIRE(table->size(2) % 8 == 0 && table->size(2) > 0 && 2 * table->size(2) <= x.size(3), name,
            ": rotary_dim must be a multiple of 16 from 16 to dim");
    REQUIRE(positions || table->size(0) >= x.size(1), name, " must have a row for every token");
    return aligned(table->requires_grad() ? table->detach() : *table);
}

Tensor check_positions(const char* name, const OptionalTensor& p, const Tensor& x)
{
    if (!p) return Tensor();
    REQUIRE(p->device() == x.device() && p->scalar_type() == at::kInt && p->dim() == 2 && p->size(0) == x.size(0) && p->size(1) == x.size(1),
            name, " must be an int32 tensor of shape [batch, tokens] on the device of q");
    return p->is_contiguous() ? *p : p->contiguous();
}

std::tuple<Tensor, Tensor> qk_norm_rotary(const Tensor& q, const Tensor& k, const OptionalTensor& q_weight_, const OptionalTensor& k_weight_,
                                          const OptionalTensor& q_table_, const OptionalTensor& k_table_,
                                          const OptionalTensor& q_positions_, const OptionalTensor& k_positions_, double eps)
{
    check_not_traced();
    check_heads("q", q, q);
    check_heads("k", k, q);
    const int64_t d = q.size(3);
    REQUIRE(k.size(0) == q.size(0) && k.size(3) == d, "k must have the batch and the dim of q");
    REQUIRE(q.size(2) > 0 && k.size(2) > 0, "q and k must have at least one head");
    REQUIRE(d >= 8 && d <= 256 && d % 8 == 0, "dim must be a multiple of 8 from 8 to 256");
    REQUIRE(q_table_.has_value() == k_table_.has_value(), "q_table and k_table must be given together");
    REQUIRE(q_table_.has_value() || (!q_positions_ && !k_positions_), "positions need tables");
    REQUIRE(eps >= 0.0, "eps must not be negative");
    const Tensor q_weight = check_weight("q_weight", q_weight_, q), k_weight = check_weight("k_weight", k_weight_, q);
    const Tensor q_positions = check_positions("q_positions", q_positions_, q), k_positions = check_positions("k_positions", k_positions_, k);
    const Tensor q_table = check_table("q_table", q_table_, q, q_positions.defined());
    const Tensor k_table = check_table("k_table", k_table_, k, k_positions.defined());
    REQUIRE(!q_table.defined() || q_table.size(2) == k_table.size(2), "q_table and k_table must have the same rotary_dim");
    const auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    variable_list y;
    if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(q_weight) || wants(k_weight))) {
        y = QkNormRotary::apply(q, k, optional(q_weight), optional(k_weight), optional(q_table), optional(k_table),
                                optional(q_positions), optional(k_positions), eps);
    } else {
        at::NoGradGuard no_grad;
        y = norm({{rows(q), q_weight, q_table, q_positions}, {rows(k), k_weight, k_table, k_positions}}, eps);
    }
    return {y[0], y[1]};
}

// --- global gradient norm and clipping -------------------------------------------

Tensor clip_grad_norm(const std::vector<Tensor>& grads, double max_norm, const std::optional<std::vector<Tensor>>& out)
{
    check_not_traced();
    REQUIRE(max_norm >= 0.0, "max_norm must not be negative");
    REQUIRE(!grads.empty(), "grads must not be empty");
    const std::vector<Tensor>& outs = out ? *out : grads;
    REQUIRE(outs.size() == grads.size(), "out must have one tensor for every gradient");
    const at::Device device = grads[0].device();
    REQUIRE(device.is_cuda(), "grads must be CUDA tensors. CPU tensors are not supported.");
    const bool tangents = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;  // asked once, not of every tensor
    std::vector<policy_grad> table(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor &g = grads[i], &o = outs[i];
        REQUIRE(known_type(g), "grads must be float32 or bfloat16");
        if (tangents) {
            check_tangent("a tensor of grads", g);
            check_tangent("a tensor of out", o);
        }
        REQUIRE(g.device() == device, "grads must all be on one device");
        REQUIRE(g.is_non_overlapping_and_dense(), "grads must be dense in memory");
        REQUIRE(o.is_same(g) || (o.device() == device && o.scalar_type() == g.scalar_type() && o.sizes() == g.sizes() && o.strides() == g.strides()),
                "out must have the shapes, types, strides and device of grads");
        table[i].grad = g.const_data_ptr();
        table[i].out = o.data_ptr();
        table[i].count = static_cast<uint64_t>(g.numel());
        table[i].dtype = dtype_of(g);
    }
    at::NoGradGuard no_grad;
    const auto n = static_cast<int64_t>(table.size());
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    const Tensor ws = scratch(policy_clip_grad_workspace_bytes(table.data(), n), norm);
    check_status(policy_clip_grad_norm(table.data(), n, static_cast<float>(max_norm), norm.data_ptr<float>(), device.index(), data(ws),
                                       stream_of(norm)),
                 "policy_clip_grad_norm");
    for (const Tensor& o : outs)
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();  // as torch's in-place operations do
    return norm;
}

}  // namespace

// What the module was built for; the loader and the build look for it in the file.
extern "C" __attribute__((used)) const char navi_policy_torch_built_for[] = "navi_policy_torch for torch " NAVI_TORCH_VERSION;

PYBIND11_MODULE(navi_policy_torch, m)
{
    using release = py::call_guard<py::gil_scoped_release>;
    m.def("cross_attention", &cross_attention, release());
    m.def("qk_norm_rotary", &qk_norm_rotary, release());
    m.def("clip_grad_norm", &clip_grad_norm, release());
}

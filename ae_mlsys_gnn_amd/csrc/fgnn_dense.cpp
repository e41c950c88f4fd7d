// The dense operators' way from torch tensors to the C ABI, in C++: checks of the operands, outputs, workspaces, and the autograd nodes.  Small layers are
// bound by the host: the norm of 64 rows with its backward pass took 124 us of it in Python (of which 49 go to any autograd function written there, and
// most of the rest to the thread that runs backward passes).  The kernels are those of libfgnn_hip.so; there is no CPU path here either.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <cmath>
#include <sstream>
#include "fgnn.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

namespace {

struct Error : std::runtime_error { using std::runtime_error::runtime_error; };
template <typename... A> [[noreturn]] void refuse(const A &...a)
{
    std::ostringstream s;
    (s << ... << a);
    throw Error(s.str());
}
void check(int rc, const char *what)
{
    if (rc != 0) refuse(what, " failed (code ", rc, "): ", fgnn_last_error());
}

int float_type(const Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return FGNN_F32;
    case at::kBFloat16: return FGNN_BF16;
    case at::kHalf: return FGNN_F16;
    default: return -1;
    }
}
int eight_type(at::ScalarType t) { return t == at::kChar ? FGNN_I8 : t == at::kFloat8_e4m3fn ? FGNN_E4M3 : -1; }
void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
// Operands are on the GPU, and torch's own operations are not being recorded or transformed: a kernel launched past jit.trace, make_fx or export would be missing from the
// record (its output a constant of it), and one launched past forward mode would drop the tangents, with no error from anyone.  torch.compile breaks its graph at
// the call and runs it as it is; functorch's tensors have no memory and are refused for that by torch.
void usable_one(const char *who, const Tensor &t)
{
    if (!t.defined()) return;
    if (!t.is_cuda()) refuse("fgnn operators run on the GPU only (got a ", t.device(), " tensor); there is no CPU path");
    if (t._fw_grad(0).defined()) refuse(who, ": derivatives in forward mode are not recorded");
}
template <typename... T> void usable(const char *who, const T &...operands)
{
    (usable_one(who, operands), ...);
    typedef c10::impl::TorchDispatchModeTLS Modes;
    typedef c10::impl::TorchDispatchModeKey Mode;
    if (torch::jit::tracer::isTracing() || (Modes::any_modes_set() && (Modes::get_mode(Mode::PROXY) || Modes::get_mode(Mode::FAKE) || Modes::get_mode(Mode::FUNCTIONAL))))
        refuse(who, ": calls are not recorded by jit.trace, make_fx or export");
}
Tensor given(const MaybeTensor &t) { return t.has_value() ? *t : Tensor(); }

// t as [rows, columns] with unit column stride; copied only where no view of that kind exists.
struct Rows { Tensor t; int64_t rows, cols, ld; };
Rows rows_of(const Tensor &t)
{
    const int64_t cols = t.size(-1), rows = c10::multiply_integers(t.sizes().slice(0, t.dim() - 1));
    if (t.is_contiguous()) return {t, rows, cols, cols};
    Tensor r = t.dim() == 2 ? t : t.reshape({rows, cols});
    if ((cols > 1 && r.stride(1) != 1) || (rows > 1 && r.stride(0) < cols)) r = r.contiguous();
    return {r, rows, cols, rows > 1 ? r.stride(0) : cols};
}
// Whether rows do not all start at 16 bytes and hold whole 16 bytes, or lie too far apart to be moved as they are: 2^23 bytes, 2^25 where the reduction goes
// from row to row (`strided`).
bool loose(const Rows &r, bool strided = false)
{
    const int64_t size = r.t.element_size();
    return (((uintptr_t)r.t.data_ptr() | r.ld * size | r.cols * size) & 15) || r.ld * size >= (strided ? 1 << 25 : 1 << 23);
}
Tensor like(const Tensor &t, at::IntArrayRef shape) { return at::empty(shape, t.options()); }
Tensor like(const Tensor &t, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, t.options().dtype(type)); }
Tensor scratch(const Tensor &t, size_t bytes) { return bytes ? at::empty({(int64_t)bytes}, t.options().dtype(at::kByte)) : Tensor(); }
std::vector<int64_t> with_last(const Tensor &t, int64_t n)
{
    std::vector<int64_t> s(t.sizes().begin(), t.sizes().end());
    s.back() = n;
    return s;
}
int as_int(int64_t v, const char *what)
{
    if (v > INT32_MAX) refuse(what, " of ", v, " columns");
    return (int)v;
}
bool wanted(const Tensor &t) { return t.defined() && t.requires_grad(); }

// Gradients that a graph was asked of (create_graph): used once more, they say that there is none.
variable_list final_gradients(const char *what, variable_list grads)
{
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (auto &g : grads) if (g.defined()) some.push_back(g.detach().requires_grad_(true));
    const int64_t n = (int64_t)some.size();
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": gradients of second order are not recorded", n);
    some = (*node)(std::move(some));
    size_t i = 0;
    for (auto &g : grads) if (g.defined()) g = some[i++];
    return grads;
}

// ------------------------------------------------------------------------------------------------ norm
struct NormOperands { Rows x, r; Tensor w; int type, wtype; };
NormOperands norm_operands(const char *who, const Tensor &x, const Tensor &w, const Tensor &r)
{
    usable(who, x, w, r);
    const int type = float_type(x);
    if (type < 0) refuse(who, ": rows of ", x.scalar_type(), "; fp32, bf16 and fp16 are supported");
    if (x.dim() == 0 || x.size(-1) == 0) refuse(who, ": no features in ", x.sizes());
    NormOperands o{{}, {}, {}, type, type};
    if (w.defined()) {
        if (w.dim() != 1 || w.size(0) != x.size(-1) || (w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat) || w.device() != x.device())
            refuse(who, ": weights ", w.sizes(), " of ", w.scalar_type(), " for rows ", x.sizes(), " of ", x.scalar_type());
        o.w = w.contiguous();
        o.wtype = float_type(w);
    }
    if (r.defined()) {
        if (r.sizes() != x.sizes() || r.scalar_type() != x.scalar_type() || r.device() != x.device())
            refuse(who, ": residual ", r.sizes(), " of ", r.scalar_type(), " beside ", x.sizes(), " of ", x.scalar_type());
        o.r = rows_of(r);
    }
    o.x = rows_of(x);
    return o;
}

struct NormOut { Tensor y, h, rstd; };
NormOut norm_forward(const Tensor &x, const Tensor &w, const Tensor &r, double eps, bool keep)
{
    const NormOperands o = norm_operands("rms_norm", x, w, r);
    const c10::OptionalDeviceGuard guard(x.device());
    NormOut out{like(x, x.sizes()), {}, {}};
    if (r.defined()) out.h = like(x, x.sizes());
    if (keep) out.rstd = like(x, {o.x.rows}, at::kFloat);
    check(fgnn_rms_norm(o.x.rows, as_int(o.x.cols, "rows"), o.type, address(o.x.t), o.x.ld, address(o.r.t), o.r.ld, address(o.w), o.wtype, (float)eps, address(out.h), address(out.y),
                        (float *)address(out.rstd), stream_of(x)), "fgnn_rms_norm");
    return out;
}

// Kept for the backward pass: h as it is handed out (x without a residual) and a scale a row; the norm itself is taken of the sum before it is rounded.
struct Norm : torch::autograd::Function<Norm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps)
    {
        const Tensor w = given(weight), r = given(residual);
        const NormOut o = norm_forward(x, w, r, eps, true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["need"] = (int64_t)(wanted(x) | wanted(w) << 1 | wanted(r) << 2);
        ctx->save_for_backward({o.h.defined() ? o.h : x, w, o.rstd});
        return o.h.defined() ? variable_list{o.y, o.h} : variable_list{o.y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const variable_list saved = ctx->get_saved_variables();
        const int64_t need = ctx->saved_data["need"].toInt();
        Tensor gy = up[0], gh = up.size() > 1 ? up[1] : Tensor();
        if ((!gy.defined() && !gh.defined()) || need == 0) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const Rows h = rows_of(saved[0]);
        const Tensor w = saved[1].defined() ? saved[1].contiguous() : Tensor();
        const int type = float_type(h.t), wtype = w.defined() ? float_type(w) : type;
        if (gy.defined()) gy = gy.contiguous();
        if (gh.defined()) gh = gh.contiguous();
        const c10::OptionalDeviceGuard guard(h.t.device());
        Tensor dx, dw, ws;
        if (need & 5) dx = like(h.t, saved[0].sizes());
        size_t bytes = 0;
        if (need & 2) {
            dw = like(w, w.sizes());
            ws = scratch(h.t, bytes = fgnn_rms_norm_backward_workspace_bytes(h.rows, (int)h.cols, type));
        }
        check(fgnn_rms_norm_backward(h.rows, (int)h.cols, type, address(gy), address(gh), address(h.t), h.ld, address(w), wtype, (const float *)address(saved[2]), address(dx), address(dw),
                                     address(ws), bytes, stream_of(h.t)), "fgnn_rms_norm_backward");
        return final_gradients("rms_norm", {need & 1 ? dx : Tensor(), dw, need & 4 ? dx : Tensor(), Tensor()});
    }
};

py::object rms_norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps)
{
    Tensor y, h;
    const Tensor w = given(weight), r = given(residual);
    {
        py::gil_scoped_release off;
        if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(r))) {
            const variable_list out = Norm::apply(x, weight, residual, eps);
            y = out[0];
            if (out.size() > 1) h = out[1];
        } else {
            const NormOut out = norm_forward(x, w, r, eps, false);
            y = out.y;
            h = out.h;
        }
    }
    return h.defined() ? (py::object)py::make_tuple(y, h) : py::cast(y);
}

py::tuple rms_norm_q8(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &residual, double eps, at::ScalarType to)
{
    const int eight = eight_type(to);
    if (eight < 0) refuse("rms_norm_q8: 8-bit output in ", to, "; torch.int8 and torch.float8_e4m3fn are supported");
    const Tensor w = given(weight), r = given(residual);
    const NormOperands o = norm_operands("rms_norm_q8", x, w, r);
    const c10::OptionalDeviceGuard guard(x.device());
    const Tensor q = like(x, x.sizes(), to), scale = like(x, x.sizes().slice(0, x.dim() - 1), at::kFloat), h = r.defined() ? like(x, x.sizes()) : Tensor();
    check(fgnn_rms_norm_q8(o.x.rows, as_int(o.x.cols, "rows"), o.type, address(o.x.t), o.x.ld, address(o.r.t), o.r.ld, address(o.w), o.wtype, (float)eps, eight, address(h), address(q),
                           (float *)address(scale), stream_of(x)), "fgnn_rms_norm_q8");
    return h.defined() ? py::make_tuple(q, scale, h) : py::make_tuple(q, scale);
}

py::tuple quantize_rows(const Tensor &x, at::ScalarType to)
{
    const int eight = eight_type(to);
    if (eight < 0) refuse("quantize_rows: 8-bit output in ", to, "; torch.int8 and torch.float8_e4m3fn are supported");
    const NormOperands o = norm_operands("quantize_rows", x, Tensor(), Tensor());
    const c10::OptionalDeviceGuard guard(x.device());
    const Tensor q = like(x, x.sizes(), to), scale = like(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
    check(fgnn_quantize_rows(o.x.rows, as_int(o.x.cols, "rows"), o.type, address(o.x.t), o.x.ld, eight, address(q), (float *)address(scale), stream_of(x)), "fgnn_quantize_rows");
    return py::make_tuple(q, scale);
}

// ------------------------------------------------------------------------------------------------ linear maps
struct Epilogue { Tensor bias; int btype; Rows res; };
Epilogue epilogue(const char *who, const Tensor &x, int64_t n, at::ScalarType dtype, int type, const Tensor &bias, const Tensor &residual)
{
    Epilogue e{{}, type, {}};
    if (bias.defined()) {
        if (bias.dim() != 1 || bias.size(0) != n || (bias.scalar_type() != dtype && bias.scalar_type() != at::kFloat) || bias.device() != x.device())
            refuse(who, ": bias ", bias.sizes(), " of ", bias.scalar_type(), " for ", n, " columns of ", dtype);
        e.bias = bias.contiguous();
        e.btype = float_type(bias);
    }
    if (residual.defined()) {
        if (residual.dim() != x.dim() || residual.sizes() != at::IntArrayRef(with_last(x, n)) || residual.scalar_type() != dtype || residual.device() != x.device())
            refuse(who, ": residual ", residual.sizes(), " of ", residual.scalar_type(), " beside ", with_last(x, n), " of ", dtype);
        e.res = rows_of(residual);
    }
    return e;
}

struct LinearOut { Tensor y, z; };
LinearOut linear_forward(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &residual, int64_t act, double slope, bool keep)
{
    usable("linear_act", x, w, bias, residual);
    const int type = float_type(x);
    if (type < 0 || w.scalar_type() != x.scalar_type())
        refuse("linear_act: rows of ", x.scalar_type(), " with weights of ", w.scalar_type(), "; fp32, bf16 and fp16, both the same, are supported");
    if (x.dim() == 0 || w.dim() != 2 || w.size(1) != x.size(-1) || w.device() != x.device()) refuse("linear_act: x ", x.sizes(), " with weights ", w.sizes());
    const int n = as_int(w.size(0), "weights"), k = as_int(w.size(1), "weights");
    const Epilogue e = epilogue("linear_act", x, n, x.scalar_type(), type, bias, residual);
    const Rows a = rows_of(x), b = rows_of(w);
    const c10::OptionalDeviceGuard guard(x.device());
    LinearOut out{like(x, with_last(x, n)), {}};
    if (keep) out.z = like(x, {a.rows, n});
    const size_t bytes = fgnn_linear_workspace_bytes(a.rows, n, k, type, loose(a) || loose(b));
    const Tensor ws = scratch(x, bytes);
    check(fgnn_linear(a.rows, n, k, type, address(a.t), a.ld, address(b.t), b.ld, address(e.bias), e.btype, address(e.res.t), e.res.ld, (int)act, (float)slope, address(out.z), address(out.y),
                      address(ws), bytes, stream_of(x)), "fgnn_linear");
    return out;
}

// Kept for the backward pass: x, W and, with an activation, its argument in the rows' type.
struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const MaybeTensor &bias, const MaybeTensor &residual, int64_t act, double slope)
    {
        const Tensor b = given(bias), r = given(residual);
        const LinearOut o = linear_forward(x, weight, b, r, act, slope, act != 0);
        ctx->saved_data["need"] = (int64_t)(wanted(x) | wanted(weight) << 1 | wanted(b) << 2 | wanted(r) << 3);
        ctx->saved_data["act"] = act;
        ctx->saved_data["slope"] = slope;
        ctx->saved_data["btype"] = (int64_t)(b.defined() ? b.scalar_type() : x.scalar_type());
        ctx->save_for_backward({x, weight, o.z});
        return o.y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const variable_list saved = ctx->get_saved_variables();
        const int64_t need = ctx->saved_data["need"].toInt();
        const int act = (int)ctx->saved_data["act"].toInt();
        const at::ScalarType bias = (at::ScalarType)ctx->saved_data["btype"].toInt();
        const Rows x = rows_of(saved[0]), w = rows_of(saved[1]);
        Rows dz = rows_of(up[0]);
        const int type = float_type(x.t), n = (int)w.rows, k = (int)w.cols;
        const bool sloped = act && (need & 3);
        const c10::OptionalDeviceGuard guard(x.t.device());
        void *stream = stream_of(x.t);
        Tensor dx, dw, db;
        if (need & 4) db = like(x.t, {n}, bias);
        if (n && (sloped || (need & 4))) {
            const Rows g = dz;
            if (sloped) {
                const int64_t width = 16 / x.t.element_size(), ld = (n + width - 1) / width * width;
                dz = Rows{like(x.t, {x.rows, ld}), x.rows, n, ld};
            }
            const size_t bytes = need & 4 ? fgnn_linear_slope_workspace_bytes(x.rows, n, type) : 0;
            const Tensor ws = scratch(x.t, bytes);
            check(fgnn_linear_slope(x.rows, n, type, address(g.t), g.ld, address(saved[2]), act, (float)ctx->saved_data["slope"].toDouble(), sloped ? address(dz.t) : nullptr, dz.ld, address(db),
                                    db.defined() ? float_type(db) : type, address(ws), bytes, stream), "fgnn_linear_slope");
        }
        if (need & 3) {
            const size_t bytes = fgnn_linear_backward_workspace_bytes(x.rows, n, k, type, loose(x, true) || loose(w, true) || (!sloped && loose(dz)));
            const Tensor ws = scratch(x.t, bytes);
            if (need & 1) {
                dx = like(x.t, saved[0].sizes());
                check(fgnn_linear_dx(x.rows, n, k, type, address(dz.t), dz.ld, sloped, address(w.t), w.ld, address(dx), address(ws), bytes, stream), "fgnn_linear_dx");
            }
            if (need & 2) {
                dw = like(x.t, {n, k});
                check(fgnn_linear_dw(x.rows, n, k, type, address(dz.t), dz.ld, sloped, address(x.t), x.ld, address(dw), address(ws), bytes, stream), "fgnn_linear_dw");
            }
        }
        return final_gradients("linear_act", {dx, dw, db, need & 8 ? up[0] : Tensor(), Tensor(), Tensor()});
    }
};

Tensor linear_act(const Tensor &x, const Tensor &weight, const MaybeTensor &bias, const MaybeTensor &residual, int64_t act, double slope)
{
    py::gil_scoped_release off;
    const Tensor b = given(bias), r = given(residual);
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(weight) || wanted(b) || wanted(r))) return Linear::apply(x, weight, bias, residual, act, slope);
    return linear_forward(x, weight, b, r, act, slope, false).y;
}

Tensor linear_q8(const Tensor &q, const Tensor &scale, const Tensor &w, const Tensor &wscale, const MaybeTensor &bias, const MaybeTensor &residual, int64_t act, double slope,
                 at::ScalarType to)
{
    const Tensor b = given(bias), r = given(residual);
    usable("linear_q8", q, scale, w, wscale, b, r);
    const int eight = eight_type(q.scalar_type()), type = to == at::kFloat ? FGNN_F32 : to == at::kBFloat16 ? FGNN_BF16 : to == at::kHalf ? FGNN_F16 : -1;
    if (eight < 0 || w.scalar_type() != q.scalar_type() || type < 0)
        refuse("linear_q8: ", q.scalar_type(), " with weights of ", w.scalar_type(), " to ", to, "; int8 or float8_e4m3fn, both the same, to fp32, bf16 or fp16 are supported");
    if (q.dim() == 0 || w.dim() != 2 || w.size(1) != q.size(-1) || scale.sizes() != q.sizes().slice(0, q.dim() - 1) || wscale.sizes() != w.sizes().slice(0, 1))
        refuse("linear_q8: q ", q.sizes(), ", scale ", scale.sizes(), ", weights ", w.sizes(), ", their scale ", wscale.sizes());
    if (scale.scalar_type() != at::kFloat || wscale.scalar_type() != at::kFloat || scale.device() != q.device() || w.device() != q.device() || wscale.device() != q.device())
        refuse("linear_q8: scales are fp32 on the operands' device");
    const int n = as_int(w.size(0), "weights"), k = as_int(w.size(1), "weights");
    const Epilogue e = epilogue("linear_q8", q, n, to, type, b, r);
    const Rows x = rows_of(q), p = rows_of(w);
    const Tensor s = scale.contiguous(), ws = wscale.contiguous();
    const c10::OptionalDeviceGuard guard(q.device());
    const Tensor y = like(q, with_last(q, n), to);
    const size_t bytes = fgnn_linear_workspace_bytes(x.rows, n, k, eight, loose(x) || loose(p));
    const Tensor work = scratch(q, bytes);
    check(fgnn_linear_q8(x.rows, n, k, eight, type, address(x.t), x.ld, (const float *)address(s), address(p.t), p.ld, (const float *)address(ws), address(e.bias), e.btype, address(e.res.t),
                         e.res.ld, (int)act, (float)slope, address(y), address(work), bytes, stream_of(q)), "fgnn_linear_q8");
    return y;
}

// ------------------------------------------------------------------------------------------------ group norm
// t as [samples, points, channels] with unit channel stride; copied only where no view of that kind exists.
struct Points { Tensor t; int64_t batch, points, cols, ld, stride; };
Points points_of(const Tensor &t)
{
    const int64_t b = t.size(0), cols = t.size(-1), n = c10::multiply_integers(t.sizes().slice(1, t.dim() - 2));
    Tensor r = t.reshape({b, n, cols});
    if ((cols > 1 && r.stride(2) != 1) || (n > 1 && r.stride(1) < cols)) r = r.contiguous();
    return {r, b, n, cols, n > 1 ? r.stride(1) : cols, b > 1 ? r.stride(0) : 0};
}
struct GroupNormOperands { Points x; Tensor w, b; int type, wtype, btype, groups; };
GroupNormOperands group_norm_operands(const Tensor &x, int64_t groups, const Tensor &w, const Tensor &b)
{
    usable("group_norm", x, w, b);
    const int type = float_type(x);
    if (type < 0) refuse("group_norm: features of ", x.scalar_type(), "; fp32, bf16 and fp16 are supported");
    if (x.dim() < 2 || x.size(-1) == 0) refuse("group_norm: features ", x.sizes(), "; [samples, ..., channels] is wanted");
    if (groups < 1 || groups > x.size(-1) || x.size(-1) % groups) refuse("group_norm: ", groups, " groups of ", x.size(-1), " channels");
    GroupNormOperands o{{}, {}, {}, type, type, type, as_int(groups, "groups")};
    const auto vector = [&](const Tensor &v, const char *what, Tensor &to, int &to_type) {
        if (!v.defined()) return;
        if (v.dim() != 1 || v.size(0) != x.size(-1) || (v.scalar_type() != x.scalar_type() && v.scalar_type() != at::kFloat) || v.device() != x.device())
            refuse("group_norm: ", what, " ", v.sizes(), " of ", v.scalar_type(), " for features ", x.sizes(), " of ", x.scalar_type());
        to = v.contiguous();
        to_type = float_type(v);
    };
    vector(w, "weights", o.w, o.wtype);
    vector(b, "bias", o.b, o.btype);
    o.x = points_of(x);
    return o;
}
struct GroupNormOut { Tensor y, mean, rstd; };
GroupNormOut group_norm_forward(const Tensor &x, int64_t groups, const Tensor &w, const Tensor &b, double eps, int64_t act, double slope)
{
    const GroupNormOperands o = group_norm_operands(x, groups, w, b);
    const c10::OptionalDeviceGuard guard(x.device());
    const int cols = as_int(o.x.cols, "features");
    GroupNormOut out{like(x, x.sizes()), like(x, {o.x.batch, groups}, at::kFloat), like(x, {o.x.batch, groups}, at::kFloat)};
    const size_t bytes = fgnn_group_norm_workspace_bytes(o.x.batch, o.x.points, cols, o.groups, o.type);
    const Tensor ws = scratch(x, bytes);
    check(fgnn_group_norm(o.x.batch, o.x.points, cols, o.groups, o.type, address(o.x.t), o.x.ld, o.x.stride, address(o.w), o.wtype, address(o.b), o.btype, (float)eps, (int)act, (float)slope,
                          address(out.y), (float *)address(out.mean), (float *)address(out.rstd), address(ws), bytes, stream_of(x)), "fgnn_group_norm");
    return out;
}

// Kept for the backward pass: x, weights, bias, and two numbers a sample and group.
struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, int64_t groups, double eps, int64_t act, double slope)
    {
        const Tensor w = given(weight), b = given(bias);
        const GroupNormOut o = group_norm_forward(x, groups, w, b, eps, act, slope);
        ctx->saved_data["need"] = (int64_t)(wanted(x) | wanted(w) << 1 | wanted(b) << 2);
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        ctx->saved_data["slope"] = slope;
        ctx->save_for_backward({x, w, b, o.mean, o.rstd});
        return o.y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const variable_list saved = ctx->get_saved_variables();
        const int64_t need = ctx->saved_data["need"].toInt();
        const Points x = points_of(saved[0]);
        const Tensor w = saved[1].defined() ? saved[1].contiguous() : Tensor(), b = saved[2].defined() ? saved[2].contiguous() : Tensor(), gy = up[0].contiguous();
        const int type = float_type(x.t), wtype = w.defined() ? float_type(w) : type, btype = b.defined() ? float_type(b) : type, cols = (int)x.cols,
                  groups = (int)ctx->saved_data["groups"].toInt();
        const c10::OptionalDeviceGuard guard(x.t.device());
        Tensor dx, dw, db;
        if (need & 1) dx = like(x.t, saved[0].sizes());
        if (need & 2) dw = like(w, w.sizes());
        if (need & 4) db = like(b, b.sizes());
        const size_t bytes = fgnn_group_norm_backward_workspace_bytes(x.batch, x.points, cols, groups, type);
        const Tensor ws = scratch(x.t, bytes);
        check(fgnn_group_norm_backward(x.batch, x.points, cols, groups, type, address(gy), address(x.t), x.ld, x.stride, address(w), wtype, address(b), btype,
                                       (int)ctx->saved_data["act"].toInt(), (float)ctx->saved_data["slope"].toDouble(), (const float *)address(saved[3]), (const float *)address(saved[4]),
                                       address(dx), address(dw), address(db), address(ws), bytes, stream_of(x.t)), "fgnn_group_norm_backward");
        return final_gradients("group_norm", {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};
Tensor group_norm(const Tensor &x, int64_t groups, const MaybeTensor &weight, const MaybeTensor &bias, double eps, int64_t act, double slope)
{
    py::gil_scoped_release off;
    const Tensor w = given(weight), b = given(bias);
    if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b))) return GroupNorm::apply(x, weight, bias, groups, eps, act, slope);
    return group_norm_forward(x, groups, w, b, eps, act, slope).y;
}

// ------------------------------------------------------------------------------------------------ embeddings
struct Lookup { Tensor tokens; Rows w; int type, wide; };
Lookup lookup_operands(const Tensor &tokens, const Tensor &weight, const std::optional<int64_t> &padding)
{
    usable("embedding", tokens, weight);
    const int type = float_type(weight);
    if (type < 0 || weight.dim() != 2 || weight.size(1) == 0) refuse("embedding: a table ", weight.sizes(), " of ", weight.scalar_type(), "; rows of fp32, bf16 and fp16 are supported");
    if ((tokens.scalar_type() != at::kInt && tokens.scalar_type() != at::kLong) || tokens.device() != weight.device())
        refuse("embedding: tokens of ", tokens.scalar_type(), " on ", tokens.device(), "; int32 and int64 on the table's device are supported");
    if (padding && (*padding < 0 || *padding >= weight.size(0))) refuse("embedding: padding ", *padding, " in a table of ", weight.size(0), " rows");
    as_int(weight.size(0), "rows of a table; columns");
    return {tokens.contiguous(), rows_of(weight), type, tokens.scalar_type() == at::kLong};
}
Tensor lookup_forward(const Tensor &tokens, const Tensor &weight, double scale, const std::optional<int64_t> &padding)
{
    const Lookup o = lookup_operands(tokens, weight, padding);
    const c10::OptionalDeviceGuard guard(weight.device());
    std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(o.w.cols);
    const Tensor y = like(weight, shape);
    check(fgnn_embedding(tokens.numel(), (int)o.w.rows, as_int(o.w.cols, "a table"), o.type, address(o.tokens), o.wide, address(o.w.t), o.w.ld, (float)scale, address(y), stream_of(weight)),
          "fgnn_embedding");
    return y;
}

// Kept for the backward pass: the tokens.
struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext *ctx, const Tensor &weight, const Tensor &tokens, double scale, std::optional<int64_t> padding)
    {
        const Tensor y = lookup_forward(tokens, weight, scale, padding);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding ? *padding : (int64_t)-1;
        ctx->saved_data["rows"] = weight.size(0);
        ctx->save_for_backward({tokens});
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const Tensor tokens = ctx->get_saved_variables()[0].contiguous();
        const Rows gy = rows_of(up[0]);
        const int rows = (int)ctx->saved_data["rows"].toInt(), cols = (int)gy.cols, type = float_type(gy.t);
        const c10::OptionalDeviceGuard guard(gy.t.device());
        const Tensor dw = like(gy.t, {rows, cols});
        const size_t bytes = fgnn_embedding_backward_workspace_bytes(gy.rows, rows, cols, type);
        const Tensor ws = scratch(gy.t, bytes);
        check(fgnn_embedding_backward(gy.rows, rows, cols, type, address(tokens), tokens.scalar_type() == at::kLong, ctx->saved_data["padding"].toInt(), address(gy.t), gy.ld,
                                      (float)ctx->saved_data["scale"].toDouble(), address(dw), address(ws), bytes, stream_of(gy.t)), "fgnn_embedding_backward");
        return final_gradients("embedding", {dw, Tensor(), Tensor(), Tensor()});
    }
};
Tensor embedding(const Tensor &tokens, const Tensor &weight, double scale, std::optional<int64_t> padding)
{
    py::gil_scoped_release off;
    if (at::GradMode::is_enabled() && wanted(weight)) return Embedding::apply(weight, tokens, scale, padding);
    return lookup_forward(tokens, weight, scale, padding);
}

// ------------------------------------------------------------------------------------------------ attention
// t [samples, positions, heads, components] with unit component stride and no negative ones; copied only where no view of that kind exists.
Tensor heads_of(const Tensor &t) { return t.size(3) > 1 && t.stride(3) != 1 ? t.contiguous() : t; }
struct AttentionOperands { Tensor q, k, v, lengths, mask; int type, batch, nq, nk, heads, kv_heads, dim, wide; float scale; };
void strides_to(int64_t *to, const Tensor &t)
{
    for (int i = 0; i < 3; ++i) to[i] = t.size(i) > 1 ? t.stride(i) : 0;
}
AttentionOperands attention_operands(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &lengths, const Tensor &mask, const std::optional<double> &scale)
{
    usable("cross_attention", q, k, v, lengths, mask);
    const int type = float_type(q);
    if (type < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
        refuse("cross_attention: queries of ", q.scalar_type(), " with keys of ", k.scalar_type(), " and values of ", v.scalar_type(), "; fp32, bf16 and fp16, all the same, are supported");
    if (q.dim() != 4 || k.dim() != 4 || k.sizes() != v.sizes() || q.size(0) != k.size(0) || q.size(3) != k.size(3) || k.device() != q.device() || v.device() != q.device())
        refuse("cross_attention: queries ", q.sizes(), ", keys ", k.sizes(), ", values ", v.sizes(), "; [samples, positions, heads, components] are wanted");
    if (k.size(2) == 0 || q.size(2) == 0 || q.size(2) % k.size(2)) refuse("cross_attention: ", q.size(2), " heads over ", k.size(2), " of keys");
    if (q.size(3) < 1 || q.size(3) > 256) refuse("cross_attention: heads of ", q.size(3), " components; up to 256 are supported");
    if (lengths.defined() && (lengths.dim() != 1 || lengths.size(0) != q.size(0) || (lengths.scalar_type() != at::kInt && lengths.scalar_type() != at::kLong) || lengths.device() != q.device()))
        refuse("cross_attention: lengths ", lengths.sizes(), " of ", lengths.scalar_type(), "; one int32 or int64 for each of ", q.size(0), " samples is wanted");
    if (mask.defined() && (mask.dim() != 2 || mask.size(0) != q.size(0) || mask.size(1) != k.size(1) || mask.scalar_type() != at::kBool || mask.device() != q.device()))
        refuse("cross_attention: mask ", mask.sizes(), " of ", mask.scalar_type(), "; a truth value for each of ", q.size(0), " x ", k.size(1), " keys is wanted");
    const double s = scale ? *scale : 1. / std::sqrt((double)q.size(3));
    if (!(s >= 1e-30 && s <= 1e30)) refuse("cross_attention: scale ", s, "; a positive number is wanted");
    return {heads_of(q), heads_of(k), heads_of(v), lengths.defined() ? lengths.contiguous() : Tensor(), mask.defined() ? mask.contiguous() : Tensor(), type, as_int(q.size(0), "samples;"),
            as_int(q.size(1), "queries;"), as_int(k.size(1), "keys;"), as_int(q.size(2), "heads;"), (int)k.size(2), (int)q.size(3), lengths.defined() && lengths.scalar_type() == at::kLong, (float)s};
}
struct AttentionOut { Tensor y, lse, rest; };
AttentionOut attention_forward(const AttentionOperands &o, bool keep, bool keep_rest)
{
    const c10::OptionalDeviceGuard guard(o.q.device());
    int64_t strides[9];
    strides_to(strides, o.q);
    strides_to(strides + 3, o.k);
    strides_to(strides + 6, o.v);
    AttentionOut out{like(o.q, o.q.sizes()), keep ? like(o.q, {o.batch, o.heads, o.nq}, at::kFloat) : Tensor(), keep_rest && o.type != FGNN_F32 ? like(o.q, o.q.sizes()) : Tensor()};
    const size_t bytes = fgnn_attention_workspace_bytes(o.batch, o.nq, o.nk, o.heads, o.kv_heads, o.dim, o.type, address(o.k), address(o.v), strides);
    const Tensor ws = scratch(o.q, bytes);
    check(fgnn_attention_kept(o.batch, o.nq, o.nk, o.heads, o.kv_heads, o.dim, o.type, address(o.q), address(o.k), address(o.v), strides, address(o.lengths), o.wide,
                              (const uint8_t *)address(o.mask), o.scale, address(out.y), address(out.rest), (float *)address(out.lse), address(ws), bytes, stream_of(o.q)), "fgnn_attention");
    return out;
}

// Kept for the backward pass: q, k, v, y, of 16-bit types what its rounding leaves (where q or k is trained), the logarithm of every query's sum, and what is seen.
struct Attention : torch::autograd::Function<Attention> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &lengths, const MaybeTensor &mask, std::optional<double> scale)
    {
        const AttentionOperands o = attention_operands(q, k, v, given(lengths), given(mask), scale);
        // (a call whose gradients are refused is refused before it runs)
        check(fgnn_attention_backward_check(o.batch, o.nq, o.nk, o.heads, o.kv_heads, o.dim, o.type, wanted(q), wanted(k) || wanted(v)), "fgnn_attention_backward");
        const AttentionOut out = attention_forward(o, true, wanted(q) || wanted(k));
        ctx->saved_data["need"] = (int64_t)(wanted(q) | wanted(k) << 1 | wanted(v) << 2);
        ctx->saved_data["scale"] = (double)o.scale;
        ctx->save_for_backward({q, k, v, out.y, out.lse, o.lengths, o.mask, out.rest});
        return out.y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list up)
    {
        const variable_list saved = ctx->get_saved_variables();
        const int64_t need = ctx->saved_data["need"].toInt();
        const Tensor q = heads_of(saved[0]), k = heads_of(saved[1]), v = heads_of(saved[2]), &y = saved[3], &lengths = saved[5], &mask = saved[6], &rest = saved[7], g = heads_of(up[0]);
        const int type = float_type(q), batch = (int)q.size(0), nq = (int)q.size(1), nk = (int)k.size(1), heads = (int)q.size(2), kv_heads = (int)k.size(2), dim = (int)q.size(3);
        const c10::OptionalDeviceGuard guard(q.device());
        int64_t strides[12];
        strides_to(strides, q);
        strides_to(strides + 3, k);
        strides_to(strides + 6, v);
        strides_to(strides + 9, g);
        Tensor dq, dk, dv;
        if (need & 1) dq = like(q, q.sizes());
        if (need & 6) {
            dk = like(k, k.sizes());
            dv = like(v, v.sizes());
        }
        const size_t bytes = fgnn_attention_backward_workspace_bytes(batch, nq, nk, heads, kv_heads, dim, type, address(q), address(k), address(v), address(g), strides);
        const Tensor ws = scratch(q, bytes);
        check(fgnn_attention_kept_backward(batch, nq, nk, heads, kv_heads, dim, type, address(q), address(k), address(v), address(y), address(rest), address(g), strides, address(lengths),
                                           lengths.defined() && lengths.scalar_type() == at::kLong, (const uint8_t *)address(mask), (float)ctx->saved_data["scale"].toDouble(),
                                           (const float *)address(saved[4]), address(dq), address(dk), address(dv), address(ws), bytes, stream_of(q)), "fgnn_attention_backward");
        return final_gradients("cross_attention", {dq, need & 2 ? dk : Tensor(), need & 4 ? dv : Tensor(), Tensor(), Tensor(), Tensor()});
    }
};
Tensor cross_attention(const Tensor &q, const Tensor &k, const Tensor &v, const MaybeTensor &lengths, const MaybeTensor &mask, std::optional<double> scale)
{
    py::gil_scoped_release off;
    if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v))) return Attention::apply(q, k, v, lengths, mask, scale);
    return attention_forward(attention_operands(q, k, v, given(lengths), given(mask), scale), false, false).y;
}

// ------------------------------------------------------------------------------------------------ orthogonalised updates
Tensor orthogonalize(const Tensor &given_g, const std::vector<float> &coefficients, double eps)
{
    usable("orthogonalize", given_g);
    const int type = float_type(given_g);
    if (type < 0 || given_g.dim() < 2) refuse("orthogonalize: matrices ", given_g.sizes(), " of ", given_g.scalar_type(), "; fp32, bf16 and fp16 are supported");
    const Tensor g = given_g.detach().contiguous();
    const int m = as_int(g.size(-2), "matrices"), n = as_int(g.size(-1), "matrices");
    const int batch = as_int(c10::multiply_integers(g.sizes().slice(0, g.dim() - 2)), "a batch");
    const c10::OptionalDeviceGuard guard(g.device());
    const Tensor out = like(g, g.sizes());
    const size_t bytes = fgnn_orthogonalize_workspace_bytes(batch, m, n);
    const Tensor ws = scratch(g, bytes);
    check(fgnn_orthogonalize(batch, m, n, type, address(g), (int)coefficients.size() / 3, coefficients.data(), (float)eps, address(out), address(ws), bytes, stream_of(g)),
          "fgnn_orthogonalize");
    return out;
}

}  // namespace

PYBIND11_MODULE(_dense, m)
{
    // raised as the package's own error
    static PyObject *error = py::object(py::module_::import("ae_mlsys_gnn_amd._lib").attr("FgnnError")).release().ptr();
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Error &e) { PyErr_SetString(error, e.what()); }
    });
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_q8", &rms_norm_q8);
    m.def("quantize_rows", &quantize_rows);
    m.def("linear_act", &linear_act);
    m.def("linear_q8", &linear_q8);
    m.def("orthogonalize", &orthogonalize);
    m.def("group_norm", &group_norm);
    m.def("embedding", &embedding);
    m.def("cross_attention", &cross_attention);
}

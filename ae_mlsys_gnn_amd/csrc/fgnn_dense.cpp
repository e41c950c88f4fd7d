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
}

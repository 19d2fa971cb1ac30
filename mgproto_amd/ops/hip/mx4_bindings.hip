// Tensor entry points of the MX4 product and of gradient clipping.

#include <torch/extension.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <tuple>
#include <vector>

#include "grad_clip.h"
#include "mx4_common.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = c10::optional<Tensor>;

// A call's argument is refused as Python would refuse it.
template <class E, class... A>
void refuse_unless(bool ok, A&&... what) {
    if (!ok) throw E(c10::str(std::forward<A>(what)...));
}
#define CHECK_TYPE(ok, ...) refuse_unless<py::type_error>(ok, __VA_ARGS__)
#define CHECK_VALUE(ok, ...) refuse_unless<py::value_error>(ok, __VA_ARGS__)

// A forward-mode derivative would be dropped without a word.
void check_no_tangent(const Tensor& t, const char* what) {
    if (!t._fw_grad(0).defined()) return;
    PyErr_SetString(PyExc_NotImplementedError, c10::str(
        what, ": no forward-mode derivative").c_str());
    throw py::error_already_set();
}

int dtype_code(const Tensor& t, const char* what) {
    CHECK_TYPE(!t.is_neg(), what, ": a view that stands for its negative; "
               "resolve_neg() it first");
    switch (t.scalar_type()) {
        case at::kFloat: return mx4::F32;
        case at::kBFloat16: return mx4::BF16;
        case at::kHalf: return mx4::F16;
        default:
            throw py::type_error(c10::str(
                what, ": float32, bfloat16 or float16, not ",
                t.scalar_type()));
    }
}

at::ScalarType scalar_type(int64_t dt) {
    TORCH_CHECK(dt >= 0 && dt <= 2, "unknown type code ", dt);
    return dt == mx4::F32 ? at::kFloat : dt == mx4::BF16 ? at::kBFloat16
                                                         : at::kHalf;
}

// at::empty, past the dispatcher: small calls are bound by the host (1x512->512 4.6 us
// -> 4.2, rounding 5.0 -> 4.4)
Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
    return at::detail::empty_cuda(shape, type, like.device(), c10::nullopt);
}

// A launch that was refused raises here, instead of leaving what the memory held.
void check_launches() { C10_HIP_CHECK(hipGetLastError()); }

hipStream_t current_stream() { return at::hip::getCurrentHIPStream(); }

// [..., K] as [M, K] with contiguous rows: a view where it can be
Tensor matrix(const Tensor& x, const char* what) {
    CHECK_VALUE(x.dim() >= 1, what, ": rows, not a number");
    CHECK_VALUE(x.is_cuda(), what, ": on ", x.device(), ", not on a GPU");
    const int64_t K = x.size(-1);
    CHECK_VALUE(K < (1L << 22), what, ": rows of at most 2^22 elements");
    int64_t M = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) M *= x.size(i);
    // the products' launches: 64 rows a block in the longest ones, 2^32 threads
    CHECK_VALUE(M < (1L << 29), what, ": fewer than 2^29 rows");
    Tensor x2 = x.dim() == 2 ? x : x.reshape({M, K});
    if ((K > 1 && x2.stride(1) != 1) || (M > 1 && x2.stride(0) < K))
        x2 = x2.contiguous();
    return x2;
}

int64_t row_stride(const Tensor& x) {
    return x.size(0) > 1 ? x.stride(0) : x.size(1);
}

// the result's shape: x's, with N for the last
std::vector<int64_t> shape_of(const Tensor& x, int64_t N) {
    auto s = x.sizes().vec();
    s.back() = N;
    return s;
}

// 4-bit rows of K elements, as mx4_common.h lays them out
void check_packed(const Tensor& codes, const Tensor& scales, int64_t K,
                  const char* what) {
    TORCH_CHECK(codes.is_cuda() && codes.device() == scales.device(), what,
                ": codes and scales on one GPU");
    TORCH_CHECK(codes.scalar_type() == at::kByte &&
                    scales.scalar_type() == at::kByte, what, ": uint8");
    TORCH_CHECK(codes.dim() == 3 && scales.dim() == 3 &&
                    codes.is_contiguous() && scales.is_contiguous(), what,
                ": contiguous codes and scales");
    TORCH_CHECK(K >= 0 && K < (1L << 22) &&
                    codes.size(0) == mx4::steps_of(K) && codes.size(2) == 64 &&
                    scales.size(0) == mx4::chunks_of(K) &&
                    scales.size(2) == 16 && codes.size(1) == scales.size(1),
                what, ": codes ", codes.sizes(), " and scales ",
                scales.sizes(), " do not hold rows of ", K);
    TORCH_CHECK(((uintptr_t)codes.data_ptr() |
                 (uintptr_t)scales.data_ptr()) % 16 == 0, what,
                ": codes and scales start on 16 bytes");
}

void check_bias(const OptTensor& bias, int64_t N, const Tensor& like) {
    if (!bias.has_value()) return;
    CHECK_VALUE(bias->dim() == 1 && bias->size(0) == N, "mx4_linear: bias ",
                bias->sizes(), " for ", N, " columns");
    CHECK_VALUE(bias->device() == like.device(), "mx4_linear: input on ",
                like.device(), ", bias on ", bias->device());
}

Tensor workspace(size_t bytes, const Tensor& like) {
    return fresh({(int64_t)std::max<size_t>(bytes, 1)}, at::kByte, like);
}

struct Packed {               // room for the blocks of a matrix
    Tensor codes, scales;
    explicit Packed(const Tensor& x2) {
        const int64_t R = x2.size(0), K = x2.size(1);
        codes = fresh({mx4::steps_of(K), R, 64}, at::kByte, x2);
        scales = fresh({mx4::chunks_of(K), R, 16}, at::kByte, x2);
    }
};

Packed pack(const Tensor& x2, int dt) {
    const int64_t R = x2.size(0), K = x2.size(1);
    Packed p(x2);
    mx4::quantize(x2.data_ptr(), dt, R, K, row_stride(x2),
                  p.codes.data_ptr<uint8_t>(), p.scales.data_ptr<uint8_t>(),
                  current_stream());
    check_launches();
    return p;
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x) {
    const int dt = dtype_code(x, "mx4_quantize");
    const Tensor x2 = matrix(x, "mx4_quantize");
    c10::DeviceGuard guard(x2.device());
    Packed p = pack(x2, dt);
    return {p.codes, p.scales};
}

Tensor dequantize(const Tensor& codes, const Tensor& scales, int64_t K,
                  int64_t dt) {
    check_packed(codes, scales, K, "mx4_dequantize");
    c10::DeviceGuard guard(codes.device());
    auto out = fresh({codes.size(1), K}, scalar_type(dt), codes);
    mx4::dequantize(codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                    codes.size(1), K, out.data_ptr(), (int)dt,
                    current_stream());
    check_launches();
    return out;
}

// The form that is asked for, or the chosen one. A launch has 2^32 threads at
// most: forms of small blocks have 256 (512) for each 16 x 16 or 32 x 32 results, the
// one that rounds on the way for 64 rows of 64 to 256 columns; tiles take turns.
int pick(int64_t form, int chosen, int64_t M, int64_t N) {
    CHECK_VALUE(form >= -1 && form < mx4::FORMS, "mx4_linear: no form ", form);
    const int f = form < 0 ? chosen : (int)form;
    int64_t rows = 128, cols = 128, most = 1L << 30;
    if (f == mx4::ROWS16 || f == mx4::HELD16) rows = cols = 16, most = 1L << 23;
    else if (f == mx4::ROWS32 || f == mx4::HELD32) rows = cols = 32, most = 1L << 24;
    else if (f == mx4::ROUNDING) rows = 64, cols = N > 128 ? 256 : 64, most = 1L << 23;
    CHECK_VALUE((M + rows - 1) / rows * ((N + cols - 1) / cols) < most,
                "mx4_linear: ", M, " x ", N, " results are too many");
    return f;
}

struct Bias {            // contiguous, and its type
    Tensor t;
    int dt = 0;
    explicit Bias(const OptTensor& b) {
        if (!b.has_value()) return;
        dt = dtype_code(*b, "mx4_linear: bias");
        t = b->contiguous();
    }
    const void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};

// Q(x) W^T + bias with held weights, no gradient
Tensor linear(const Tensor& x, const Tensor& wc, const Tensor& ws, int64_t K,
              const OptTensor& bias, int64_t form) {
    const int dt = dtype_code(x, "mx4_linear: input");
    const Tensor x2 = matrix(x, "mx4_linear: input");
    const int64_t M = x2.size(0), N = wc.size(1);
    CHECK_VALUE(x2.size(1) == K, "mx4_linear: input ", x.sizes(),
                " and weight [", N, ", ", K, "] do not match");
    CHECK_VALUE(x.device() == wc.device(), "mx4_linear: input on ", x.device(),
                ", weight on ", wc.device());
    check_packed(wc, ws, K, "mx4_linear: weight");
    check_bias(bias, N, x);
    c10::DeviceGuard guard(x.device());
    auto y = fresh(shape_of(x, N), x.scalar_type(), x);
    if (!M || !N) return y;
    const Bias b(bias);
    const int64_t ldx = row_stride(x2);
    const int f = pick(form, mx4::linear_form(M, K, N), M, N);
    Tensor work;
    if (const size_t bytes = mx4::linear_bytes(f, M, K))
        work = workspace(bytes, x);
    mx4::linear(x2.data_ptr(), dt, M, K, ldx, wc.data_ptr<uint8_t>(),
                ws.data_ptr<uint8_t>(), N, b.ptr(), b.dt, y.data_ptr(), f,
                work.defined() ? work.data_ptr() : nullptr, current_stream());
    check_launches();
    return y;
}

Tensor product_q(const Tensor& xc, const Tensor& xs, int64_t K,
                 const Tensor& wc, const Tensor& ws, const OptTensor& bias,
                 std::vector<int64_t> shape, int dt, int64_t form) {
    const int64_t M = xc.size(1), N = wc.size(1);
    check_bias(bias, N, xc);
    auto y = fresh(shape, scalar_type(dt), xc);
    if (!M || !N) return y;
    const Bias b(bias);
    const int chosen = mx4::linear_q_form(M, K, N);
    const int f = pick(form < 0 || form >= mx4::HELD16 ? form : chosen, chosen, M, N);
    mx4::linear_q(xc.data_ptr<uint8_t>(), xs.data_ptr<uint8_t>(), M, K,
                  wc.data_ptr<uint8_t>(), ws.data_ptr<uint8_t>(), N, b.ptr(),
                  b.dt, y.data_ptr(), dt, f, current_stream());
    check_launches();
    return y;
}

// the same from rows held in 4 bits
Tensor linear_q(const Tensor& xc, const Tensor& xs, int64_t K,
                const Tensor& wc, const Tensor& ws, const OptTensor& bias,
                int64_t dt, int64_t form) {
    check_packed(xc, xs, K, "mx4_linear: input");
    check_packed(wc, ws, K, "mx4_linear: weight");
    CHECK_VALUE(xc.device() == wc.device(), "mx4_linear: one GPU for all");
    scalar_type(dt);
    c10::DeviceGuard guard(xc.device());
    return product_q(xc, xs, K, wc, ws, bias, {xc.size(1), wc.size(1)}, (int)dt,
                     form);
}

// Q(x) Q(w)^T + bias, and what its gradients want of it
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> linear_train(
        const Tensor& x, const Tensor& w, const OptTensor& bias) {
    const int dt = dtype_code(x, "mx4_linear: input");
    const int wdt = dtype_code(w, "mx4_linear: weight");
    const Tensor x2 = matrix(x, "mx4_linear: input");
    const int64_t K = x2.size(1);
    CHECK_VALUE(w.dim() == 2 && w.size(1) == K, "mx4_linear: input ",
                x.sizes(), " and weight ", w.sizes(), " do not match");
    CHECK_VALUE(x.device() == w.device(), "mx4_linear: input on ", x.device(),
                ", weight on ", w.device());
    c10::DeviceGuard guard(x.device());
    const Tensor w2 = matrix(w, "mx4_linear: weight");
    Packed pw(w2), px(x2);
    mx4::quantize_two(
        w2.data_ptr(), wdt, w2.size(0), row_stride(w2),
        pw.codes.data_ptr<uint8_t>(), pw.scales.data_ptr<uint8_t>(),
        x2.data_ptr(), dt, x2.size(0), row_stride(x2),
        px.codes.data_ptr<uint8_t>(), px.scales.data_ptr<uint8_t>(), K,
        current_stream());
    check_launches();
    Tensor y = product_q(px.codes, px.scales, K, pw.codes, pw.scales, bias,
                         shape_of(x, w.size(0)), dt, -1);
    return {y, px.codes, px.scales, pw.codes, pw.scales};
}

// Gradients of the product: to the input (type dx_dt) where weights are given,
// to the weight (dw_dt) where rows are, to the bias (db_dt); -1 leaves one out.
std::tuple<OptTensor, OptTensor, OptTensor> linear_backward(
        const Tensor& grad, const OptTensor& wc, const OptTensor& ws,
        const OptTensor& xc, const OptTensor& xs, int64_t K, int64_t dx_dt,
        int64_t dw_dt, int64_t db_dt, int64_t form) {
    CHECK_VALUE(grad.is_cuda() && grad.dim() >= 1,
                "mx4_linear: output gradient: rows on the GPU");
    CHECK_VALUE(form >= -1 && form < mx4::GRAD_FORMS, "mx4_linear: no form ",
                form);
    mx4::GradArgs a{};
    a.g_dt = dtype_code(grad, "mx4_linear: output gradient");
    a.N = grad.size(-1), a.M = 1, a.K = K;
    for (int64_t i = 0; i + 1 < grad.dim(); ++i) a.M *= grad.size(i);
    CHECK_VALUE(a.M < (1L << 29) && a.N < (1L << 22) && K >= 0 &&
                    K < (1L << 22), "mx4_linear: output gradient: too large");
    if (dx_dt >= 0) {
        CHECK_VALUE(wc.has_value() && ws.has_value(),
                    "mx4_linear: no weight for the input's gradient");
        check_packed(*wc, *ws, K, "mx4_linear: weight");
        CHECK_VALUE(wc->size(1) == a.N && grad.device() == wc->device(),
                    "mx4_linear: output gradient does not match the weight");
        a.wc = wc->data_ptr<uint8_t>(), a.ws = ws->data_ptr<uint8_t>();
    }
    if (dw_dt >= 0) {
        CHECK_VALUE(xc.has_value() && xs.has_value(),
                    "mx4_linear: no rows for the weight's gradient");
        check_packed(*xc, *xs, K, "mx4_linear: input");
        CHECK_VALUE(xc->size(1) == a.M && grad.device() == xc->device(),
                    "mx4_linear: output gradient does not match the input");
        a.xc = xc->data_ptr<uint8_t>(), a.xs = xs->data_ptr<uint8_t>();
    }
    c10::DeviceGuard guard(grad.device());
    const Tensor g = grad.contiguous();
    OptTensor dx, dw, db;
    // a sum over nothing is 0
    auto make = [&](std::vector<int64_t> shape, int64_t dt, int64_t over,
                    OptTensor& t, void*& ptr, int& code) {
        if (dt < 0) return;
        t = fresh(shape, scalar_type(dt), g);
        code = (int)dt;
        if (!t->numel()) return;
        if (over) ptr = t->data_ptr();
        else t->zero_();
    };
    make(shape_of(grad, K), dx_dt, a.N, dx, a.dx, a.dx_dt);
    make({a.N, K}, dw_dt, a.M, dw, a.dw, a.dw_dt);
    make({a.N}, db_dt, a.M, db, a.db, a.db_dt);
    if (!a.dx && !a.dw && !a.db) return {dx, dw, db};
    a.K = std::max<int64_t>(K, 1);        // only db is left where K is 0
    a.g = g.data_ptr();
    a.aligned = (uintptr_t)a.g % 16 == 0;
    Tensor work;
    if (const size_t bytes = mx4::grads_bytes(a, (int)form))
        work = workspace(bytes, g);
    mx4::grads(a, (int)form, work.defined() ? work.data_ptr() : nullptr,
               current_stream());
    check_launches();
    return {dx, dw, db};
}

// The differentiable product. The node is native: a small layer's step is
// bound by the host, and a Python node costs it twice what this one does.
// The weight is w, or held in 4 bits (wc, ws).
struct LinearNode : public torch::autograd::Function<LinearNode> {
    using Context = torch::autograd::AutogradContext;
    using List = torch::autograd::variable_list;

    static Tensor forward(Context* ctx, const Tensor& x, const OptTensor& w,
                          const OptTensor& bias, const OptTensor& wc,
                          const OptTensor& ws, int64_t K) {
        const bool need_x = x.requires_grad();
        const bool need_w = w.has_value() && w->requires_grad();
        const bool need_b = bias.has_value() && bias->requires_grad();
        Tensor y, xc, xs, c = wc.value_or(Tensor()), s = ws.value_or(Tensor());
        if (need_w) {        // the rounded rows are kept, a quarter of bf16
            std::tie(y, xc, xs, c, s) = linear_train(x, *w, bias);
        } else {
            if (w.has_value()) std::tie(c, s) = quantize(*w);
            y = linear(x, c, s, K, bias, -1);
        }
        if (!need_x) c = s = Tensor();
        ctx->save_for_backward({c, s, xc, xs});
        auto code = [](const Tensor& t) {
            return (int64_t)dtype_code(t, "mx4_linear");
        };
        ctx->saved_data["K"] = K;
        ctx->saved_data["types"] = std::vector<int64_t>{
            need_x ? code(x) : -1, need_w ? code(*w) : -1,
            need_b ? code(*bias) : -1};
        return y;
    }

    static List backward(Context* ctx, List grads) {
        const bool again = at::GradMode::is_enabled() &&
                           grads[0].requires_grad();
        const List t = ctx->get_saved_variables();
        const auto types = ctx->saved_data["types"].toIntVector();
        List out(6);
        {
            at::AutoGradMode off(false);
            const auto [dx, dw, db] = linear_backward(
                grads[0].resolve_neg(), t[0], t[1], t[2], t[3],
                ctx->saved_data["K"].toInt(), types[0], types[1], types[2], -1);
            out[0] = dx.value_or(Tensor());
            out[1] = dw.value_or(Tensor());
            out[2] = db.value_or(Tensor());
        }
        if (again) {         // a second derivative is refused where it is taken
            for (auto& d : out) {
                if (!d.defined()) continue;
                auto refuse = std::make_shared<torch::autograd::DelayedError>(
                    "mx4_linear is differentiable once", 1);
                d = (*refuse)(List{d.detach().set_requires_grad(true)})[0];
            }
        }
        return out;
    }
};

bool needs_grad(const Tensor& x, const OptTensor& w, const OptTensor& bias) {
    check_no_tangent(x, "mx4_linear: input");
    if (w.has_value()) check_no_tangent(*w, "mx4_linear: weight");
    if (bias.has_value()) check_no_tangent(*bias, "mx4_linear: bias");
    return at::GradMode::is_enabled() &&
           (x.requires_grad() || (w.has_value() && w->requires_grad()) ||
            (bias.has_value() && bias->requires_grad()));
}

// Q(x) W^T + bias, held weights
Tensor linear_held(const Tensor& x, const Tensor& wc, const Tensor& ws,
                   int64_t K, const OptTensor& bias, int64_t form) {
    if (needs_grad(x, c10::nullopt, bias) && form < 0)
        return LinearNode::apply(x, c10::nullopt, bias, wc, ws, K);
    return linear(x, wc, ws, K, bias, form);
}

// Q(x) Q(w)^T + bias, a float weight
Tensor linear_float(const Tensor& x, const Tensor& w, const OptTensor& bias) {
    dtype_code(x, "mx4_linear: input");
    dtype_code(w, "mx4_linear: weight");
    CHECK_VALUE(x.dim() >= 1, "mx4_linear: input: rows, not a number");
    CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(-1), "mx4_linear: input ",
                x.sizes(), " and weight ", w.sizes(), " do not match");
    CHECK_VALUE(x.device() == w.device(), "mx4_linear: input on ", x.device(),
                ", weight on ", w.device());
    check_bias(bias, w.size(0), x);
    if (needs_grad(x, w, bias))
        return LinearNode::apply(x, w, bias, c10::nullopt, c10::nullopt,
                                 x.size(-1));
    const auto [c, s] = quantize(w);
    return linear(x, c, s, x.size(-1), bias, -1);
}

// ---------------------------------------------------------------------------
// gradient clipping
// ---------------------------------------------------------------------------

void check_list(const std::vector<Tensor>& ts, const char* what) {
    for (const auto& t : ts) {
        CHECK_TYPE(t.layout() == at::kStrided, what, ": dense tensors, not ",
                   t.layout());
        CHECK_VALUE(t.device() == ts[0].device(), what, ": tensors on ",
                    ts[0].device(), " and ", t.device());
        CHECK_VALUE(t.is_cuda(), what, ": on ", t.device(), ", not on a GPU");
        check_no_tangent(t, what);
        dtype_code(t, what);
    }
}

// the end of a tensor's memory; gaps count
uintptr_t end_of(const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return (uintptr_t)t.data_ptr() + (last + 1) * t.element_size();
}

// A written tensor may share memory with no other one, but for its own source
// within its own place, in the same type.
void check_apart(const std::vector<Tensor>& grads, const std::vector<Tensor>& outs) {
    struct Span { uintptr_t lo, hi; size_t i; bool out; };
    std::vector<Span> s;
    s.reserve(grads.size() * 2);
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor &g = grads[i], &o = outs[i];
        if (!o.numel()) continue;
        const uintptr_t lo = (uintptr_t)o.data_ptr(), hi = end_of(o);
        s.push_back({lo, hi, i, true});
        if ((uintptr_t)g.data_ptr() != lo || g.scalar_type() != o.scalar_type() ||
            end_of(g) > hi)
            s.push_back({(uintptr_t)g.data_ptr(), end_of(g), i, false});
    }
    std::sort(s.begin(), s.end(),
              [](const Span& a, const Span& b) { return a.lo < b.lo; });
    uintptr_t any = 0, out = 0;          // ends of what came before
    for (const auto& e : s) {
        TORCH_CHECK(!(e.lo < out || (e.out && e.lo < any)),
                    "clip_grads_: a tensor that is written shares memory with "
                    "another one (number ", e.i, ")");
        any = std::max(any, e.hi);
        if (e.out) out = std::max(out, e.hi);
    }
}

int norm_kind(double p) {
    if (p == 2.0) return gradclip::L2;
    if (p == 1.0) return gradclip::L1;
    CHECK_VALUE(std::isinf(p) && p > 0, "norm_type: 1, 2 or inf, not ", p);
    return gradclip::LINF;
}

Tensor grad_norm(const std::vector<Tensor>& grads, double p) {
    const int kind = norm_kind(p);
    TORCH_CHECK(!grads.empty(), "grad_norm: an empty list");
    check_list(grads, "grad_norm");
    c10::DeviceGuard guard(grads[0].device());
    std::vector<gradclip::Item> items;
    std::vector<Tensor> kept;
    items.reserve(grads.size());
    for (const auto& t : grads) {
        Tensor c = t;
        if (!t.is_non_overlapping_and_dense()) {
            c = t.contiguous();
            kept.push_back(c);
        }
        const int dt = dtype_code(c, "grad_norm");
        items.push_back({c.data_ptr(), nullptr, c.numel(), dt, dt});
    }
    auto norm = fresh({}, at::kFloat, grads[0]);
    const gradclip::List list(items);
    auto work = fresh({(int64_t)list.workspace_doubles()}, at::kDouble, norm);
    list.norm(kind, norm.data_ptr<float>(), work.data_ptr<double>(),
              current_stream());
    check_launches();
    return norm;
}

Tensor clip_grads(const std::vector<Tensor>& grads,
                  const std::vector<Tensor>& outs, double max_norm, double p) {
    const int kind = norm_kind(p);
    TORCH_CHECK(!grads.empty(), "clip_grads_: an empty list");
    CHECK_VALUE(max_norm >= 0, "clip_grads_: max_norm ", max_norm);
    CHECK_VALUE(grads.size() == outs.size(), "clip_grads_: ", grads.size(),
                " gradients, ", outs.size(), " outputs");
    check_list(grads, "clip_grads_");
    check_list(outs, "clip_grads_: out");
    CHECK_VALUE(grads[0].device() == outs[0].device(),
                "clip_grads_: gradients on ", grads[0].device(), ", out on ",
                outs[0].device());
    c10::DeviceGuard guard(grads[0].device());
    std::vector<gradclip::Item> items;
    std::vector<Tensor> kept;
    items.reserve(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor &g = grads[i], &o = outs[i];
        CHECK_VALUE(g.sizes() == o.sizes(), "clip_grads_: out ", o.sizes(),
                    " for a gradient ", g.sizes());
        TORCH_CHECK(o.is_non_overlapping_and_dense(), "clip_grads_: tensor ",
                    i, " is written and has gaps or shares elements with "
                    "itself");
        Tensor src = g;
        if (g.strides() != o.strides()) {    // laid out as the output is
            src = at::empty_like(o, o.options().dtype(g.scalar_type()));
            src.copy_(g);
            kept.push_back(src);
        }
        items.push_back({src.data_ptr(), o.data_ptr(), src.numel(),
                         dtype_code(g, "clip_grads_"),
                         dtype_code(o, "clip_grads_: out")});
    }
    check_apart(grads, outs);
    auto norm = fresh({}, at::kFloat, grads[0]);
    const gradclip::List list(items);
    auto work = fresh({(int64_t)list.workspace_doubles()}, at::kDouble, norm);
    list.clip(kind, max_norm, norm.data_ptr<float>(), work.data_ptr<double>(),
              current_stream());
    check_launches();
    for (const auto& o : outs)           // written behind autograd's back
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    return norm;
}

}  // namespace

void register_mx4(pybind11::module& m) {
    m.def("mx4_quantize", &quantize, "rows to MX4 codes and scales");
    m.def("mx4_dequantize", &dequantize, "MX4 codes and scales to values");
    m.def("mx4_linear", &linear_held, "Q(x) W^T + bias", py::arg("x"),
          py::arg("codes"), py::arg("scales"), py::arg("K"), py::arg("bias"),
          py::arg("form") = -1);
    m.def("mx4_linear_q", &linear_q, "X W^T + bias from 4-bit rows",
          py::arg("xcodes"), py::arg("xscales"), py::arg("K"),
          py::arg("codes"), py::arg("scales"), py::arg("bias"),
          py::arg("dtype"), py::arg("form") = -1);
    m.def("mx4_linear_float", &linear_float, "Q(x) Q(w)^T + bias");
    m.def("mx4_linear_backward", &linear_backward,
          "gradients to the input, the weight and the bias", py::arg("grad"),
          py::arg("codes"), py::arg("scales"), py::arg("xcodes"),
          py::arg("xscales"), py::arg("K"), py::arg("dx_dtype"),
          py::arg("dw_dtype"), py::arg("db_dtype"), py::arg("form") = -1);
    m.def("grad_norm", &grad_norm, "global norm of a list of tensors");
    m.def("clip_grads", &clip_grads,
          "a list scaled to a global norm of at most max_norm; returns the norm");
}

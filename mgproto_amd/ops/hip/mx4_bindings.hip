// Tensor entry points of the MX4 product and of gradient clipping.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <tuple>
#include <vector>

#include "grad_clip.h"
#include "mx4_common.h"

namespace {

using at::Tensor;

int dtype_code(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return mx4::F32;
        case at::kBFloat16: return mx4::BF16;
        case at::kHalf: return mx4::F16;
        default:
            TORCH_CHECK(false, what, ": float32, bfloat16 or float16, not ",
                        t.scalar_type());
    }
}

at::ScalarType scalar_type(int64_t dt) {
    TORCH_CHECK(dt >= 0 && dt <= 2, "unknown type code ", dt);
    return dt == mx4::F32 ? at::kFloat : dt == mx4::BF16 ? at::kBFloat16
                                                         : at::kHalf;
}

hipStream_t current_stream() { return at::hip::getCurrentHIPStream(); }

// rows of elements next to each other, at any distance
void check_rows(const Tensor& x, const char* what) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2, what, ": a matrix on the GPU");
    TORCH_CHECK(x.size(1) <= 1 || x.stride(1) == 1, what,
                ": rows must be contiguous");
    TORCH_CHECK(x.size(1) < (1L << 30), what, ": rows too long");
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

void check_bias(const c10::optional<Tensor>& bias, int64_t N,
                const Tensor& like) {
    if (!bias.has_value()) return;
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N &&
                    bias->is_contiguous() && bias->device() == like.device(),
                "bias: contiguous, ", N, " values, on the same GPU");
}

Tensor workspace(size_t bytes, const Tensor& like) {
    return at::empty({(int64_t)std::max<size_t>(bytes, 1)},
                     like.options().dtype(at::kByte));
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x) {
    check_rows(x, "mx4_quantize");
    const int dt = dtype_code(x, "mx4_quantize");
    c10::DeviceGuard guard(x.device());
    const int64_t R = x.size(0), K = x.size(1);
    auto opt = x.options().dtype(at::kByte);
    auto codes = at::empty({mx4::steps_of(K), R, 64}, opt);
    auto scales = at::empty({mx4::chunks_of(K), R, 16}, opt);
    mx4::quantize(x.data_ptr(), dt, R, K, R > 1 ? x.stride(0) : K,
                  codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                  current_stream());
    return {codes, scales};
}

Tensor dequantize(const Tensor& codes, const Tensor& scales, int64_t K,
                  int64_t dt) {
    check_packed(codes, scales, K, "mx4_dequantize");
    c10::DeviceGuard guard(codes.device());
    auto out = at::empty({codes.size(1), K},
                         codes.options().dtype(scalar_type(dt)));
    mx4::dequantize(codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                    codes.size(1), K, out.data_ptr(), (int)dt,
                    current_stream());
    return out;
}

// what one tile of 16 x 16 a block can number
void check_tiles(int64_t M, int64_t N) {
    TORCH_CHECK((M + 15) / 16 * ((N + 15) / 16) < (1L << 31),
                "mx4_linear: ", M, " x ", N, " results are too many");
}

int pick(int64_t form, int chosen) {
    TORCH_CHECK(form >= -1 && form < mx4::FORMS, "mx4_linear: no form ", form);
    return form < 0 ? chosen : (int)form;
}

Tensor linear(const Tensor& x, const Tensor& wc, const Tensor& ws,
              const c10::optional<Tensor>& bias, int64_t form) {
    check_rows(x, "mx4_linear: input");
    const int64_t M = x.size(0), K = x.size(1), N = wc.size(1);
    check_packed(wc, ws, K, "mx4_linear: weight");
    TORCH_CHECK(x.device() == wc.device(), "mx4_linear: one GPU for all");
    check_bias(bias, N, x);
    const int dt = dtype_code(x, "mx4_linear: input");
    c10::DeviceGuard guard(x.device());
    check_tiles(M, N);
    auto y = at::empty({M, N}, x.options());
    if (!M || !N) return y;
    const int64_t ldx = M > 1 ? x.stride(0) : K;
    const bool aligned = (uintptr_t)x.data_ptr() % 16 == 0 &&
                         ldx * x.element_size() % 16 == 0;
    const int f = pick(form, mx4::linear_form(M, K, N, dt, aligned));
    Tensor work;
    if (const size_t bytes = mx4::linear_bytes(f, M, K))
        work = workspace(bytes, x);
    mx4::linear(x.data_ptr(), dt, M, K, ldx, wc.data_ptr<uint8_t>(),
                ws.data_ptr<uint8_t>(), N, bias ? bias->data_ptr() : nullptr,
                bias ? dtype_code(*bias, "mx4_linear: bias") : 0, y.data_ptr(),
                f, work.defined() ? work.data_ptr() : nullptr,
                current_stream());
    return y;
}

Tensor linear_q(const Tensor& xc, const Tensor& xs, int64_t K,
                const Tensor& wc, const Tensor& ws,
                const c10::optional<Tensor>& bias, int64_t dt, int64_t form) {
    check_packed(xc, xs, K, "mx4_linear: input");
    check_packed(wc, ws, K, "mx4_linear: weight");
    TORCH_CHECK(xc.device() == wc.device(), "mx4_linear: one GPU for all");
    const int64_t M = xc.size(1), N = wc.size(1);
    check_bias(bias, N, xc);
    c10::DeviceGuard guard(xc.device());
    check_tiles(M, N);
    auto y = at::empty({M, N}, xc.options().dtype(scalar_type(dt)));
    if (M && N)
        mx4::linear_q(xc.data_ptr<uint8_t>(), xs.data_ptr<uint8_t>(), M, K,
                      wc.data_ptr<uint8_t>(), ws.data_ptr<uint8_t>(), N,
                      bias ? bias->data_ptr() : nullptr,
                      bias ? dtype_code(*bias, "mx4_linear: bias") : 0,
                      y.data_ptr(), (int)dt,
                      pick(form, mx4::linear_q_form(M, K, N)),
                      current_stream());
    return y;
}

void check_grad(const Tensor& g) {
    TORCH_CHECK(g.is_cuda() && g.dim() == 2 && g.is_contiguous(),
                "mx4_linear: output gradient: a contiguous matrix on the GPU");
    TORCH_CHECK(g.size(0) < (1L << 31) && g.size(1) < (1L << 30),
                "mx4_linear: output gradient: too large");
}

Tensor grad_input(const Tensor& g, const Tensor& wc, const Tensor& ws,
                  int64_t K, int64_t dt) {
    check_grad(g);
    check_packed(wc, ws, K, "mx4_linear: weight");
    const int64_t M = g.size(0), N = g.size(1);
    TORCH_CHECK(wc.size(1) == N && g.device() == wc.device(),
                "mx4_linear: output gradient does not match the weight");
    const int gd = dtype_code(g, "mx4_linear: output gradient");
    c10::DeviceGuard guard(g.device());
    auto dx = at::empty({M, K}, g.options().dtype(scalar_type(dt)));
    if (!M || !K) return dx;
    if (!N) return dx.zero_();
    const bool aligned = (uintptr_t)g.data_ptr() % 16 == 0;
    auto work = workspace(mx4::grad_input_bytes(M, N, K, gd, aligned), g);
    mx4::grad_input(g.data_ptr(), gd, aligned, M, N, K,
                    wc.data_ptr<uint8_t>(), ws.data_ptr<uint8_t>(),
                    dx.data_ptr(), (int)dt, work.data_ptr(), current_stream());
    return dx;
}

Tensor grad_weight(const Tensor& g, const Tensor& xc, const Tensor& xs,
                   int64_t K, int64_t dt) {
    check_grad(g);
    check_packed(xc, xs, K, "mx4_linear: input");
    const int64_t M = g.size(0), N = g.size(1);
    TORCH_CHECK(xc.size(1) == M && g.device() == xc.device(),
                "mx4_linear: output gradient does not match the input");
    const int gd = dtype_code(g, "mx4_linear: output gradient");
    c10::DeviceGuard guard(g.device());
    auto dw = at::empty({N, K}, g.options().dtype(scalar_type(dt)));
    if (!N || !K) return dw;
    if (!M) return dw.zero_();
    auto work = workspace(mx4::grad_weight_bytes(M, N, K, gd), g);
    mx4::grad_weight(g.data_ptr(), gd, M, N, K, xc.data_ptr<uint8_t>(),
                     xs.data_ptr<uint8_t>(), dw.data_ptr(), (int)dt,
                     work.data_ptr(), current_stream());
    return dw;
}

Tensor col_sum(const Tensor& g, int64_t dt) {
    check_grad(g);
    const int64_t M = g.size(0), N = g.size(1);
    const int gd = dtype_code(g, "mx4_linear: output gradient");
    c10::DeviceGuard guard(g.device());
    auto out = at::empty({N}, g.options().dtype(scalar_type(dt)));
    if (!N) return out;
    if (!M) return out.zero_();
    auto work = workspace(mx4::col_sum_bytes(M, N), g);
    mx4::col_sum(g.data_ptr(), gd, M, N, out.data_ptr(), (int)dt,
                 work.data_ptr(), current_stream());
    return out;
}

// ---------------------------------------------------------------------------
// gradient clipping
// ---------------------------------------------------------------------------

void check_list(const std::vector<Tensor>& ts, const char* what) {
    for (const auto& t : ts) {
        TORCH_CHECK(t.layout() == at::kStrided && t.is_cuda(), what,
                    ": dense tensors on the GPU");
        TORCH_CHECK(t.device() == ts[0].device(), what, ": one GPU for all");
        dtype_code(t, what);
    }
}

// A written tensor may share memory with no other one, but for its own source
// in the same place and of the same type.
void check_apart(const std::vector<gradclip::Item>& items) {
    struct Span { uintptr_t lo, hi; size_t i; bool out; };
    std::vector<Span> s;
    s.reserve(items.size() * 2);
    auto width = [](int dt) { return dt == mx4::F32 ? 4 : 2; };
    for (size_t i = 0; i < items.size(); ++i) {
        const auto& it = items[i];
        if (!it.n) continue;
        s.push_back({(uintptr_t)it.dst,
                     (uintptr_t)it.dst + it.n * width(it.dst_dt), i, true});
        if (it.src != it.dst || it.src_dt != it.dst_dt)
            s.push_back({(uintptr_t)it.src,
                         (uintptr_t)it.src + it.n * width(it.src_dt), i, false});
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
    TORCH_CHECK(std::isinf(p) && p > 0, "norm_type: 1, 2 or inf, not ", p);
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
    auto norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    auto work = at::empty({(int64_t)gradclip::workspace_doubles(items)},
                          norm.options().dtype(at::kDouble));
    gradclip::norm(items, kind, 0.0, norm.data_ptr<float>(),
                   work.data_ptr<double>(), current_stream());
    return norm;
}

Tensor clip_grads(const std::vector<Tensor>& grads,
                  const std::vector<Tensor>& outs, double max_norm, double p) {
    const int kind = norm_kind(p);
    TORCH_CHECK(!grads.empty(), "clip_grads_: an empty list");
    TORCH_CHECK(max_norm >= 0, "clip_grads_: max_norm is negative or NaN");
    TORCH_CHECK(grads.size() == outs.size(), "clip_grads_: ", grads.size(),
                " gradients, ", outs.size(), " outputs");
    check_list(grads, "clip_grads_");
    check_list(outs, "clip_grads_: out");
    TORCH_CHECK(grads[0].device() == outs[0].device(),
                "clip_grads_: one GPU for all");
    c10::DeviceGuard guard(grads[0].device());
    std::vector<gradclip::Item> items;
    std::vector<Tensor> kept;
    items.reserve(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor &g = grads[i], &o = outs[i];
        TORCH_CHECK(g.sizes() == o.sizes(), "clip_grads_: out ", i,
                    " has another shape");
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
    check_apart(items);
    auto norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    auto work = at::empty({(int64_t)gradclip::workspace_doubles(items)},
                          norm.options().dtype(at::kDouble));
    const hipStream_t stream = current_stream();
    gradclip::norm(items, kind, max_norm, norm.data_ptr<float>(),
                   work.data_ptr<double>(), stream);
    gradclip::scale(items, work.data_ptr<double>(), stream);
    return norm;
}

}  // namespace

void register_mx4(pybind11::module& m) {
    m.def("mx4_quantize", &quantize, "rows to MX4 codes and scales");
    m.def("mx4_dequantize", &dequantize, "MX4 codes and scales to values");
    namespace py = pybind11;
    m.def("mx4_linear", &linear, "Q(x) W^T + bias", py::arg("x"),
          py::arg("codes"), py::arg("scales"), py::arg("bias"),
          py::arg("form") = -1);
    m.def("mx4_linear_q", &linear_q, "X W^T + bias from 4-bit rows",
          py::arg("xcodes"), py::arg("xscales"), py::arg("K"),
          py::arg("codes"), py::arg("scales"), py::arg("bias"),
          py::arg("dtype"), py::arg("form") = -1);
    m.def("mx4_grad_input", &grad_input, "g W");
    m.def("mx4_grad_weight", &grad_weight, "g^T X");
    m.def("col_sum", &col_sum, "column sums of a matrix");
    m.def("grad_norm", &grad_norm, "global norm of a list of tensors");
    m.def("clip_grads", &clip_grads,
          "a list scaled to a global norm of at most max_norm; returns the norm");
}

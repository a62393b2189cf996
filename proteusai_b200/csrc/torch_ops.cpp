// The PyTorch side of the feed-forward products: argument checks, buffers and autograd nodes around the C entry points pai_linear_* and
// pai_gated_* of libproteus_b200.so, whose addresses the Python loader hands over (bind): this module links no kernel.
//
// It is C++ because small products are bound by the host: with autograd nodes in Python a small forward + backward took 119 us of the host and a
// forward pass alone 12.3; here 77 and 6.
#include <ATen/autocast_mode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <string>

#include "../../include/proteus_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&pai_status_str) status_str;
    decltype(&pai_dense_saved_bytes) saved_bytes;
    decltype(&pai_dense_bwd_workspace_bytes) workspace_bytes;
    decltype(&pai_linear_fwd) linear_fwd;
    decltype(&pai_gated_fwd) gated_fwd;
    decltype(&pai_linear_bwd) linear_bwd;
    decltype(&pai_gated_bwd) gated_bwd;
    decltype(&pai_copy_rows16) copy_rows;
} api;

void bind(const std::map<std::string, uintptr_t> &at) {
    auto set = [&](auto &fn, const char *name) { fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(at.at(name)); };
    set(api.status_str, "pai_status_str");
    set(api.saved_bytes, "pai_dense_saved_bytes");
    set(api.workspace_bytes, "pai_dense_bwd_workspace_bytes");
    set(api.linear_fwd, "pai_linear_fwd");
    set(api.gated_fwd, "pai_gated_fwd");
    set(api.linear_bwd, "pai_linear_bwd");
    set(api.gated_bwd, "pai_gated_bwd");
    set(api.copy_rows, "pai_copy_rows16");
}

void check(int status, const char *what) { TORCH_CHECK(status == 0, what, " failed: ", api.status_str(status), " (status ", status, ")"); }

void *address(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
int dtype_of(const Tensor &t) { return t.scalar_type() == at::kHalf ? PAI_FP16 : PAI_BF16; }
int is_fp32(const Tensor &b) { return b.defined() && b.scalar_type() == at::kFloat; }
void *stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
Tensor bytes(size_t n, const Tensor &like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

// t [rows, cols], or a copy, with contiguous columns and rows that do not overlap
Tensor whole_rows(const Tensor &t) {
    if ((t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= t.size(1) || t.size(0) == 1)) return t;
    return t.contiguous();
}

// The products' operands as they are read: 16-byte aligned rows.  Those whose rows are not (odd widths, odd offsets) lie as copies in `copies`, one
// buffer and one launch for all; `copies` of the forward pass serves the backward pass.
struct Operands {
    const void *p[3];
    int64_t ld[3];
    Tensor copies;

    Operands(std::initializer_list<Tensor> ts, const Tensor &kept = Tensor()) : copies(kept) {
        const void *src[3];
        void *dst[3];
        int64_t ld_src[3], ld_dst[3];
        long long rows[3];
        int cols[3], n = 0, i = 0;
        int64_t elements = 0;
        for (const Tensor &t : ts) {
            p[i] = t.defined() ? t.data_ptr() : nullptr, ld[i] = t.defined() ? t.stride(0) : 0;
            if (t.defined() && t.size(0) > 0 && (((uintptr_t)p[i] & 15) != 0 || ((ld[i] & 7) != 0 && t.size(0) > 1))) {
                src[n] = p[i], ld_src[n] = ld[i], rows[n] = t.size(0), cols[n] = (int)t.size(1);
                ld_dst[n] = (t.size(1) + 7) / 8 * 8;
                dst[n] = reinterpret_cast<void *>(elements * 2);  // (offset until the buffer is there)
                p[i] = nullptr, ld[i] = n++;
                elements += t.size(0) * ld_dst[n - 1];
            }
            ++i;
        }
        if (n == 0) return;
        const bool fill = !copies.defined();
        if (fill) copies = at::empty({elements}, ts.begin()->options());
        for (int k = 0; k < n; ++k) dst[k] = (char *)copies.data_ptr() + (size_t)dst[k];
        i = 0;
        for (const Tensor &t : ts) {
            if (t.defined() && t.size(0) > 0 && !p[i]) {
                const int k = (int)ld[i];
                p[i] = dst[k], ld[i] = ld_dst[k];
            }
            ++i;
        }
        if (fill) check(api.copy_rows(n, src, ld_src, dst, ld_dst, rows, cols, stream()), "pai_copy_rows16");
    }
};

// y [m, n] from x [m, k] and w [n, k] (o: their operands); `saved` receives the pre-activations if wanted.  Gated: o.p[2] is the second weight.
Tensor forward(const Operands &o, const Tensor &x, int64_t n, bool gated, const Tensor &b, const Tensor &b2, const Tensor &r, int act, Tensor *saved) {
    const int64_t m = x.size(0), k = x.size(1);
    const Tensor y = at::empty({m, n}, x.options());
    if (m == 0) return y;
    void *at = nullptr;
    if (saved && (gated || act != PAI_ACT_NONE)) {
        *saved = bytes(api.saved_bytes(m, (int)n, (int)k, gated, dtype_of(x)), x);
        at = saved->data_ptr();
    }
    if (gated)
        check(api.gated_fwd(o.p[0], o.ld[0], o.p[1], o.ld[1], o.p[2], o.ld[2], address(b), address(b2), is_fp32(b) || is_fp32(b2), y.data_ptr(), n, at,
                            m, (int)n, (int)k, act, dtype_of(x), stream()),
              "pai_gated_fwd");
    else
        check(api.linear_fwd(o.p[0], o.ld[0], o.p[1], o.ld[1], address(b), is_fp32(b), address(r), r.defined() ? r.stride(0) : 0, y.data_ptr(), n, at,
                             m, (int)n, (int)k, act, dtype_of(x), stream()),
              "pai_linear_fwd");
    return y;
}

// a gradient's buffer, if it is wanted (zeros where there are no rows to sum)
Tensor gradient(bool want, const Tensor &like, at::IntArrayRef shape, bool rows) {
    if (!want) return Tensor();
    return rows ? at::empty(shape, like.options()) : at::zeros(shape, like.options());
}

Tensor or_none(const std::optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }
// (autograd's edges count the tensors that are there)
std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

void first_order_only() {
    TORCH_CHECK(!at::GradMode::is_enabled(), "fused_ops.linear and gated_linear have first-order gradients only: no create_graph");
}

// What the forward pass saved has the form that its kernel writes; a backward pass under another choice of kernels (pai_tune_set in between) would
// take it for the other form and read past its end.
void check_saved(const Tensor &saved, int64_t m, int64_t n, int64_t k, bool gated, const Tensor &x) {
    TORCH_CHECK(!saved.defined() || (size_t)saved.numel() == api.saved_bytes(m, (int)n, (int)k, gated, dtype_of(x)),
                "fused_ops: the kernels' tuning changed between the forward pass and its backward pass");
}

// A leaf's accumulator runs on the stream that was current when its first graph was built, and lives as long as a graph that uses it.  If that is the
// default stream, the engine would draw it into the capture, which CUDA does not allow and the process does not survive: refused before that.
void check_capture(const Tensor &x) {
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    const c10::Stream none = c10::cuda::getDefaultCUDAStream(x.device().index()).unwrap();
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    for (const auto &edge : node->next_edges())
        if (edge.function && edge.function->name() == "torch::autograd::AccumulateGrad") {
            const auto at = edge.function->stream();
            TORCH_CHECK(!at || *at != none, "fused_ops: a backward pass is being captured while another graph of the same leaves lives that was built on "
                                            "the default stream; drop that graph first, or build it on a side stream");
        }
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &w_, const std::optional<Tensor> &b_, const std::optional<Tensor> &r_,
                          int64_t act) {
        const c10::cuda::CUDAGuard guard(x_.device());
        const Tensor b = or_none(b_), r = or_none(r_);
        const Tensor x = whole_rows(x_), w = whole_rows(w_);
        const Operands o({x, w});
        Tensor saved;
        const bool need = ctx->needs_input_grad(0) || ctx->needs_input_grad(1) || (b.defined() && ctx->needs_input_grad(2));
        const Tensor y = ::forward(o, x, w.size(0), false, b, Tensor(), r, (int)act, need ? &saved : nullptr);
        ctx->save_for_backward({x, w, b, saved, o.copies});
        ctx->saved_data["act"] = act;
        ctx->saved_data["edges"] = (int64_t)(b.defined() ? 1 : 0) | (int64_t)(r.defined() ? 2 : 0);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const Tensor &dy = grads[0];
        const int64_t edges = ctx->saved_data["edges"].toInt();
        const bool has_b = edges & 1, has_r = edges & 2;
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(2);
        const Tensor dr = has_r && ctx->needs_input_grad(has_b ? 3 : 2) ? dy : Tensor();
        if (!dy.defined() || !(need_x || need_w || need_b)) return {Tensor(), Tensor(), Tensor(), dr, Tensor()};
        first_order_only();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
        const c10::cuda::CUDAGuard guard(x.device());
        const int64_t m = x.size(0), k = x.size(1), n = w.size(0), act = ctx->saved_data["act"].toInt();
        check_capture(x);
        check_saved(saved[3], m, n, k, false, x);
        const Tensor dx = gradient(need_x, x, {m, k}, true), dw = gradient(need_w, w, {n, k}, m > 0), db = gradient(need_b, b, {n}, m > 0);
        if (m > 0) {
            const Operands o({x, w}, saved[4]);
            const Tensor d = whole_rows(dy);
            const bool product = act == PAI_ACT_NONE && (need_x || need_w);  // dy itself is an operand
            const Operands od({product ? d : Tensor()});
            const size_t size = api.workspace_bytes(m, (int)n, (int)k, 0);
            const Tensor ws = bytes(size, x);
            check(api.linear_bwd(product ? od.p[0] : d.data_ptr(), product ? od.ld[0] : d.stride(0), o.p[0], o.ld[0], o.p[1], o.ld[1], address(saved[3]),
                                 address(dx), k,
                                 address(dw), address(db), is_fp32(b), ws.data_ptr(), size, m, (int)n, (int)k, (int)act, dtype_of(x), stream()),
                  "pai_linear_bwd");
        }
        return {dx, dw, db, dr, Tensor()};
    }
};

struct Gated : torch::autograd::Function<Gated> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &wg_, const Tensor &wu_, const std::optional<Tensor> &bg_,
                          const std::optional<Tensor> &bu_, int64_t act) {
        const c10::cuda::CUDAGuard guard(x_.device());
        const Tensor bg = or_none(bg_), bu = or_none(bu_);
        const Tensor x = whole_rows(x_), wg = whole_rows(wg_), wu = whole_rows(wu_);
        const Operands o({x, wg, wu});
        Tensor saved;
        const Tensor h = ::forward(o, x, wg.size(0), true, bg, bu, Tensor(), (int)act, &saved);
        ctx->save_for_backward({x, wg, wu, bg, bu, saved, o.copies});
        ctx->saved_data["act"] = act;
        return h;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const Tensor &dh = grads[0];
        if (!dh.defined()) return variable_list(6);
        first_order_only();
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &bg = saved[3], &bu = saved[4];
        const c10::cuda::CUDAGuard guard(x.device());
        const int64_t m = x.size(0), k = x.size(1), n = wg.size(0), act = ctx->saved_data["act"].toInt();
        check_capture(x);
        check_saved(saved[5], m, n, k, true, x);
        const Tensor dx = gradient(ctx->needs_input_grad(0), x, {m, k}, true);
        const Tensor dwg = gradient(ctx->needs_input_grad(1), wg, {n, k}, m > 0), dwu = gradient(ctx->needs_input_grad(2), wu, {n, k}, m > 0);
        const Tensor dbg = gradient(bg.defined() && ctx->needs_input_grad(3), bg, {n}, m > 0);
        const Tensor dbu = gradient(bu.defined() && ctx->needs_input_grad(bg.defined() ? 4 : 3), bu, {n}, m > 0);
        if (m > 0) {
            const Operands o({x, wg, wu}, saved[6]);
            const Tensor d = whole_rows(dh);
            const size_t size = api.workspace_bytes(m, (int)n, (int)k, 1);
            const Tensor ws = bytes(size, x);
            check(api.gated_bwd(d.data_ptr(), d.stride(0), o.p[0], o.ld[0], o.p[1], o.ld[1], o.p[2], o.ld[2], address(saved[5]), address(dx), k, address(dwg), address(dwu), address(dbg), address(dbu), is_fp32(bg) || is_fp32(bu),
                                ws.data_ptr(), size, m, (int)n, (int)k, (int)act, dtype_of(x), stream()),
                  "pai_gated_bwd");
        }
        return {dx, dwg, dwu, dbg, dbu, Tensor()};
    }
};

// ---- arguments --------------------------------------------------------------------------------------------------------
bool given(const Tensor &t) { return t.defined(); }

// The checks both operators share (undefined: left out); ws: one or two weights.
void check_arguments(const char *what, const Tensor &x, at::ArrayRef<Tensor> ws, at::ArrayRef<Tensor> bs, const Tensor &r) {
    for (const auto &list : {at::ArrayRef<Tensor>(x), ws, bs, at::ArrayRef<Tensor>(r)})
        for (const Tensor &t : list) TORCH_CHECK(!given(t) || t.is_cuda(), what, " needs CUDA tensors: there is no CPU path");
    for (const auto &list : {ws, bs, at::ArrayRef<Tensor>(r)})
        for (const Tensor &t : list) TORCH_CHECK(!given(t) || t.device() == x.device(), what, ": all tensors must be on one device");
    const auto dt = x.scalar_type();
    for (const Tensor &w : ws)
        TORCH_CHECK_TYPE((dt == at::kBFloat16 || dt == at::kHalf) && w.scalar_type() == dt, what,
                         ": x and weights must all be bfloat16 or all float16, not ", dt, " and ", w.scalar_type());
    for (const Tensor &w : ws)
        TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && w.sizes() == ws[0].sizes() && w.size(1) == x.size(-1), what,
                          ": x [..., d_in] and weights [d_out, d_in] do not fit: ", x.sizes(), " and ", w.sizes());
    TORCH_CHECK_VALUE(ws[0].size(0) > 0 && ws[0].size(1) > 0, what, ": weights must not be empty: ", ws[0].sizes());
    const Tensor *first = nullptr;
    for (const Tensor &b : bs)
        if (given(b)) {
            if (!first) first = &b;
            TORCH_CHECK_VALUE(b.dim() == 1 && b.size(0) == ws[0].size(0), what, ": a bias must have shape [", ws[0].size(0), "], not ", b.sizes());
            TORCH_CHECK_TYPE((b.scalar_type() == dt || b.scalar_type() == at::kFloat) && b.scalar_type() == first->scalar_type(), what,
                             ": biases must all be ", dt, " or all float32, not ", b.scalar_type());
        }
    if (given(r)) {
        TORCH_CHECK_TYPE(r.scalar_type() == dt, what, ": residual must be ", dt, ", not ", r.scalar_type());
        bool same = r.dim() == x.dim() && r.size(-1) == ws[0].size(0);
        for (int64_t i = 0; same && i + 1 < x.dim(); ++i) same = r.size(i) == x.size(i);
        TORCH_CHECK_VALUE(same, what, ": residual must have the output's shape, x's with ", ws[0].size(0), " columns; got ", r.sizes(), " beside ",
                          x.sizes());
    }
}

Tensor cast(const Tensor &t, at::ScalarType dt, bool keep_fp32 = false) {
    return !given(t) || t.scalar_type() == dt || !t.is_floating_point() || (keep_fp32 && t.scalar_type() == at::kFloat) ? t : t.to(dt);
}
bool autocast() { return at::autocast::is_autocast_enabled(at::kCUDA); }
Tensor flat(const Tensor &t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }
Tensor shaped(const Tensor &y, const Tensor &x) {
    if (x.dim() == 2) return y;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = y.size(1);
    return y.view(shape);
}
Tensor contiguous(const Tensor &b) { return given(b) ? b.contiguous() : b; }
bool recording(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : ts)
        if (given(t) && t.requires_grad()) return true;
    return false;
}
Tensor linear(Tensor x, Tensor w, const std::optional<Tensor> &b_, int64_t act, const std::optional<Tensor> &r_) {
    Tensor b = or_none(b_), r = or_none(r_);
    if (autocast()) {
        const auto dt = at::autocast::get_autocast_dtype(at::kCUDA);
        x = cast(x, dt), w = cast(w, dt), b = cast(b, dt, true), r = cast(r, dt);
    }
    check_arguments("linear", x, w, b, r);
    b = contiguous(b);
    const Tensor x2 = flat(x);
    if (given(r)) {
        r = flat(r);
        if (r.stride(1) != 1 && r.size(1) != 1) r = r.contiguous();
    }
    if (recording({x2, w, b, r})) return shaped(Linear::apply(x2, w, maybe(b), maybe(r), act), x);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xr = whole_rows(x2), wr = whole_rows(w);
    return shaped(forward(Operands({xr, wr}), xr, wr.size(0), false, b, Tensor(), r, (int)act, nullptr), x);
}

Tensor gated_linear(Tensor x, Tensor wg, Tensor wu, const std::optional<Tensor> &bg_, const std::optional<Tensor> &bu_, int64_t act) {
    Tensor bg = or_none(bg_), bu = or_none(bu_);
    if (autocast()) {
        const auto dt = at::autocast::get_autocast_dtype(at::kCUDA);
        x = cast(x, dt), wg = cast(wg, dt), wu = cast(wu, dt), bg = cast(bg, dt, true), bu = cast(bu, dt, true);
    }
    check_arguments("gated_linear", x, {wg, wu}, {bg, bu}, Tensor());
    bg = contiguous(bg), bu = contiguous(bu);
    const Tensor x2 = flat(x);
    if (recording({x2, wg, wu, bg, bu})) return shaped(Gated::apply(x2, wg, wu, maybe(bg), maybe(bu), act), x);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor xr = whole_rows(x2), wgr = whole_rows(wg), wur = whole_rows(wu);
    return shaped(forward(Operands({xr, wgr, wur}), xr, wgr.size(0), true, bg, bu, Tensor(), (int)act, nullptr), x);
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
    m.def("bind", &bind);
    m.def("linear", &linear, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("gated_linear", &gated_linear, pybind11::call_guard<pybind11::gil_scoped_release>());
}

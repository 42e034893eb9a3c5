// Torch binding of the block norms, the fp8 quantisation and the fp8 product:
//   rmsnorm.block_norm, rmsnorm.block_norm_backward, proj.fp8_quantize, proj.fp8_matmul
// Errors surface as RuntimeError; launches go to torch's current HIP stream of
// the tensors' device.
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include "../../include/gdn_amd.h"

namespace {

using at::Tensor;
using Opt = std::optional<Tensor>;

void* stream_of(const Tensor& t) {
    return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(t.get_device()).stream());
}

void check_status(int st, const char* who) {
    TORCH_CHECK(st == GDN_OK, who, ": ", gdn_status_string(st), ": ", gdn_last_error());
}

bool given(const Opt& t) { return t.has_value() && t->defined(); }

// An operand as rows of its last axis: how many, and the elements from one to the next.
struct Rows {
    void* ptr = nullptr;
    int64_t rows = 0, ld = 0;
};
Rows rows_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() >= 1, name, " must have at least one axis");
    const int64_t n = t.dim(), D = t.size(n - 1);
    TORCH_CHECK(D <= 1 || t.stride(n - 1) == 1, name, " must have adjacent elements along its last axis");
    Rows r;
    r.ptr = t.data_ptr();
    r.rows = 1;
    r.ld = D;
    if (t.numel() == 0) return r;
    for (int64_t i = n - 2; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (r.rows == 1)
            r.ld = t.stride(i);
        else
            TORCH_CHECK(t.stride(i) == r.ld * r.rows, name, " must have one stride between its rows");
        r.rows *= t.size(i);
    }
    TORCH_CHECK(r.ld >= D, name, " must not have rows that overlap");
    return r;
}

int type_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name, " must be bfloat16 or float32");
    return t.scalar_type() == at::kFloat ? GDN_F32 : GDN_BF16;
}

void check_like(const Tensor& t, const Tensor& y, const char* name) {
    TORCH_CHECK(t.device() == y.device(), name, " must be on y's device");
    TORCH_CHECK(t.sizes() == y.sizes(), name, " must have y's shape");
}

int act_of(const std::string& act) {
    if (act == "none") return GDN_ACT_NONE;
    if (act == "sigmoid") return GDN_ACT_SIGMOID;
    if (act == "silu") return GDN_ACT_SILU;
    if (act == "tanh") return GDN_ACT_TANH;
    TORCH_CHECK(false, "act must be none, sigmoid, silu or tanh, got ", act);
}

// What block_norm and its backward share: y's rows, the optional operands.
struct Operands {
    Rows y, residual, gate;
    int64_t R = 0, D = 0, rows_per_gate = 1;
    int ty = 0, tr = 0, tp = 0;
    const void *post_gamma = nullptr, *gamma = nullptr, *scale = nullptr;
};

Operands operands(const Tensor& y, const Opt& residual, const Opt& gate, const Opt& post_gamma, const Opt& gamma, const Opt& scale) {
    TORCH_CHECK(y.is_cuda(), "y must be a GPU tensor");
    TORCH_CHECK(y.dim() >= 1 && y.size(-1) > 0, "y must be [..., D]");
    Operands o;
    o.y = rows_of(y, "y");
    o.R = y.numel() / y.size(-1);
    o.D = y.size(-1);
    o.ty = o.tr = type_of(y, "y");
    if (given(residual)) {
        check_like(*residual, y, "residual");
        o.residual = rows_of(*residual, "residual");
        o.tr = type_of(*residual, "residual");
    }
    if (given(gate)) {
        TORCH_CHECK(gate->device() == y.device() && gate->scalar_type() == y.scalar_type(), "gate must have y's device and type");
        if (gate->sizes() == y.sizes()) {
            o.rows_per_gate = 1;
        } else if (gate->dim() == 1 && gate->size(0) == o.D) {
            o.rows_per_gate = std::max<int64_t>(o.R, 1);
        } else {
            TORCH_CHECK(gate->dim() == 2 && y.dim() > 2 && gate->size(0) == y.size(0) && gate->size(1) == o.D,
                        "gate must have y's shape, or be [B, D] for y [B, ..., D], or [D]");
            o.rows_per_gate = std::max<int64_t>(y.size(0) > 0 ? o.R / y.size(0) : 1, 1);
        }
        o.gate = rows_of(*gate, "gate");
    }
    o.tp = -1;
    auto param = [&](const Opt& t, const char* name) -> const void* {
        if (!given(t)) return nullptr;
        TORCH_CHECK(t->device() == y.device() && t->is_contiguous() && t->numel() == o.D, name, " must be D contiguous entries on y's device");
        const int tp = type_of(*t, name);
        TORCH_CHECK(o.tp < 0 || o.tp == tp, "post_gamma, gamma and scale must have one type");
        o.tp = tp;
        return t->data_ptr();
    };
    o.post_gamma = param(post_gamma, "post_gamma");
    o.gamma = param(gamma, "gamma");
    o.scale = param(scale, "scale");
    if (o.tp < 0) o.tp = o.tr;
    return o;
}

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// An output on t's device, without the dispatcher's way round (a third of a
// small call's host time).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& t) {
    return at::detail::empty_cuda(sizes, type, t.device(), std::nullopt);
}

// Scales of M rows in KB blocks as the product reads them: a block's adjacent.
Tensor down_columns(int64_t M, int64_t KB, at::ScalarType type, const Tensor& t) {
    const int64_t Mp = up(M, 16);
    Tensor s = at::detail::empty_strided_cuda({Mp, KB}, {1, Mp}, type, t.device());
    if (Mp != M) s.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({M, KB}), at::IntArrayRef({1, Mp}));
    return s;
}

std::vector<Opt> block_norm(const Tensor& y, const Opt& residual, const Opt& gate, const Opt& post_gamma, const Opt& gamma,
                            const Opt& scale, double residual_scale, const std::string& act, double eps, bool quantize,
                            bool store_h, bool stats, bool inplace) {
    TORCH_CHECK(!inplace || !given(residual) || !at::GradMode::is_enabled() || !residual->requires_grad(),
                "block_norm: inplace would write over a residual that requires grad (no gradients are recorded here)");
    const Operands o = operands(y, residual, gate, post_gamma, gamma, scale);
    const int a = act_of(act);
    TORCH_CHECK(store_h || quantize || given(gamma), "block_norm: store_h=False leaves nothing to write");
    TORCH_CHECK(!inplace || (given(residual) && store_h), "block_norm: inplace writes h over residual");
    const c10::DeviceGuard guard(y.device());
    std::vector<Opt> out(stats ? 6 : 4);
    Rows h, n;
    if (store_h) {
        out[0] = inplace ? *residual : fresh(y.sizes(), (given(residual) ? *residual : y).scalar_type(), y);
        h = rows_of(*out[0], "h");
    }
    if (given(gamma) && !quantize) {
        out[1] = fresh(y.sizes(), y.scalar_type(), y);
        n = rows_of(*out[1], "n");
    }
    uint8_t *codes = nullptr, *scales = nullptr;
    int64_t ldc = 0, lds = 0;
    if (quantize) {
        ldc = up(o.D, 128);
        out[2] = fresh({o.R, ldc}, at::kFloat8_e4m3fn, y);
        out[3] = down_columns(o.R, ldc / 128, at::kFloat8_e8m0fnu, y);
        codes = static_cast<uint8_t*>(out[2]->data_ptr());
        scales = static_cast<uint8_t*>(out[3]->data_ptr());
        lds = up(o.R, 16);
    }
    float *ry = nullptr, *rh = nullptr;
    if (stats) {
        if (given(post_gamma)) ry = (out[4] = fresh({o.R}, at::kFloat, y))->data_ptr<float>();
        if (given(gamma)) rh = (out[5] = fresh({o.R}, at::kFloat, y))->data_ptr<float>();
    }
    if (o.R == 0) return out;
    check_status(gdn_block_norm_hip(o.y.ptr, o.y.ld, o.residual.ptr, o.residual.ld, o.gate.ptr, o.gate.ld, o.rows_per_gate,
                                    o.post_gamma, o.gamma, o.scale, static_cast<float>(residual_scale), a,
                                    static_cast<float>(eps), h.ptr, h.ld, n.ptr, n.ld, codes, ldc, scales, lds, ry, rh, o.R, o.D,
                                    o.ty, o.tr, o.tp, stream_of(y)),
                 "block_norm");
    if (inplace && !residual->is_inference()) residual->unsafeGetTensorImpl()->bump_version();  // a graph that saved it raises
    return out;
}

std::vector<Opt> block_norm_backward(const Opt& dh, const Opt& dn, const Tensor& y, const Opt& residual, const Opt& gate,
                                     const Opt& post_gamma, const Opt& gamma, const Opt& scale, double residual_scale,
                                     const std::string& act, const Opt& rstd_y, const Opt& rstd_h) {
    const Operands o = operands(y, residual, gate, post_gamma, gamma, scale);
    const int a = act_of(act);
    TORCH_CHECK(given(dh) || given(dn), "block_norm_backward: dh or dn is needed");
    Rows rdh, rdn;
    if (given(dh)) {
        check_like(*dh, y, "dh");
        TORCH_CHECK(type_of(*dh, "dh") == o.tr, "dh must have h's type");
        rdh = rows_of(*dh, "dh");
    }
    if (given(dn)) {
        check_like(*dn, y, "dn");
        TORCH_CHECK(type_of(*dn, "dn") == o.ty, "dn must have y's type");
        TORCH_CHECK(given(gamma), "dn needs gamma");
        rdn = rows_of(*dn, "dn");
    }
    auto rstd = [&](const Opt& t, bool needed, const char* name) -> const float* {
        if (!needed) return nullptr;
        TORCH_CHECK(given(t) && t->device() == y.device() && t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == o.R,
                    name, " must be the forward pass's, float32 with an entry a row");
        return t->data_ptr<float>();
    };
    // a gamma without dn has no part in h: its gradient is zeros
    const bool normed = given(dn);
    const float* const ry = rstd(rstd_y, given(post_gamma), "rstd_y");
    const float* const rh = rstd(rstd_h, normed, "rstd_h");
    const c10::DeviceGuard guard(y.device());
    std::vector<Opt> out(6);
    auto like = [&](const Opt& t) { return fresh(t->sizes(), t->scalar_type(), y); };
    if (given(residual)) out[0] = like(residual);
    out[1] = fresh(y.sizes(), y.scalar_type(), y);
    if (given(gate)) out[2] = like(gate);
    if (given(post_gamma)) out[3] = like(post_gamma);
    if (given(gamma)) out[4] = normed ? like(gamma) : at::zeros(gamma->sizes(), gamma->options());
    if (given(scale)) out[5] = like(scale);
    if (o.R == 0) {
        for (auto& t : out)
            if (given(t)) t->zero_();
        return out;
    }
    const bool sums = given(post_gamma) || normed || given(scale) || (given(gate) && o.rows_per_gate > 1);
    const size_t bytes = sums ? gdn_block_norm_bwd_workspace_bytes(o.R, o.D, given(gate) ? o.rows_per_gate : 1) : 0;
    const Tensor ws = fresh({static_cast<int64_t>(bytes)}, at::kByte, y);
    auto ptr = [&](int i) { return given(out[i]) ? out[i]->data_ptr() : nullptr; };
    check_status(gdn_block_norm_bwd_hip(rdh.ptr, rdh.ld, rdn.ptr, rdn.ld, o.y.ptr, o.y.ld, o.residual.ptr, o.residual.ld,
                                        o.gate.ptr, o.gate.ld, o.rows_per_gate, o.post_gamma, normed ? o.gamma : nullptr, o.scale,
                                        static_cast<float>(residual_scale), a, ry, rh, ptr(0), ptr(1), ptr(2), ptr(3),
                                        normed ? ptr(4) : nullptr, ptr(5), o.R, o.D, o.ty, o.tr, o.tp,
                                        bytes ? ws.data_ptr() : nullptr, bytes, stream_of(y)),
                 "block_norm_backward");
    return out;
}

int format_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kFloat8_e5m2, name, " must be float8_e4m3fn or float8_e5m2");
    return t.scalar_type() == at::kFloat8_e4m3fn ? GDN_E4M3 : GDN_E5M2;
}

std::vector<Tensor> fp8_quantize(const Tensor& x, int64_t block_rows, at::ScalarType dtype, bool rows, bool columns) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a GPU tensor [M, K]");
    TORCH_CHECK(x.size(1) <= 1 || x.stride(1) == 1, "x must have adjacent elements along its last axis");
    TORCH_CHECK(dtype == at::kFloat8_e4m3fn || dtype == at::kFloat8_e5m2, "dtype must be float8_e4m3fn or float8_e5m2");
    TORCH_CHECK(block_rows == 1 || block_rows == 128, "block_rows must be 1 or 128");
    TORCH_CHECK(rows || columns, "fp8_quantize: neither rows nor columns");
    const int type = type_of(x, "x");
    const int64_t M = x.size(0), K = x.size(1), Mp = up(M, 128), Kp = up(K, 128), ld = M > 1 ? x.stride(0) : std::max<int64_t>(K, 1);
    const c10::DeviceGuard guard(x.device());
    std::vector<Tensor> out;
    uint8_t* ptr[4] = {};
    int64_t lds[2] = {};
    auto make = [&](int at, int64_t m, int64_t mp, int64_t kp) {
        out.push_back(fresh({m, kp}, dtype, x));
        ptr[at] = static_cast<uint8_t*>(out.back().data_ptr());
        if (block_rows == 1) {
            out.push_back(down_columns(m, kp / 128, at::kFloat8_e8m0fnu, x));
            lds[at / 2] = up(m, 16);
        } else {
            out.push_back(fresh({mp / 128, kp / 128}, at::kFloat8_e8m0fnu, x));
            lds[at / 2] = kp / 128;
        }
        ptr[at + 1] = static_cast<uint8_t*>(out.back().data_ptr());
    };
    if (rows) make(0, M, Mp, Kp);
    if (columns) make(2, K, Kp, Mp);
    if (M == 0 || K == 0) {  // nothing but the padding's shape
        for (auto& t : out) t.view(at::kByte).fill_(0);
        return out;
    }
    check_status(gdn_fp8_quantize_hip(x.data_ptr(), ld, type, M, K, static_cast<int>(block_rows),
                                      dtype == at::kFloat8_e4m3fn ? GDN_E4M3 : GDN_E5M2, ptr[0], Kp, ptr[1], lds[0], ptr[2], Mp,
                                      ptr[3], lds[1], stream_of(x)),
                 "fp8_quantize");
    return out;
}

// Scales [M, KB] of a row and block each, with a block's adjacent and 16 apart
// from the next: as given where they are, else laid out so.
Tensor scale_rows(const Tensor& s, int64_t* ld) {
    const int64_t M = s.size(0), KB = s.size(1), e = s.element_size();
    const int64_t step = KB > 1 ? s.stride(1) : up(M, 16);
    if ((M <= 1 || s.stride(0) == 1) && step % 16 == 0 && step >= M && reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0 &&
        static_cast<int64_t>(s.storage().nbytes()) >= (s.storage_offset() + (KB - 1) * step + up(M, 16)) * e) {
        *ld = step;
        return s;
    }
    auto t = down_columns(M, KB, s.scalar_type(), s);
    *ld = up(M, 16);
    t.view(e == 1 ? at::kByte : at::kFloat).copy_(s.view(e == 1 ? at::kByte : at::kFloat));
    return t;
}

Tensor fp8_matmul(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, at::ScalarType out_dtype) {
    TORCH_CHECK(a.is_cuda() && a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1), "a, b must be GPU tensors [M, K], [N, K]");
    TORCH_CHECK(a_scale.device() == a.device() && b.device() == a.device() && b_scale.device() == a.device(),
                "the operands must be on one device");
    const int fa = format_of(a, "a"), fb = format_of(b, "b");
    const int64_t M = a.size(0), N = b.size(0), K = a.size(1);
    TORCH_CHECK(K > 0 && K % 128 == 0, "K must be a multiple of 128, got ", K);
    TORCH_CHECK(a.stride(1) == 1 && b.stride(1) == 1, "a, b must have adjacent elements along their last axis");
    TORCH_CHECK(out_dtype == at::kBFloat16 || out_dtype == at::kFloat, "out_dtype must be bfloat16 or float32");
    const int64_t KB = K / 128, NB = (N + 127) / 128;
    TORCH_CHECK(a_scale.scalar_type() == at::kFloat8_e8m0fnu && a_scale.dim() == 2 && a_scale.size(0) == M && a_scale.size(1) == KB,
                "a_scale must be float8_e8m0fnu [M, K / 128]");
    TORCH_CHECK(b_scale.scalar_type() == at::kFloat8_e8m0fnu || b_scale.scalar_type() == at::kFloat, "b_scale must be float8_e8m0fnu or float32");
    TORCH_CHECK(b_scale.dim() == 2 && (b_scale.size(0) == N || b_scale.size(0) == NB) && b_scale.size(1) == KB,
                "b_scale must be [N, K / 128] or [ceil(N / 128), K / 128]");
    const c10::DeviceGuard guard(a.device());
    auto out = fresh({M, N}, out_dtype, a);
    if (M == 0 || N == 0) return out;
    int64_t lda_s = 0, ldb_s = 0;
    const Tensor as = scale_rows(a_scale, &lda_s);
    const bool blocks = b_scale.size(0) == NB;
    Tensor bs = b_scale;
    if (!blocks) {
        bs = scale_rows(b_scale, &ldb_s);
    } else {
        if (KB > 1 && bs.stride(1) != 1) bs = bs.contiguous();
        ldb_s = NB > 1 ? bs.stride(0) : KB;
    }
    check_status(gdn_fp8_matmul_hip(static_cast<const uint8_t*>(a.data_ptr()), M > 1 ? a.stride(0) : K, fa,
                                    static_cast<const uint8_t*>(as.data_ptr()), lda_s, static_cast<const uint8_t*>(b.data_ptr()),
                                    N > 1 ? b.stride(0) : K, fb, bs.data_ptr(), ldb_s, blocks ? 128 : 1,
                                    bs.scalar_type() == at::kFloat ? GDN_F32 : GDN_E8M0, out.data_ptr(), N,
                                    out_dtype == at::kFloat ? GDN_F32 : GDN_BF16, M, N, K, stream_of(a)),
                 "fp8_matmul");
    return out;
}

// Whether a node's stream is one that a capture on the current stream must not
// wait for or write to: another than the current one, and not part of a capture.
bool outside_capture(const c10::Stream& s) {
    if (s.id() == c10::hip::getCurrentHIPStream(s.device_index()).id()) return false;
    if (s.id() == 0) return true;  // the default stream cannot be captured (nor asked while another is)
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const c10::hip::HIPStream stream(c10::hip::HIPStream::UNCHECKED, s);
    if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) {
        (void)hipGetLastError();
        return true;
    }
    return status != hipStreamCaptureStatusActive;
}

// The nodes that the running backward pass has to run (empty outside of one), by
// name, and whether each belongs to a stream outside of the current capture.
std::vector<std::pair<std::string, bool>> backward_nodes() {
    std::vector<std::pair<std::string, bool>> out;
    const auto* const nodes = torch::autograd::get_current_graph_task_nodes_in_graph();
    if (!nodes) return out;
    const auto* const wanted = torch::autograd::get_current_graph_task_exec_info();  // empty: all of them
    for (auto* const node : *nodes) {
        if (wanted && !wanted->empty()) {
            const auto it = wanted->find(node);
            if (it == wanted->end() || !it->second.should_execute()) continue;
        }
        const auto stream = node->stream();
        out.emplace_back(node->name(), stream.has_value() && outside_capture(*stream));
    }
    return out;
}

}  // namespace

void bind_block_ops(pybind11::module_& top, pybind11::module_& rmsnorm, pybind11::module_& proj) {
    namespace py = pybind11;
    top.def("_backward_nodes", &backward_nodes);
    const py::object none = py::none();
    rmsnorm.def("block_norm", &block_norm,
                "u = RMSNorm(y) post_gamma; h = residual + residual_scale scale act(gate) u; n = RMSNorm(h) gamma.\n"
                "y [..., D]; residual of y's shape; gate of y's shape, [B, D] (one a sequence of y [B, ..., D]) or [D]; "
                "post_gamma, gamma, scale [D]; what is None is left out.  Returns [h, n, codes, scales] "
                "(+ [rstd_y, rstd_h] with stats, for block_norm_backward), None where not made: quantize gives n (h without "
                "gamma) as e4m3 codes [R, D padded to 128] with e8m0 scales [R, blocks] instead of n; store_h=False leaves h "
                "out, inplace writes it over residual (as an in-place operation: a graph that saved the residual can no longer "
                "run backward; one that requires grad is refused while gradients are recorded).",
                py::arg("y"), py::arg("residual") = none, py::arg("gate") = none, py::arg("post_gamma") = none,
                py::arg("gamma") = none, py::arg("scale") = none, py::arg("residual_scale") = 1.0, py::arg("act") = "none",
                py::arg("eps") = 1e-6, py::arg("quantize") = false, py::arg("store_h") = true, py::arg("stats") = false,
                py::arg("inplace") = false);
    rmsnorm.def("block_norm_backward", &block_norm_backward,
                "Gradients of block_norm: [dresidual, dy, dgate, dpost_gamma, dgamma, dscale], None for absent inputs.  dh, dn "
                "(either may be None): those of h and n; rstd_y, rstd_h: block_norm's with stats.  At most 65535 gate rows that "
                "several rows share.",
                py::arg("dh"), py::arg("dn"), py::arg("y"), py::arg("residual") = none, py::arg("gate") = none,
                py::arg("post_gamma") = none, py::arg("gamma") = none, py::arg("scale") = none,
                py::arg("residual_scale") = 1.0, py::arg("act") = "none", py::arg("rstd_y") = none, py::arg("rstd_h") = none);
    proj.def("fp8_quantize", &fp8_quantize,
             "x [M, K] (bf16 or fp32) to 8-bit codes with a power-of-two scale for each block of block_rows (1 or 128) x 128: "
             "[codes, scales] along the rows (codes [M, K padded to 128]), and / or along the columns (codes of x^T "
             "[K, M padded to 128]), in that order.  Scales: float8_e8m0fnu, a row of codes or 128 of them by blocks.",
             py::arg("x"), py::arg("block_rows") = 1, py::arg("dtype") = at::kFloat8_e4m3fn, py::arg("rows") = true,
             py::arg("columns") = false);
    proj.def("fp8_matmul", &fp8_matmul,
             "out [M, N] = (a a_scale) (b b_scale)^T for codes a [M, K], b [N, K] (float8_e4m3fn or float8_e5m2, K a multiple "
             "of 128) with a scale a block of 128: a_scale float8_e8m0fnu [M, K / 128]; b_scale float8_e8m0fnu or float32 "
             "[N, K / 128] or, a 128 x 128 block each, [ceil(N / 128), K / 128].  fp32 results sum every product in full; for "
             "bf16 results the instruction drops up to 2^-10 of the product of the largest codes of a block, which matters where "
             "large products of a block cancel.  Scales of a row and block each "
             "are read as fp8_quantize lays them out; others are copied into that layout first.",
             py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("out_dtype") = at::kBFloat16);
}

// Torch binding of the 4-bit quantisation and the product with 4-bit weights:
//   proj.fp4_quantize, proj.fp4_fp8_quantize, proj.fp4_dequantize, proj.fp4_matmul, proj.fp4_linear
// Errors surface as RuntimeError; launches go to torch's current HIP stream of
// the tensors' device.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "bindings_common.hpp"

namespace {

constexpr auto kFp4 = at::kFloat4_e2m1fn_x2;

// Scales [M, KB, 4] of M rows as the product reads them: a row's four bytes of a block
// of 128 adjacent, then the rows, 16 at a time.
Tensor words(int64_t M, int64_t KB, const Tensor& t) {
    const int64_t Mp = up(M, 16);
    Tensor s = at::detail::empty_strided_cuda({Mp, KB, 4}, {4, 4 * Mp, 1}, at::kFloat8_e8m0fnu, t.device());
    if (Mp != M) s.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({M, KB, 4}), at::IntArrayRef({4, 4 * Mp, 1}));
    return s;
}

// Scales [M, KB, 4] or [M, 4 KB]: as given where they lie so, else laid out so.
Tensor word_rows(const Tensor& given, int64_t M, int64_t KB, int64_t* ld, const char* name) {
    TORCH_CHECK(given.scalar_type() == at::kFloat8_e8m0fnu && ((given.dim() == 3 && given.size(2) == 4 && given.size(1) == KB) ||
                                                              (given.dim() == 2 && given.size(1) == 4 * KB)) && given.size(0) == M,
                name, " must be float8_e8m0fnu [", M, ", ", KB, ", 4] or [", M, ", ", 4 * KB, "]");
    if (given.dim() == 3) {
        const int64_t step = KB > 1 ? given.stride(1) : 4 * up(M, 16);
        if (given.stride(2) == 1 && (M <= 1 || given.stride(0) == 4) && step % 16 == 0 && step >= 4 * M &&
            reinterpret_cast<uintptr_t>(given.data_ptr()) % 16 == 0 &&
            static_cast<int64_t>(given.storage().nbytes()) >= given.storage_offset() + (KB - 1) * step + 4 * up(M, 4)) {
            *ld = step / 4;
            return given;
        }
    }
    Tensor t = words(M, KB, given);
    *ld = up(M, 16);
    t.view(at::kByte).copy_((given.dim() == 3 ? given : given.unflatten(1, {KB, 4})).view(at::kByte));
    return t;
}

std::vector<Tensor> fp4_quantize(const Tensor& x, int64_t block_rows, bool rows, bool columns) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a GPU tensor [M, K]");
    TORCH_CHECK(x.size(1) <= 1 || x.stride(1) == 1, "x must have adjacent elements along its last axis");
    TORCH_CHECK(block_rows == 1 || block_rows == 32, "block_rows must be 1 or 32");
    TORCH_CHECK(rows || columns, "fp4_quantize: neither rows nor columns");
    const int type = type_of(x, "x");
    const int64_t M = x.size(0), K = x.size(1), ld = M > 1 ? x.stride(0) : std::max<int64_t>(K, 1);
    TORCH_CHECK(M == 0 || ld >= K, "x must not have rows that overlap");
    const c10::DeviceGuard guard(x.device());
    std::vector<Tensor> out;
    uint8_t* ptr[4] = {};
    auto make = [&](int at, int64_t m, int64_t k) {
        const int64_t kp = up(k, 256);
        out.push_back(fresh({m, kp / 2}, kFp4, x));
        ptr[at] = static_cast<uint8_t*>(out.back().data_ptr());
        out.push_back(words(m, kp / 128, x));
        ptr[at + 1] = static_cast<uint8_t*>(out.back().data_ptr());
    };
    if (rows) make(0, M, K);
    if (columns) make(2, K, M);
    if (M == 0 || K == 0) return out;  // no values: codes and scales are empty too
    check_status(gdn_fp4_quantize_hip(x.data_ptr(), ld, type, M, K, static_cast<int>(block_rows), ptr[0], up(K, 256) / 2, ptr[1], up(M, 16),
                                      ptr[2], up(M, 256) / 2, ptr[3], up(K, 16), stream_of(x)),
                 "fp4_quantize");
    return out;
}

std::vector<Tensor> fp4_fp8_quantize(const Tensor& x) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2, "x must be a GPU tensor [M, K]");
    TORCH_CHECK(x.size(1) <= 1 || x.stride(1) == 1, "x must have adjacent elements along its last axis");
    const int type = type_of(x, "x");
    const int64_t M = x.size(0), K = x.size(1), ld = M > 1 ? x.stride(0) : std::max<int64_t>(K, 1), Kp = up(K, 256), Mp = up(M, 128);
    TORCH_CHECK(M == 0 || ld >= K, "x must not have rows that overlap");
    const c10::DeviceGuard guard(x.device());
    std::vector<Tensor> out = {fresh({M, Kp / 2}, kFp4, x), words(M, Kp / 128, x), fresh({K, Mp}, at::kFloat8_e4m3fn, x),
                               down_columns(K, Mp / 128, at::kFloat8_e8m0fnu, x)};
    if (M == 0 || K == 0) return out;  // no values: codes and scales are empty too
    const auto ptr = [&](int i) { return static_cast<uint8_t*>(out[i].data_ptr()); };
    check_status(gdn_fp4_fp8_quantize_hip(x.data_ptr(), ld, type, M, K, ptr(0), Kp / 2, ptr(1), up(M, 16), ptr(2), Mp, ptr(3), up(K, 16), stream_of(x)),
                 "fp4_fp8_quantize");
    return out;
}

// Codes [M, K / 2] as rows: the bytes from one to the next.
int64_t code_rows(const Tensor& t, const char* name) {
    TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have adjacent elements along its last axis");
    TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must not have rows that overlap");
    return t.size(0) > 1 ? t.stride(0) : up(std::max<int64_t>(t.size(1), 1), 16);
}

Tensor fp4_dequantize(const Tensor& codes, const Tensor& scales, std::optional<int64_t> columns, at::ScalarType dtype) {
    TORCH_CHECK(codes.is_cuda() && codes.dim() == 2 && codes.scalar_type() == kFp4, "codes must be a GPU tensor [M, K / 2] of float4_e2m1fn_x2");
    TORCH_CHECK(scales.device() == codes.device(), "scales must be on codes' device");
    TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kFloat, "dtype must be bfloat16 or float32");
    TORCH_CHECK(codes.size(1) % 64 == 0, "codes must have rows of whole 128 values");
    const int64_t M = codes.size(0), K = columns.value_or(2 * codes.size(1));
    TORCH_CHECK(K >= 0 && K <= 2 * codes.size(1), "columns=", K, " of ", 2 * codes.size(1));
    const c10::DeviceGuard guard(codes.device());
    int64_t lds = 0;
    const Tensor s = word_rows(scales, M, codes.size(1) / 64, &lds, "scales");
    auto out = fresh({M, K}, dtype, codes);
    if (M == 0 || K == 0) return out;
    check_status(gdn_fp4_dequantize_hip(static_cast<const uint8_t*>(codes.data_ptr()), code_rows(codes, "codes"),
                                        static_cast<const uint8_t*>(s.data_ptr()), lds, out.data_ptr(), K, dtype == at::kFloat ? GDN_F32 : GDN_BF16, M,
                                        K, stream_of(codes)),
                 "fp4_dequantize");
    return out;
}

Tensor fp4_matmul(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, at::ScalarType out_dtype) {
    TORCH_CHECK(a.is_cuda() && a.dim() == 2 && b.dim() == 2, "a, b must be GPU tensors of codes [M, K], [N, K]");
    TORCH_CHECK(a_scale.device() == a.device() && b.device() == a.device() && b_scale.device() == a.device(), "the operands must be on one device");
    TORCH_CHECK(b.scalar_type() == kFp4, "b must be float4_e2m1fn_x2");
    const bool fp4 = a.scalar_type() == kFp4;
    TORCH_CHECK(fp4 || a.scalar_type() == at::kFloat8_e4m3fn || a.scalar_type() == at::kFloat8_e5m2, "a must be float4_e2m1fn_x2, float8_e4m3fn or float8_e5m2");
    const int format = fp4 ? GDN_E2M1 : format_of(a, "a");
    TORCH_CHECK(out_dtype == at::kBFloat16 || out_dtype == at::kFloat, "out_dtype must be bfloat16 or float32");
    const int64_t M = a.size(0), N = b.size(0), K = fp4 ? 2 * a.size(1) : a.size(1);
    TORCH_CHECK(K > 0 && K % (fp4 ? 256 : 128) == 0, "K must be a multiple of ", fp4 ? 256 : 128, ", got ", K);
    TORCH_CHECK(2 * b.size(1) == up(K, 256), "b must have rows of ", up(K, 256), " values (K up to the next multiple of 256), got ", 2 * b.size(1));
    const int64_t lda = code_rows(a, "a"), ldb = code_rows(b, "b"), KB = K / 128;
    TORCH_CHECK(fp4 || (a_scale.scalar_type() == at::kFloat8_e8m0fnu && a_scale.dim() == 2 && a_scale.size(0) == M && a_scale.size(1) == KB),
                "a_scale must be float8_e8m0fnu [M, K / 128]");
    const c10::DeviceGuard guard(a.device());
    int64_t lda_s = 0, ldb_s = 0;
    const Tensor as = fp4 ? word_rows(a_scale, M, KB, &lda_s, "a_scale") : scale_rows(a_scale, &lda_s);
    const Tensor bs = word_rows(b_scale, N, up(K, 256) / 128, &ldb_s, "b_scale");
    auto out = fresh({M, N}, out_dtype, a);
    if (M == 0 || N == 0) return out;
    check_status(gdn_fp4_matmul_hip(static_cast<const uint8_t*>(a.data_ptr()), lda, format, static_cast<const uint8_t*>(as.data_ptr()), lda_s,
                                    static_cast<const uint8_t*>(b.data_ptr()), ldb, static_cast<const uint8_t*>(bs.data_ptr()), ldb_s,
                                    out.data_ptr(), N, out_dtype == at::kFloat ? GDN_F32 : GDN_BF16, M, N, K, stream_of(a)),
                 "fp4_matmul");
    return out;
}

// x [M, K] with a row's elements adjacent, as the quantisation reads them; expanded
// and transposed ones are copied.
Tensor adjacent(const Tensor& x) {
    return x.stride(1) == 1 && x.stride(0) >= x.size(1) ? x : x.contiguous();
}

// Refuses a backward pass that is being captured into a graph and has yet to reach nodes
// of eager work, such as the gradient accumulators of leaves that an eager graph keeps
// alive: they belong to the eager work's stream, which autograd would draw into the
// capture, and that ends the process.
void check_capture() {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    std::string outside;
    for (const auto& node : gdn_bindings::backward_nodes())
        if (node.second && outside.find(node.first) == std::string::npos) outside += (outside.empty() ? "" : ", ") + node.first;
    TORCH_CHECK(outside.empty(), "a backward pass is captured while an eager autograd graph of the same leaves is alive: drop (or detach) "
                                 "the eager results before the capture (", outside, ")");
}

// The linear layer with its gradients, in C++: forward and backward take 96 us of host time,
// through Python's autograd 133; the kernels of 2683 x 2048 x 2048 take 95.
class Fp4Linear : public torch::autograd::Function<Fp4Linear> {
public:
    // weight: a tensor to quantise here, or none, with w its codes and scales (and those of
    // its transpose, or undefined ones).  record: whether gradients are recorded.
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Opt& weight, std::vector<Tensor> w, int64_t N, bool fp4,
                          bool record) {
        const bool need_x = record && x.requires_grad(), need_w = record && given(weight) && weight->requires_grad();
        const int64_t K = x.size(-1);
        const Tensor x2 = adjacent(x.reshape({-1, K}));
        // x's codes for y and, from the same read, those that dW takes
        const std::vector<Tensor> q = !fp4    ? gdn_bindings::fp8_quantize(x2, 1, at::kFloat8_e4m3fn, true, need_w)
                                      : need_w ? fp4_fp8_quantize(x2)
                                               : fp4_quantize(x2, 1, true, false);
        if (given(weight)) {
            w = fp4_quantize(adjacent(weight->detach()), 32, true, need_x);
            w.resize(4);
        }
        ctx->save_for_backward({need_w ? q[2] : Tensor(), need_w ? q[3] : Tensor(), need_x ? w[2] : Tensor(), need_x ? w[3] : Tensor()});
        ctx->saved_data["need_x"] = need_x;
        ctx->saved_data["need_w"] = need_w;
        ctx->saved_data["sizes"] = x.sizes().vec();
        ctx->saved_data["N"] = N;
        ctx->saved_data["types"] = std::vector<int64_t>{static_cast<int64_t>(x.scalar_type()), static_cast<int64_t>(given(weight) ? weight->scalar_type() : x.scalar_type())};
        auto sizes = x.sizes().vec();
        sizes.back() = N;
        return at::_unsafe_view(fp4_matmul(q[0], q[1], w[0], w[1], x.scalar_type()), sizes);  // no view: a caller may write to it
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        torch::autograd::variable_list out(6);
        {
            const at::NoGradGuard no_grad;
            compute(ctx, grads[0], out);
        }
        if (!at::GradMode::is_enabled()) return out;
        // a graph of the gradients is recorded: using it for second derivatives raises
        for (auto& t : out)
            if (t.defined()) {
                t.requires_grad_();
                t = (*std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice fp4_linear, which has first derivatives alone", 1))({t})[0];
            }
        return out;
    }

private:
    static void compute(torch::autograd::AutogradContext* ctx, const Tensor& dy, torch::autograd::variable_list& out) {
        check_capture();
        const auto saved = ctx->get_saved_variables();
        const bool need_x = ctx->saved_data["need_x"].toBool() && ctx->needs_input_grad(0);
        const bool need_w = ctx->saved_data["need_w"].toBool() && ctx->needs_input_grad(1);
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const auto types = ctx->saved_data["types"].toIntVector();
        const auto tx = static_cast<at::ScalarType>(types[0]), tw = static_cast<at::ScalarType>(types[1]);
        const int64_t N = ctx->saved_data["N"].toInt(), K = sizes.back();
        if (!dy.defined() || (!need_x && !need_w)) return;
        if (dy.numel() == 0) {  // no tokens, or no columns
            if (need_x) out[0] = at::zeros(sizes, dy.options().dtype(tx));
            if (need_w) out[1] = at::zeros({N, K}, dy.options().dtype(tw));
            return;
        }
        const auto d = gdn_bindings::fp8_quantize(adjacent(dy.reshape({-1, N})), 1, at::kFloat8_e5m2, need_x, need_w);
        if (need_x) out[0] = at::_unsafe_view(fp4_matmul(d[0], d[1], saved[2], saved[3], tx), sizes);
        if (need_w) out[1] = gdn_bindings::fp8_matmul(d[d.size() - 2], d.back(), saved[0], saved[1], tw);
    }
};

Tensor fp4_linear(const Tensor& x, const Opt& weight, const Opt& codes, const Opt& scales, const Opt& codes_t, const Opt& scales_t, int64_t N, bool fp4) {
    TORCH_CHECK(x.is_cuda(), "x must be a GPU tensor");
    TORCH_CHECK(given(weight) ? weight->dim() == 2 && x.dim() >= 1 && weight->size(0) == N && weight->size(1) == x.size(-1) : given(codes) && given(scales),
                "fp4_linear: a weight [N, K] for x [..., K], or its codes and scales");
    std::vector<Tensor> w;
    for (const auto* const t : {&codes, &scales, &codes_t, &scales_t}) w.push_back(given(*t) ? **t : Tensor());
    return Fp4Linear::apply(x, weight, w, N, fp4, at::GradMode::is_enabled());
}

}  // namespace

void bind_fp4_ops(pybind11::module_& proj) {
    namespace py = pybind11;
    proj.def("fp4_quantize", &fp4_quantize,
             "x [M, K] (bf16 or fp32) to 4-bit codes (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6) with a power-of-two scale for each block of "
             "block_rows (1 or 32) x 32: [codes, scales] along the rows (float4_e2m1fn_x2 [M, K padded to 256, / 2]; float8_e8m0fnu [M, "
             "padded K / 128, 4]), and / or along the columns (of x^T), in that order.  With block_rows=32 both stand for the same values.",
             py::arg("x"), py::arg("block_rows") = 1, py::arg("rows") = true, py::arg("columns") = false);
    proj.def("fp4_fp8_quantize", &fp4_fp8_quantize,
             "From one read of x [M, K]: [codes, scales] of fp4_quantize(x) and those along the columns of fp8_quantize(x, rows=False, "
             "columns=True), what a training step with 4-bit activations takes of x.",
             py::arg("x"));
    proj.def("fp4_dequantize", &fp4_dequantize,
             "What 4-bit codes [M, K / 2] with scales [M, K / 128, 4] (or [M, K / 32]) stand for: [M, columns] (all of them without "
             "columns), bfloat16 or float32, exactly.",
             py::arg("codes"), py::arg("scales"), py::arg("columns") = py::none(), py::arg("dtype") = at::kBFloat16);
    proj.def("fp4_matmul", &fp4_matmul,
             "out [M, N] = (a a_scale) (b b_scale)^T for 4-bit codes b [N, K padded to 256, / 2] with a scale a row and 32 values, and a "
             "either 4-bit codes [M, K / 2] with scales alike or float8_e4m3fn / float8_e5m2 codes [M, K] with a scale a row and 128, "
             "a_scale [M, K / 128] (what block_norm and fp8_quantize write).  Scales of 4-bit codes: float8_e8m0fnu [rows, K / 128, 4] or "
             "[rows, K / 32].  With 8-bit codes fp32 results sum every product in full; for bf16 results the instruction drops what lies "
             "below 2^-17 of the largest of 128 products.  With 4-bit codes each 128 products are added with an error of at most 2^-21 of "
             "the largest among them, their sums of 32, the sum so far and the new one, whatever the result's type.  Scales are read as fp4_quantize and fp8_quantize lay them out; others are "
             "copied into that layout first.",
             py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("out_dtype") = at::kBFloat16);
    proj.def("fp4_linear", &fp4_linear,
             "x [..., K] times a weight [N, K]^T on 4-bit codes of the weight and 8-bit (fp4: 4-bit) ones of x, with gradients: what "
             "blocks.fp4_linear calls.  weight, or codes and scales (and codes_t, scales_t for the gradient of x).",
             py::arg("x"), py::arg("weight"), py::arg("codes"), py::arg("scales"), py::arg("codes_t"), py::arg("scales_t"), py::arg("N"), py::arg("fp4"));
}

// What the bindings of the block norms, the 8-bit and 4-bit projections and the
// gradients' norm share: streams, status, types, outputs and layouts of scales.
#pragma once

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "../../include/gdn_amd.h"

// Defined in bindings_block.cpp.
namespace gdn_bindings {
std::vector<at::Tensor> fp8_quantize(const at::Tensor& x, int64_t block_rows, at::ScalarType dtype, bool rows, bool columns);
at::Tensor fp8_matmul(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b, const at::Tensor& b_scale, at::ScalarType out_dtype);
std::vector<std::pair<std::string, bool>> backward_nodes();
}  // namespace gdn_bindings

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

int type_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name, " must be bfloat16 or float32");
    return t.scalar_type() == at::kFloat ? GDN_F32 : GDN_BF16;
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

int format_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kFloat8_e5m2, name, " must be float8_e4m3fn or float8_e5m2");
    return t.scalar_type() == at::kFloat8_e4m3fn ? GDN_E4M3 : GDN_E5M2;
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

}  // namespace

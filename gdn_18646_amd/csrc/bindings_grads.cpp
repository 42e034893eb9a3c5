// Torch binding of the gradients' norm and clipping: grads.norm, grads.clip.
// Errors surface as RuntimeError; launches go to torch's current HIP stream of
// the tensors' device.
#include <c10/hip/HIPCachingAllocator.h>

#include "bindings_common.hpp"

namespace {

// A tensor whose elements fill one piece of memory, in any order, and stand for
// themselves alone: a forward-mode tangent would not be carried along.
void check_dense(const Tensor& t, const Tensor& first, const char* name, size_t i) {
    TORCH_CHECK(!t._fw_grad(0).defined(), name, "[", i, "] has a forward-mode tangent, which the norm and the clipping do not carry");
    TORCH_CHECK(t.is_cuda() && t.device() == first.device(), name, "[", i, "] must be a GPU tensor on the others' device");
    TORCH_CHECK(t.is_non_overlapping_and_dense(), name, "[", i, "] must fill its memory without gaps or overlaps");
}

struct Call {
    std::vector<gdn_grad_t> grads;
    Tensor norm;
    c10::DataPtr workspace;  // the allocator's own: a tensor costs more host time
    size_t bytes = 0;
};
Call call_of(const std::vector<Tensor>& grads) {
    TORCH_CHECK(!grads.empty(), "grads: no tensors");
    Call c;
    c.grads.resize(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor& t = grads[i];
        check_dense(t, grads[0], "grads", i);
        c.grads[i] = {t.data_ptr(), nullptr, t.numel(), type_of(t, "grads"), GDN_BF16};
    }
    return c;
}
void allocate(Call& c, const Tensor& t) {
    c.norm = fresh({}, at::kFloat, t);
    c.bytes = gdn_grad_norm_workspace_bytes(static_cast<int64_t>(c.grads.size()));
    c.workspace = c10::hip::HIPCachingAllocator::get()->allocate(c.bytes);
}

Tensor norm(const std::vector<Tensor>& grads) {
    Call c = call_of(grads);
    const c10::DeviceGuard guard(grads[0].device());
    allocate(c, grads[0]);
    check_status(gdn_grad_norm_hip(c.grads.data(), static_cast<int64_t>(c.grads.size()), c.norm.data_ptr<float>(), c.workspace.get(), c.bytes,
                                   stream_of(grads[0])),
                 "grad_norm");
    return c.norm;
}

// Whether the elements of two tensors of one shape lie in the same order.
bool same_order(const Tensor& a, const Tensor& b) {
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
    return true;
}

Tensor clip(const std::vector<Tensor>& grads, double max_norm, const std::optional<std::vector<Tensor>>& out) {
    TORCH_CHECK(max_norm >= 0, "max_norm must be at least 0, got ", max_norm);
    Call c = call_of(grads);
    const std::vector<Tensor>& to = out ? *out : grads;
    TORCH_CHECK(to.size() == grads.size(), grads.size(), " grads and ", to.size(), " out");
    for (size_t i = 0; i < to.size(); ++i) {
        const Tensor& t = to[i];
        TORCH_CHECK(!at::GradMode::is_enabled() || !t.requires_grad(), "clip would write over a tensor that requires grad (no gradients are recorded here): tensor ", i);
        if (out) {
            check_dense(t, grads[0], "out", i);
            TORCH_CHECK(t.sizes() == grads[i].sizes() && (t.numel() == 0 || same_order(t, grads[i])), "out[", i, "] must have grads[", i, "]'s shape and order of axes");
        }
        c.grads[i].out = t.data_ptr();
        c.grads[i].type_out = type_of(t, "out");
    }
    const c10::DeviceGuard guard(grads[0].device());
    allocate(c, grads[0]);
    check_status(gdn_clip_grad_norm_hip(c.grads.data(), static_cast<int64_t>(c.grads.size()), max_norm, c.norm.data_ptr<float>(),
                                        c.workspace.get(), c.bytes, stream_of(grads[0])),
                 "clip_grad_norm");
    for (const Tensor& t : to)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // a graph that saved it raises
    return c.norm;
}

}  // namespace

void bind_grad_ops(pybind11::module_& grads) {
    namespace py = pybind11;
    grads.def("norm", &norm,
              "The 2-norm of all tensors' elements together (a list of bf16 and fp32 tensors on one GPU, each filling its memory), a float32 "
              "tensor of no axes.  Sums in 64 bits, in a fixed order; an element counts as often as it is given.",
              py::arg("grads"));
    grads.def("clip", &clip,
              "grads times min(1, max_norm / (norm + 1e-6)), in place or into out (tensors of the same shapes and orders of axes, bf16 or fp32); "
              "returns the norm before.  What is written may not share memory with another tensor of the call.  Counts as an in-place "
              "operation on what it writes.",
              py::arg("grads"), py::arg("max_norm"), py::arg("out") = py::none());
}

// Compiled binding of litegs_amd/stochastic.py (host-only C++ over the C ABI): outputs and workspaces from ATen, launches on torch's current
// HIP stream, dropout's gradient as a C++ autograd node.  Through Python's autograd and ctypes a forward and a backward pass of dropout
// took 120 us of host time, here 42 (the engine alone takes 34 for a product with a constant); arguments are checked by the Python functions, which also work without this module.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <mutex>
#include <optional>
#include "litegs_hip.h"

namespace {

using at::Tensor;
typedef std::optional<Tensor> OptTensor;

inline void* cur_stream() { return (void*)c10::hip::getCurrentHIPStream().stream(); }
inline void check(int rc, const char* what) { TORCH_CHECK(rc == 0, "litegs_amd: ", what, " failed with hipError ", rc); }

inline int dtype_code(const Tensor& t, const char* what)
{
    switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: TORCH_CHECK(false, what, ": float32, float16 or bfloat16 GPU tensor required (no CPU path)");
    }
    return -1;
}
inline const int64_t* words(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr<int64_t>() : nullptr; }

// Whether torch's calls are being recorded (a trace, a proxy or functional mode) or only their shapes worked out (a fake mode).  The kernels here
// write into empty tensors behind the dispatcher's back, so that a recording would hold the empty tensor alone.
bool traced()
{
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    if (torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) return true;
    return Modes::stack_len() > 0 && (Modes::get_mode(Key::PROXY).has_value() || Modes::get_mode(Key::FAKE).has_value() || Modes::get_mode(Key::FUNCTIONAL).has_value());
}

struct Mask {                          // which elements a call keeps: the arguments of lg_dropout behind the type
    int64_t lead, M;
    double p;
    int64_t seed, offset, S;
};

Tensor dropout(const Tensor& x, const Mask& m, const OptTensor& offset_dev, const OptTensor& chunk_ids);

// A linear map that is its own transpose: the gradient is the same call on the gradient, to any order.  A node of its own and no
// torch::autograd::Function, whose context (a dictionary of boxed values) took as long as the launch.
struct DropoutBackward : public torch::autograd::Node {
    Mask mask;
    bool by_tensor = false, by_chunk = false;
    torch::autograd::SavedVariable offset_dev, chunk_ids;              // a step counter advanced in between is reported by autograd, not used

    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[0].defined()) return { Tensor() };
        return { dropout(grads[0], mask, by_tensor ? OptTensor(offset_dev.unpack()) : OptTensor(), by_chunk ? OptTensor(chunk_ids.unpack()) : OptTensor()) };
    }
    void release_variables() override
    {
        std::lock_guard<std::mutex> lock(mutex_);
        offset_dev.reset_data();
        chunk_ids.reset_data();
    }
    std::string name() const override { return "DropoutBackward"; }
};

Tensor dropout(const Tensor& x, const Mask& m, const OptTensor& offset_dev, const OptTensor& chunk_ids)
{
    TORCH_CHECK(!torch::autograd::isFwGradDefined(x), "dropout: no forward-mode derivative");
    TORCH_CHECK(!traced(), "dropout: cannot be traced (the kernel would not be part of the trace)");        // (a backward pass comes here without the Python function)
    const bool graph = at::GradMode::is_enabled() && x.requires_grad();
    Tensor y;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        const c10::OptionalDeviceGuard guard(at::device_of(x));
        const Tensor c = x.contiguous();
        y = at::empty(c.sizes(), c.options());
        check(lg_dropout(c.data_ptr(), y.data_ptr(), dtype_code(c, "dropout"), m.lead, m.M, m.p, m.seed, m.offset, words(offset_dev), words(chunk_ids), (int)m.S, cur_stream()), "dropout");
    }
    if (graph) {
        std::shared_ptr<DropoutBackward> node(new DropoutBackward(), torch::autograd::deleteNode);
        node->mask = m;
        node->by_tensor = offset_dev.has_value();
        node->by_chunk = chunk_ids.has_value();
        if (node->by_tensor) node->offset_dev = torch::autograd::SavedVariable(*offset_dev, false);
        if (node->by_chunk) node->chunk_ids = torch::autograd::SavedVariable(*chunk_ids, false);
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        torch::autograd::set_history(y, node);
    }
    return y;
}

Tensor dropout_call(const Tensor& x, int64_t lead, int64_t M, double p, int64_t seed, int64_t offset, const OptTensor& offset_dev, const OptTensor& chunk_ids, int64_t S)
{
    return dropout(x, Mask{ lead, M, p, seed, offset, S }, offset_dev, chunk_ids);
}

// std: normal draws into `out`, else uniform ones
void random_draw(const OptTensor& std_, Tensor out, int64_t seed, int64_t offset, const OptTensor& offset_dev)
{
    const c10::OptionalDeviceGuard guard(at::device_of(out));
    check(lg_random_draw(std_.has_value() ? std_->data_ptr() : nullptr, out.data_ptr(), dtype_code(out, "random_draw"), out.numel(), seed, offset, words(offset_dev), cur_stream()), "random_draw");
}

void sample(const Tensor& scores, const Tensor& u, Tensor out, int64_t n, bool distinct, bool logits, double temperature, int64_t top_k, double top_p, double min_p)
{
    const c10::OptionalDeviceGuard guard(at::device_of(scores));
    const int64_t R = scores.size(0), V = scores.size(1);
    const long long bytes = lg_sample_temp_bytes(R, V, n, dtype_code(scores, "sample"), distinct, top_k, top_p);
    Tensor temp;
    if (bytes) temp = at::empty({ bytes }, scores.options().dtype(at::kByte));
    check(lg_sample(scores.data_ptr(), dtype_code(scores, "sample"), scores.stride(0), (const float*)u.data_ptr(), u.stride(0), R, V, n, distinct, logits, temperature, top_k,
                    top_p, min_p, out.data_ptr<int64_t>(), bytes ? temp.data_ptr() : nullptr, bytes, cur_stream()), distinct ? "sample_distinct" : "sample");
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("traced", &traced);
    m.def("dropout", &dropout_call);
    m.def("random_draw", &random_draw);
    m.def("sample", &sample);
}

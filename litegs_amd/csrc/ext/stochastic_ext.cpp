// Compiled binding of litegs_amd/stochastic.py (host-only C++ over the C ABI): outputs and workspaces from ATen, launches on torch's current
// HIP stream, dropout's gradient as a C++ autograd function.  Through Python's autograd and ctypes a forward and a backward pass of dropout
// took 120 us of host time, here 47 (the engine alone takes 36 for a product with a constant); arguments are checked by the Python functions, which also work without this module.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
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

// a linear map that is its own transpose: the gradient is the same call on the gradient, to any order
struct Dropout : public torch::autograd::Function<Dropout> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, int64_t lead, int64_t M, double p, int64_t seed, int64_t offset,
                          const OptTensor& offset_dev, const OptTensor& chunk_ids, int64_t S)
    {
        ctx->saved_data["k"] = std::vector<int64_t>{ lead, M, seed, offset, S };
        ctx->saved_data["p"] = p;
        // a step counter advanced in between is reported by autograd, not used
        ctx->save_for_backward({ offset_dev.has_value() ? *offset_dev : Tensor(), chunk_ids.has_value() ? *chunk_ids : Tensor() });
        const c10::OptionalDeviceGuard guard(at::device_of(x));
        const Tensor c = x.contiguous();
        Tensor y = at::empty(c.sizes(), c.options());
        check(lg_dropout(c.data_ptr(), y.data_ptr(), dtype_code(c, "dropout"), lead, M, p, seed, offset, words(offset_dev), words(chunk_ids), (int)S, cur_stream()), "dropout");
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        const std::vector<int64_t> k = ctx->saved_data["k"].toIntVector();
        const torch::autograd::variable_list saved = ctx->get_saved_variables();
        auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        const Tensor none;
        Tensor g = Dropout::apply(grads[0], k[0], k[1], ctx->saved_data["p"].toDouble(), k[2], k[3], opt(saved[0]), opt(saved[1]), k[4]);
        return { g, none, none, none, none, none, none, none, none };
    }
};

Tensor dropout(const Tensor& x, int64_t lead, int64_t M, double p, int64_t seed, int64_t offset, const OptTensor& offset_dev, const OptTensor& chunk_ids, int64_t S)
{
    return Dropout::apply(x, lead, M, p, seed, offset, offset_dev, chunk_ids, S);
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
    m.def("dropout", &dropout);
    m.def("random_draw", &random_draw);
    m.def("sample", &sample);
}

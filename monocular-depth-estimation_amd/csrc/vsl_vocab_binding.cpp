// The Python package's side of include/vsloss_vocab_torch.h.  The library's functions are not linked in: they come from
// the libvsloss.so that the package has loaded.
#include <torch/extension.h>
#include <torch/csrc/Exceptions.h>

#include "vsloss_vocab_torch.h"

namespace {

// Without the interpreter's lock; ValueError for malformed arguments, torch's own errors as torch raises them, the
// package's error for what the library returns.
template <typename F>
auto run(const char* module, F&& call) {
  HANDLE_TH_ERRORS
  try {
    const py::gil_scoped_release no_gil;
    return call();
  } catch (const std::runtime_error& e) {
    const std::string text = e.what();
    PyErr_SetString(py::module_::import(module).attr("VslError").ptr(), text.c_str());
    throw py::error_already_set();
  }
  END_HANDLE_TH_ERRORS_PYBIND
}

}  // namespace

PYBIND11_MODULE(vsl_vocab_binding, m) {
  static std::string abi;   // the module that holds VslError
  m.def("errors_from", [](const std::string& name) { abi = name; });
  m.def("top_logits", [](const torch::Tensor& logits, int64_t k, double temperature) {
    return run(abi.c_str(), [&] { return vsl::top_logits(logits, k, temperature); });
  });
  m.def("topk_distillation_loss", [](const torch::Tensor& logits, const torch::Tensor& values, const torch::Tensor& indices,
                                     const std::optional<torch::Tensor>& lse, double temperature,
                                     const std::optional<torch::Tensor>& weights, const std::string& reduction) {
    return run(abi.c_str(), [&] { return vsl::topk_distillation_loss(logits, values, indices, lse, temperature, weights, reduction); });
  });
  m.def("linear_cross_entropy", [](const torch::Tensor& hidden, const torch::Tensor& weight, const torch::Tensor& target,
                                   const std::optional<torch::Tensor>& bias, int64_t ignore_index, double z_loss,
                                   const std::string& reduction) {
    return run(abi.c_str(), [&] { return vsl::linear_cross_entropy(hidden, weight, target, bias, ignore_index, z_loss, reduction); });
  });
}

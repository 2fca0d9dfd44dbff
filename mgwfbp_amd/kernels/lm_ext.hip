// Python bindings of the language-model kernels.
#include <torch/extension.h>

#include <tuple>
#include <vector>

namespace mgx {

torch::Tensor grad_norm(const std::vector<torch::Tensor>& grads);
std::tuple<std::vector<torch::Tensor>, torch::Tensor> clip_grads(
    const std::vector<torch::Tensor>& grads, double max_norm, double eps);
torch::Tensor clip_grads_(const std::vector<torch::Tensor>& grads,
                          double max_norm, double eps);

}  // namespace mgx

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("grad_norm", &mgx::grad_norm, "L2 norm over a list of gradients");
  m.def("clip_grads", &mgx::clip_grads,
        "New gradients scaled to a global norm, and the norm");
  m.def("clip_grads_", &mgx::clip_grads_,
        "Scale gradients in place to a global norm; returns the norm");
}

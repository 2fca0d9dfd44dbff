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

torch::Tensor embedding(const torch::Tensor& tokens,
                        const torch::Tensor& weight, double scale,
                        int64_t padding, bool twice);
torch::Tensor cross_entropy(const torch::Tensor& logits,
                            const torch::Tensor& targets, int64_t ignore,
                            int64_t reduction, bool scaled, bool twice);
std::vector<torch::Tensor> token_log_probs(const torch::Tensor& logits,
                                           const torch::Tensor& targets,
                                           int64_t k, int64_t ignore);

}  // namespace mgx

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("grad_norm", &mgx::grad_norm, "L2 norm over a list of gradients");
  m.def("clip_grads", &mgx::clip_grads,
        "New gradients scaled to a global norm, and the norm");
  m.def("clip_grads_", &mgx::clip_grads_,
        "Scale gradients in place to a global norm; returns the norm");
  m.def("embedding", &mgx::embedding,
        "Rows of a table by token, scaled (differentiable)",
        py::arg("tokens"), py::arg("weight"), py::arg("scale"),
        py::arg("padding"), py::arg("twice") = false);
  m.def("cross_entropy", &mgx::cross_entropy,
        "Cross entropy of logits and class indices (differentiable)",
        py::arg("logits"), py::arg("targets"), py::arg("ignore"),
        py::arg("reduction"), py::arg("scaled"), py::arg("twice") = false);
  m.def("token_log_probs", &mgx::token_log_probs,
        "Log probabilities of given tokens, entropy, best alternatives");
}

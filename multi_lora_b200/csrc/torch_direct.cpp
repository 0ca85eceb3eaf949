// The operators of the paged serving step as functions of a Python module (_mlora_direct.so): the same C++ functions as
// torch.ops.mlora.* without the dispatcher's argument handling. A library of its own, since it needs
// Python and the operators' library (_mlora_torch.so) does not.
#include <torch/csrc/utils/pybind.h>

#include "torch_ops_paged.h"

PYBIND11_MODULE(_mlora_direct, m) {
  m.def("plan_paged_step", &mlora_torch::plan_paged_step);
  m.def("write_paged_kv", &mlora_torch::write_paged_kv);
  m.def("paged_attention", &mlora_torch::paged_attention);
  m.def("verify_draft", &mlora_torch::verify_draft);
}

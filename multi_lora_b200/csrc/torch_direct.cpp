// The operators of the paged serving step as functions of a Python module (_mlora_direct.so): the same C++ functions as
// torch.ops.mlora.* without the dispatcher's argument handling. A library of its own, since it needs
// Python and the operators' library (_mlora_torch.so) does not.
//
// Where the dispatcher would do more than call that function (a dispatch mode, a tensor subclass, a profiler, a graph
// for gradients), the call goes through it.
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/utils/pybind.h>

#include "torch_ops_paged.h"

namespace {

// A call runs without the GIL: a launch waits where the queue of launches is full. (0.1 to 0.2 us a call; pybind11's
// own guard looks its thread state up besides.)
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

struct Seen {
  c10::DispatchKeySet keys;
  bool requires_grad = false;
};
void look(Seen& s, const at::Tensor& t) {
  s.keys = s.keys | t.key_set();
  s.requires_grad |= t.requires_grad();
}
void look(Seen& s, const c10::optional<at::Tensor>& t) {
  if (t.has_value()) look(s, *t);
}
template <typename T>
void look(Seen&, const T&) {}  // a number

// Keys of plain CUDA tensors: for these the dispatcher has the CUDA function, or passes on to it.
constexpr c10::DispatchKeySet kPlain({c10::DispatchKey::Dense, c10::DispatchKey::BackendSelect,
                                      c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutogradFunctionality,
                                      c10::DispatchKey::AutocastCUDA});

// `graph`: whether a result could be part of a graph. The step's whole numbers and the cache, which
// would hold the graphs of all steps together, are not.
template <typename R, typename... A>
auto either(R (*fn)(A...), const char* name, bool graph) {
  const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<R(A...)>();
  // Arguments come by reference and are copied where the function takes a copy: a tensor's second reference
  // comes and goes with the GIL, which costs a call without it that destroys one 0.4 us.
  return [fn, op, graph](const std::decay_t<A>&... a) -> R {
    Seen s;
    (look(s, a), ...);
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    const auto more = ((s.keys | tls.included_) - tls.excluded_) - kPlain;
    if (graph && s.requires_grad && at::GradMode::is_enabled()) return op.call(a...);
    if (more.highestFunctionalityKey() == c10::DispatchKey::Undefined && !at::hasCallbacks())
      return fn(a...);
    if (graph) return op.call(a...);
    const at::AutoDispatchBelowADInplaceOrView no_graph;
    return op.call(a...);
  };
}

}  // namespace

PYBIND11_MODULE(_mlora_direct, m) {
  const auto def = [&](const char* name, auto fn) { m.def(name, fn, pybind11::call_guard<NoGil>()); };
  def("plan_paged_step", either(&mlora_torch::plan_paged_step, "mlora::plan_paged_step", false));
  def("write_paged_kv", either(&mlora_torch::write_paged_kv, "mlora::write_paged_kv", false));
  def("paged_attention", either(&mlora_torch::paged_attention, "mlora::paged_attention", true));
  def("verify_draft", either(&mlora_torch::verify_draft, "mlora::verify_draft", false));
}

// text_nodes.cpp — host-side help for the text encoder's operators (attention.py, dense.rms_norm_residual).
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/extension.h>

#include "torch_nodes.h"

namespace irxn {

// The first of `leaves` whose gradient accumulator lives on another stream than the current one of its device, or -1. The autograd engine
// makes an accumulator's stream wait for the backward that feeds it, and the accumulator keeps the stream of the first graph that used the
// leaf for as long as any such graph lives. Inside a capture that wait would draw a stream that is not being captured into it: the runtime
// ends the process when the capture ends.
static int64_t foreign_leaf(const std::vector<c10::optional<at::Tensor>>& leaves) {
  for (size_t i = 0; i < leaves.size(); ++i) {
    const auto& t = leaves[i];
    if (!t.has_value() || !t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto acc = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!acc) continue;
    const auto s = acc->stream();
    if (s.has_value() && *s != c10::impl::VirtualGuardImpl(t->device().type()).getStream(t->device())) return (int64_t)i;
  }
  return -1;
}

void register_text(pybind11::module& m) { m.def("foreign_leaf", &foreign_leaf); }

}  // namespace irxn

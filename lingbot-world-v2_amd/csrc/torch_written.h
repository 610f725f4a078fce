// torch.ops.lbw: an op that writes into tensors of its caller counts the write in their versions, so that a
// backward pass which saved one of them before raises instead of computing with what was written over it.
#pragma once

#include <ATen/ATen.h>
#include <torch/library.h>

#include <array>
#include <string>

namespace {

template <typename T>
void count_write(bool, const T&) {}
inline void count_write(bool written, const at::Tensor& t) {
  // (tensors of inference mode have no version)
  if (written && t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
inline void count_write(bool written, const std::optional<at::Tensor>& t) {
  if (t.has_value()) count_write(written, *t);
}

// The ADInplaceOrView kernel of an op: the op below it, then one more version for each argument that its schema
// marks as written. `f` is its GPU kernel, for the argument types.
template <typename F, F* f>
struct CountWrites;
template <typename... A, void (*f)(A...)>
struct CountWrites<void(A...), f> {
  static std::string& name() {
    static std::string n;
    return n;
  }
  static void call(c10::DispatchKeySet ks, A... a) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name().c_str(), "").typed<void(A...)>();
    static const auto written = [] {
      std::array<bool, sizeof...(A)> w{};
      for (size_t i = 0; i < w.size(); ++i) {
        const auto* alias = op.schema().arguments()[i].alias_info();
        w[i] = alias != nullptr && alias->isWrite();
      }
      return w;
    }();
    op.redispatch(ks & c10::after_ADInplaceOrView_keyset, a...);
    size_t i = 0;
    (count_write(written[i++], a), ...);
  }
  static void add(torch::Library& m, const char* op) {
    name() = std::string("lbw::") + op;
    m.impl(op, TORCH_FN(call));
  }
};
#define LBW_COUNT_WRITES(m, op) CountWrites<decltype(op), &op>::add(m, #op)

}  // namespace

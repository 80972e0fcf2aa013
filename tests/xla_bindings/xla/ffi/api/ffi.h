// The stub of XLA's FFI API (tests/xla_stub) with its registrations: as XLA's own, a handler's
// binding lists what the call decodes (its context, operands, attributes and results, in their
// order), and the handler has to take exactly those. Checked when it is compiled.
#pragma once

#include <type_traits>

#include "../../../../xla_stub/xla/ffi/api/ffi.h"

namespace xla::ffi {

template <typename T>
struct Context;
template <typename T>
struct Context<PlatformStream<T>> {
  using type = T;
};

template <typename... Ts>
struct Binding {
  using Handler = Error(Ts...);
  template <typename T>
  Binding<Ts..., typename Context<T>::type> Ctx();
  template <typename T>
  Binding<Ts..., T> Arg();
  template <typename T>
  Binding<Ts..., T> Attr(const char* name);
  template <typename T>
  Binding<Ts..., Result<T>> Ret();
  Binding<Ts..., xla::ffi::RemainingArgs> RemainingArgs();
  Binding<Ts..., xla::ffi::RemainingRets> RemainingRets();
};
struct Ffi {
  static Binding<> Bind();
};

}  // namespace xla::ffi

#undef XLA_FFI_DEFINE_HANDLER_SYMBOL
#define XLA_FFI_DEFINE_HANDLER_SYMBOL(name, impl, binding)                     \
  static_assert(std::is_same_v<decltype(binding)::Handler, decltype(impl)>, \
                #name ": the binding is not its handler's")

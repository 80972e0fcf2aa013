// The names of XLA's FFI API that bux_amd/xla/xla_ffi.cc uses, with just enough behind them
// to call its handlers as functions on buffers a test makes up. A handler's registration
// expands to nothing.
#pragma once

#include <cstddef>
#include <cstdint>
#include <optional>
#include <string>
#include <utility>
#include <vector>

namespace xla::ffi {

enum class DataType { U8, S32, BF16, F32 };
enum class ErrorCode { kOk, kInvalidArgument, kInternal };

class Error {
 public:
  Error(ErrorCode code, std::string message) : code_(code), message_(std::move(message)) {}
  static Error Success() { return Error(ErrorCode::kOk, ""); }
  bool success() const { return code_ == ErrorCode::kOk; }
  ErrorCode errc() const { return code_; }
  const std::string& message() const { return message_; }

 private:
  ErrorCode code_;
  std::string message_;
};

class AnyBuffer {
 public:
  AnyBuffer(DataType type, std::vector<int64_t> dims, void* data = nullptr)
      : type_(type), dims_(std::move(dims)), data_(data) {}
  DataType element_type() const { return type_; }
  const std::vector<int64_t>& dimensions() const { return dims_; }
  size_t element_count() const {
    size_t n = 1;
    for (int64_t d : dims_) n *= static_cast<size_t>(d);
    return n;
  }
  size_t size_bytes() const {
    return element_count() * (type_ == DataType::U8 ? 1 : type_ == DataType::BF16 ? 2 : 4);
  }
  void* untyped_data() const { return data_; }

 private:
  DataType type_;
  std::vector<int64_t> dims_;
  void* data_;
};

template <typename T>
class Result {
 public:
  Result(T value) : value_(std::move(value)) {}
  T* operator->() { return &value_; }
  T& operator*() { return value_; }

 private:
  T value_;
};

template <typename T>
struct PlatformStream {};

template <typename T>
class ErrorOr {
 public:
  ErrorOr(T value) : value_(std::move(value)), has_(true) {}
  ErrorOr() = default;
  bool has_value() const { return has_; }
  T& value() { return *value_; }

 private:
  std::optional<T> value_;
  bool has_ = false;
};

// A handler's operands and results past its named ones.
class RemainingArgs {
 public:
  explicit RemainingArgs(std::vector<AnyBuffer> buffers) : buffers_(std::move(buffers)) {}
  size_t size() const { return buffers_.size(); }
  template <typename T>
  ErrorOr<T> get(size_t i) const {
    return i < buffers_.size() ? ErrorOr<T>(buffers_[i]) : ErrorOr<T>();
  }

 private:
  std::vector<AnyBuffer> buffers_;
};
class RemainingRets {
 public:
  explicit RemainingRets(std::vector<AnyBuffer> buffers) : buffers_(std::move(buffers)) {}
  size_t size() const { return buffers_.size(); }
  template <typename T>
  ErrorOr<Result<T>> get(size_t i) const {
    return i < buffers_.size() ? ErrorOr<Result<T>>(Result<T>(buffers_[i])) : ErrorOr<Result<T>>();
  }

 private:
  std::vector<AnyBuffer> buffers_;
};

}  // namespace xla::ffi

#define XLA_FFI_DEFINE_HANDLER_SYMBOL(name, impl, binding)

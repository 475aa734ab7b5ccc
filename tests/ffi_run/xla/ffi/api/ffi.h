// TEST STAND-IN, not XLA's header: buffers with dimensions, so that the handlers of train_gpt_b200/xla_ffi/xla_ffi.cc can be CALLED on a
// machine without jaxlib (tests/ffi_stub is the one that checks their types).
#pragma once
#include <cstddef>
#include <cstdint>
#include <string>
#include <utility>
#include <vector>

namespace xla::ffi {

enum DataType { BF16, F8E4M3FN, F32, S32, U8, U32 };
enum class ErrorCode { kOk, kInvalidArgument, kInternal };

class Error {
 public:
  Error() = default;
  Error(ErrorCode c, std::string m) : code(c), message(std::move(m)) {}
  static Error Success() { return Error(); }
  ErrorCode code = ErrorCode::kOk;
  std::string message;
};

template <typename T>
struct Span {
  const T* p = nullptr;
  size_t n = 0;
  size_t size() const { return n; }
  const T& operator[](size_t i) const { return p[i]; }
  const T& back() const { return p[n - 1]; }
};

template <DataType> struct NativeOf { using type = uint8_t; };
template <> struct NativeOf<F32> { using type = float; };
template <> struct NativeOf<S32> { using type = int32_t; };
template <> struct NativeOf<U32> { using type = uint32_t; };
template <> struct NativeOf<BF16> { using type = uint16_t; };

template <DataType D>
class Buffer {
 public:
  using Native = typename NativeOf<D>::type;
  Buffer() = default;
  Buffer(std::vector<int64_t> d) : dims_(std::move(d)) {}
  Span<int64_t> dimensions() const { return {dims_.data(), dims_.size()}; }
  size_t element_count() const {
    size_t n = 1;
    for (int64_t d : dims_) n *= size_t(d);
    return n;
  }
  void* untyped_data() const { return reinterpret_cast<void*>(4096); }
  Native* typed_data() const { return reinterpret_cast<Native*>(4096); }

 private:
  std::vector<int64_t> dims_;
};

template <typename T>
class Result {
 public:
  Result(std::vector<int64_t> d) : v_(std::move(d)) {}
  T* operator->() { return &v_; }
  T& operator*() { return v_; }

 private:
  T v_;
};
template <DataType D> using ResultBuffer = Result<Buffer<D>>;
template <typename T> struct PlatformStream {};

}  // namespace xla::ffi

#define XLA_FFI_DEFINE_HANDLER_SYMBOL(name, impl, binding)

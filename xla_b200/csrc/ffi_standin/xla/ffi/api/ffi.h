// Stand-in for the C++ side of XLA's FFI, for builds without an XLA checkout: the classes through which
// ffi_handlers.cc reads a call frame, over the declarations of c_api.h beside this file.
#ifndef B200SD_FFI_STANDIN_FFI_H_
#define B200SD_FFI_STANDIN_FFI_H_

#include <cstdio>
#include <cstring>
#include <exception>
#include <initializer_list>
#include <optional>
#include <string>
#include <string_view>
#include <type_traits>
#include <utility>

#include "xla/ffi/api/c_api.h"

namespace xla::ffi {

enum class ErrorCode : int {};

class Error {
 public:
  Error() = default;
  Error(ErrorCode code, std::string message) : code_(static_cast<int>(code)), message_(std::move(message)) {}
  static Error Success() { return Error(); }
  bool failure() const { return code_ != 0; }
  int code() const { return code_; }
  const std::string& message() const { return message_; }

 private:
  int code_ = 0;
  std::string message_;
};

template <typename T>
class ErrorOr {
 public:
  ErrorOr(T value) : value_(std::move(value)) {}   // NOLINT: implicit, as is usual for such a type
  ErrorOr(Error error) : error_(std::move(error)) {}
  bool has_value() const { return value_.has_value(); }
  const Error& error() const { return error_; }
  const T& operator*() const { return *value_; }
  const T* operator->() const { return &*value_; }

 private:
  std::optional<T> value_;
  Error error_;
};

template <typename T>
class Span {
 public:
  Span(T* data, size_t size) : data_(data), size_(size) {}
  size_t size() const { return size_; }
  T& operator[](size_t i) const { return data_[i]; }
  T* begin() const { return data_; }
  T* end() const { return data_ + size_; }

 private:
  T* data_;
  size_t size_;
};

enum class DataType : int32_t {
  S8 = XLA_FFI_DataType_S8,
  S32 = XLA_FFI_DataType_S32,
  U8 = XLA_FFI_DataType_U8,
  F16 = XLA_FFI_DataType_F16,
  F32 = XLA_FFI_DataType_F32,
  BF16 = XLA_FFI_DataType_BF16,
  F8E5M2 = XLA_FFI_DataType_F8E5M2,
  F8E4M3FN = XLA_FFI_DataType_F8E4M3FN,
  F8E8M0FNU = XLA_FFI_DataType_F8E8M0FNU,
};

class AnyBuffer {
 public:
  explicit AnyBuffer(const XLA_FFI_Buffer* b) : b_(b) {}
  DataType element_type() const { return static_cast<DataType>(b_->dtype); }
  Span<const int64_t> dimensions() const { return {b_->dims, static_cast<size_t>(b_->rank)}; }
  void* untyped_data() const { return b_->data; }
  size_t element_count() const {
    size_t n = 1;
    for (int64_t d : dimensions()) n *= static_cast<size_t>(d);
    return n;
  }
  size_t size_bytes() const {
    switch (b_->dtype) {
      case XLA_FFI_DataType_S64: case XLA_FFI_DataType_F64: return 8 * element_count();
      case XLA_FFI_DataType_S32: case XLA_FFI_DataType_F32: return 4 * element_count();
      case XLA_FFI_DataType_F16: case XLA_FFI_DataType_BF16: return 2 * element_count();
      default: return element_count();
    }
  }

 private:
  const XLA_FFI_Buffer* b_;
};

class RemainingArgs {
 public:
  explicit RemainingArgs(const XLA_FFI_Args* a) : a_(a) {}
  size_t size() const { return static_cast<size_t>(a_->size); }
  template <typename T>
  ErrorOr<AnyBuffer> get(size_t i) const {
    if (i >= size()) return Error(static_cast<ErrorCode>(3), "operand " + std::to_string(i) + " is missing");
    return AnyBuffer(static_cast<const XLA_FFI_Buffer*>(a_->args[i]));
  }

 private:
  const XLA_FFI_Args* a_;
};

// A result; dereferenced to the buffer it is written to.
class ResultBuffer {
 public:
  explicit ResultBuffer(AnyBuffer b) : b_(b) {}
  const AnyBuffer& operator*() const { return b_; }
  const AnyBuffer* operator->() const { return &b_; }

 private:
  AnyBuffer b_;
};

class RemainingRets {
 public:
  explicit RemainingRets(const XLA_FFI_Rets* r) : r_(r) {}
  size_t size() const { return static_cast<size_t>(r_->size); }
  template <typename T>
  ErrorOr<ResultBuffer> get(size_t i) const {
    if (i >= size()) return Error(static_cast<ErrorCode>(3), "result " + std::to_string(i) + " is missing");
    return ResultBuffer(AnyBuffer(static_cast<const XLA_FFI_Buffer*>(r_->rets[i])));
  }

 private:
  const XLA_FFI_Rets* r_;
};

class Dictionary {
 public:
  explicit Dictionary(const XLA_FFI_Attrs* a) : a_(a) {}
  template <typename T>
  bool contains(std::string_view name) const { return get<T>(name).has_value(); }
  template <typename T>
  ErrorOr<T> get(std::string_view name) const {
    for (int64_t i = 0; i < a_->size; ++i) {
      if (std::string_view(a_->names[i]->ptr, a_->names[i]->len) != name) continue;
      if constexpr (std::is_same_v<T, Span<const int64_t>>) {
        if (a_->types[i] != XLA_FFI_AttrType_ARRAY) break;
        const auto* v = static_cast<const XLA_FFI_Array*>(a_->attrs[i]);
        if (v->dtype != XLA_FFI_DataType_S64) break;
        return T(static_cast<const int64_t*>(v->data), v->size);
      } else {
        if (a_->types[i] != XLA_FFI_AttrType_SCALAR) break;
        const auto* v = static_cast<const XLA_FFI_Scalar*>(a_->attrs[i]);
        if (v->dtype != TypeOf<T>()) break;
        T out;
        std::memcpy(&out, v->value, sizeof(T));
        return out;
      }
    }
    return Error(static_cast<ErrorCode>(3), "no attribute " + std::string(name) + " of the type asked for");
  }

 private:
  template <typename T>
  static constexpr XLA_FFI_DataType TypeOf() {
    if constexpr (std::is_same_v<T, bool>) return XLA_FFI_DataType_PRED;
    else if constexpr (std::is_same_v<T, int32_t>) return XLA_FFI_DataType_S32;
    else if constexpr (std::is_same_v<T, int64_t>) return XLA_FFI_DataType_S64;
    else if constexpr (std::is_same_v<T, float>) return XLA_FFI_DataType_F32;
    else return XLA_FFI_DataType_F64;
  }
  const XLA_FFI_Attrs* a_;
};

enum class Traits : uint32_t { kCmdBufferCompatible = XLA_FFI_HANDLER_TRAITS_COMMAND_BUFFER_COMPATIBLE };
template <typename Stream>
struct PlatformStream {};

// What a handler is bound to: its stage, and nothing more -- the parameters of the function say what it takes.
struct Binding {
  XLA_FFI_ExecutionStage stage;
  template <typename T>
  constexpr Binding Ctx() const { return *this; }
  constexpr Binding RemainingArgs() const { return *this; }
  constexpr Binding RemainingRets() const { return *this; }
  constexpr Binding Attrs() const { return *this; }
};
inline uint32_t TraitBits(std::initializer_list<Traits> traits = {}) {
  uint32_t bits = 0;
  for (Traits t : traits) bits |= static_cast<uint32_t>(t);
  return bits;
}

struct Ffi {
  static constexpr Binding Bind() { return {XLA_FFI_ExecutionStage_EXECUTE}; }
  static constexpr Binding BindInstantiate() { return {XLA_FFI_ExecutionStage_INSTANTIATE}; }
  static constexpr Binding BindInitialize() { return {XLA_FFI_ExecutionStage_INITIALIZE}; }
  static XLA_FFI_Error* RegisterStaticHandler(const XLA_FFI_Api* api, std::string_view name, std::string_view platform,
                                              XLA_FFI_Handler_Bundle bundle, XLA_FFI_Handler_Traits traits) {
    XLA_FFI_Handler_Register_Args a{};
    a.struct_size = sizeof(a);
    a.name = {name.data(), name.size()};
    a.platform = {platform.data(), platform.size()};
    a.bundle = bundle;
    a.traits = traits;
    return api->XLA_FFI_Handler_Register(&a);
  }
};

inline XLA_FFI_Error* Report(const XLA_FFI_Api* api, int code, const char* message) {
  XLA_FFI_Error_Create_Args a{};
  a.struct_size = sizeof(a);
  a.message = message;
  a.errc = static_cast<XLA_FFI_Error_Code>(code);
  return api->XLA_FFI_Error_Create(&a);
}

// One call of a handler.  No exception leaves it.  A frame of another layout is not read, not even for what an error would
// have to be made with: a runtime that asks the handler for its version, as all do before they register one, gets none and
// refuses it.
template <typename Fn>
XLA_FFI_Error* Invoke(const XLA_FFI_CallFrame* f, Fn fn, Binding binding, uint32_t traits) {
  if (f->struct_size != XLA_FFI_CallFrame_STRUCT_SIZE) {
    std::fprintf(stderr, "libb200_scaled_dot was built without XLA's FFI headers and cannot be called by XLA; rebuild it with XLA_ROOT=<xla checkout>\n");
    return nullptr;
  }
  for (XLA_FFI_Extension_Base* e = f->extension_start; e != nullptr; e = e->next) {
    if (e->type != XLA_FFI_Extension_Metadata) continue;
    XLA_FFI_Metadata* m = reinterpret_cast<XLA_FFI_Metadata_Extension*>(e)->metadata;
    m->api_version = {XLA_FFI_Api_Version_STRUCT_SIZE, XLA_FFI_API_MAJOR, XLA_FFI_API_MINOR};
    m->traits = traits;
    return nullptr;
  }
  try {
    if (f->stage != binding.stage) return Report(f->api, 3, "handler called for another stage than its own");
    const RemainingArgs args(&f->args);
    const RemainingRets rets(&f->rets);
    const Dictionary attrs(&f->attrs);
    Error error;
    if constexpr (std::is_invocable_v<Fn>) {
      error = fn();
    } else if constexpr (std::is_invocable_v<Fn, class RemainingArgs, class RemainingRets, Dictionary>) {
      error = fn(args, rets, attrs);
    } else {
      XLA_FFI_Stream_Get_Args s{};
      s.struct_size = sizeof(s);
      s.ctx = f->ctx;
      if (XLA_FFI_Error* e = f->api->XLA_FFI_Stream_Get(&s)) return e;
      error = fn(static_cast<cudaStream_t>(s.stream), args, rets, attrs);
    }
    return error.failure() ? Report(f->api, error.code(), error.message().c_str()) : nullptr;
  } catch (const std::exception& e) {
    return Report(f->api, XLA_FFI_Error_Code_INTERNAL, e.what());
  }
}

}  // namespace xla::ffi

#define XLA_FFI_DEFINE_HANDLER_SYMBOL(symbol, function, binding, ...)                                         \
  extern "C" XLA_FFI_Error* symbol(XLA_FFI_CallFrame* frame) {                                                \
    return xla::ffi::Invoke(frame, function, binding, xla::ffi::TraitBits(__VA_ARGS__));                      \
  }

#endif  // B200SD_FFI_STANDIN_FFI_H_

// What the C entry points share (api.hip, api_f8.hip): how a call fails, and how it cuts up a workspace.
#pragma once
#include <exception>

#include "common.hpp"

namespace mi_moe {

int fail(const char *fmt, ...) __attribute__((format(printf, 1, 2)));  // keeps the message for mi_moe_last_error, tells the handler; 1

// No exception leaves an entry point: every extern "C" body is a function-try-block that ends in this.
#define MI_CATCH(name)                                                                  \
  catch (const std::exception &ex_) { return fail(name ": %s", ex_.what()); }           \
  catch (...) { return fail(name ": unknown C++ exception"); }

inline int hip_fail(const char *what, hipError_t e) {
  return fail("%s: %s", what, hipGetErrorString(e));
}

#define MI_HIP(call)                                   \
  do {                                                 \
    hipError_t e_ = (call);                            \
    if (e_ != hipSuccess) return hip_fail(#call, e_);  \
  } while (0)

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline size_t align_up(size_t v, size_t a = 256) { return (v + a - 1) / a * a; }

// carve consecutive 256-byte aligned regions out of a workspace; the first one starts at the next
// 256-byte boundary (every *_workspace_size reserves 256 bytes for that)
struct Carver {
  char *base;
  size_t off = 0;
  explicit Carver(void *p)
      : base(reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(p) + 255u) & ~(uintptr_t)255u)) {}
  template <typename T>
  T *take(size_t n) {
    T *p = reinterpret_cast<T *>(base + off);
    off += align_up(n * sizeof(T));
    return p;
  }
};

}  // namespace mi_moe

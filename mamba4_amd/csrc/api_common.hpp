// What the C entry points of every source share: the thread's error message,
// launches with the profiling log, the device's compute units, and workspaces.
#pragma once

#include <cstddef>
#include <cstdint>
#include <exception>
#include <string>

#include <hip/hip_runtime.h>

#include "../../include/mamba4_memread.h"

namespace m4 {

int api_fail(int code, const std::string& msg);
void api_clear();
int api_compute_units();
int api_launch(const char* name, hipStream_t stream, void (*body)(void*), void* context);

// Launch `body` on `stream`, timed by the profiling log when that is on.
template <typename F>
int api_launch(const char* name, hipStream_t stream, F&& body) {
  return api_launch(name, stream, [](void* f) { (*static_cast<F*>(f))(); }, &body);
}

// A C entry point's body: no C++ exception leaves it.
template <typename F>
int api_entry(const char* name, F&& body) noexcept {
  try {
    api_clear();
    return body();
  } catch (const std::exception& e) {
    try {
      return api_fail(M4MR_EHIP, std::string(name) + ": " + e.what());
    } catch (...) {
      return M4MR_EHIP;
    }
  } catch (...) {
    return M4MR_EHIP;
  }
}

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Consecutive pieces of one workspace (sizes only, if base is NULL).
struct Carver {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += align256(count * sizeof(T));
    return p;
  }
};

inline bool bad_workspace(const void* base, size_t given, size_t need, std::string* why) {
  if (need == 0) return false;
  if (!base || given < need) {
    *why = "workspace too small";
    return true;
  }
  if (reinterpret_cast<uintptr_t>(base) & 255) {
    *why = "workspace must be 256-byte aligned";
    return true;
  }
  return false;
}

}  // namespace m4

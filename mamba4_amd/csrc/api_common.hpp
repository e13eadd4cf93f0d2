// What the C entry points of every source share: the thread's error message,
// launches with the profiling log, and the device's compute units.
#pragma once

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

}  // namespace m4

// Errors of the C ABI: every entry point runs its body under guarded(), which turns an exception into a status code
// and this thread's message (aeisu_last_error).
#pragma once
#include <hip/hip_runtime.h>

#include <new>
#include <stdexcept>
#include <string>

#include "aeisu_amd.h"

namespace aeisu {

struct Error : std::runtime_error {
  int code;
  Error(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};
[[noreturn]] inline void fail(int code, const std::string& msg) { throw Error(code, msg); }
inline void check_hip(hipError_t e, const char* what) {
  if (e != hipSuccess) fail(AEISU_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}
// As check_hip; with AEISU_EAGER_VALIDATE=1 in the environment it also waits for the stream (engine.cpp).
void check_launch(hipError_t e, const char* what, hipStream_t s);

extern thread_local std::string g_last_error;

template <typename Fn>
int guarded(Fn fn) {
  try {
    fn();
    g_last_error.clear();
    return AEISU_OK;
  } catch (const Error& e) {
    g_last_error = e.what();
    return e.code;
  } catch (const std::bad_alloc&) {
    g_last_error = "host allocation failed";
    return AEISU_ERR_HIP;
  } catch (const std::exception& e) {
    g_last_error = e.what();
    return AEISU_ERR_HIP;
  }
}

}  // namespace aeisu

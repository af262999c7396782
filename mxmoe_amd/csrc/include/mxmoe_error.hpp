// What the entry points report failures with.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

namespace mxmoe {

// text of the calling thread's last failing call
inline std::string& last_error() {
  static thread_local std::string e;
  return e;
}
// `code` with its text
inline int refuse(int code, const char* what) {
  last_error() = what;
  return code;
}
// 0, or the failure of the launches before it
inline int launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return 0;
  last_error() = std::string("kernel launch failed: ") + hipGetErrorString(e);
  return 4;
}

}  // namespace mxmoe

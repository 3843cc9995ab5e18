// Exceptions of the C++ layer become return codes plus a thread-local message at the extern "C" boundary.
#pragma once
#include <exception>
#include <string>

namespace spnc_hip {

std::string& lastError();  // of the calling thread (c_api.cpp)

template <typename Fn>
int guarded(Fn&& fn) {
  try {
    lastError().clear();
    fn();
    return 0;
  } catch (const std::exception& e) {
    lastError() = e.what();
    return 1;
  } catch (...) {
    lastError() = "unknown error";
    return 1;
  }
}

}  // namespace spnc_hip

// What the C entries share.
#pragma once

#include <string>

#include "../../include/tiso.h"

namespace tiso {

// Records the calling thread's error message (for tiso_last_error) and returns code (tiso.cu).
int report_error(int code, const std::string& msg);

// An entry's body: no C++ exception (the host out of memory) leaves it.
template <typename F>
int guarded(F&& body) noexcept {
  try {
    return body();
  } catch (...) {
    return TISO_ERR_CUDA;
  }
}

}  // namespace tiso

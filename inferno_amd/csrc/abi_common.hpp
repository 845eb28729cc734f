// Helpers of the extern "C" entry points: workspace carving, the device check
// and the workspace check.
#pragma once
#include <string>

#include "common.hpp"

namespace inferno {

inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

inline size_t align_up(size_t v) { return (v + 255) & ~size_t(255); }

// Carves aligned sub-buffers out of a caller workspace.
struct Carver {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t count) {
    T* p = reinterpret_cast<T*>(base ? base + used : nullptr);
    used += align_up(count * sizeof(T));
    return p;
  }
};

// The reference returns Ok(None) ("unsupported here, the caller may fall
// back") when no native device backs the backend (backend.rs:6688-6692 and
// the non-Metal branches); the counterpart here is INFERNO_UNSUPPORTED when
// the process sees no HIP device. Argument errors are reported before this
// check, as the reference validates before it looks for the device.
inline int require_device() {
  static const int count = [] {
    int n = 0;
    return hipGetDeviceCount(&n) == hipSuccess ? n : 0;
  }();
  if (count > 0) return INFERNO_OK;
  set_error("no HIP device is available (unsupported here; the caller may fall back)");
  return INFERNO_UNSUPPORTED;
}

inline int need_ws(void* ws, size_t have, size_t need) {
  if (need > 0 && (ws == nullptr || have < need)) {
    set_error("workspace too small: need " + std::to_string(need) + " bytes");
    return INFERNO_ERR_SIZE;
  }
  return INFERNO_OK;
}

}  // namespace inferno

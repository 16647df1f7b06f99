// entry.h -- what every C entry point is wrapped in.
#pragma once
#include <exception>

#include "runtime.h"

namespace attnb {

// Runs an entry point's body inside an NVTX range named after the entry point
// (visible in Nsight timelines; free when no tool is attached) and turns its
// exceptions into a status code plus the thread's last-error message.
template <class F>
int guarded(const char* name, F&& f) {
  NvtxRange range(name);
  try {
    f();
    return ATTNB_OK;
  } catch (const Error& e) {
    return set_last_error(e.code, e.msg);
  } catch (const std::exception& e) {
    return set_last_error(ATTNB_ERR_RUNTIME, e.what());
  } catch (...) {
    return set_last_error(ATTNB_ERR_RUNTIME, "unknown error");
  }
}

inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

}  // namespace attnb

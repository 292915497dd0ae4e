// A call's workspace: the caller's, checked, or the library's scratch for the
// stream.
#pragma once

#include <string>

#include "common.h"

namespace mfx {

// Sets *out to `need` bytes, 256-byte aligned (nothing for 0).
inline int take_workspace(void* given, size_t given_bytes, size_t need, const char* query, hipStream_t s, char** out) {
  *out = nullptr;
  if (need == 0) return MFX_OK;
  if (given) {
    if (given_bytes < need) return fail(MFX_E_WORKSPACE, std::string("workspace smaller than ") + query + "()");
    if ((uintptr_t)given % 256) return fail(MFX_E_INVALID, "workspace must be 256-byte aligned");
    *out = static_cast<char*>(given);
    return MFX_OK;
  }
  *out = static_cast<char*>(device_scratch(need, s));
  return *out ? MFX_OK : MFX_E_HIP;
}

inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace mfx

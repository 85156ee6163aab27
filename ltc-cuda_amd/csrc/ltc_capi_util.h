// What the C entry points of the sequence, token and model operators share.
#pragma once

#include <string>

#include "../../include/ltc_capi.h"
#include "ltc_seq_internal.h"

namespace ltc {

// Workgroups of one launch: the runtime counts threads, up to 512 each, in 32 bits.
constexpr long long kMaxGroups = (1LL << 32) / 512 - 1;

// Pieces of a workspace or of the saved buffer, each on 256 bytes; base null:
// sizes only.
struct Pieces {
  char* base;
  long long off = 0;
  template <class T>
  T* take(long long n) {
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += (n * (long long)sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

inline int check_workspace(long long need, const void* ws, long long have) {
  if (need > 0 && (ws == nullptr || have < need))
    return host_fail(LTC_EINVAL, "workspace too small: need " + std::to_string(need) + " bytes, got " +
                                     std::to_string(ws ? have : 0));
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return host_fail(LTC_EINVAL, "workspace must be 256-byte aligned");
  return LTC_OK;
}

inline bool known_type(int t) { return t == LTC_F32 || t == LTC_BF16 || t == LTC_F16; }
inline int type_bytes(int t) { return t == LTC_F32 ? 4 : 2; }

}  // namespace ltc

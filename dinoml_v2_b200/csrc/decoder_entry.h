// What the C entries of the decoder operators have in common.  The workspaces' bookkeeping and the messages allocate on the host: no exception leaves an entry.
#pragma once
#include "gguf_common.cuh"

namespace b200gguf {
int set_error(int rc, const char* where);
}

template <typename F> static int entry(const char* where, F f) noexcept {
  try {
    return b200gguf::set_error(f(), where);
  } catch (...) {
  }
  try {
    return b200gguf::set_error(b200gguf::RC_LAUNCH, where);
  } catch (...) {
    return b200gguf::RC_LAUNCH;
  }
}

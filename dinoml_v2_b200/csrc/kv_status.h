// The status words of the cache's kernels on a device, as the host reads them.  Two words, since one would be whoever came first: a call that pointed outside of
// the cache would hide a wait that gave up, and with it that the attention's counters have to be emptied.  Host code over the CUDA runtime only.
#pragma once
#include <cuda_runtime_api.h>

namespace b200gguf {
namespace kv {

enum : int { ST_KV_RANGE = 10 };            // word 0: a block table entry, a length, a start or a begin pointed outside of the cache or of the rows
enum : int { ST_KV_TIMEOUT = 16 };          // word 1: a wait of the attention gave up
constexpr int kStatusWords = 2;

// The status, read once; reset() where a wait gave up.  -1: it could not be read.
template <typename Reset> inline int take_status(int* words, Reset reset) {
  int value[kStatusWords] = {};
  if (words == nullptr || cudaMemcpy(value, words, sizeof(value), cudaMemcpyDeviceToHost) != cudaSuccess) return -1;
  if (value[0] != 0 || value[1] != 0) cudaMemset(words, 0, sizeof(value));
  if (value[1] != 0) reset();
  return value[1] != 0 ? value[1] : value[0];
}

}  // namespace kv
}  // namespace b200gguf

// Attention of many rows over the 8-bit cache (kernel: kv_attention_many.cuh).
#include "kv_attention_many.cuh"

namespace b200gguf {
namespace kv {

int attention_many(AttnParams& a, int type, cudaStream_t s) {
  if (type == DINOML_B200_KV_INT8)
    return a.c.dim == 64 ? many::launch<DINOML_B200_KV_INT8, 64>(a, s) : many::launch<DINOML_B200_KV_INT8, 128>(a, s);
  return a.c.dim == 64 ? many::launch<DINOML_B200_KV_E4M3, 64>(a, s) : many::launch<DINOML_B200_KV_E4M3, 128>(a, s);
}

}  // namespace kv
}  // namespace b200gguf

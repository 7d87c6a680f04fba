// Attention of many rows over the 8-bit cache (kernel: kv_attention_many.cuh).
#include "kv_attention_many.cuh"

namespace b200gguf {
namespace kv {

template <int TYPE> static int launch_shape(AttnParams& a, cudaStream_t s) {
  if (a.dtype == DINO_F32) return a.c.dim == 64 ? many::launch<TYPE, 64, 2>(a, s) : many::launch<TYPE, 128, 2>(a, s);
  switch (a.c.dim) {
    case 64: return many::launch<TYPE, 64, 1>(a, s);
    case 128: return many::launch<TYPE, 128, 1>(a, s);
    default: return many::launch<TYPE, 256, 1>(a, s);
  }
}

int attention_many(AttnParams& a, int type, cudaStream_t s) {
  return type == DINOML_B200_KV_INT8 ? launch_shape<DINOML_B200_KV_INT8>(a, s) : launch_shape<DINOML_B200_KV_E4M3>(a, s);
}

}  // namespace kv
}  // namespace b200gguf

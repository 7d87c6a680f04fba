// Attention of few rows over caches of type int8 (kernel: kv_attention_few.cuh).
#include "kv_attention_few.cuh"

namespace b200gguf {
namespace kv {

int attention_few_int8(AttnParams& a, int tiles, cudaStream_t s) { return few::launch_shape<DINOML_B200_KV_INT8>(a, tiles, s); }

}  // namespace kv
}  // namespace b200gguf

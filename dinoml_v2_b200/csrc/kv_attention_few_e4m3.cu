// Attention of few rows over caches of type e4m3 (kernel: kv_attention_few.cuh).
#include "kv_attention_few.cuh"

namespace b200gguf {
namespace kv {

int attention_few_e4m3(AttnParams& a, int tiles, cudaStream_t s) { return few::launch_shape<DINOML_B200_KV_E4M3>(a, tiles, s); }

}  // namespace kv
}  // namespace b200gguf

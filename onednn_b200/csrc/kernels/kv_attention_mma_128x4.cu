#include "kv_attention_mma.cuh"

namespace b200 {
namespace kv_mma {
template int run<128, 4>(const b200_kv_attention_params_t &, int, cudaStream_t);
} // namespace kv_mma
} // namespace b200

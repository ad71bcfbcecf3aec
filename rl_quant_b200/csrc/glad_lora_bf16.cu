// The adapter kernels (glad_lora.cuh) for rows of bf16.
#include "glad_lora.cuh"

namespace glad {
namespace lora {
template cudaError_t run<__nv_bfloat16>(Params, bool, cudaStream_t);
template cudaError_t run_outer<__nv_bfloat16>(OuterPair, int, cudaStream_t);
template bool wants_transposed<__nv_bfloat16>(const Params&);
}  // namespace lora
}  // namespace glad

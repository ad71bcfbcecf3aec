// The adapter kernels (glad_lora.cuh) for rows of f32.
#include "glad_lora.cuh"

namespace glad {
namespace lora {
template cudaError_t run<float>(Params, bool, cudaStream_t);
template cudaError_t run_outer<float>(OuterPair, int, cudaStream_t);
template bool wants_transposed<float>(const Params&);
}  // namespace lora
}  // namespace glad

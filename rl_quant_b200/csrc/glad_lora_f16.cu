// The adapter kernels (glad_lora.cuh) for rows of f16.
#include "glad_lora.cuh"

namespace glad {
namespace lora {
template cudaError_t run<__half>(Params, bool, cudaStream_t);
template cudaError_t run_outer<__half>(OuterPair, int, cudaStream_t);
template bool wants_transposed<__half>(const Params&);
}  // namespace lora
}  // namespace glad

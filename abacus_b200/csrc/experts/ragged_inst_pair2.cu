#include "ragged_kernel.cuh"

namespace abacus {
namespace ragged {
template cudaError_t launch_shape<2, true>(const Params&, const Shape&, long long, int, cudaStream_t);
}  // namespace ragged
}  // namespace abacus

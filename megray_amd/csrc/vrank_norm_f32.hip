// The norm behind a fold and its backward, partial activations of type FLOAT32.
#include "vrank_norm_impl.hpp"

namespace MegRay {
namespace vrank {

NormKernels norm_kernels_f32(NormVariant v, uint32_t nranks, bool lines, bool q8) {
    return detail::norm_kernels_for<float, float>(v, nranks, lines, q8);
}

}  // namespace vrank
}  // namespace MegRay

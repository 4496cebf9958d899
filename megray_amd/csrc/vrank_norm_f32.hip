// The norm behind a fold and its backward, partial activations of type FLOAT32.
#include "vrank_norm_impl.hpp"

namespace MegRay {
namespace vrank {

NormKernels norm_kernels_f32(NormVariant v, bool stream32, bool q8) {
    return detail::norm_kernels<float>(v, stream32, q8);
}

}  // namespace vrank
}  // namespace MegRay

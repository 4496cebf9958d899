// The norm behind a fold and its backward, partial activations of type FLOAT16.
#include "vrank_norm_impl.hpp"

namespace MegRay {
namespace vrank {

NormKernels norm_kernels_f16(NormVariant v, bool stream32, bool q8) {
    return detail::norm_kernels<_Float16>(v, stream32, q8);
}

}  // namespace vrank
}  // namespace MegRay

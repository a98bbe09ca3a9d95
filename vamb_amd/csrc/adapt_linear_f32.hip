// Instantiations of the shared-projection kernel on float32 tensors (adapt_linear.hpp).
#include "adapt_linear.hpp"

namespace vh {
namespace adapt {
void launch_linear_f32(const LinArgs& a, bool backward, hipStream_t s) {
    if (backward) launch_rank<float, true, true, 3>(a, s);
    else launch_rank<float, false, false, 3>(a, s);
}
}  // namespace adapt
}  // namespace vh

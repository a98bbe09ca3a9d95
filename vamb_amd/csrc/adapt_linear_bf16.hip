// Instantiations of the shared-projection kernel on bf16 tensors (adapt_linear.hpp).
#include "adapt_linear.hpp"

namespace vh {
namespace adapt {
void launch_linear_bf16(const LinArgs& a, bool backward, hipStream_t s) {
    if (backward && a.x_planes == 2) launch_rank<bf16_t, true, true, 2>(a, s);
    else if (backward) launch_rank<bf16_t, true, true, 1>(a, s);
    else if (a.dma) launch_rank<bf16_t, false, true, 1>(a, s);
    else launch_rank<bf16_t, false, false, 1>(a, s);
}
}  // namespace adapt
}  // namespace vh

// k_ragged_f32.hip -- the products over rows in groups (ragged.hpp) for f32 operands.
#include "ragged_launch.hpp"

namespace tfh {
namespace ragged {
int32_t launch_f32(int kind, const Args& a, void* stream) { return launch_product<float>(kind, a, stream); }
}  // namespace ragged
}  // namespace tfh

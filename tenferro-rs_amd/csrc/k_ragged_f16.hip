// k_ragged_f16.hip -- the products over rows in groups (ragged.hpp) for f16 operands.
#include "ragged_launch.hpp"

namespace tfh {
namespace ragged {
int32_t launch_f16(int kind, const Args& a, void* stream) { return launch_product<_Float16>(kind, a, stream); }
}  // namespace ragged
}  // namespace tfh

// k_ragged_f64.hip -- the products over rows in groups (ragged.hpp) for f64 operands.
#include "ragged_launch.hpp"

namespace tfh {
namespace ragged {
int32_t launch_f64(int kind, const Args& a, void* stream) { return launch_product<double>(kind, a, stream); }
}  // namespace ragged
}  // namespace tfh

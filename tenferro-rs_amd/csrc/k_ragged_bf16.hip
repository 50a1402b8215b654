// k_ragged_bf16.hip -- the products over rows in groups (ragged.hpp) for bf16 operands.
#include "ragged_launch.hpp"

namespace tfh {
namespace ragged {
int32_t launch_bf16(int kind, const Args& a, void* stream) { return launch_product<__bf16>(kind, a, stream); }
}  // namespace ragged
}  // namespace tfh

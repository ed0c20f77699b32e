// q4_f32.hip -- the 4-bit products of f32 rows.
#include "q4_kernel.hpp"

namespace clear {
CLEAR_Q4_ROWS(float)
}  // namespace clear

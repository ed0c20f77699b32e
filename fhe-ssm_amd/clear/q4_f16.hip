// q4_f16.hip -- the 4-bit products of f16 rows.
#include "q4_kernel.hpp"

namespace clear {
CLEAR_Q4_ROWS(f16)
}  // namespace clear

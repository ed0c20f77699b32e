// q4_bf16.hip -- the 4-bit products of bf16 rows.
#include "q4_kernel.hpp"

namespace clear {
CLEAR_Q4_ROWS(bf16)
}  // namespace clear

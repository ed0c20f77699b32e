// clear.cpp -- the error text of libfhe_ssm_clear.so.
#include "clear.hpp"

namespace clear {
char* error_text() {
    static thread_local char text[kErrorText] = "";
    return text;
}
}  // namespace clear

extern "C" const char* fhe_ssm_clear_last_error(void) { return clear::error_text(); }

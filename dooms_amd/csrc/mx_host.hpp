// What the files of the C ABI layer share on the host.
#pragma once

#include <stdint.h>

namespace mx {

// Keeps the message for mx_attn_last_error() on this thread and returns the code.
int32_t set_error(int32_t code, const char * message);

}  // namespace mx

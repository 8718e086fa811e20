// i8.h -- what the 8-bit operators' files share (k_i8.cu, k_i8_linear.cu).
#pragma once

#include "nncu.h"

namespace nncu
{

// The product of checked arguments (k_i8_linear.cu); a cudaError_t value.
int launch_i8_linear(const nncu_i8_linear& l, void* stream);
// How many bounded waits of products ran out on the current device, read on `stream` and waited for; a cudaError_t value.
int i8_waits_out(unsigned* count, void* stream);

} // namespace nncu

// i8.h -- what the 8-bit operators' files share (k_i8.cu, k_i8_linear.cu).
#pragma once

#include "nncu.h"

namespace nncu
{

// The product of checked arguments (k_i8_linear.cu); a cudaError_t value.
int launch_i8_linear(const nncu_i8_linear& l, void* stream);
// The current device's error word of the products, cleared where it is set; a cudaError_t value.
int i8_error_word(int* word);

} // namespace nncu

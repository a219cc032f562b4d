// The product of one 8-bit matrix with a few rows (int8_few.hip).
#pragma once

#include "int8_product.h"

namespace qmoe_i8 {

// Arguments checked by the caller; one expert, no table.
int few_product(const Product& a, hipStream_t st);

}  // namespace qmoe_i8

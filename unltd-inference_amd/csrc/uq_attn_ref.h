// The running reference of the paged attention's softmax, shared by the
// kernels and the CPU emulation. A weight is held as 2^(x + a), x = score log2 e
// and -a the largest x so far, less a shift (what is left of f16's range above
// 2^0 for the weights' second terms).
//
// x is a sum of products with queries that hold the mantissa of kq_scale log2 e
// already, times a power of two: without a rounding, so that x + a is rounded
// once and the largest weight is 2^shift whatever the scores' size, as long as
// shift is not lost in a. From kFar on it would be rounded to steps of a half
// and more (and from 2^25 on to more than f16 has above the shift): there the
// reference is -x itself, and the largest weight 2^0.
#pragma once

#include "uq_bits.h"

namespace uq {

constexpr float kFar = 0x1p22f;

UQ_HD float reference(float top, float shift) { return (fabsf(top) < kFar ? shift : 0.0f) - top; }

}  // namespace uq

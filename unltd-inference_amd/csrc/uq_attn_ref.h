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

// The factor 2^e of a query's scores, a normal number: a score of zero stays
// zero, a masked score's -infinity stays one. What the limits change are
// scores of no size, or so far apart that one weight is all: sums of products
// of f16 terms are zero or 2^-48 to 2^41 in size (an f32 cache's queries take
// what the limits leave).
UQ_HD float score_factor(int e) { return ldexpf(1.0f, e < -126 ? -126 : e > 127 ? 127 : e); }

UQ_HD float reference(float top, float shift) { return (fabsf(top) < kFar ? shift : 0.0f) - top; }

}  // namespace uq

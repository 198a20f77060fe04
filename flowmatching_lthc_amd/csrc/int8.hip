// MI355X (gfx950) kernels and C ABI of the workspace branch's inference in 8-bit integers: rows in 8 bits with a scale each, the
// RMS norm with such an output, linear and gated linear layers on such rows.  Declarations are in include/lthc.h.

#include "common.inc"

// Rows in 8 bits and back, RMS norm with the residual's addition and an output in 8 bits.
#include "int8_rows.inc"
// Linear and gated linear layers.
#include "int8_linear.inc"

// MI355X (gfx950) kernels and C ABI of a training step's operators next to the interface and the workspace branch:
// rotary positions with several axes, the gated linear layer and AdamW over many tensors.  Declarations are in
// include/lthc.h.

#include "common.inc"

// Rotary positions with several axes.
#include "axial_rope.inc"
// AdamW, the norm of all gradients.
#include "adamw.inc"
// The gated linear layer and its backward.
#include "gated_linear.inc"

// mg_linear_f32.hip — the linear layer's kernels for 32-bit floats
#define MG_LINEAR_T float
#include "mg_linear_tu.inc"

// mg_linear_f16.hip — the linear layer's kernels for f16
#define MG_LINEAR_T f16
#include "mg_linear_tu.inc"

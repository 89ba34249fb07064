// mg_linear_bf16.hip — the linear layer's kernels for bf16
#define MG_LINEAR_T bf16
#include "mg_linear_tu.inc"

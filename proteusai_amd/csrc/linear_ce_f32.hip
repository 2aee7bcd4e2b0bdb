// The matrix products of the loss over a vocabulary on fp32 operands, as three pieces of bf16.
#define CE_TYPE 2
#define CE_LAUNCH launch_f32
#define CE_LAUNCH_BOTH launch_both_f32
#include "linear_ce_body.inc"

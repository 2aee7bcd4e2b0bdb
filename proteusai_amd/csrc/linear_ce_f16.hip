// The matrix products of the loss over a vocabulary on fp16 operands.
#define CE_TYPE 1
#define CE_LAUNCH launch_f16
#define CE_LAUNCH_BOTH launch_both_f16
#include "linear_ce_body.inc"

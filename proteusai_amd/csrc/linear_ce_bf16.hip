// The matrix products of the loss over a vocabulary on bf16 operands.
#define CE_TYPE 0
#define CE_LAUNCH launch_bf16
#define CE_LAUNCH_BOTH launch_both_bf16
#include "linear_ce_body.inc"

// The loss for heads of few words (linear_ce_small.hip), and what a token's loss is made of, for it and the general path (linear_ce.hip).
#pragma once

#include <hip/hip_runtime.h>
#include "linear_ce_internal.h"

namespace proteus_ce {

constexpr int SMALL_WORDS = 64;

#define CE_HIDDEN __attribute__((visibility("hidden")))
CE_HIDDEN size_t small_kept_bytes(const proteus_ce_args& a);
CE_HIDDEN size_t small_forward_bytes(const proteus_ce_args& a);
CE_HIDDEN size_t small_backward_bytes(const proteus_ce_args& a);
CE_HIDDEN int small_forward(const proteus_ce_args& a, float* loss, void* kept, void* ws, hipStream_t st);
CE_HIDDEN int small_backward(const proteus_ce_args& a, const float* dloss, const void* kept, void* dx, void* dweight, void* dbias, void* ws, hipStream_t st);

// log(1 + exp(others - own)) from the other words' largest logit and their sum of exponentials less it, and 1 - the own word's probability: neither loses anything where own and others differ by orders of magnitude.
// No others (a single word, or all the rest at -infinity): 0 and 0.  A logit of +infinity, own or not: NaN; none above LOWEST, the own included, so that there is nothing to be a share of: NaN.
__device__ __forceinline__ float loss_of(const float shift, const float total, const float wanted, float& missed)
{
    float ahead = total > 0.0f || total != total ? shift + logf(total) - wanted : wanted >= LOWEST ? -__builtin_inff() : __builtin_nanf("");
    if (total == __builtin_inff() || wanted == __builtin_inff()) ahead = __builtin_nanf("");
    missed = 1.0f / (1.0f + expf(-ahead));
    return ahead == ahead ? fmaxf(ahead, 0.0f) + log1pf(expf(-fabsf(ahead))) : ahead;
}

}  // namespace proteus_ce

// The gated feed-forward block's products in 16 bits (gated_mlp_bf16.hip) and its element-wise parts, for gated_mlp.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include "proteus_hip.h"

namespace proteus_gated {

// act(x) and its derivative, in fp32.
enum Act { SILU = PROTEUS_ACT_SILU, GELU = PROTEUS_ACT_GELU, RELU = PROTEUS_ACT_RELU, SIGMOID = PROTEUS_ACT_SIGMOID };

__device__ __forceinline__ float sigmoid(const float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f)); }

// Phi(-ax) for results in 16 bits: exp(-ax^2 / 2) t P(t), t = 1 / (1 + 0.376 ax).  P of degree 4 is the one of the least largest relative error from 0 to 13.5, a linear
// program over its coefficients: 2.8e-5, and 4e-5 with fp32's roundings, 1/100 of half a step in bf16 however small the tail is.  (From 13.2 on the exponential is below fp32's
// smallest normal number, and zero.)  A formula of bounded absolute error would do for cdf, but not for x cdf far below zero.
__device__ __forceinline__ float short_tail(const float ax)
{
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(ax, 0.376f, 1.0f));
    float p = __builtin_fmaf(t, -0.0911193951f, 0.1993228273f);
    p = __builtin_fmaf(t, p, 0.0842667374f);
    p = __builtin_fmaf(t, p, 0.1580532683f);
    return __builtin_fmaf(t, p, 0.1494627864f) * t * __builtin_amdgcn_exp2f(ax * ax * (-0.5f * 1.44269504f));
}

// EXACT: to fp32's rounding; else off by less than 2^-12 of the terms, 1/16 of half a step in bf16.
template <bool EXACT> __device__ __forceinline__ void activate(const int act, const float x, float& value, float& slope)
{
    if (act == RELU) { value = x > 0.0f ? x : x < 0.0f ? 0.0f : x; slope = x > 0.0f ? 1.0f : 0.0f; return; }       // (NaN stays)
    if (act == GELU) {
        const float ax = fabsf(x);
        const float tail = EXACT ? 0.5f * erfcf(ax * 0.70710678118654752f) : short_tail(ax), cdf = x < 0.0f ? tail : 1.0f - tail;
        value = x < -40.0f ? 0.0f : x * cdf;
        slope = ax > 40.0f ? cdf : __builtin_fmaf(x, 0.39894228040143268f * (EXACT ? expf(-0.5f * x * x) : __builtin_amdgcn_exp2f(x * x * (-0.5f * 1.44269504f))), cdf);
        return;
    }
    const float s = EXACT ? 1.0f / (1.0f + expf(-x)) : sigmoid(x);
    value = act == SILU ? x * s : s;
    slope = act == SILU ? s * __builtin_fmaf(x, 1.0f - s, 1.0f) : s * (1.0f - s);
}

enum Epilogue { PLAIN, GATED, GATED_KEPT, GATED_GRAD };

// One product in bf16, fp32 sums.  NT: C[m][n] = sum_k A[m][k] B[n][k]; NN: B[k][n]; TN: A[k][m] B[k][n].
//   PLAIN        C = sums + bias
//   GATED        NT, B [2 N][K] (gates, then values), C = act(sums of n) * (sums of N + n), bias [2 N] before that; _KEPT: the sums themselves too, to 20 bits each, the
//                upper 16 in z [M][2 N], the next four in rest [M][N] (the gate's below the value's): rounded to bf16 they would put as much into dz as its own rounding does, and
//                gradients would be 1.3 times as far off; a pass takes 1 to 4 % longer for it
//   GATED_GRAD   NN, sums = dh: z and rest are read, C = dz [M][2 N] = (dh * value * act'(gate) | dh * act(gate)), and column sums of it per 32-row block of a wave
//                go to `columns` [rows of blocks][2 N] where that is given
struct Product {
    const uint16_t *A, *B, *bias;
    uint16_t *C, *z;
    uint8_t* rest;
    float* columns;
    int M, N, K;
    int64_t lda, ldb, ldc;
    int form, epilogue, act;
    float* part;                                    // PLAIN: what product_bytes asks for
};
// What is left to add up behind products: the shares of K of up to three, and up to two column sums, in one launch.
struct Ends {
    struct Shares { const float* part; const uint16_t* bias; uint16_t* C; int64_t n, ldc; int shares, N; };
    struct Columns { const float* part; uint16_t* out; int rows, C; };                               // out [C] = sums of part [rows][C]
    Shares shares[3];
    Columns columns[2];
    int count, column_count;
};
// Tiles of a product and its shares of K, of `steps` steps each.
struct Plan { int tile, shares, steps; };
size_t product_bytes(int form, int M, int N, int K);
int column_rows(int M, int N, int K);               // rows of blocks of a GATED_GRAD
int product(const Product& p, Ends& ends, hipStream_t st);                     // C is not whole before finish, and p.part its own until then
// The three products behind dz, one after the other or in one launch: dy^T h [O][F], dz^T x [2 F][D], dz W [rows][D], and the bytes of each one's part.
struct Behind { Plan plan[3]; bool together; size_t part[3]; };
Behind behind(int rows, int D, int F, int O);
struct Columns { const uint16_t* a; float* part; uint16_t* out; int64_t rows; int C; };              // out [C] = sums of a [rows][C], or a NULL; part [column_shares][C]
int64_t column_shares(int64_t rows);
int products_behind(const Behind& b, const Product (&p)[3], const Columns& columns, Ends& ends, hipStream_t st);      // those with a C; M, N and K as above
int finish(Ends& ends, hipStream_t st);

}  // namespace proteus_gated

// The matrix products of the loss (linear_ce_body.inc, an instance for each type of operands) for its host side (linear_ce.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include "proteus_hip.h"

namespace proteus_ce {

// of a shift, and its largest is minus this: what lies lower takes no part beside it, what lies higher (in 16-bit types) gives a NaN, and its product with log2(e) is a number, too
constexpr float LOWEST = -2.0e38f;

// What a product makes of its tile.  With n the number of tokens that count, which only the device knows:
//   STATS  x W^T + b, [n][N]: of every row of 32 columns times the wave's, the largest, the sum of exponentials and the sum, the token's own word apart
//   GRAD   x W^T + b again: its gradient, in 16 bits (F32: three of them), and sums over rows of it
//   DX     P W, [n][N]
//   DW     P^T x, [M][N], over n tokens
enum Role { STATS, GRAD, DX, DW };
enum Tile { T256, T128, T64, T64_FINE };            // rows: 256, 128, 64, 64; columns: 256, 128, 128, 128.  FINE: DX and DW of 16-bit types from P in two pieces

struct Row { float shift, scale, own; int target; };          // GRAD: exp(logit - shift) * scale; what the own word has instead

struct Args {
    const uint16_t *A, *B;                          // 16-bit operands, fp32 ones as three pieces of bf16
    int64_t piece_a, piece_b, lda, ldb;             // elements from one piece to the next, and from one row
    const uint16_t *x_all;                          // the features where all tokens count (NULL: the same): the tensor itself instead of a copy of its rows
    const int* count;                               // n
    int all;                                        // all tokens
    int M, N, K;                                    // GRAD, STATS, DX: M = all; DW: K = all
    int a_cols;                                     // DW: columns of A that may be read
    int group;                                      // tiles along m that go side by side
    int shares;                                     // of K
    const float* bias;                              // fp32, -infinity behind the last column up to a whole tile; or NULL
    int first;                                      // word of column 0
    // STATS
    const int* target;                              // of the tokens that count, -1: none that there is
    float2* part;                                   // [column group][all]
    float* part_sum;                                // or NULL
    float* wanted;                                  // [all]
    // GRAD
    const Row* row;
    const float* weight;                            // of each token
    uint16_t* P;                                    // [all][ldp], pieces piece_p apart; columns up to the next multiple of 8 are zeros
    int64_t ldp, piece_p;
    int fine;                                       // (16-bit types, T64) as two pieces
    float even;                                     // what smoothing takes from every word, times the token's weight
    float* columns;                                 // [row group][N], or NULL
    // DX, DW
    void* C;                                        // rows of ldc, in the operands' type
    int64_t ldc;
    float* slab;                                    // or (not NULL) sums as they are, [share][M or all][N]
    int adds;                                       // to what is there
    const float* scale;                             // of C
    const int* rows;                                // row of C for a token (where not all of them count)
};

constexpr int rows_of(const int t) { return t == T256 ? 256 : t == T128 ? 128 : 64; }
constexpr int columns_of(const int t) { return t == T256 ? 256 : 128; }
constexpr int column_group(const int t) { return columns_of(t) / 2; }          // columns of a wave
constexpr int row_group(const int t) { return rows_of(t) / 2; }

// blocks: a multiple of 8
typedef int Launch(const Args& a, int role, int tile, unsigned blocks, hipStream_t st);
__attribute__((visibility("hidden"))) Launch launch_bf16, launch_f16, launch_f32;
// DX and DW side by side, in tiles of 128 x 128 (fp32: 64 x 128)
typedef int LaunchBoth(const Args& dx, const Args& dw, unsigned blocks_dx, unsigned blocks_dw, bool dw_first, hipStream_t st);
__attribute__((visibility("hidden"))) LaunchBoth launch_both_bf16, launch_both_f16, launch_both_f32;

}  // namespace proteus_ce

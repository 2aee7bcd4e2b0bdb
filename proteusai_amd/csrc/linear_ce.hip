// Softmax cross entropy over a vocabulary from features and words' weights, and its gradients (gfx950): what goes on around the matrix products of linear_ce_body.inc.
//
//   l = x W^T + b;   lse_i = log sum_j exp l_ij;   loss_i = lse_i - (1 - e) l_it - e / V sum_j l_ij   (t: the token's word, e: label_smoothing)
//   dl_ij = (exp(l_ij - lse_i) - (1 - e) [j = t] - e / V) g_i;   dx = dl W;   dW = dl^T x;   db = sum_i dl
//
// Logits are never in memory: the forward pass keeps four numbers a token, the backward makes the logits again, a piece of the vocabulary at a time, and writes their gradient for it (16 bits;
// P_BYTES at most, whatever the sizes, but for 2048 words of it), from which that piece of dW and its share of dx follow.  8 n D V operations where 6 are the least; keeping n V logits in 16 bits instead
// would cost 2 bytes written, read, and scaled for each 2 D operations.
//
// Tokens that are left out (ignore_index) are left out altogether: a first launch numbers those that count, collects their features one behind the other (unless all count) and leaves their number on the
// device, for the products.  What lies in the others' features, NaN or not, is not read.
//
// Bound by the products.  A pass, forward and backward: 16384 tokens, 2048 features, 65536 words in bf16 13.3 to 14.1 ms, by the card (8 n D V at 1320 to 1250 TFLOP/s; library products of these sizes run at 1090 to 1290), 5003 (4753 of which
// count), 712, 20011 0.63 ms (860), 2000, 768, 8001 in fp16 145 us (680), 2048 (1843), 512, 1000 in fp32 88 us (86; 510 of pieces); what goes on around them takes 4 to 10 us a launch, 25 for the losses of 16384 x 65536 and 40 for the sums of its dx.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include <algorithm>
#include "linear_ce_internal.h"
#include "linear_ce_small.h"

namespace {

using namespace proteus_ce;

constexpr int THREADS = 256;
constexpr int64_t P_BYTES = 1024ll << 20;           // of the logits' gradient at a time (16384 x 2048 x 65536, which has 2 GB of it, on one card: 13.8 ms; at 512 MB 14.0, at 2 GB 13.7).  All tokens at once, whatever their number
constexpr int LEAST_WORDS = 2048;                   // of a piece of the vocabulary: dx is read and written once for each, 8 bytes beside 4096 operations in each of its columns
constexpr int MOST_SHARES = 32;
constexpr int64_t MOST_TILES = (1 << 24) - 8;       // in a launch with a workgroup to a tile, which may have 2^32 - 1 threads (2^20 tokens of 64 features and 2^17 words are one more)
constexpr int FINE_ROWS = 64;                       // up to so many tokens (one tile's; those that are left out count, as the host does not know them) P is two 16-bit numbers: where few terms make a gradient its rounding does not average out beside the
                                                    // result's own (2 x 136 x 30693 in bf16: gradients 2.8e-3 off, the result's rounding alone 1.9e-3).  64 x 1024 x 5000: 57 / 60 us a pass, 64 x 2048 x 65536 308 / 354
constexpr float F16_SCALE = 32768.0f;               // fp16 ends at 6e-8: the logits' gradients, 1 at most, are written as large as they fit

struct f16_t { _Float16 v; };
struct bf16_t { __bf16 v; };
__device__ __forceinline__ float value(const f16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const bf16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const float x) { return x; }
__device__ __forceinline__ void put(float* to, const float x) { *to = x; }
__device__ __forceinline__ void put(f16_t* to, const float x) { to->v = (_Float16)x; }
__device__ __forceinline__ void put(bf16_t* to, const float x) { to->v = (__bf16)x; }

// fp32 as three bf16 numbers, four elements at a time
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float  f32x4  __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void split(f32x4 x, uint16_t* to, const int64_t piece)
{
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const bf16x4 r = __builtin_convertvector(x, bf16x4);
        *reinterpret_cast<bf16x4*>(to + p * piece) = r;
        x -= __builtin_convertvector(r, f32x4);
    }
}

// What the first launch works out and leaves, for the forward pass or for the backward.
struct Prepare {
    const void* x; const void* bias; const int64_t* target;
    int64_t ignored;
    int rows, D, V, type, per, row_blocks;          // per: rows of a workgroup
    int* count; int* index;                         // n, and the row of each token that counts
    uint16_t* features; int64_t ld, piece;          // their features (fp32: three pieces, always; else where not all count)
    float* bias_out; int bias_words;                // fp32, -infinity from V on; NULL: not needed
    int bias_blocks, split_blocks;                  // workgroups behind those of the rows
    const float* words_in; uint16_t* words_out;        // fp32 weights as three pieces, rows of ld (zeros behind the last column)
    // forward
    int* words;                                     // the word of each token that counts, -1: no word
    float* loss;                                    // of each row: zero for those left out; or NULL
    uint32_t* ticket;
    // backward
    const Row* kept; const float* dloss; int per_token, mean;
    Row* row; float* weight; float* scale;
    float target_even, size;                        // what smoothing gives the own word; what P is enlarged by
    void* dx;                                       // zeros for rows left out; or NULL
};

// put(row, chunk, get(row, chunk)) for all chunks of 16 bytes of `rows` rows, eight reads of a thread on their way at once
template <typename GET, typename PUT> __device__ __forceinline__ void each_chunk(const int chunks, const int rows, const GET& get, const PUT& put)
{
    constexpr int AHEAD = 8;
    for (int i0 = threadIdx.x; i0 < rows * chunks; i0 += AHEAD * THREADS) {    // (256 rows of 2^14 chunks at most: an int holds them)
        uint4 v[AHEAD];
        int k[AHEAD], c[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int i = min(i0 + a * THREADS, rows * chunks - 1);
            k[a] = i / chunks;
            c[a] = i - k[a] * chunks;
            v[a] = get(k[a], c[a]);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) if (i0 + a * THREADS < rows * chunks) put(k[a], c[a], v[a]);
    }
}

// Every workgroup counts all tokens by itself (8 bytes each, from the L2 cache), so that one launch does it: the tokens before its own rows, and all.  Backward, loss by token: the largest weight, too.
template <typename T, bool BACKWARD>
__global__ __launch_bounds__(THREADS)
void prepare_kernel(const Prepare p)
{
    __shared__ int before_s[4], all_s[4];
    __shared__ float most_s[4];
    __shared__ int place[THREADS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (sizeof(T) == 4 && (int)blockIdx.x >= p.row_blocks + p.bias_blocks) {
        const int64_t chunks = p.ld / 4, all = (int64_t)p.V * chunks, stride = (int64_t)p.split_blocks * THREADS;
        constexpr int AHEAD = 4;
        for (int64_t i0 = ((int64_t)blockIdx.x - p.row_blocks - p.bias_blocks) * THREADS + threadIdx.x; i0 < all; i0 += AHEAD * stride) {
            f32x4 v[AHEAD];
            int64_t r[AHEAD], c[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int64_t i = min(i0 + k * stride, all - 1);
                r[k] = i / chunks;
                c[k] = (i - r[k] * chunks) * 4;
                v[k] = c[k] < p.D ? *reinterpret_cast<const f32x4*>(p.words_in + r[k] * p.D + c[k]) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) if (i0 + k * stride < all) split(v[k], p.words_out + r[k] * p.ld + c[k], (int64_t)p.V * p.ld);
        }
        return;
    }
    if ((int)blockIdx.x >= p.row_blocks) {
        const int i = ((int)blockIdx.x - p.row_blocks) * THREADS + threadIdx.x;
        if (i < p.bias_words) p.bias_out[i] = i >= p.V ? -__builtin_inff() : p.bias ? value(static_cast<const T*>(p.bias)[i]) : 0.0f;
        return;
    }
    const int r0 = blockIdx.x * p.per, r1 = min(p.rows, r0 + p.per);
    int before = 0, all = 0;
    float most = 0.0f;
    constexpr int AHEAD = 8;                        // loads sent off together
    const bool weights = BACKWARD && p.per_token;
    for (int i0 = threadIdx.x; i0 < p.rows; i0 += AHEAD * THREADS) {
        int64_t word[AHEAD];
        float g[AHEAD] = {};
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) { const int i = i0 + k * THREADS; word[k] = p.target[min(i, p.rows - 1)]; }
        if (weights)
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) { const int i = i0 + k * THREADS; g[k] = p.dloss[min(i, p.rows - 1)]; }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + k * THREADS;
            const bool counts = i < p.rows && word[k] != p.ignored;
            before += counts && i < r0;
            all += counts;
            const float size = fabsf(g[k]);
            most = fmaxf(most, counts && size < __builtin_inff() ? size : 0.0f);
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        before += __shfl_xor(before, o);
        all += __shfl_xor(all, o);
        most = fmaxf(most, __shfl_xor(most, o));
    }
    if (lane == 0) { before_s[wave] = before; all_s[wave] = all; most_s[wave] = most; }
    __syncthreads();
    before = before_s[0] + before_s[1] + before_s[2] + before_s[3];
    all = all_s[0] + all_s[1] + all_s[2] + all_s[3];
    most = fmaxf(fmaxf(most_s[0], most_s[1]), fmaxf(most_s[2], most_s[3]));
    // a power of two that makes the largest weight at most 1, so that what is written of P in 16 bits has the range it needs
    int e = 0;
    if (weights && most > 0.0f) e = min(max((int)(__builtin_bit_cast(uint32_t, most) >> 23) - 126, -126), 126);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *p.count = all;
        if (!BACKWARD) *p.ticket = 0;
        else *p.scale = (all == 0 ? 0.0f : p.per_token ? __builtin_amdgcn_ldexpf(1.0f, e) : p.mean ? *p.dloss / (float)all : *p.dloss) / p.size;
    }
    for (int base = r0; base < r1; base += THREADS) {
        const int r = base + threadIdx.x;
        const int64_t word = r < r1 ? p.target[r] : p.ignored;
        const bool counts = word != p.ignored;
        const uint64_t ballot = __ballot(counts);
        __syncthreads();
        if (lane == 0) before_s[wave] = __popcll(ballot);
        __syncthreads();
        int at = before + __popcll(ballot & ((1ull << lane) - 1));
        for (int w = 0; w < 4; ++w) {
            if (w < wave) at += before_s[w];
            before += before_s[w];
        }
        place[threadIdx.x] = counts ? at : -1;
        __syncthreads();
        // (read before the features, used behind them)
        Row k = {};
        float g = 1.0f;
        if (BACKWARD && counts) {
            k = p.kept[at];
            if (weights) g = p.dloss[r];
        }
        // the features of these rows, and zeros for the gradient of those that are left out
        const int rows = min(THREADS, r1 - base);
        auto left_out = [&](const int row, const int chunk) {
            if (BACKWARD && p.dx) *reinterpret_cast<uint4*>(static_cast<char*>(p.dx) + ((int64_t)(base + row) * p.D) * sizeof(T) + 16 * chunk) = make_uint4(0, 0, 0, 0);
        };
        if constexpr (sizeof(T) == 4) {
            each_chunk((int)(p.ld / 4), rows, [&](const int k, const int c) {
                return place[k] >= 0 && 4 * c < p.D ? *reinterpret_cast<const uint4*>(static_cast<const float*>(p.x) + (int64_t)(base + k) * p.D + 4 * c) : make_uint4(0, 0, 0, 0);
            }, [&](const int k, const int c, const uint4 v) {
                if (place[k] >= 0) split(__builtin_bit_cast(f32x4, v), p.features + (int64_t)place[k] * p.ld + 4 * c, p.piece);
                else if (4 * c < p.D) left_out(k, c);
            });
        } else if (all < p.rows) {
            each_chunk(p.D / 8, rows, [&](const int k, const int c) {
                return place[k] >= 0 ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + (int64_t)(base + k) * p.D + 8 * c) : make_uint4(0, 0, 0, 0);
            }, [&](const int k, const int c, const uint4 v) {
                if (place[k] >= 0) *reinterpret_cast<uint4*>(p.features + (int64_t)place[k] * p.ld + 8 * c) = v;
                else left_out(k, c);
            });
        }
        if (counts) {
            p.index[at] = r;
            if (!BACKWARD) p.words[at] = word >= 0 && word < p.V ? (int)word : -1;
            else {
                const float weight = (weights ? __builtin_amdgcn_ldexpf(g, -e) : 1.0f) * p.size;
                p.row[at] = Row{k.shift, k.scale * weight, (p.target_even - k.own) * weight, k.target};
                p.weight[at] = weight;
            }
        } else if (!BACKWARD && r < r1 && p.loss) p.loss[r] = 0.0f;
    }
}

// The losses from what the products left of each column group: 32 tokens a workgroup, every 8th group a thread.  The last workgroup adds up the workgroups' sums, in their order.
// (The hardware's exponential will do: of arguments x <= 0 it is off by 2^-23 + |x| 2^-24 of itself, so that a term exp(x) is off by less than 2^-22 of the largest.)
struct Losses {
    const float2* part; const float* part_sum; const float* wanted; const int* words; const int* count; const int* index;
    int all, groups, V, reduction;
    float e;
    float* loss; Row* kept;                         // kept: or NULL
    double* sums; uint32_t* ticket;
};
constexpr int LOSS_ROWS = 32, SLICES = THREADS / LOSS_ROWS;
__global__ __launch_bounds__(THREADS)
void loss_kernel(const Losses p)
{
    __shared__ float most_s[SLICES][LOSS_ROWS], total_s[SLICES][LOSS_ROWS], sum_s[SLICES][LOSS_ROWS];
    __shared__ double block_s[THREADS];
    __shared__ bool last;
    const int n = *p.count, r = threadIdx.x % LOSS_ROWS, slice = threadIdx.x / LOSS_ROWS, row = blockIdx.x * LOSS_ROWS + r, from = min(row, p.all - 1);
    const int word = slice == 0 ? p.words[from] : 0, to = slice == 0 ? p.index[from] : 0;      // (behind the last that counts: nothing that is used)
    const float own = slice == 0 ? p.wanted[from] : 0.0f;
    float most = LOWEST, total = 0.0f, sum = 0.0f;
    constexpr int AHEAD = 8;                        // loads sent off together
    for (int g0 = slice; g0 < p.groups && row < n; g0 += AHEAD * SLICES) {
        float2 v[AHEAD];
        float t[AHEAD] = {};
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) { const int g = g0 + k * SLICES; v[k] = p.part[(int64_t)min(g, p.groups - 1) * p.all + row]; }
        if (p.part_sum)
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) { const int g = g0 + k * SLICES; t[k] = p.part_sum[(int64_t)min(g, p.groups - 1) * p.all + row]; }
        float m = most;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (g0 + k * SLICES >= p.groups) { v[k] = make_float2(LOWEST, 0.0f); t[k] = 0.0f; }
            m = fmaxf(m, v[k].x);
        }
        total *= __expf(most - m);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) { total += v[k].y * __expf(v[k].x - m); sum += t[k]; }
        most = m;
    }
    most_s[slice][r] = most; total_s[slice][r] = total; sum_s[slice][r] = sum;
    __syncthreads();
    double mine = 0.0;
    if (slice == 0 && row < n) {
        for (int s = 1; s < SLICES; ++s) most = fmaxf(most, most_s[s][r]);
        total = 0.0f; sum = 0.0f;
        for (int s = 0; s < SLICES; ++s) { total += total_s[s][r] * __expf(most_s[s][r] - most); sum += sum_s[s][r]; }
        const float wanted = word >= 0 ? own : __builtin_nanf("");
        float missed, loss = loss_of(most, total, wanted, missed);
        if (p.e != 0.0f && loss < __builtin_inff()) loss += p.e * wanted - p.e / (float)p.V * sum;        // (a word at -infinity is infinitely wrong already)
        if (p.kept) p.kept[row] = Row{most, missed / (total != 0.0f ? total : 1.0f), missed, word};
        if (p.reduction == PROTEUS_CE_NONE) p.loss[to] = loss;
        mine = loss;
    }
    if (p.reduction == PROTEUS_CE_NONE) return;
    block_s[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < LOSS_ROWS; ++i) s += block_s[i];
        p.sums[blockIdx.x] = s;
        __threadfence();
        last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double s = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += THREADS) s += __builtin_nontemporal_load(p.sums + i);
    block_s[threadIdx.x] = s;
    __syncthreads();
    for (int o = THREADS / 2; o; o >>= 1) {
        if ((int)threadIdx.x < o) block_s[threadIdx.x] += block_s[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *p.loss = (float)(p.reduction == PROTEUS_CE_MEAN ? block_s[0] / (double)n : block_s[0]);
}

// Sums of shares of dx (a token's row of it) and dW, and of the bias's gradient over groups of rows.
struct Ends {
    const int* count; const int* index; const float* scale;
    int all, D, V;
    const float* dx_slab; int dx_shares; void* dx;
    const float* dw_slab; int dw_shares; void* dw;
    const float* columns; int group; int piece; void* db;      // [piece of the vocabulary][row group][its words]
    int first[4];                                   // workgroups of each
};
template <typename T>
__global__ __launch_bounds__(THREADS)
void ends_kernel(const Ends p)
{
    __shared__ float s[8][32];
    const int n = *p.count, block = blockIdx.x;
    const float scale = *p.scale;
    const int job = block >= p.first[2] ? 2 : block >= p.first[1] ? 1 : 0;
    if (job == 2) {
        const int w = (block - p.first[2]) * 32 + (threadIdx.x & 31), g0 = threadIdx.x >> 5;
        const int groups = (n + p.group - 1) / p.group, most = (p.all + 255) / 256 * 256 / p.group;
        float v = 0.0f;
        if (w < p.V) {
            const int piece = w / p.piece, words = min(p.piece, p.V - piece * p.piece);
            const float* const from = p.columns + (int64_t)piece * p.piece * most + (w - piece * p.piece);
#pragma unroll 8
            for (int g = g0; g < groups; g += 8) v += from[(int64_t)g * words];
        }
        s[g0][threadIdx.x & 31] = v;
        __syncthreads();
        if (g0 == 0 && w < p.V) {
            for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x];
            put(static_cast<T*>(p.db) + w, v * scale);
        }
        return;
    }
    const int blocks = p.first[job + 1] - p.first[job];
    const int64_t rows = job ? p.V : n, chunks = p.D / 4, stride = (job ? (int64_t)p.V : (int64_t)p.all) * p.D;
    const float* const slab = job ? p.dw_slab : p.dx_slab;
    const int shares = job ? p.dw_shares : p.dx_shares;
    T* const out = static_cast<T*>(job ? p.dw : p.dx);
    for (int64_t i = (int64_t)(block - p.first[job]) * THREADS + threadIdx.x; i < rows * chunks; i += (int64_t)blocks * THREADS) {
        const int64_t r = i / chunks, c = (i - r * chunks) * 4;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < shares; ++k) v += *reinterpret_cast<const f32x4*>(slab + k * stride + r * p.D + c);
        T* const to = out + (job ? r : (int64_t)p.index[r]) * p.D + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) put(to + e, v[e] * scale);
    }
}

// ---------------------------------------------------------------------------------------------------- plans

int64_t up(const int64_t x, const int64_t by) { return (x + by - 1) / by * by; }
int pieces_of(const int type) { return type == PROTEUS_DTYPE_F32 ? 3 : 1; }
bool all_pieces(const int type, const int tile) { return type == PROTEUS_DTYPE_F32 && tile == T64; }         // of fp32 in a step; else a product of two pieces at a time
int segments_of(const int type, const int tile) { return type == PROTEUS_DTYPE_F32 && tile != T64 ? 6 : 1; }
int64_t tiles_of(const int t, const int64_t M, const int64_t N) { return ((M + rows_of(t) - 1) / rows_of(t)) * ((N + columns_of(t) - 1) / columns_of(t)); }

struct Plan { int tile, shares; };

// What a product takes, us, as measured: rounds of workgroups by the time of one (one tile of 256 x 256 to a compute unit; two of 128 x 128; three of 64 x 128, in fp32 one), a step of 64 k and an epilogue each, and
// what the first tile waits for that the later ones find done.
double cost_of(const int type, const int t, const int role, const int64_t tiles, const int64_t steps)
{
    static const double end256[4] = {5.5, 9.0, 2.5, 2.5}, first256[4] = {8.0, 7.0, 4.0, 4.0}, end128[4] = {3.0, 5.0, 1.0, 1.0}, end64[4] = {1.5, 3.0, 1.0, 1.0}, full64[4] = {0.93, 0.93, 1.25, 1.4};
    if (t == T256) return 2.0 + first256[role] + (double)((tiles + 255) / 256) * ((tiles < 128 ? 1.15 : 1.6) * steps + end256[role]);
    if (all_pieces(type, t)) {                      // (half a chip's loads do not fill the caches' bandwidth yet)
        static const double alone[4] = {0.88, 0.92, 1.03, 1.23}, full[4] = {1.15, 1.25, 1.38, 1.42}, end[4] = {4.2, 6.0, 3.0, 4.0};
        const int64_t rest = tiles % 256;
        return 2.0 + (tiles / 256) * (full[role] * steps + end[role]) + (rest == 0 ? 0.0 : (rest <= 128 ? alone : full)[role] * steps + end[role]);
    }
    const int together = t == T128 ? 512 : 768;
    const double alone = (t == T128 ? 0.55 : 0.42) * steps + (t == T128 ? end128 : end64)[role], full = (t == T128 ? 1.02 : full64[role]) * steps + (t == T128 ? end128 : end64)[role];
    const int64_t whole = tiles / together, rest = tiles % together;
    // (two to a unit of 64 x 128: two thirds of three)
    return 2.0 + whole * full + (rest == 0 ? 0.0 : rest <= 256 ? alone : t == T64 && rest <= 512 ? std::max(alone, full * 0.75) : full);
}

Plan plan_of(const int role, const int64_t M, const int64_t N, const int64_t K, const int type, const bool shared, double* const cost = nullptr, const int only = -1)
{
    const int64_t steps = (K + 63) / 64;
    Plan best = {T128, 1};
    double least = 1e30;
    for (int t = only < 0 ? T256 : only; t <= (only < 0 ? T64 : only); ++t)
        for (int s = 1; s <= (shared ? MOST_SHARES : 1); ++s) {
            const int64_t per = s == 1 ? steps : up((steps + s - 1) / s, 2);
            if ((s > 1 && per < (all_pieces(type, t) ? 2 : 4)) || (t != T256 && tiles_of(t, M, N) * s > MOST_TILES)) break;
            const double c = cost_of(type, t, role, tiles_of(t, M, N) * s, per * segments_of(type, t)) + (s > 1 ? 2.5 + (double)M * N * 8 * s / 8e6 : 0.0);
            if (c < least) { least = c; best = {t, s}; }
        }
    if (cost) *cost = least;
    return best;
}

// The two gradients behind P: one after the other, or side by side in one launch of 128 x 128 (fp32: 64 x 128), the longer workgroups first, in such shares that all are done soonest.
// Alone the tiles of either seldom fill the chip.  2000 x 768 x 8001 in fp16: 158 us a pass one after the other, 150 side by side; 2048 x 512 x 1000 in fp32 121 and 115 (then on tiles of 128); 5003 x 712 x 20011, where
// they do, stays as it was.
struct Behind { bool together, dw_first; Plan dx, dw; };
// When `n` jobs of `length` and then `n2` of `length2`, which are shorter, are done by 256
double done(const int64_t n, const double length, const int64_t n2, const double length2)
{
    const int64_t late = n % 256;                   // units with one of the first more than the others
    const double early = (double)(n / 256) * length, all_first = early + (late ? length : 0.0);
    double t = std::max(all_first, (n * length + n2 * length2) / 256);          // at least
    for (int k = 0; k < 4; ++k) {                   // the others' ends in turn, until there are enough
        const int64_t by_early = (int64_t)((t - early) / length2 + 1e-6), by_late = (int64_t)((t - early - length) / length2 + 1e-6);
        if ((256 - late) * by_early + late * by_late >= n2) break;
        t = std::min(early + (by_early + 1) * length2, late ? early + length + (by_late + 1) * length2 : 1e30);
    }
    return t;
}
Behind behind(const int64_t rows, const int64_t D, const int64_t words, const int type, const bool shared_dw)
{
    double cost_dx, cost_dw;
    Behind b = {false, false, plan_of(DX, rows, D, words, type, true, &cost_dx), plan_of(DW, words, D, rows, type, shared_dw, &cost_dw)};
    const int t = type == PROTEUS_DTYPE_F32 ? T64 : T128;
    const int64_t steps[2] = {(words + 63) / 64, (rows + 63) / 64}, tiles[2] = {tiles_of(t, rows, D), tiles_of(t, words, D)}, size[2] = {rows * D, words * D};
    double least = cost_dx + cost_dw;
    for (int limit = t == T64 ? 2 : 4; limit <= 16384; limit += limit < 16 ? 2 : limit / 4) {
        double all = 0.0, longest = 0.0, sums = 0.0, length[2];
        int shares[2];
        for (int i = 0; i < 2; ++i) {
            shares[i] = i == 1 && !shared_dw ? 1 : (int)std::min<int64_t>((steps[i] + limit - 1) / limit, MOST_SHARES);
            const int64_t per = shares[i] == 1 ? steps[i] : up((steps[i] + shares[i] - 1) / shares[i], 2);
            all += (double)(tiles[i] * shares[i]) * (0.53 * per + 1.0) / 256;
            length[i] = t == T64 ? 1.38 * per + 3.0 : 1.05 * per + 2.0;
            longest = std::max(longest, length[i]);
            if (shares[i] > 1) sums += (double)size[i] * 8 * shares[i] / 8e6;
        }
        const int l = length[1] > length[0];        // the longer ones first
        const double work = t == T128 ? std::max(all, longest) : done(tiles[l] * shares[l], length[l], tiles[1 - l] * shares[1 - l], length[1 - l]);
        const double c = 4.0 + work + sums + (sums > 0.0 ? 2.5 : 0.0);
        if (c < least) { least = c; b = {true, l == 1, {t, shares[0]}, {t, shares[1]}}; }
    }
    return b;
}

// All that a call's sizes determine.
struct Sizes {
    int64_t rows, D, V, ld;                         // ld: of pieces
    int type, pieces, p_pieces, groups;
    bool fine;
    Plan stats, grad, dx, dw;
    bool together, dw_first;
    int64_t width, parts, ldp;                      // of the vocabulary's pieces
    Sizes(const proteus_ce_args& a)
    {
        rows = a.rows; D = a.d; V = a.vocab; type = a.dtype; pieces = pieces_of(type);
        ld = pieces > 1 ? up(D, 8) : D;
        fine = pieces == 1 && rows <= FINE_ROWS;
        p_pieces = fine ? 2 : pieces;
        stats = plan_of(STATS, rows, V, ld, type, false);
        groups = (int)((V + columns_of(stats.tile) - 1) / columns_of(stats.tile) * 2);
        const int64_t most = std::max<int64_t>(LEAST_WORDS, P_BYTES / (rows * 2 * p_pieces) / 256 * 256);
        parts = (V + most - 1) / most;
        width = parts == 1 ? V : up((V + parts - 1) / parts, 256);
        parts = (V + width - 1) / width;
        ldp = up(width, 64);
        grad = plan_of(GRAD, rows, width, ld, type, false, nullptr, fine ? T64 : -1);
        Behind b;
        if (!fine) b = behind(rows, D, width, type, parts == 1);
        else b = {false, false, {T64_FINE, plan_of(DX, rows, D, width, type, true, nullptr, T64).shares}, {T64_FINE, 1}};
        together = b.together; dw_first = b.dw_first; dx = b.dx; dw = b.dw;
    }
    int64_t row_groups() const { return up(rows, 256) / row_group(grad.tile); }
    bool dx_apart() const { return dx.shares > 1 || parts > 1; }            // sums over pieces and shares before they are rounded
    bool padded(const bool bias) const { return bias || V % 256; }
};

// A workspace's parts, one behind the other.
struct Space {
    char* at; size_t used = 0;
    template <typename T> T* take(const int64_t count)
    {
        T* const p = at ? reinterpret_cast<T*>(at + used) : nullptr;
        used += (size_t)up(count * (int64_t)sizeof(T), 256);
        return p;
    }
};

struct Common { int* count; int* index; uint16_t* features; uint16_t* weights; float* bias; };
Common common(Space& s, const Sizes& z)
{
    Common c;
    c.count = s.take<int>(64);
    c.index = s.take<int>(z.rows);
    c.features = s.take<uint16_t>(z.rows * z.ld * z.pieces);
    c.weights = z.pieces > 1 ? s.take<uint16_t>(z.V * z.ld * z.pieces) : nullptr;
    c.bias = s.take<float>(up(z.V, 256) + 256);
    return c;
}

struct Forward { Common c; int* words; float2* part; float* part_sum; float* wanted; double* sums; };
Forward forward_space(Space& s, const Sizes& z, const bool smoothing)
{
    Forward f;
    f.c = common(s, z);
    f.words = s.take<int>(z.rows);
    f.part = s.take<float2>(z.groups * z.rows);
    f.part_sum = smoothing ? s.take<float>(z.groups * z.rows) : nullptr;
    f.wanted = s.take<float>(z.rows);
    f.sums = s.take<double>((z.rows + LOSS_ROWS - 1) / LOSS_ROWS);
    return f;
}

struct Backward { Common c; Row* row; float* weight; uint16_t* P; float* columns; float* dx_slab; float* dw_slab; };
Backward backward_space(Space& s, const Sizes& z, const bool bias)
{
    Backward b;
    b.c = common(s, z);
    b.row = s.take<Row>(z.rows);
    b.weight = s.take<float>(z.rows);
    b.P = s.take<uint16_t>(z.rows * z.ldp * z.p_pieces);
    b.columns = bias ? s.take<float>(z.row_groups() * up(z.V, 4)) : nullptr;
    b.dx_slab = z.dx_apart() ? s.take<float>((int64_t)z.dx.shares * z.rows * z.D) : nullptr;
    b.dw_slab = z.dw.shares > 1 ? s.take<float>((int64_t)z.dw.shares * z.V * z.D) : nullptr;
    return b;
}

int check(const proteus_ce_args* p)
{
    if (!p) return PROTEUS_ERR_NULL_POINTER;
    const proteus_ce_args& a = *p;
    if (a.dtype != PROTEUS_DTYPE_F32 && a.dtype != PROTEUS_DTYPE_BF16 && a.dtype != PROTEUS_DTYPE_F16) return PROTEUS_ERR_BAD_OPERAND_TYPE;
    if (a.rows < 1 || a.rows > (1 << 24) || a.vocab < 1 || a.vocab > (1 << 24) || a.d < 1 || a.d > (1 << 16) || a.d % (a.dtype == PROTEUS_DTYPE_F32 ? 4 : 8)) return PROTEUS_ERR_BAD_SHAPE;
    if (!(a.label_smoothing >= 0.0f && a.label_smoothing <= 1.0f)) return PROTEUS_ERR_BAD_SHAPE;
    if (a.reduction != PROTEUS_CE_NONE && a.reduction != PROTEUS_CE_MEAN && a.reduction != PROTEUS_CE_SUM) return PROTEUS_ERR_UNSUPPORTED;
    return 0;
}
int check_pointers(const proteus_ce_args& a, const void* ws, const size_t ws_bytes, const size_t wanted)
{
    if (!a.x || !a.weight || !a.target || !ws) return PROTEUS_ERR_NULL_POINTER;
    if ((uintptr_t)a.x % 16 || (uintptr_t)a.weight % 16 || (uintptr_t)a.bias % 16 || (uintptr_t)a.target % 8 || (uintptr_t)ws % 256) return PROTEUS_ERR_BAD_ALIGNMENT;
    return ws_bytes < wanted ? PROTEUS_ERR_TOO_LARGE : 0;
}

unsigned blocks_of(const int tile, const int64_t M, const int64_t N, const int shares)
{
    const int64_t per_xcd = (tiles_of(tile, M, N) * shares + 7) / 8;
    return 8u * (unsigned)(tile == T256 ? std::min<int64_t>(per_xcd, 32) : per_xcd);                           // (32 compute units of an XCD)
}
int launch(const Args& a, const int role, const Plan& plan, const int type, const int64_t M, hipStream_t st)
{
    return (type == PROTEUS_DTYPE_BF16 ? launch_bf16 : type == PROTEUS_DTYPE_F16 ? launch_f16 : launch_f32)(a, role, plan.tile, blocks_of(plan.tile, M, a.N, plan.shares), st);
}

Prepare prepare_of(const proteus_ce_args& a, const Sizes& z, const Common& c)
{
    Prepare p = {};
    p.x = a.x; p.bias = a.bias; p.target = a.target; p.ignored = a.ignore_index;
    p.rows = (int)z.rows; p.D = (int)z.D; p.V = (int)z.V; p.type = z.type;
    p.per = (int)std::max<int64_t>(16, (z.rows + 511) / 512);
    p.row_blocks = (p.rows + p.per - 1) / p.per;
    p.count = c.count; p.index = c.index; p.features = c.features; p.ld = z.ld; p.piece = z.rows * z.ld;
    if (z.padded(a.bias)) { p.bias_out = c.bias; p.bias_words = (int)up(z.V, 256); p.bias_blocks = (p.bias_words + THREADS - 1) / THREADS; }
    if (c.weights) {
        p.words_in = static_cast<const float*>(a.weight); p.words_out = c.weights;
        p.split_blocks = (int)std::min<int64_t>((z.V * (z.ld / 4) + 4 * THREADS - 1) / (4 * THREADS), 2048);
    }
    return p;
}
template <bool BACKWARD> int go_prepare(const Prepare& p, hipStream_t st)
{
    const dim3 grid((unsigned)(p.row_blocks + p.bias_blocks + p.split_blocks)), block(THREADS);
    if (p.type == PROTEUS_DTYPE_F32)       hipLaunchKernelGGL((prepare_kernel<float, BACKWARD>), grid, block, 0, st, p);
    else if (p.type == PROTEUS_DTYPE_BF16) hipLaunchKernelGGL((prepare_kernel<bf16_t, BACKWARD>), grid, block, 0, st, p);
    else                                   hipLaunchKernelGGL((prepare_kernel<f16_t, BACKWARD>), grid, block, 0, st, p);
    return (int)hipGetLastError();
}
// x W^T for the words from `first` on
Args logits_of(const proteus_ce_args& a, const Sizes& z, const Common& c, const int64_t first, const int64_t words)
{
    Args g = {};
    g.A = c.features; g.lda = z.ld; g.piece_a = z.rows * z.ld;
    g.x_all = z.pieces > 1 ? nullptr : static_cast<const uint16_t*>(a.x);
    g.B = (c.weights ? c.weights : static_cast<const uint16_t*>(a.weight)) + first * z.ld; g.ldb = z.ld; g.piece_b = z.V * z.ld;
    g.count = c.count; g.all = (int)z.rows;
    g.M = (int)z.rows; g.N = (int)words; g.K = (int)z.ld;
    g.group = 8; g.shares = 1;
    g.bias = z.padded(a.bias) ? c.bias + first : nullptr;
    g.first = (int)first;
    return g;
}

}  // namespace

// Heads of few words: their own kernels.  A pass on the device, theirs and the general path's, us, bf16: 8192 tokens of 512 features, 20 words 28 / 68, 64 words 45 / 70; 65536 of 1024, 20 words 155 / 297, 64 words
// 338 / 305 (the only one of 54 sizes where they lose more than 2 %); 64 of 512, 20 words 19 / 39.  fp32: 8192 of 512, 20 words 29 / 114, 64 words 45 / 117.
static bool small(const proteus_ce_args& a) { return a.vocab <= SMALL_WORDS; }

extern "C" size_t proteus_linear_ce_kept_bytes(const proteus_ce_args* args)
{
    if (check(args)) return 0;
    return small(*args) ? small_kept_bytes(*args) : (size_t)args->rows * sizeof(Row);
}

extern "C" size_t proteus_linear_ce_fwd_bytes(const proteus_ce_args* args)
{
    if (check(args)) return 0;
    if (small(*args)) return small_forward_bytes(*args);
    Space s = {nullptr};
    forward_space(s, Sizes(*args), args->label_smoothing != 0.0f);
    return s.used;
}

extern "C" size_t proteus_linear_ce_bwd_bytes(const proteus_ce_args* args)
{
    if (check(args)) return 0;
    if (small(*args)) return small_backward_bytes(*args);
    Space s = {nullptr};
    backward_space(s, Sizes(*args), args->bias != nullptr);
    return s.used;
}

extern "C" int proteus_linear_ce_fwd(const proteus_ce_args* args, float* loss, void* kept, size_t kept_bytes, void* ws, size_t ws_bytes, void* stream)
{
    if (const int rc = check(args)) return rc;
    const proteus_ce_args& a = *args;
    if (const int rc = check_pointers(a, ws, ws_bytes, proteus_linear_ce_fwd_bytes(args))) return rc;
    if (!loss) return PROTEUS_ERR_NULL_POINTER;
    if ((uintptr_t)loss % 4 || (uintptr_t)kept % 16) return PROTEUS_ERR_BAD_ALIGNMENT;
    if (kept && kept_bytes < proteus_linear_ce_kept_bytes(args)) return PROTEUS_ERR_TOO_LARGE;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (small(a)) return small_forward(a, loss, kept, ws, st);
    const Sizes z(a);
    Space s = {static_cast<char*>(ws)};
    const Forward f = forward_space(s, z, a.label_smoothing != 0.0f);
    Prepare p = prepare_of(a, z, f.c);
    p.words = f.words;
    p.loss = a.reduction == PROTEUS_CE_NONE ? loss : nullptr;
    p.ticket = reinterpret_cast<uint32_t*>(f.c.count + 1);
    if (const int rc = go_prepare<false>(p, st)) return rc;
    Args g = logits_of(a, z, f.c, 0, z.V);
    g.target = f.words; g.part = f.part; g.part_sum = f.part_sum; g.wanted = f.wanted;
    if (const int rc = launch(g, STATS, z.stats, z.type, z.rows, st)) return rc;
    Losses l = {};
    l.part = f.part; l.part_sum = f.part_sum; l.wanted = f.wanted; l.words = f.words; l.count = f.c.count; l.index = f.c.index;
    l.all = (int)z.rows; l.groups = z.groups; l.V = (int)z.V; l.reduction = a.reduction; l.e = a.label_smoothing;
    l.loss = loss; l.kept = static_cast<Row*>(kept); l.sums = f.sums; l.ticket = p.ticket;
    hipLaunchKernelGGL(loss_kernel, dim3((unsigned)((z.rows + LOSS_ROWS - 1) / LOSS_ROWS)), dim3(THREADS), 0, st, l);
    return (int)hipGetLastError();
}

extern "C" int proteus_linear_ce_bwd(const proteus_ce_args* args, const float* dloss, const void* kept, size_t kept_bytes, void* dx, void* dweight, void* dbias, void* ws, size_t ws_bytes, void* stream)
{
    if (const int rc = check(args)) return rc;
    const proteus_ce_args& a = *args;
    if (const int rc = check_pointers(a, ws, ws_bytes, proteus_linear_ce_bwd_bytes(args))) return rc;
    if (!dloss || !kept || (dbias && !a.bias)) return PROTEUS_ERR_NULL_POINTER;
    if ((uintptr_t)dloss % 4 || (uintptr_t)kept % 16 || (uintptr_t)dx % 16 || (uintptr_t)dweight % 16 || (uintptr_t)dbias % 16) return PROTEUS_ERR_BAD_ALIGNMENT;
    if (kept_bytes < proteus_linear_ce_kept_bytes(args)) return PROTEUS_ERR_TOO_LARGE;
    if (!dx && !dweight && !dbias) return 0;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (small(a)) return small_backward(a, dloss, kept, dx, dweight, dbias, ws, st);
    const Sizes z(a);
    Space s = {static_cast<char*>(ws)};
    const Backward b = backward_space(s, z, a.bias != nullptr);
    const int itemsize = z.type == PROTEUS_DTYPE_F32 ? 4 : 2;
    Prepare p = prepare_of(a, z, b.c);
    p.kept = static_cast<const Row*>(kept); p.dloss = dloss; p.per_token = a.reduction == PROTEUS_CE_NONE; p.mean = a.reduction == PROTEUS_CE_MEAN;
    p.row = b.row; p.weight = b.weight; p.scale = reinterpret_cast<float*>(b.c.count + 2);
    const float even = a.label_smoothing / (float)a.vocab;
    p.target_even = a.label_smoothing - even; p.size = z.type == PROTEUS_DTYPE_F16 ? F16_SCALE : 1.0f;
    p.dx = dx;
    if (const int rc = go_prepare<true>(p, st)) return rc;
    for (int64_t i = 0; i < z.parts; ++i) {
        const int64_t first = i * z.width, words = std::min(z.width, z.V - first);
        Args g = logits_of(a, z, b.c, first, words);
        g.row = b.row; g.weight = b.weight; g.P = b.P; g.ldp = z.ldp; g.piece_p = z.rows * z.ldp; g.fine = z.fine; g.even = even;
        g.columns = dbias ? b.columns + first * z.row_groups() : nullptr;
        if (const int rc = launch(g, GRAD, z.grad, z.type, z.rows, st)) return rc;
        Args gx = {}, gw = {};
        gx.A = b.P; gx.lda = z.ldp; gx.piece_a = z.rows * z.ldp;
        gx.B = g.B; gx.ldb = z.ld; gx.piece_b = z.V * z.ld;
        gx.count = b.c.count; gx.all = (int)z.rows;
        gx.M = (int)z.rows; gx.N = (int)z.D; gx.K = (int)words; gx.group = 8; gx.shares = z.dx.shares;
        gx.slab = b.dx_slab; gx.adds = i > 0;
        gx.C = dx; gx.ldc = z.D; gx.scale = p.scale; gx.rows = b.c.index;
        gw.A = b.P; gw.lda = z.ldp; gw.piece_a = z.rows * z.ldp; gw.a_cols = (int)up(words, 8);
        gw.B = b.c.features; gw.ldb = z.ld; gw.piece_b = z.rows * z.ld; gw.x_all = g.x_all;
        gw.count = b.c.count; gw.all = (int)z.rows;
        gw.M = (int)words; gw.N = (int)z.D; gw.K = (int)z.rows; gw.group = 8; gw.shares = z.dw.shares;
        gw.slab = b.dw_slab;
        gw.C = static_cast<char*>(dweight) + first * z.D * itemsize; gw.ldc = z.D; gw.scale = p.scale;
        if (dx && dweight && z.together) {
            const auto both = z.type == PROTEUS_DTYPE_BF16 ? launch_both_bf16 : z.type == PROTEUS_DTYPE_F16 ? launch_both_f16 : launch_both_f32;
            if (const int rc = both(gx, gw, blocks_of(z.dx.tile, z.rows, z.D, z.dx.shares), blocks_of(z.dw.tile, words, z.D, z.dw.shares), z.dw_first, st)) return rc;
            continue;
        }
        if (dx) if (const int rc = launch(gx, DX, z.dx, z.type, z.rows, st)) return rc;
        if (dweight) if (const int rc = launch(gw, DW, z.dw, z.type, words, st)) return rc;
    }
    Ends e = {};
    e.count = b.c.count; e.index = b.c.index; e.scale = p.scale;
    e.all = (int)z.rows; e.D = (int)z.D; e.V = (int)z.V;
    e.dx_slab = b.dx_slab; e.dx_shares = z.dx.shares; e.dx = dx;
    e.dw_slab = b.dw_slab; e.dw_shares = z.dw.shares; e.dw = dweight;
    e.columns = b.columns; e.group = row_group(z.grad.tile); e.piece = (int)z.width; e.db = dbias;
    e.first[1] = dx && b.dx_slab ? (int)std::min<int64_t>((z.rows * (z.D / 4) + THREADS - 1) / THREADS, 4096) : 0;
    e.first[2] = e.first[1] + (dweight && b.dw_slab ? (int)std::min<int64_t>((z.V * (z.D / 4) + THREADS - 1) / THREADS, 4096) : 0);
    e.first[3] = e.first[2] + (dbias ? (int)((z.V + 31) / 32) : 0);
    if (!e.first[3]) return 0;
    const dim3 grid((unsigned)e.first[3]), block(THREADS);
    if (z.type == PROTEUS_DTYPE_F32)       hipLaunchKernelGGL((ends_kernel<float>), grid, block, 0, st, e);
    else if (z.type == PROTEUS_DTYPE_BF16) hipLaunchKernelGGL((ends_kernel<bf16_t>), grid, block, 0, st, e);
    else                                   hipLaunchKernelGGL((ends_kernel<f16_t>), grid, block, 0, st, e);
    return (int)hipGetLastError();
}

extern "C" int proteus_linear_ce_check(const proteus_ce_args* args) { return check(args); }

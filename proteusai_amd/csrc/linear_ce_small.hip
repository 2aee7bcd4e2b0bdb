// Softmax cross entropy from features for heads of up to 64 words (gfx950): the operator of linear_ce.hip where its tiles of 128 and 256 words would be mostly empty.
//
// Products on the fp32 matrix instructions (32 x 32 x 2), whatever the operands' type: 16-bit ones are exact in fp32, nothing is rounded before the results are, and few words cost less than reading the
// features does.  Bound by launches and memory: 8192 tokens of 512 features in fp32, 20 words: forward 10 us (17 MB read, 1.6 TB/s), backward 15 (34 MB, 2.2), their sums 4 each.
//
// Forward.  A workgroup has 32 tokens; its waves take a quarter of the features each, straight from memory into registers (a lane's token, 16 bytes of its row), and add up in LDS.  The probabilities
// less the targets' are kept for the backward, 4 bytes a word: little beside the features' rows, and what saves the logits' second product.
//
// Backward.  A workgroup has 128 features of every G-th block of 32 tokens: its words' weights and the sums of dW stay in registers, dx leaves as it is made, and a second launch adds up the G sums of dW
// and db.  The order of sums is fixed.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include <algorithm>
#include "linear_ce_internal.h"
#include "linear_ce_small.h"

namespace {

using namespace proteus_ce;

constexpr int THREADS = 256, TOKENS = 32, COLUMNS = 128;
constexpr int64_t HEAD = 256;                       // bytes in front of what is kept: the number of tokens that count

typedef float f32x16 __attribute__((ext_vector_type(16)));
struct f16_t { _Float16 v; };
struct bf16_t { __bf16 v; };
__device__ __forceinline__ float value(const f16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const bf16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const float x) { return x; }
template <typename T> __device__ __forceinline__ T rounded(const float x) { T r; r.v = (decltype(r.v))x; return r; }
template <> __device__ __forceinline__ float rounded<float>(const float x) { return x; }
template <typename T, int N> struct __align__(N * sizeof(T)) Pack { T e[N]; };

// Reads without branches: what lies outside comes back as zeros.
constexpr uint32_t OUTSIDE = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, const int64_t bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)min(bytes, (int64_t)0x7ffffff0), 0x00020000); }
template <typename T> using PackOf = Pack<T, 16 / sizeof(T)>;
template <typename T> __device__ __forceinline__ PackOf<T> sixteen_bytes(const __amdgpu_buffer_rsrc_t r, const uint32_t at)
{
    return __builtin_bit_cast(PackOf<T>, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
}
template <typename T> __device__ __forceinline__ float one(const __amdgpu_buffer_rsrc_t r, const uint32_t at)
{
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
    else return value(__builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0)));
}

__device__ __forceinline__ f32x16 product(const float a, const float b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

struct SmallForward {
    const void *x, *weight, *bias;
    const int64_t* target;
    int64_t ignored;
    int rows, D, V, reduction, chunks;              // chunks of a wave's share of the features
    float e;
    float* loss;                                    // by token; else
    double* sums; int* counts;                      // of each workgroup
    float* kept;                                    // [rows][V], or NULL
};

template <typename T, int NV>
__global__ __launch_bounds__(THREADS)
void small_forward_kernel(const SmallForward p)
{
    constexpr int E = 16 / sizeof(T), PITCH = TOKENS + 1;
    __shared__ float logits[4][NV * 32 * PITCH];
    __shared__ float most_s[8][TOKENS], total_s[8][TOKENS], sum_s[8][TOKENS], wanted_s[TOKENS], loss_s[TOKENS];
    __shared__ float out[TOKENS * NV * 32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int m0 = blockIdx.x * TOKENS, m = m0 + col;
    const bool counts = m < p.rows && p.target[m] != p.ignored;
    if (!__syncthreads_or(counts)) {                // nothing to do but to say so
        if (threadIdx.x < TOKENS && m < p.rows && p.loss) p.loss[m] = 0.0f;
        if (p.kept) for (int i = threadIdx.x; i < min(TOKENS, p.rows - m0) * p.V; i += THREADS) p.kept[(int64_t)m0 * p.V + i] = 0.0f;
        if (threadIdx.x == 0 && p.sums) { p.sums[blockIdx.x] = 0.0; p.counts[blockIdx.x] = 0; }
        return;
    }
    f32x16 acc[NV] = {};
    {
        const __amdgpu_buffer_rsrc_t rx = buffer_of(static_cast<const T*>(p.x) + (int64_t)m0 * p.D, (int64_t)min(TOKENS, p.rows - m0) * p.D * sizeof(T)), rw = buffer_of(p.weight, (int64_t)p.V * p.D * sizeof(T));
        const int k0 = wave * p.chunks * 2 * E + half * E;
        constexpr int DEEP = NV == 1 ? 8 : 4;       // chunks whose loads are sent off together
        for (int c0 = 0; c0 < p.chunks; c0 += DEEP) {
            PackOf<T> a[DEEP], b[DEEP][NV];
#pragma unroll
            for (int c = 0; c < DEEP; ++c) {
                const int k = k0 + (c0 + c) * 2 * E;
                const bool in = k < p.D && c0 + c < p.chunks;
                a[c] = sixteen_bytes<T>(rx, in && counts ? (uint32_t)(col * p.D + k) * (uint32_t)sizeof(T) : OUTSIDE);
#pragma unroll
                for (int v = 0; v < NV; ++v) b[c][v] = sixteen_bytes<T>(rw, in && v * 32 + col < p.V ? (uint32_t)((v * 32 + col) * p.D + k) * (uint32_t)sizeof(T) : OUTSIDE);
            }
#pragma unroll
            for (int c = 0; c < DEEP; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int v = 0; v < NV; ++v) acc[v] = product(value(b[c][v].e[e]), value(a[c].e[e]), acc[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int r = 0; r < 16; ++r) logits[wave][(v * 32 + 8 * (r / 4) + 4 * half + r % 4) * PITCH + col] = acc[v][r];
    __syncthreads();
    // a token to 8 threads, every 8th word to one
    const int t = threadIdx.x & 31, slice = threadIdx.x >> 5, mt = m0 + t;
    const int64_t target = mt < p.rows ? p.target[mt] : p.ignored;
    const bool mine = mt < p.rows && target != p.ignored;
    float l[NV * 4], most = LOWEST, total = 0.0f, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) {
        const int w = i * 8 + slice, at = w * PITCH + t;
        l[i] = w < p.V ? (logits[0][at] + logits[1][at]) + (logits[2][at] + logits[3][at]) + (p.bias ? value(static_cast<const T*>(p.bias)[w]) : 0.0f) : -__builtin_inff();
        if (w < p.V) sum += l[i];
        if (w == target) wanted_s[t] = l[i];
        else most = fmaxf(most, l[i]);
    }
#pragma unroll
    for (int i = 0; i < NV * 4; ++i) total += i * 8 + slice == target ? 0.0f : expf(l[i] - most);
    most_s[slice][t] = most; total_s[slice][t] = total; sum_s[slice][t] = sum;
    __syncthreads();
    float shift = most_s[0][t];
#pragma unroll
    for (int s = 1; s < 8; ++s) shift = fmaxf(shift, most_s[s][t]);
    total = 0.0f; sum = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) { total += total_s[s][t] * expf(most_s[s][t] - shift); sum += sum_s[s][t]; }
    const float wanted = target >= 0 && target < p.V ? wanted_s[t] : __builtin_nanf("");
    float missed;
    float loss = loss_of(shift, total, wanted, missed);
    const float even = p.e / (float)p.V;
    if (p.e != 0.0f && loss < __builtin_inff()) loss += p.e * wanted - even * sum;        // (a word at -infinity is infinitely wrong already)
    if (p.kept) {
        const float scale = missed / (total != 0.0f ? total : 1.0f);
#pragma unroll
        for (int i = 0; i < NV * 4; ++i) {
            const int w = i * 8 + slice;
            const float g = w == target ? p.e - even - missed : expf(l[i] - shift) * scale - even;
            if (w < p.V) out[t * p.V + w] = mine ? g : 0.0f;
        }
    }
    if (slice == 0) {
        if (p.loss && mt < p.rows) p.loss[mt] = mine ? loss : 0.0f;
        loss_s[t] = mine ? loss : 0.0f;
    }
    const int number = __syncthreads_count(slice == 0 && mine);
    if (p.kept) for (int i = threadIdx.x; i < min(TOKENS, p.rows - m0) * p.V; i += THREADS) p.kept[(int64_t)m0 * p.V + i] = out[i];
    if (threadIdx.x == 0 && p.sums) {
        double s = 0.0;
        for (int i = 0; i < TOKENS; ++i) s += loss_s[i];
        p.sums[blockIdx.x] = s;
        p.counts[blockIdx.x] = number;
    }
}

// The sum or mean over workgroups, in a fixed order.
__global__ __launch_bounds__(THREADS)
void small_total_kernel(const double* __restrict__ sums, const int* __restrict__ counts, const int blocks, const int mean, float* __restrict__ loss, int* __restrict__ number)
{
    __shared__ double s_s[THREADS];
    __shared__ int n_s[THREADS];
    double s = 0.0;
    int n = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < blocks; i += THREADS) { s += sums[i]; n += counts[i]; }
    s_s[threadIdx.x] = s; n_s[threadIdx.x] = n;
    __syncthreads();
    for (int o = THREADS / 2; o; o >>= 1) {
        if ((int)threadIdx.x < o) { s_s[threadIdx.x] += s_s[threadIdx.x + o]; n_s[threadIdx.x] += n_s[threadIdx.x + o]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *loss = (float)(mean ? s_s[0] / (double)n_s[0] : s_s[0]);
        if (number) *number = n_s[0];
    }
}

struct SmallBackward {
    const void *x, *weight;
    const int64_t* target;
    int64_t ignored;
    int rows, D, V, reduction, groups;
    const float* dloss; const int* number; const float* kept;
    void* dx; float* dw; float* db;                 // dw, db: [group][V][D], [group][V]; each or NULL
};

template <typename T, int NV>
__global__ __launch_bounds__(THREADS)
void small_backward_kernel(const SmallBackward p)
{
    constexpr int PITCH = NV * 32 + 1;
    __shared__ float P[TOKENS * PITCH];
    __shared__ bool there_s[TOKENS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int group = blockIdx.x % p.groups, c0 = blockIdx.x / p.groups * COLUMNS + wave * 32, c = c0 + col;
    const int steps = (p.V + 1) / 2, blocks = (p.rows + TOKENS - 1) / TOKENS;
    const float all = p.reduction == PROTEUS_CE_NONE ? 1.0f : p.reduction == PROTEUS_CE_MEAN ? *p.dloss / (float)*p.number : *p.dloss;
    float w[NV * 16];                               // weights of word 2 s + half
    const __amdgpu_buffer_rsrc_t rw = buffer_of(p.weight, (int64_t)p.V * p.D * sizeof(T));
#pragma unroll
    for (int s = 0; s < NV * 16; ++s) w[s] = one<T>(rw, p.dx && 2 * s + half < p.V && c < p.D ? (uint32_t)((2 * s + half) * p.D + c) * (uint32_t)sizeof(T) : OUTSIDE);
    f32x16 dw[NV] = {};
    float db = 0.0f;
    for (int b = group; b < blocks; b += p.groups) {
        const int m0 = b * TOKENS, tokens = min(TOKENS, p.rows - m0);
        __syncthreads();
        if (threadIdx.x < TOKENS) there_s[threadIdx.x] = (int)threadIdx.x < tokens && p.target[m0 + threadIdx.x] != p.ignored;
        __syncthreads();
        for (int i = threadIdx.x; i < TOKENS * NV * 32; i += THREADS) {
            const int t = i / (NV * 32), v = i % (NV * 32);
            const bool in = v < p.V && there_s[t];
            const float g = in ? p.kept[(int64_t)(m0 + t) * p.V + v] : 0.0f;
            P[t * PITCH + v] = in ? g * (p.reduction == PROTEUS_CE_NONE ? p.dloss[m0 + t] : all) : 0.0f;
        }
        float x[16];
        const __amdgpu_buffer_rsrc_t rx = buffer_of(static_cast<const T*>(p.x) + (int64_t)m0 * p.D, (int64_t)tokens * p.D * sizeof(T));
#pragma unroll
        for (int s = 0; s < 16; ++s) x[s] = one<T>(rx, p.dw && there_s[2 * s + half] && c < p.D ? (uint32_t)((2 * s + half) * p.D + c) * (uint32_t)sizeof(T) : OUTSIDE);
        __syncthreads();
        if (p.db && blockIdx.x / p.groups == 0 && (int)threadIdx.x < p.V)
            for (int t = 0; t < TOKENS; ++t) db += P[t * PITCH + threadIdx.x];
        if (p.dx) {
            f32x16 dx = {};
            for (int s = 0; s < NV * 16; ++s) if (s < steps) dx = product(w[s], P[col * PITCH + 2 * s + half], dx);
            if (col < tokens) {
                T* const to = static_cast<T*>(p.dx) + (int64_t)(m0 + col) * p.D;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int at = c0 + 8 * q + 4 * half;
                    if (at < p.D) *reinterpret_cast<Pack<T, 4>*>(to + at) = Pack<T, 4>{{rounded<T>(dx[4 * q]), rounded<T>(dx[4 * q + 1]), rounded<T>(dx[4 * q + 2]), rounded<T>(dx[4 * q + 3])}};
                }
            }
        }
        if (p.dw)
#pragma unroll
            for (int s = 0; s < 16; ++s)
#pragma unroll
                for (int v = 0; v < NV; ++v) dw[v] = product(P[(2 * s + half) * PITCH + v * 32 + col], x[s], dw[v]);
    }
    if (p.dw && c < p.D)
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int word = v * 32 + 8 * (r / 4) + 4 * half + r % 4;
                if (word < p.V) p.dw[((int64_t)group * p.V + word) * p.D + c] = dw[v][r];
            }
    if (p.db && blockIdx.x / p.groups == 0 && (int)threadIdx.x < p.V) p.db[group * p.V + threadIdx.x] = db;
}

// Sums over groups: 32 elements a workgroup, every 8th group a thread.
template <typename T>
__global__ __launch_bounds__(THREADS)
void small_sums_kernel(const float* __restrict__ dw, const float* __restrict__ db, const int groups, const int64_t n_w, const int n_b, T* __restrict__ out_w, T* __restrict__ out_b)
{
    __shared__ float s[8][32];
    const int64_t blocks_w = dw ? (n_w + 31) / 32 : 0;
    const bool of_b = blockIdx.x >= blocks_w;
    const float* const from = of_b ? db : dw;
    const int64_t n = of_b ? n_b : n_w, i = (of_b ? (int64_t)blockIdx.x - blocks_w : (int64_t)blockIdx.x) * 32 + (threadIdx.x & 31);
    float v = 0.0f;
    if (i < n)
#pragma unroll 8
        for (int g = threadIdx.x >> 5; g < groups; g += 8) v += from[g * n + i];
    s[threadIdx.x >> 5][threadIdx.x & 31] = v;
    __syncthreads();
    if (threadIdx.x >= 32 || i >= n) return;
    for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x];
    (of_b ? out_b : out_w)[i] = rounded<T>(v);
}

int blocks_of(const int64_t rows) { return (int)((rows + TOKENS - 1) / TOKENS); }
// Workgroups of the backward: two to a compute unit, and four where that leaves each 8 blocks of tokens or more (512 features, 20 words in bf16: 65536 tokens 77 / 57 us; 8192, whose groups' sums would be twice as
// much beside two blocks each, 15.2 and 3.8 as it is, 15.6 and 4.0).  Of more than 32 words a unit holds three: 65536 tokens, 64 words 134 us, with more of them 144.
int groups_of(const proteus_ce_args& a)
{
    const int across = (a.d + COLUMNS - 1) / COLUMNS, blocks = blocks_of(a.rows);
    return std::max(1, std::min(blocks, std::max(512 / across, a.vocab <= 32 ? std::min(1024 / across, blocks / 8) : 0)));
}

template <typename T> int forward_of(const SmallForward& p, hipStream_t st)
{
    const dim3 grid((unsigned)blocks_of(p.rows)), block(THREADS);
    if (p.V <= 32) hipLaunchKernelGGL((small_forward_kernel<T, 1>), grid, block, 0, st, p);
    else           hipLaunchKernelGGL((small_forward_kernel<T, 2>), grid, block, 0, st, p);
    return (int)hipGetLastError();
}
template <typename T> int backward_of(const SmallBackward& p, void* dweight, void* dbias, hipStream_t st)
{
    const dim3 grid((unsigned)((p.dx || p.dw ? (p.D + COLUMNS - 1) / COLUMNS : 1) * p.groups)), block(THREADS);
    if (p.V <= 32) hipLaunchKernelGGL((small_backward_kernel<T, 1>), grid, block, 0, st, p);
    else           hipLaunchKernelGGL((small_backward_kernel<T, 2>), grid, block, 0, st, p);
    if (const int rc = (int)hipGetLastError()) return rc;
    const int64_t n = (p.dw ? ((int64_t)p.V * p.D + 31) / 32 : 0) + (p.db ? (p.V + 31) / 32 : 0);
    if (!n) return 0;
    hipLaunchKernelGGL((small_sums_kernel<T>), dim3((unsigned)n), block, 0, st, p.dw, p.db, p.groups, (int64_t)p.V * p.D, p.V, static_cast<T*>(dweight), static_cast<T*>(dbias));
    return (int)hipGetLastError();
}

}  // namespace

size_t proteus_ce::small_kept_bytes(const proteus_ce_args& a) { return (size_t)HEAD + (size_t)a.rows * a.vocab * 4; }
size_t proteus_ce::small_forward_bytes(const proteus_ce_args& a) { return (size_t)blocks_of(a.rows) * 12 + 256; }
size_t proteus_ce::small_backward_bytes(const proteus_ce_args& a) { return (size_t)groups_of(a) * ((size_t)a.vocab * a.d + a.vocab) * 4 + 256; }

int proteus_ce::small_forward(const proteus_ce_args& a, float* loss, void* kept, void* ws, hipStream_t st)
{
    SmallForward p = {};
    p.x = a.x; p.weight = a.weight; p.bias = a.bias; p.target = a.target; p.ignored = a.ignore_index;
    p.rows = (int)a.rows; p.D = a.d; p.V = a.vocab; p.reduction = a.reduction; p.e = a.label_smoothing;
    const int unit = a.dtype == PROTEUS_DTYPE_F32 ? 8 : 16;
    p.chunks = ((a.d + unit - 1) / unit + 3) / 4;
    const bool by_token = a.reduction == PROTEUS_CE_NONE;
    p.loss = by_token ? loss : nullptr;
    p.sums = by_token ? nullptr : static_cast<double*>(ws);
    p.counts = reinterpret_cast<int*>(static_cast<double*>(ws) + blocks_of(a.rows));
    p.kept = kept ? reinterpret_cast<float*>(static_cast<char*>(kept) + HEAD) : nullptr;
    const int rc = a.dtype == PROTEUS_DTYPE_F32 ? forward_of<float>(p, st) : a.dtype == PROTEUS_DTYPE_BF16 ? forward_of<bf16_t>(p, st) : forward_of<f16_t>(p, st);
    if (rc || by_token) return rc;
    hipLaunchKernelGGL(small_total_kernel, dim3(1), dim3(THREADS), 0, st, p.sums, p.counts, blocks_of(a.rows), (int)(a.reduction == PROTEUS_CE_MEAN), loss, static_cast<int*>(kept));
    return (int)hipGetLastError();
}

int proteus_ce::small_backward(const proteus_ce_args& a, const float* dloss, const void* kept, void* dx, void* dweight, void* dbias, void* ws, hipStream_t st)
{
    SmallBackward p = {};
    p.x = a.x; p.weight = a.weight; p.target = a.target; p.ignored = a.ignore_index;
    p.rows = (int)a.rows; p.D = a.d; p.V = a.vocab; p.reduction = a.reduction; p.groups = groups_of(a);
    p.dloss = dloss; p.number = static_cast<const int*>(kept); p.kept = reinterpret_cast<const float*>(static_cast<const char*>(kept) + HEAD);
    p.dx = dx;
    p.dw = dweight ? static_cast<float*>(ws) : nullptr;
    p.db = dbias ? static_cast<float*>(ws) + (size_t)p.groups * p.V * p.D : nullptr;
    return a.dtype == PROTEUS_DTYPE_F32 ? backward_of<float>(p, dweight, dbias, st) : a.dtype == PROTEUS_DTYPE_BF16 ? backward_of<bf16_t>(p, dweight, dbias, st) : backward_of<f16_t>(p, dweight, dbias, st);
}

// Root-mean-square norm of every head's queries and keys and their rotation by position, in one pass, and its gradient (gfx950).
//
//   r = 1 / sqrt(mean(x^2) + eps),  u = x r w,  y = u turned: each pair (a, b) of features becomes (a cos - b sin, b cos + a sin), angle position * base^(-2i/d)
//   backward: t = dy turned back;  dw = sum over tokens t x r;  m = t w;  dx = r (m - x r mean(m x r))
//
// Bound by memory: every element is read once and written once (backward: read twice, x and dy), nothing is kept between the directions but the inputs. A lane holds
// 16 elements of a head, eight of either half, so that both partners of a rotated pair are its own in either order of pairing; d / 16 lanes make up a head and add up
// among themselves.  A lane stays with its head (its weights and the sums of their gradients in registers) and walks over tokens.
//
// Cosine and sine depend on the token and the pair alone: a workgroup works them out once for its next tokens (up to 16), in LDS, for all heads of queries and keys.
// The angle is taken in turns, in fp64, where position * frequency is good to 2^-52 of its size (half a step each for the frequency and for the product), and only what
// is left of it beyond whole turns is rounded to fp32: positions beyond 10^5 would lose the angle itself in fp32.
//
// us and TB/s: 2 x 16384 tokens, 8 heads of queries and of keys, 128 features, bf16, forward 50 and 5.4, backward 90 and 4.5 (a copy of 1 GiB 5.0; lines that two passes of a kernel share are in the
// caches); 8 x 1024 padded tokens of a fused projection, 3 x 8 heads of 64, fp32 to bf16, 13.9 and 22.8; 512 tokens and 64 single ones 4.3 and 4.2, a launch.
//
// Sums over tokens: each workgroup leaves its own (its lanes' sums added up in LDS in a fixed order), and a second launch adds them up: the same bits on every call.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "proteus_hip.h"

namespace {

constexpr int THREADS = 256, TOKENS = 16;           // tokens of a step, at most
constexpr int MOST_BLOCKS = 2048, MOST_SUMS = 768;  // workgroups, two rounds of four to a compute unit and (backward, each with sums of its own) one of three
constexpr int FINAL_THREADS = 1024, FINAL_COLUMNS = 16;

struct Part {                                       // queries, keys or (copied) values
    const char *x, *dy;
    char* y;                                        // y, or dx
    int64_t xs[3], ds[3], ys[3];                    // bytes from one batch item, head, token to the next
    const void* w;
};
struct Args {
    Part part[3];
    int heads_q, normed, rows;                      // rows: heads of queries | keys | values; the first two kinds are normed
    int group;                                      // rows of a workgroup
    const int64_t* positions;                       // or NULL: 0 .. N - 1
    int64_t positions_z;
    const uint8_t* mask;
    int N, tokens, step;                            // batch items * N; tokens of a step
    uint32_t per_item; int per_item_shift;          // token / N = token * per_item >> shift, for tokens below 2^31
    float eps;
    int interleaved, weight_type, per_head;
    float* sums;                                    // backward: [workgroup][queries, keys][d], per head [workgroup][head][d]
    double turns[64];                               // per position
};

struct f16_t { _Float16 v; };
struct bf16_t { __bf16 v; };
__device__ __forceinline__ float value(const float x) { return x; }
__device__ __forceinline__ float value(const f16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const bf16_t x) { return (float)x.v; }
template <typename T> __device__ __forceinline__ T rounded(const float x) { T r; r.v = (decltype(r.v))x; return r; }
template <> __device__ __forceinline__ float rounded<float>(const float x) { return x; }
// Eight elements from either half of a head, as they lie in memory.
template <typename T> struct Raw {
    uint4 v[sizeof(T)];                             // (16 sizeof(T) bytes of a lane)
    __device__ __forceinline__ void load(const char* p, const int second)
    {
        constexpr int H = sizeof(T) / 2;
#pragma unroll
        for (int i = 0; i < H; ++i) { v[i] = reinterpret_cast<const uint4*>(p)[i]; v[H + i] = reinterpret_cast<const uint4*>(p + second)[i]; }
    }
    __device__ __forceinline__ void values(float* a, float* b) const
    {
        struct { T e[16]; } r;
        __builtin_memcpy(&r, v, sizeof(r));
#pragma unroll
        for (int i = 0; i < 8; ++i) { a[i] = value(r.e[i]); b[i] = value(r.e[8 + i]); }
    }
    static __device__ __forceinline__ void store(char* p, const int second, const float* a, const float* b)
    {
        constexpr int H = sizeof(T) / 2;
        struct { T e[16]; } r;
#pragma unroll
        for (int i = 0; i < 8; ++i) { r.e[i] = rounded<T>(a[i]); r.e[8 + i] = rounded<T>(b[i]); }
        uint4 v[2 * H];
        __builtin_memcpy(v, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < H; ++i) { reinterpret_cast<uint4*>(p)[i] = v[i]; reinterpret_cast<uint4*>(p + second)[i] = v[H + i]; }
    }
};

// The lane's 16 elements of a weight [d] (rows of which may lie at any multiple of an element)
__device__ __forceinline__ void weights(const Args& g, const void* w, const int64_t first, const int second, float* to)
{
    auto all = [&](auto e) {
        using T = decltype(e);
        const T* const p = static_cast<const T*>(w) + first;
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i] = value(p[i < 8 ? i : second + i - 8]);
    };
    if (!w) {
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i] = 1.0f;
    }
    else if (g.weight_type == PROTEUS_DTYPE_F32)  all(float{});
    else if (g.weight_type == PROTEUS_DTYPE_BF16) all(bf16_t{});
    else                                          all(f16_t{});
}

// cos and sin of an angle in turns, |turns| <= 1/2: the rest of the nearest quarter, exact, through the series at 0 (|angle| <= pi/4: up to its 9th power the sine's
// next term is below 2e-9, up to the 8th the cosine's below 3e-8), and the quarter by swaps and signs.
__device__ __forceinline__ void turned(const float turns, float& c, float& s)
{
    const float quarter = rintf(4.0f * turns), x = __builtin_fmaf(quarter, -0.25f, turns) * 6.283185307f, y = x * x;
    float sn = __builtin_fmaf(y, 2.7557319e-6f, -1.9841270e-4f), cs = __builtin_fmaf(y, 2.4801587e-5f, -1.3888889e-3f);
    sn = __builtin_fmaf(y, sn, 8.3333333e-3f);
    cs = __builtin_fmaf(y, cs, 4.1666667e-2f);
    sn = __builtin_fmaf(y, sn, -1.6666667e-1f);
    cs = __builtin_fmaf(y, cs, -0.5f);
    sn = __builtin_fmaf(x * y, sn, x);
    cs = __builtin_fmaf(y, cs, 1.0f);
    const int k = (int)quarter;
    const float a = k & 1 ? sn : cs, b = k & 1 ? cs : sn;
    c = (k + 1) & 2 ? -a : a;
    s = k & 2 ? -b : b;
}

// Sum over the L lanes of a head.
template <int L> __device__ __forceinline__ float head_sum(float v)
{
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// Pairs turned by +angle (SIGN 1) or back (-1).  a: elements 8l .. 8l + 7 of a head, b: d / 2 + 8l ...
template <int SIGN> __device__ __forceinline__ void turn(float* a, float* b, const float* c, const float* s, const int interleaved)
{
    auto pair = [&](float& x, float& y, const int i) {
        const float sn = SIGN * s[i], u = x * c[i] - y * sn, v = y * c[i] + x * sn;
        x = u; y = v;
    };
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { pair(a[2 * i], a[2 * i + 1], i); pair(b[2 * i], b[2 * i + 1], 4 + i); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) pair(a[i], b[i], i);
    }
}

template <int D> struct Lds {
    float cos_[TOKENS][D / 2], sin_[TOKENS][D / 2];
};

__device__ __forceinline__ int item_of(const Args& g, const int token) { return (int)((uint64_t)(uint32_t)token * g.per_item >> g.per_item_shift); }

// cos and sin of the next tokens (at + 0 .. count - 1).
template <int D> __device__ __forceinline__ void prepare(const Args& g, Lds<D>& s, const int at, const int count)
{
    for (int i = threadIdx.x; i < count * (D / 2); i += THREADS) {
        const int t = i / (D / 2), f = i % (D / 2);
        const int z = item_of(g, at + t), n = at + t - z * g.N;
        const double angle = (double)(g.positions ? g.positions[z * g.positions_z + n] : (int64_t)n) * g.turns[f];
        turned((float)(angle - rint(angle)), s.cos_[t][f], s.sin_[t][f]);
    }
}

template <int D> __device__ __forceinline__ void angles(const Args& g, const Lds<D>& s, const int t, const int l, float* c, float* sn)
{
    const int first = g.interleaved ? 4 * l : 8 * l, second = g.interleaved ? D / 4 + 4 * l : 8 * l + 4;
    *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(&s.cos_[t][first]);
    *reinterpret_cast<float4*>(c + 4) = *reinterpret_cast<const float4*>(&s.cos_[t][second]);
    *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(&s.sin_[t][first]);
    *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(&s.sin_[t][second]);
}

template <int D, typename T, typename U, bool BACKWARD>
__global__ __launch_bounds__(THREADS)
void qk_kernel(const Args g)
{
    constexpr int L = D / 16, LANES = THREADS / L;
    __shared__ __align__(16) union { Lds<D> tokens; float sums[LANES][D]; } s;
    const int l = threadIdx.x % L, lane = threadIdx.x / L;
    const int row = blockIdx.y * g.group + lane % g.group, sub = lane / g.group, subs = LANES / g.group;
    const bool busy = sub < subs && row < g.rows;
    const bool normed = row < g.normed;
    const int kind = row < g.heads_q ? 0 : normed ? 1 : 2, head = row - (kind == 0 ? 0 : kind == 1 ? g.heads_q : g.normed);
    const Part& p = g.part[kind];
    constexpr int SECOND_T = D / 2 * sizeof(T), SECOND_U = D / 2 * sizeof(U);
    const char *const x0 = p.x + head * p.xs[1] + 8 * l * sizeof(T), *const d0 = BACKWARD ? p.dy + head * p.ds[1] + 8 * l * sizeof(U) : nullptr;
    using V = typename std::conditional<BACKWARD, T, U>::type;
    char* const y0 = p.y + head * p.ys[1] + 8 * l * sizeof(V);
    // a token's inputs, on their way while the angles are worked out and while the token before is
    Raw<T> next_x;
    Raw<U> next_d;
    int64_t next_at;                                // of the results
    bool next_padded;
    auto fetch = [&](const int token) {
        const int64_t z = item_of(g, token), n = token - z * g.N;
        next_padded = g.mask && g.mask[token];
        next_at = z * p.ys[0] + n * p.ys[2];
        if (next_padded) return;
        if (!BACKWARD || normed) next_x.load(x0 + z * p.xs[0] + n * p.xs[2], SECOND_T);
        if (BACKWARD) next_d.load(d0 + z * p.ds[0] + n * p.ds[2], SECOND_U);
    };
    float w[16], dw[16] = {};
    bool first = true;
    for (int at = blockIdx.x * g.step; at < g.tokens; at += gridDim.x * g.step) {
        const int count = min(g.step, g.tokens - at);
        const bool any = busy && sub < count;
        if (any) fetch(at + sub);
        if (first && busy && normed) weights(g, p.w, (g.per_head ? head * D : 0) + 8 * l, D / 2, w);
        first = false;
        prepare<D>(g, s.tokens, at, count);
        __syncthreads();
        for (int t = sub; any && t < count; t += subs) {
            const bool padded = next_padded;
            const Raw<T> raw_x = next_x;
            const Raw<U> raw_d = next_d;
            char* const y = y0 + next_at;
            if (t + subs < count) fetch(at + t + subs);
            float a[8], b[8];
            if (padded) {
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.0f;
            } else if (!BACKWARD) {
                raw_x.values(a, b);
                if (normed) {
                    float c[8], sn[8], ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
                    const float r = rsqrtf(head_sum<L>(ss) * (1.0f / D) + g.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) { a[i] *= r * w[i]; b[i] *= r * w[8 + i]; }
                    angles<D>(g, s.tokens, t, l, c, sn);
                    turn<1>(a, b, c, sn, g.interleaved);
                }
            } else {
                raw_d.values(a, b);
                if (normed) {
                    float xa[8], xb[8], ss = 0.0f, mx = 0.0f;
                    raw_x.values(xa, xb);
                    {
                        float c[8], sn[8];
                        angles<D>(g, s.tokens, t, l, c, sn);
                        turn<-1>(a, b, c, sn, g.interleaved);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss += xa[i] * xa[i] + xb[i] * xb[i];
                    const float r = rsqrtf(head_sum<L>(ss) * (1.0f / D) + g.eps);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        xa[i] *= r; xb[i] *= r;
                        dw[i] += a[i] * xa[i]; dw[8 + i] += b[i] * xb[i];
                        a[i] *= w[i]; b[i] *= w[8 + i];
                        mx += a[i] * xa[i] + b[i] * xb[i];
                    }
                    mx = head_sum<L>(mx) * (1.0f / D);
#pragma unroll
                    for (int i = 0; i < 8; ++i) { a[i] = r * (a[i] - xa[i] * mx); b[i] = r * (b[i] - xb[i] * mx); }
                }
            }
            Raw<V>::store(y, D / 2 * sizeof(V), a, b);
        }
        __syncthreads();
    }
    if (!BACKWARD || !g.sums) return;
    // ---- the workgroup's sums for the weights' gradients ----
#pragma unroll
    for (int i = 0; i < 16; ++i) s.sums[lane][8 * l + (i < 8 ? i : D / 2 + i - 8)] = dw[i];    // (idle lanes' are zero)
    __syncthreads();
    if (g.per_head) {
        for (int i = threadIdx.x; i < g.group * D; i += THREADS) {
            const int k = i / D, e = i % D, at = blockIdx.y * g.group + k;
            float v = 0.0f;
            for (int u = 0; u < subs; ++u) v += s.sums[u * g.group + k][e];
            if (at < g.normed) g.sums[((int64_t)blockIdx.x * g.normed + at) * D + e] = v;
        }
    } else {
        for (int i = threadIdx.x; i < 2 * D; i += THREADS) {
            const int which = i / D, e = i % D;
            float v = 0.0f;
            for (int k = 0; k < g.group; ++k) {
                const int at = blockIdx.y * g.group + k;
                if (at < g.normed && (at >= g.heads_q) == (which == 1))
                    for (int u = 0; u < subs; ++u) v += s.sums[u * g.group + k][e];
            }
            g.sums[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * D + i] = v;
        }
    }
}

// Column sums of [rows][columns] to the two weights' gradients (the first `columns_q` columns are the queries'), which may be left out.
__global__ __launch_bounds__(FINAL_THREADS)
void qk_sums_kernel(const float* __restrict__ sums, const int rows, const int columns, const int columns_q, void* dq, void* dk, const int type)
{
    constexpr int COLUMNS = FINAL_COLUMNS, GROUPS = FINAL_THREADS / COLUMNS;
    __shared__ float part[GROUPS][COLUMNS];
    const int c = blockIdx.x * COLUMNS + threadIdx.x % COLUMNS, group = threadIdx.x / COLUMNS;
    float v = 0.0f;
    if (c < columns)
#pragma unroll 8
        for (int r = group; r < rows; r += GROUPS) v += sums[(int64_t)r * columns + c];
    part[group][threadIdx.x % COLUMNS] = v;
    __syncthreads();
    if (group != 0 || c >= columns) return;
    for (int k = 1; k < GROUPS; ++k) v += part[k][threadIdx.x];
    void* const out = c < columns_q ? dq : dk;
    const int i = c < columns_q ? c : c - columns_q;
    if (!out) return;
    if (type == PROTEUS_DTYPE_F32)       static_cast<float*>(out)[i] = v;
    else if (type == PROTEUS_DTYPE_BF16) static_cast<bf16_t*>(out)[i] = rounded<bf16_t>(v);
    else                                 static_cast<f16_t*>(out)[i] = rounded<f16_t>(v);
}

bool known(const int type) { return type == PROTEUS_DTYPE_F32 || type == PROTEUS_DTYPE_BF16 || type == PROTEUS_DTYPE_F16; }
int size_of(const int type) { return type == PROTEUS_DTYPE_F32 ? 4 : 2; }

struct Sizes { int rows, group, groups, subs; };
// Rows of a workgroup: all of them, or a share of the fewest shares that leave a tenth of the lanes idle at most (24 rows of 64 as one 48 busy, as two 60).
Sizes sizes(const int heads_q, const int heads_k, const int heads_v, const int d)
{
    const int rows = heads_q + heads_k + heads_v, lanes = THREADS / (d / 16), fewest = (rows + lanes - 1) / lanes;
    int best = fewest, most = 0;
    for (int groups = fewest; groups <= fewest + 3 && groups <= rows; ++groups) {
        const int group = (rows + groups - 1) / groups, busy = lanes / group * rows / groups;      // (of a workgroup, on average)
        if (busy > most) { most = busy; best = groups; }
        if (busy * 10 >= lanes * 9) break;
    }
    const int group = (rows + best - 1) / best;
    return {rows, group, best, lanes / group};
}
// Workgroups along the tokens, and tokens of a step: a step as long as its workgroup's lanes take at once where there are few tokens, so that these spread over the chip,
// else four of that (at most TOKENS), over which the working out of the angles and the barriers are spread.
int blocks_of(const int64_t tokens, const Sizes& s, const int most, int& step)
{
    step = s.subs < TOKENS ? s.subs : TOKENS;
    while (step * 2 <= TOKENS && tokens > (int64_t)step * 512) step *= 2;
    const int64_t n = (tokens + step - 1) / step, limit = most / s.groups > 0 ? most / s.groups : 1;
    return (int)(n < limit ? n : limit);
}

int check(const proteus_qk_args* a, const bool backward)
{
    if (!a || !a->x[0] || !a->x[1] || !a->y[0] || !a->y[1] || (backward && (!a->dy[0] || !a->dy[1]))) return PROTEUS_ERR_NULL_POINTER;
    if (a->heads_v < 0 || (a->heads_v > 0 && (!(backward || a->x[2]) || !a->y[2] || (backward && !a->dy[2])))) return a->heads_v < 0 ? PROTEUS_ERR_BAD_SHAPE : PROTEUS_ERR_NULL_POINTER;
    if (a->d_head != 32 && a->d_head != 64 && a->d_head != 128) return PROTEUS_ERR_BAD_HEAD_DIM;
    if (a->Z <= 0 || a->N <= 0 || a->heads_q <= 0 || a->heads_k <= 0 || a->N > (1 << 30) || (int64_t)a->Z * a->N >= (1LL << 31) - TOKENS * (int64_t)MOST_BLOCKS
        || a->heads_q > 8192 || a->heads_k > 8192 || a->heads_v > 8192) return PROTEUS_ERR_BAD_SHAPE;
    if (!(a->eps >= 0.0f) || !(a->base > 0.0) || !(a->base <= 1.7e308)) return PROTEUS_ERR_BAD_SHAPE;
    if (!known(a->x_type) || !known(a->y_type) || !known(a->weight_type)) return PROTEUS_ERR_BAD_OPERAND_TYPE;
    if (a->x_type != a->y_type && a->x_type != PROTEUS_DTYPE_F32) return PROTEUS_ERR_BAD_OPERAND_TYPE;
    for (int i = 0; i < (a->heads_v > 0 ? 3 : 2); ++i) {
        const bool x = !(backward && i == 2);       // (values' inputs are not read again)
        const int in = backward ? a->y_type : a->x_type, out = backward ? a->x_type : a->y_type;
        if ((x && (uintptr_t)a->x[i] % 16) || (uintptr_t)a->y[i] % 16 || (backward && (uintptr_t)a->dy[i] % 16)) return PROTEUS_ERR_BAD_ALIGNMENT;
        for (int k = 0; k < 3; ++k)
            if ((x && a->x_strides[i][k] % (16 / size_of(a->x_type))) || a->y_strides[i][k] % (16 / size_of(out)) || (backward && a->dy_strides[i][k] % (16 / size_of(in))))
                return PROTEUS_ERR_BAD_ALIGNMENT;
    }
    for (int i = 0; i < 2; ++i) if (a->weight[i] && (uintptr_t)a->weight[i] % size_of(a->weight_type)) return PROTEUS_ERR_BAD_ALIGNMENT;
    if (a->positions && (uintptr_t)a->positions % 8) return PROTEUS_ERR_BAD_ALIGNMENT;
    return 0;
}

Args kernel_args(const proteus_qk_args& a, const bool backward, const Sizes& s)
{
    Args g = {};
    const int in = size_of(a.x_type), y = backward ? in : size_of(a.y_type);
    for (int i = 0; i < 3; ++i) {
        Part& p = g.part[i];
        p.x = static_cast<const char*>(a.x[i]); p.dy = static_cast<const char*>(a.dy[i]); p.y = static_cast<char*>(a.y[i]);
        for (int k = 0; k < 3; ++k) { p.xs[k] = a.x_strides[i][k] * in; p.ds[k] = a.dy_strides[i][k] * size_of(a.y_type); p.ys[k] = a.y_strides[i][k] * y; }
        p.w = i < 2 ? a.weight[i] : nullptr;
    }
    g.heads_q = a.heads_q; g.normed = a.heads_q + a.heads_k; g.rows = s.rows; g.group = s.group;
    g.positions = a.positions; g.positions_z = a.positions_stride; g.mask = a.mask;
    g.N = a.N; g.tokens = a.Z * a.N; g.eps = a.eps;
    // shift = 31 + ceil(log2 N), factor = ceil(2^shift / N) < 2^32 (N = 1: 2^31): what it is too large by, below N / 2^shift, times a token stays below 1
    g.per_item_shift = 31;
    while ((1u << (g.per_item_shift - 31)) < (uint32_t)a.N) ++g.per_item_shift;
    g.per_item = (uint32_t)(((1ull << g.per_item_shift) + a.N - 1) / a.N);
    g.interleaved = a.interleaved != 0; g.weight_type = a.weight_type; g.per_head = a.per_head != 0;
    // Frequencies as powers in 64 bits of mantissa, rounded to fp64 once: 63 products behind one another are off by less than 2^-54 (the exponential of a rounded
    // logarithm, in fp64, by up to 2^-49.7).
    const long double step = exp2l(-2.0L * log2l((long double)a.base) / a.d_head);
    long double turns = 0.159154943091895335768883763372514362L;
    for (int i = 0; i < a.d_head / 2; ++i, turns *= step) g.turns[i] = (double)turns;
    return g;
}

template <bool BACKWARD, int D>
int launch_typed(const Args& g, const dim3 grid, const int x, const int y, hipStream_t st)
{
    const dim3 block(THREADS);
    if (x == PROTEUS_DTYPE_F32 && y == PROTEUS_DTYPE_F32)       hipLaunchKernelGGL((qk_kernel<D, float, float, BACKWARD>), grid, block, 0, st, g);
    else if (x == PROTEUS_DTYPE_F32 && y == PROTEUS_DTYPE_BF16) hipLaunchKernelGGL((qk_kernel<D, float, bf16_t, BACKWARD>), grid, block, 0, st, g);
    else if (x == PROTEUS_DTYPE_F32)                            hipLaunchKernelGGL((qk_kernel<D, float, f16_t, BACKWARD>), grid, block, 0, st, g);
    else if (x == PROTEUS_DTYPE_BF16)                           hipLaunchKernelGGL((qk_kernel<D, bf16_t, bf16_t, BACKWARD>), grid, block, 0, st, g);
    else                                                        hipLaunchKernelGGL((qk_kernel<D, f16_t, f16_t, BACKWARD>), grid, block, 0, st, g);
    return (int)hipGetLastError();
}
template <bool BACKWARD>
int launch(const Args& g, const dim3 grid, const proteus_qk_args& a, hipStream_t st)
{
    return a.d_head == 32 ? launch_typed<BACKWARD, 32>(g, grid, a.x_type, a.y_type, st) : a.d_head == 64 ? launch_typed<BACKWARD, 64>(g, grid, a.x_type, a.y_type, st)
                                                                                         : launch_typed<BACKWARD, 128>(g, grid, a.x_type, a.y_type, st);
}

}  // namespace

extern "C" int proteus_qk_norm_rotate_check(const proteus_qk_args* args, int backward) { return check(args, backward != 0); }

extern "C" int proteus_qk_norm_rotate_fwd(const proteus_qk_args* args, void* stream)
{
    if (const int rc = check(args, false)) return rc;
    const Sizes s = sizes(args->heads_q, args->heads_k, args->heads_v, args->d_head);
    Args g = kernel_args(*args, false, s);
    const int blocks = blocks_of(g.tokens, s, MOST_BLOCKS, g.step);
    return launch<false>(g, dim3(blocks, s.groups), *args, reinterpret_cast<hipStream_t>(stream));
}

extern "C" size_t proteus_qk_norm_rotate_bwd_workspace_bytes(int Z, int N, int heads_q, int heads_k, int heads_v, int d_head, int per_head)
{
    if (Z <= 0 || N <= 0 || heads_q <= 0 || heads_k <= 0 || heads_v < 0 || (d_head != 32 && d_head != 64 && d_head != 128)) return 0;
    const Sizes s = sizes(heads_q, heads_k, heads_v, d_head);
    int step;
    const size_t blocks = blocks_of((int64_t)Z * N, s, MOST_SUMS, step);
    return blocks * (per_head ? (size_t)(heads_q + heads_k) : 2 * (size_t)s.groups) * d_head * sizeof(float);
}

extern "C" int proteus_qk_norm_rotate_bwd(const proteus_qk_args* args, void* dq_weight, void* dk_weight, void* ws, size_t ws_bytes, void* stream)
{
    if (const int rc = check(args, true)) return rc;
    const bool sums = dq_weight || dk_weight;
    if (((uintptr_t)dq_weight | (uintptr_t)dk_weight) % size_of(args->weight_type) || (uintptr_t)ws % 16) return PROTEUS_ERR_BAD_ALIGNMENT;
    if (sums && !ws) return PROTEUS_ERR_NULL_POINTER;
    if (sums && ws_bytes < proteus_qk_norm_rotate_bwd_workspace_bytes(args->Z, args->N, args->heads_q, args->heads_k, args->heads_v, args->d_head, args->per_head))
        return PROTEUS_ERR_TOO_LARGE;
    const Sizes s = sizes(args->heads_q, args->heads_k, args->heads_v, args->d_head);
    Args g = kernel_args(*args, true, s);
    const int blocks = blocks_of(g.tokens, s, MOST_SUMS, g.step);
    g.sums = sums ? static_cast<float*>(ws) : nullptr;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (const int rc = launch<true>(g, dim3(blocks, s.groups), *args, st)) return rc;
    if (!sums) return 0;
    const int columns = (g.per_head ? g.normed : 2) * args->d_head, columns_q = (g.per_head ? g.heads_q : 1) * args->d_head;
    hipLaunchKernelGGL(qk_sums_kernel, dim3((columns + FINAL_COLUMNS - 1) / FINAL_COLUMNS), dim3(FINAL_THREADS), 0, st, g.sums, blocks * (g.per_head ? 1 : s.groups), columns, columns_q,
                       dq_weight, dk_weight, args->weight_type);
    return (int)hipGetLastError();
}

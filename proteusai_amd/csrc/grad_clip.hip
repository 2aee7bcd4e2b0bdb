// The norm over the gradients of a training step, and the gradients scaled to at most a given norm (gfx950).
//
//   norm = (sum over all elements |g|^p)^(1/p), p = 1, 2 or infinity;   out = g * min(1, max_norm / (norm + 1e-6))
//
// Two passes over the gradients, whatever the number of tensors: a launch takes a table of up to 320 of them among its arguments (4 KB; 190 where results go
// elsewhere), so that nothing is copied to the device and a captured graph holds all that it reads.  The first pass leaves a sum per workgroup; every workgroup
// of the second adds all of these up in their order and so knows the factor, which saves the launch of a reduction between the two.  Nothing depends on
// the order in which workgroups run: the same bits on every call.
//
// Squares and sums are fp64: fp32's squares leave its range from 2^64 on and below 2^-75, and a sum of 10^9 of them its precision; at the rate at which
// memory delivers elements the vector units have four times the time that takes.
//
// Tensors are cut into chunks of one size, dealt to the workgroups in turn (runs of consecutive chunks for each: 350 million bf16 gradients 645 us, so 619).  Bound by memory:
// those, scaled into fp32, 164 us of the first pass (4.3 TB/s) and 452 of the second (4.7 TB/s, last to first); a copy of 1 GiB runs at 5.0.  12.6 million fp32 gradients of 34 tensors, from the
// caches, 10.6 and 17.9; 500 tensors of 1200 elements 15 us of the device in four launches, 45 of the host.  Addresses are only as aligned as the elements: tensors
// of odd sizes lie one behind the other in buckets, and unaligned 16-byte loads and stores cost less than a path for every alignment.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "proteus_hip.h"

namespace {

constexpr int THREADS = 512, WAVES = THREADS / 64;
constexpr int MOST_BLOCKS = 1024;                   // of a launch: what the chip holds at four to a compute unit
constexpr int IN_PLACE = 320, APART = 190;          // tensors of a launch
constexpr uint64_t ADDRESS = (1ull << 48) - 1;

// address of a tensor's elements | elements in its last chunk - 1; the first chunk of every tensor, and the end
template <int MOST, bool TO> struct Table {
    uint64_t from[MOST];
    uint64_t to[TO ? MOST : 1];
    uint32_t first[MOST + 1];
    int count;
    int chunk;                                      // elements
};
static_assert(sizeof(Table<IN_PLACE, false>) <= 4000 && sizeof(Table<APART, true>) <= 4000, "kernel arguments");

enum Kind { ONE = 1, TWO = 2, LARGEST = 3 };

struct f16_t { _Float16 v; };
struct bf16_t { __bf16 v; };
__device__ __forceinline__ float value(const f16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const bf16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const float x) { return x; }
template <typename T> __device__ __forceinline__ T rounded(const float x) { T r; r.v = (decltype(r.v))x; return r; }
template <> __device__ __forceinline__ float rounded<float>(const float x) { return x; }

// elements in global memory (told so, since their addresses come as numbers), at any alignment of theirs
#define GC_GLOBAL __attribute__((address_space(1)))
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T, int N> struct Pack {
    T e[N];
    static constexpr int WORDS = N * sizeof(T) / 16;                           // of 16 bytes
    struct All { words4 w[WORDS]; };
    static __device__ __forceinline__ Pack load(const GC_GLOBAL T* p)
    {
        All a;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) a.w[i] = reinterpret_cast<const GC_GLOBAL words4*>(p)[i];
        return __builtin_bit_cast(Pack, a);
    }
    __device__ __forceinline__ void store(GC_GLOBAL T* p) const
    {
        const All a = __builtin_bit_cast(All, *this);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) reinterpret_cast<GC_GLOBAL words4*>(p)[i] = a.w[i];
    }
};
template <int BYTES> struct Bits { using type = uint16_t; };
template <> struct Bits<4> { using type = uint32_t; };
template <typename T> __device__ __forceinline__ T one(const GC_GLOBAL T* p) { using B = typename Bits<sizeof(T)>::type; return __builtin_bit_cast(T, *reinterpret_cast<const GC_GLOBAL B*>(p)); }
template <typename T> __device__ __forceinline__ void put(GC_GLOBAL T* p, const T v) { using B = typename Bits<sizeof(T)>::type; *reinterpret_cast<GC_GLOBAL B*>(p) = __builtin_bit_cast(B, v); }
template <typename T> __device__ __forceinline__ GC_GLOBAL T* elements(const uint64_t address) { return reinterpret_cast<GC_GLOBAL T*>(address & ADDRESS); }

// A running result of one kind; the largest is held as the bits of |x|, whose order is that of the numbers, with NaN above infinity.
template <int KIND> struct Running {
    double sum = 0.0;
    __device__ __forceinline__ void add(const float x)
    {
        const double d = x;
        sum = KIND == TWO ? __builtin_fma(d, d, sum) : sum + fabs(d);
    }
    __device__ __forceinline__ void join(const double other) { sum += other; }
    __device__ __forceinline__ double get() const { return sum; }
};
template <> struct Running<LARGEST> {
    uint32_t most = 0;
    __device__ __forceinline__ void add(const float x) { most = max(most, __builtin_bit_cast(uint32_t, x) & 0x7fffffffu); }
    __device__ __forceinline__ void join(const double other) { add((float)other); }
    __device__ __forceinline__ double get() const { return (double)__builtin_bit_cast(float, most); }
};

// All threads' results together, in a fixed order; every thread gets it.
template <int KIND> __device__ __forceinline__ double block_total(Running<KIND> r, double* lds)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) r.join(__shfl_xor(r.get(), o));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = r.get();
    __syncthreads();
    Running<KIND> all;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all.join(lds[w]);
    return all.get();
}

// fn(tensor, first element, elements) for every gridDim.x-th chunk, first to last or (BACK) last to first.
template <bool BACK, typename TABLE, typename F> __device__ __forceinline__ void chunks(const TABLE& t, const F& fn)
{
    const uint32_t all = t.first[t.count];
    for (uint32_t i = blockIdx.x; i < all; i += gridDim.x) {
        const uint32_t c = BACK ? all - 1 - i : i;
        int lo = 0, hi = t.count;                   // first[lo] <= c < first[hi]
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (t.first[mid] <= c) lo = mid; else hi = mid; }
        fn(lo, (uint64_t)(c - t.first[lo]) * t.chunk, c + 1 == t.first[lo + 1] ? (uint32_t)(t.from[lo] >> 48) + 1 : (uint32_t)t.chunk);
    }
}

template <typename T, int KIND>
__global__ __launch_bounds__(THREADS, 8)
void norm_kernel(const Table<IN_PLACE, false> t, double* __restrict__ sums)
{
    __shared__ double lds[WAVES];
    constexpr int E = 16 / (int)sizeof(T), DEEP = 4;
    using P = Pack<T, E>;
    Running<KIND> r;
    chunks<false>(t, [&](const int i, const uint64_t at, const uint32_t n) {
        const GC_GLOBAL T* const x = elements<T>(t.from[i]) + at;
        uint32_t k = threadIdx.x * E;
        for (; k + (DEEP - 1) * THREADS * E + E <= n; k += DEEP * THREADS * E) {
            P v[DEEP];
#pragma unroll
            for (int j = 0; j < DEEP; ++j) v[j] = P::load(x + k + j * THREADS * E);
#pragma unroll
            for (int j = 0; j < DEEP; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) r.add(value(v[j].e[e]));
        }
        for (; k + E <= n; k += THREADS * E) {
            const P v = P::load(x + k);
#pragma unroll
            for (int e = 0; e < E; ++e) r.add(value(v.e[e]));
        }
        for (; k < n; ++k) r.add(value(one(x + k)));      // (of one thread, the others are past the end)
    });
    const double s = block_total<KIND>(r, lds);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// The norm from all workgroups' sums.
template <int KIND> __device__ __forceinline__ float whole_norm(const double* __restrict__ sums, const int n, double* lds)
{
    Running<KIND> r;
    for (int i = threadIdx.x; i < n; i += THREADS) r.join(sums[i]);
    const double s = block_total<KIND>(r, lds);
    return (float)(KIND == TWO ? sqrt(s) : s);
}

__device__ __forceinline__ float norm_of(const int kind, const double* sums, const int n, double* lds)
{
    return kind == TWO ? whole_norm<TWO>(sums, n, lds) : kind == ONE ? whole_norm<ONE>(sums, n, lds) : whole_norm<LARGEST>(sums, n, lds);
}

__global__ __launch_bounds__(THREADS)
void last_kernel(const double* __restrict__ sums, const int n, const int kind, float* __restrict__ norm)
{
    __shared__ double lds[WAVES];
    const float v = norm_of(kind, sums, n, lds);
    if (threadIdx.x == 0) *norm = v;
}

template <typename T, typename U, int MOST, bool TO>
__global__ __launch_bounds__(THREADS)
void scale_kernel(const Table<MOST, TO> t, const double* __restrict__ sums, const int n_sums, const int kind, const float max_norm, float* __restrict__ norm, const int writes_norm)
{
    __shared__ double lds[WAVES];
    const float v = norm_of(kind, sums, n_sums, lds);
    if (writes_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
    const float ratio = max_norm / (v + 1e-6f), factor = ratio > 1.0f ? 1.0f : ratio;      // (NaN stays)
    if (!TO && factor == 1.0f) return;              // within the bound and in place: nothing changes
    constexpr int E = 16 / (int)(sizeof(T) < sizeof(U) ? sizeof(T) : sizeof(U)), DEEP = 4;     // 16 bytes of the smaller type
    using P = Pack<T, E>;
    using Q = Pack<U, E>;
    // last to first: the end of what the first pass read is nearest
    chunks<true>(t, [&](const int i, const uint64_t at, const uint32_t n) {
        const GC_GLOBAL T* const x = elements<T>(t.from[i]) + at;
        GC_GLOBAL U* const y = elements<U>(TO ? t.to[i] : t.from[i]) + at;
        auto scaled = [&](const P& p) {
            Q q;
#pragma unroll
            for (int e = 0; e < E; ++e) q.e[e] = rounded<U>(value(p.e[e]) * factor);
            return q;
        };
        uint32_t k = threadIdx.x * E;
        for (; k + (DEEP - 1) * THREADS * E + E <= n; k += DEEP * THREADS * E) {
            P p[DEEP];
#pragma unroll
            for (int j = 0; j < DEEP; ++j) p[j] = P::load(x + k + j * THREADS * E);
#pragma unroll
            for (int j = 0; j < DEEP; ++j) scaled(p[j]).store(y + k + j * THREADS * E);
        }
        for (; k + E <= n; k += THREADS * E) scaled(P::load(x + k)).store(y + k);
        for (; k < n; ++k) put(y + k, rounded<U>(value(one(x + k)) * factor));
    });
}

int size_of(const int type) { return type == PROTEUS_DTYPE_F32 ? 4 : 2; }

// Elements of a chunk: a sweep of the workgroup at least, and as many as leave 512 of them (each workgroup of the second pass adds up all workgroups' sums: 12.6 million
// fp32 gradients in chunks of 4096, 16384 and 32768 29.3, 27.0 and 25.5 us).
int chunk_of(const uint64_t elements)
{
    int c = 4096;
    while (c < 65536 && elements / c > 512) c *= 2;
    return c;
}

// One launch's tensors: of one pair of types, from `next` on.  fills the table and moves `next` behind them; returns the chunks (0: none left).
struct Call {
    const void* const* from; void* const* to; const int64_t* numel; const int* from_type; const int* to_type; int count;
};

template <int MOST, bool TO>
uint32_t fill(Table<MOST, TO>& t, const Call& c, const int ft, const int tt, int& i, int64_t& done)
{
    // (a tensor whose chunks would not fit 31 bits goes over several entries or launches)
    uint64_t elements = 0;
    int j = i;
    for (int n = 0; j < c.count && n < MOST; ++j) if (c.numel[j] > 0 && c.from_type[j] == ft && (!TO || c.to_type[j] == tt)) { elements += c.numel[j]; ++n; }
    t.chunk = chunk_of(elements);
    t.count = 0;
    uint32_t chunks = 0;
    while (i < c.count && t.count < MOST) {
        if (!(c.numel[i] > 0 && c.from_type[i] == ft && (!TO || c.to_type[i] == tt))) { ++i; continue; }
        const int64_t left = c.numel[i] - done, room = (int64_t)(0x7fffffffu - chunks) * t.chunk;
        if (room == 0) break;
        const int64_t n = left < room ? left : room;
        const uint32_t k = (uint32_t)((n + t.chunk - 1) / t.chunk);
        const uint64_t rest = (uint64_t)(n - (int64_t)(k - 1) * t.chunk - 1) << 48;
        t.from[t.count] = ((uint64_t)(uintptr_t)c.from[i] + (uint64_t)done * size_of(ft)) | rest;
        if (TO) t.to[t.count] = (uint64_t)(uintptr_t)c.to[i] + (uint64_t)done * size_of(tt);
        t.first[t.count++] = chunks;
        chunks += k;
        done += n;
        if (done < c.numel[i]) break;
        ++i;
        done = 0;
    }
    t.first[t.count] = chunks;
    return chunks;
}

unsigned blocks_of(const uint32_t chunks) { return chunks < (uint32_t)MOST_BLOCKS ? chunks : (unsigned)MOST_BLOCKS; }

// fn(table, chunks) for every launch over the tensors of one pair of types
template <int MOST, bool TO, typename F>
int launches(const Call& c, const int ft, const int tt, const F& fn)
{
    Table<MOST, TO> t;
    int i = 0;
    int64_t done = 0;
    for (;;) {
        const uint32_t k = fill(t, c, ft, tt, i, done);
        if (!k) return 0;
        const int rc = fn(t, k);
        if (rc) return rc;
    }
}

template <typename T> void launch_norm(const int kind, const unsigned grid, hipStream_t st, const Table<IN_PLACE, false>& t, double* sums)
{
    if (kind == TWO)      hipLaunchKernelGGL((norm_kernel<T, TWO>), dim3(grid), dim3(THREADS), 0, st, t, sums);
    else if (kind == ONE) hipLaunchKernelGGL((norm_kernel<T, ONE>), dim3(grid), dim3(THREADS), 0, st, t, sums);
    else                  hipLaunchKernelGGL((norm_kernel<T, LARGEST>), dim3(grid), dim3(THREADS), 0, st, t, sums);
}

int check(const Call& c, const int norm_type, const float max_norm, const float* norm, const void* ws, const size_t ws_bytes)
{
    if (c.count < 0 || (c.count > 0 && (!c.from || !c.numel || !c.from_type)) || !norm || (c.to && !c.to_type)) return c.count < 0 ? PROTEUS_ERR_BAD_SHAPE : PROTEUS_ERR_NULL_POINTER;
    if (norm_type != PROTEUS_NORM_1 && norm_type != PROTEUS_NORM_2 && norm_type != PROTEUS_NORM_INF) return PROTEUS_ERR_UNSUPPORTED;
    if (c.to && !(max_norm >= 0.0f)) return PROTEUS_ERR_BAD_SHAPE;
    for (int i = 0; i < c.count; ++i) {
        if (c.numel[i] < 0 || c.numel[i] >= (1LL << 46)) return PROTEUS_ERR_BAD_SHAPE;
        for (int side = 0; side < (c.to ? 2 : 1); ++side) {
            const int type = side ? c.to_type[i] : c.from_type[i];
            if (type != PROTEUS_DTYPE_F32 && type != PROTEUS_DTYPE_BF16 && type != PROTEUS_DTYPE_F16) return PROTEUS_ERR_BAD_OPERAND_TYPE;
            if (c.numel[i] == 0) continue;
            const uint64_t p = (uint64_t)(uintptr_t)(side ? c.to[i] : c.from[i]);
            if (!p) return PROTEUS_ERR_NULL_POINTER;
            if (p % size_of(type) || p + (uint64_t)c.numel[i] * size_of(type) > ADDRESS) return PROTEUS_ERR_BAD_ALIGNMENT;
        }
    }
    if (!ws) return PROTEUS_ERR_NULL_POINTER;
    if ((uintptr_t)ws % 8) return PROTEUS_ERR_BAD_ALIGNMENT;
    if (ws_bytes < proteus_clip_grads_workspace_bytes(c.count)) return PROTEUS_ERR_TOO_LARGE;
    return 0;
}

}  // namespace

// Sums of every launch: the tensors of each of three types by 320, and a launch more for each 2^31 chunks of 65536 elements (2^47: none).
extern "C" size_t proteus_clip_grads_workspace_bytes(int count)
{
    if (count < 0) return 0;
    return (size_t)(count / IN_PLACE + 3) * MOST_BLOCKS * sizeof(double);
}

extern "C" int proteus_clip_grads_check(const void* const* grads, void* const* out, const int64_t* numel, const int* types, const int* out_types, int count,
                                        int norm_type, float max_norm, const float* norm, const void* ws, size_t ws_bytes)
{
    return check(Call{grads, out, numel, types, out_types, count}, norm_type, max_norm, norm, ws, ws_bytes);
}

extern "C" int proteus_clip_grads(const void* const* grads, void* const* out, const int64_t* numel, const int* types, const int* out_types, int count,
                                  int norm_type, float max_norm, float* norm, void* ws, size_t ws_bytes, void* stream)
{
    const Call c = {grads, out, numel, types, out_types, count};
    if (const int rc = check(c, norm_type, max_norm, norm, ws, ws_bytes)) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    double* const sums = static_cast<double*>(ws);
    const int kind = norm_type == PROTEUS_NORM_1 ? ONE : norm_type == PROTEUS_NORM_2 ? TWO : LARGEST;
    int n = 0, rc;
    bool present[3] = {};
    for (int i = 0; i < count; ++i) present[types[i]] = true;
    static_assert(PROTEUS_DTYPE_F32 >= 0 && PROTEUS_DTYPE_F32 < 3 && PROTEUS_DTYPE_BF16 >= 0 && PROTEUS_DTYPE_BF16 < 3 && PROTEUS_DTYPE_F16 >= 0 && PROTEUS_DTYPE_F16 < 3, "");
    for (const int ft : {PROTEUS_DTYPE_F32, PROTEUS_DTYPE_BF16, PROTEUS_DTYPE_F16}) {
        if (!present[ft]) continue;
        rc = launches<IN_PLACE, false>(c, ft, ft, [&](const Table<IN_PLACE, false>& t, const uint32_t k) {
            const unsigned grid = blocks_of(k);
            if (ft == PROTEUS_DTYPE_F32)       launch_norm<float>(kind, grid, st, t, sums + n);
            else if (ft == PROTEUS_DTYPE_BF16) launch_norm<bf16_t>(kind, grid, st, t, sums + n);
            else                               launch_norm<f16_t>(kind, grid, st, t, sums + n);
            n += (int)grid;
            return (int)hipGetLastError();
        });
        if (rc) return rc;
    }
    bool written = false;                           // the norm, by the first launch that scales
    bool in_place = out != nullptr;
    for (int i = 0; in_place && i < count; ++i) in_place = out[i] == grads[i] && out_types[i] == types[i];
    for (const int ft : {PROTEUS_DTYPE_F32, PROTEUS_DTYPE_BF16, PROTEUS_DTYPE_F16})
        for (const int tt : {PROTEUS_DTYPE_F32, PROTEUS_DTYPE_BF16, PROTEUS_DTYPE_F16}) {
            if (!out || !present[ft] || (in_place && ft != tt)) continue;
            auto go = [&](auto from, auto to) {
                using T = decltype(from); using U = decltype(to);
                auto scale = [&](const auto kernel, const auto& t, const uint32_t k) {
                    hipLaunchKernelGGL(kernel, dim3(blocks_of(k)), dim3(THREADS), 0, st, t, sums, n, kind, max_norm, norm, (int)!written);
                    written = true;
                    return (int)hipGetLastError();
                };
                if constexpr (sizeof(T) == sizeof(U)) if (in_place)
                    return launches<IN_PLACE, false>(c, ft, ft, [&](const Table<IN_PLACE, false>& t, const uint32_t k) { return scale(scale_kernel<T, T, IN_PLACE, false>, t, k); });
                return launches<APART, true>(c, ft, tt, [&](const Table<APART, true>& t, const uint32_t k) { return scale(scale_kernel<T, U, APART, true>, t, k); });
            };
            auto to = [&](auto from) { return tt == PROTEUS_DTYPE_F32 ? go(from, float{}) : tt == PROTEUS_DTYPE_BF16 ? go(from, bf16_t{}) : go(from, f16_t{}); };
            rc = ft == PROTEUS_DTYPE_F32 ? to(float{}) : ft == PROTEUS_DTYPE_BF16 ? to(bf16_t{}) : to(f16_t{});
            if (rc) return rc;
        }
    if (!written) {
        hipLaunchKernelGGL(last_kernel, dim3(1), dim3(THREADS), 0, st, sums, n, kind, norm);
        return (int)hipGetLastError();
    }
    return 0;
}

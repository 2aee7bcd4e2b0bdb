// A step of AdamW over many tensors, moments in 32 bits or in 8 (gfx950).
//
//   g = grad * min(1, max_norm / (norm + 1e-6));   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// One pass over everything: a launch takes a table of up to some hundred tensors among its arguments (4 KB), so that nothing is copied to the device and a captured graph holds all that it
// reads.  Tensors are cut into chunks of one size, dealt to the workgroups in turn.  The clipping's factor is applied on the way: gradients are read once and not written.
//
// Moments in 8 bits.  A row of 1056 bytes holds 512 elements of a tensor: 512 codes of m, 512 of r = sqrt(v), 16 scales of m, 16 of r.  A code is an e4m3 number (4 bits of exponent, 3 of
// mantissa), a scale the exponent of a power of two (e8m0), one for 32 elements: the least by which the largest of them is at most 448, e4m3's largest, so that multiplying by it is exact.  The root
// is kept because v spans twice m's range.  A decay of 0.1 % a step is far below the distance of two codes (6 to 12 %): rounded to nearest a moment would never
// leave its code, so what is cut off is rounded up with its own probability, from 16 bits of a hash of the seed, the step, the tensor's number and the element's.  A root that is not
// zero keeps the smallest code at least: a zero would make the next update of that element as large as a first one; where its square is below the least of fp32 (roots below 2^-75) it decays by itself, by
// sqrt(b2).  What is not finite becomes NaN, for its own element alone; the update itself uses the moments before they are rounded.
//
// A wave has 256 elements of a row at a time, four to a lane: whole lines of every operand, and the 32 elements of a scale are 8 lanes, which agree on their largest in
// three steps within the row of lanes.
//
// Bound by memory: 12.6 million fp32 parameters 65 us (5.4 TB/s), moments in 8 bits 41 (5.0, with the launch that counts the step); 350 million fp32 ones with bf16 gradients 1814 (5.0), bf16 with fp32 master weights
// and moments in 8 bits 1167 (4.8); a copy of 1 GiB runs at 5.07.  500 tensors of 1200 elements take six launches of 6 us, and 80 of the host
// (the optimizer's step() in front of it 250 more).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include "proteus_hip.h"

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int MOST_BLOCKS = 2048;                   // of a launch: what the chip holds at eight to a compute unit
constexpr int ROW = PROTEUS_ADAMW_ROW, CODES = 512;
constexpr uint64_t ADDRESS = (1ull << 48) - 1;

struct Scalars {
    const float* lr;                                // on the GPU, or NULL
    const int64_t* step;                            // steps done, on the GPU, or NULL
    const float* norm;                              // or NULL
    double lr_, decay, log_b1, log_b2;              // for what has to be worked out here
    float b1, b2, c1, c2, eps, max_norm;            // c = 1 - b
    float keep, size, root;                         // 1 - lr decay, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), where both are known
    float decays;                                   // sqrt(b2)
    uint32_t seed;
    int64_t number;                                 // of this step
};

template <bool EIGHT, bool MASTER> struct Table {
    static constexpr int MOST = (3808 - (int)sizeof(Scalars)) / (8 * (EIGHT ? 3 : 4) + (MASTER ? 8 : 0) + 4 + (EIGHT ? 4 : 0));
    uint64_t p[MOST];                               // address of chunk 0 | elements in the last chunk - 1
    uint64_t g[MOST];                               // address | elements of chunk 0 in front of the tensor's first
    uint64_t m[MOST];                               // or the rows
    uint64_t v[EIGHT ? 1 : MOST];
    uint64_t w[MASTER ? MOST : 1];
    uint32_t first[MOST + 1];                       // first chunk of every tensor, and the end
    uint32_t tensor[EIGHT ? MOST : 1];              // its number in the call
    int count;
    int chunk;                                      // elements
    Scalars s;
};

struct f16_t { _Float16 v; };
struct bf16_t { __bf16 v; };
__device__ __forceinline__ float value(const f16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const bf16_t x) { return (float)x.v; }
__device__ __forceinline__ float value(const float x) { return x; }
template <typename T> __device__ __forceinline__ T rounded(const float x) { T r; r.v = (decltype(r.v))x; return r; }
template <> __device__ __forceinline__ float rounded<float>(const float x) { return x; }

#define AW_GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ __forceinline__ AW_GLOBAL T* elements(const uint64_t address) { return reinterpret_cast<AW_GLOBAL T*>(address & ADDRESS); }
template <int BYTES> struct Bits { using type = uint16_t; };
template <> struct Bits<4> { using type = uint32_t; };

// Four elements at any alignment of theirs, or `from` to `to` - 1 of them at a tensor's ends.  PAST: not to be kept in the caches.
template <typename T> struct Quad {
    typedef uint32_t words __attribute__((ext_vector_type(sizeof(T)), aligned(2)));
    T e[4];
    template <bool PAST> static __device__ __forceinline__ Quad load(const AW_GLOBAL T* p)
    {
        const AW_GLOBAL words* const w = reinterpret_cast<const AW_GLOBAL words*>(p);
        return __builtin_bit_cast(Quad, PAST ? __builtin_nontemporal_load(w) : *w);
    }
    static __device__ __forceinline__ Quad load(const AW_GLOBAL T* p, const int from, const int to)
    {
        using B = typename Bits<sizeof(T)>::type;
        Quad q = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i >= from && i < to) q.e[i] = __builtin_bit_cast(T, reinterpret_cast<const AW_GLOBAL B*>(p)[i]);
        return q;
    }
    template <bool PAST> __device__ __forceinline__ void store(AW_GLOBAL T* p) const
    {
        AW_GLOBAL words* const w = reinterpret_cast<AW_GLOBAL words*>(p);
        if (PAST) __builtin_nontemporal_store(__builtin_bit_cast(words, *this), w);
        else      *w = __builtin_bit_cast(words, *this);
    }
    __device__ __forceinline__ void store(AW_GLOBAL T* p, const int from, const int to) const
    {
        using B = typename Bits<sizeof(T)>::type;
#pragma unroll
        for (int i = 0; i < 4; ++i) if (i >= from && i < to) reinterpret_cast<AW_GLOBAL B*>(p)[i] = __builtin_bit_cast(B, e[i]);
    }
};
static_assert(sizeof(Quad<float>::words) == 16 && sizeof(Quad<bf16_t>::words) == 8, "");

// What all elements of a launch share.
struct Shared { float factor, keep, size, root; uint32_t key; };

// A mix of 32 bits: shifts, and products with odd numbers that C. Wellons searched for an even spread and published in 2018.
__device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x ^= x >> 16; x *= 0x7feb352du;
    x ^= x >> 15; x *= 0x846ca68bu;
    return x ^ (x >> 16);
}

__device__ __forceinline__ Shared shared_of(const Scalars& s)
{
    Shared h = {1.0f, s.keep, s.size, s.root, 0};
    const int64_t t = s.step ? *s.step + 1 : s.number;
    if (s.norm) {
        const float ratio = s.max_norm / (*s.norm + 1e-6f);
        h.factor = ratio > 1.0f ? 1.0f : ratio;     // (NaN stays)
    }
    if (s.lr || s.step) {
        const double lr = s.lr ? (double)*s.lr : s.lr_;
        h.keep = (float)(1.0 - lr * s.decay);
        h.size = (float)(lr / -expm1((double)t * s.log_b1));
        h.root = (float)(1.0 / sqrt(-expm1((double)t * s.log_b2)));
    }
    h.key = mix(s.seed + (uint32_t)t * 0x9e3779b1u);
    return h;
}

// `least`: of the root, where the square that it is taken from is below fp32's least
__device__ __forceinline__ void update(const Scalars& s, const Shared& h, float& p, const float grad, float& m, float& v, float& root, const float least)
{
    const float g = grad * h.factor;
    {
        // (products rounded before their sum, as the formula's: where 0.9 m + 0.1 g is a code's own border, a sum of one rounded and one unrounded product lands beside it)
#pragma clang fp contract(off)
        m = s.b1 * m + s.c1 * g;
        v = s.b2 * v + s.c2 * g * g;
    }
    root = sqrtf(v);
    root = root == 0.0f ? least : root;
    p = p * h.keep - h.size * m / (root * h.root + s.eps);
    asm("" : "+v"(p));                              // (an fp32 number: left to itself the compiler has the last product and sum rounded to fp16 at once, which is not what the master weight rounds to)
}

// fn(tensor, first element, elements, chunk 0) for every gridDim.x-th chunk
template <typename TABLE, typename F> __device__ __forceinline__ void chunks(const TABLE& t, const F& fn)
{
    const uint32_t all = t.first[t.count];
    for (uint32_t c = blockIdx.x; c < all; c += gridDim.x) {
        int lo = 0, hi = t.count;                   // first[lo] <= c < first[hi]
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (t.first[mid] <= c) lo = mid; else hi = mid; }
        fn(lo, (uint64_t)(c - t.first[lo]) * t.chunk, c + 1 == t.first[lo + 1] ? (uint32_t)(t.p[lo] >> 48) + 1 : (uint32_t)t.chunk, c == t.first[lo]);
    }
}

// Chunk 0 begins up to 31 elements in front of a tensor that does not begin on a multiple of 32 of them (in a bucket of odd sizes), so that a wave's accesses are whole lines
// (of 16-bit operands halves of them).  PAST: all operands begin with a line, and none but the parameters' is read again before the next step.  12.6 million fp32 parameters 77 us, past the caches 65 (parameters,
// too: 71); 350 million with bf16 gradients in buckets of odd sizes 1955 as they lie (past the caches 2177), 1814 so, 1835 with whole lines of the gradients, too, and past the caches.
template <typename P, typename G, bool MASTER, bool PAST>
__global__ __launch_bounds__(THREADS)
void adamw_kernel(const Table<false, MASTER> t)
{
    const Shared h = shared_of(t.s);
    chunks(t, [&](const int i, const uint64_t at, const uint32_t n, const bool first) {
        AW_GLOBAL P* const p = elements<P>(t.p[i]) + at;
        const AW_GLOBAL G* const g = elements<G>(t.g[i]) + at;
        AW_GLOBAL float* const m = elements<float>(t.m[i]) + at;
        AW_GLOBAL float* const v = elements<float>(t.v[i]) + at;
        AW_GLOBAL float* const w = MASTER ? elements<float>(t.w[i]) + at : nullptr;
        const int begin = first ? (int)(t.g[i] >> 48) : 0;
        auto step = [&](Quad<float>& wq, Quad<P>& pq, const Quad<G>& gq, Quad<float>& mq, Quad<float>& vq) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = MASTER ? wq.e[e] : value(pq.e[e]), root;
                update(t.s, h, x, value(gq.e[e]), mq.e[e], vq.e[e], root, 0.0f);
                wq.e[e] = x;
                pq.e[e] = rounded<P>(x);
            }
        };
        for (uint32_t k = threadIdx.x * 4; k < n; k += THREADS * 4) {
            const int from = begin - (int)k, to = (int)min(n - k, 4u);
            Quad<P> pq = {};
            Quad<float> wq = {};
            if (from <= 0 && to == 4) {
                if constexpr (MASTER) wq = Quad<float>::template load<PAST>(w + k); else pq = Quad<P>::template load<PAST>(p + k);
                const Quad<G> gq = Quad<G>::template load<PAST>(g + k);
                Quad<float> mq = Quad<float>::template load<PAST>(m + k), vq = Quad<float>::template load<PAST>(v + k);
                step(wq, pq, gq, mq, vq);
                pq.template store<false>(p + k);
                if constexpr (MASTER) wq.template store<PAST>(w + k);
                mq.template store<PAST>(m + k);
                vq.template store<PAST>(v + k);
            } else if (from < 4) {
                if constexpr (MASTER) wq = Quad<float>::load(w + k, from, to); else pq = Quad<P>::load(p + k, from, to);
                const Quad<G> gq = Quad<G>::load(g + k, from, to);
                Quad<float> mq = Quad<float>::load(m + k, from, to), vq = Quad<float>::load(v + k, from, to);
                step(wq, pq, gq, mq, vq);
                pq.store(p + k, from, to);
                if constexpr (MASTER) wq.store(w + k, from, to);
                mq.store(m + k, from, to);
                vq.store(v + k, from, to);
            }
        }
    });
}

// The largest of 8 lanes' numbers: neighbours, pairs, and the two halves mirrored onto one another.
__device__ __forceinline__ uint32_t largest_of_8(uint32_t x)
{
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));
}

// Four codes and their scale, as values.
__device__ __forceinline__ void decode(const uint32_t codes, const int scale, float (&x)[4])
{
#ifdef __HIP_DEVICE_COMPILE__
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
    const float y[4] = {a[0], a[1], b[0], b[1]};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_amdgcn_ldexpf(y[e], scale - 127);
#endif
}

// The scale for a group of 8 lanes, and the codes of this lane's four: |x| in e4m3 has the lowest exponents of fp32 (2^-120 of it), so that adding random bits below the mantissa's three
// and cutting off is the rounding, subnormals included.
template <bool LEAST> __device__ __forceinline__ uint32_t encode(const float (&x)[4], const uint32_t (&random)[4], int& scale)
{
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu;
        most = max(most, b < 0x7f800000u ? b : 0u);
    }
    most = largest_of_8(most);
    scale = max((int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u), 0);
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_ldexpf(__builtin_fabsf(x[e]), 7 - scale));
        uint32_t c = min((b + (random[e] << 4)) >> 20, 0x7fu);
        if (LEAST) c = max(c, x[e] > 0.0f ? 1u : 0u);
        else       c |= __builtin_bit_cast(uint32_t, x[e]) >> 24 & 0x80u;
        codes |= c << (8 * e);
    }
    return codes;
}

template <typename P, typename G, bool MASTER, bool PAST>
__global__ __launch_bounds__(THREADS)
void adamw8_kernel(const Table<true, MASTER> t)
{
    const Shared h = shared_of(t.s);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    chunks(t, [&](const int i, const uint64_t at, const uint32_t n, bool) {
        AW_GLOBAL P* const p = elements<P>(t.p[i]) + at;
        const AW_GLOBAL G* const g = elements<G>(t.g[i]) + at;
        AW_GLOBAL float* const w = MASTER ? elements<float>(t.w[i]) + at : nullptr;
        AW_GLOBAL uint8_t* const rows = elements<uint8_t>(t.m[i]) + at / CODES * ROW;
        const uint32_t key = mix(h.key + t.tensor[i] * 0x85ebca6bu + (uint32_t)(at >> 32) * 0xc2b2ae35u);        // (a chunk lies within 2^32 elements: both are powers of two)
        for (uint32_t r = wave; r * CODES < n; r += WAVES)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t k = r * CODES + half * 256 + lane * 4;
                AW_GLOBAL uint8_t* const row = rows + (uint64_t)r * ROW + half * 256 + lane * 4;
                AW_GLOBAL uint8_t* const scales = rows + (uint64_t)r * ROW + 2 * CODES + half * 8 + (lane >> 3);
                const int left = (int)min(n - min(k, n), 4u);
                Quad<P> pq = {};
                Quad<float> wq = {};
                Quad<G> gq;
                if (left == 4) {
                    if constexpr (MASTER) wq = Quad<float>::template load<PAST>(w + k); else pq = Quad<P>::template load<PAST>(p + k);
                    gq = Quad<G>::template load<PAST>(g + k);
                } else {
                    if constexpr (MASTER) wq = Quad<float>::load(w + k, 0, left); else pq = Quad<P>::load(p + k, 0, left);
                    gq = Quad<G>::load(g + k, 0, left);
                }
                float m[4], root[4];
                decode(*reinterpret_cast<const AW_GLOBAL uint32_t*>(row), scales[0], m);
                decode(*reinterpret_cast<const AW_GLOBAL uint32_t*>(row + CODES), scales[16], root);
                uint32_t random1[4], random2[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = e < left;       // (nothing but zeros behind the last element)
                    m[e] = in ? m[e] : 0.0f;
                    float x = MASTER ? wq.e[e] : value(pq.e[e]), v = in ? root[e] * root[e] : 0.0f;
                    update(t.s, h, x, value(gq.e[e]), m[e], v, root[e], in ? root[e] * t.s.decays : 0.0f);
                    wq.e[e] = x;
                    pq.e[e] = rounded<P>(x);
                    const uint32_t random = mix(key ^ ((uint32_t)at + k + e));
                    random1[e] = random & 0xffffu;
                    random2[e] = random >> 16;
                }
                int s1, s2;
                const uint32_t c1 = encode<false>(m, random1, s1), c2 = encode<true>(root, random2, s2);
                *reinterpret_cast<AW_GLOBAL uint32_t*>(row) = c1;
                *reinterpret_cast<AW_GLOBAL uint32_t*>(row + CODES) = c2;
                if ((lane & 7) == 0) {
                    scales[0] = (uint8_t)s1;
                    scales[16] = (uint8_t)s2;
                }
                if (left == 4) {
                    pq.template store<false>(p + k);
                    if constexpr (MASTER) wq.template store<PAST>(w + k);
                } else {
                    pq.store(p + k, 0, left);
                    if constexpr (MASTER) wq.store(w + k, 0, left);
                }
            }
    });
}

// (The last workgroup of a step's launch cannot do it for less: 2048 of them telling one address that they are through take 15 us, a launch 4.)
__global__ void count_kernel(int64_t* step) { *step += 1; }

int size_of(const int type) { return type == PROTEUS_DTYPE_F32 ? 4 : 2; }

// Elements of a chunk: two sweeps of a workgroup at least, and up to 8192 as long as they leave two chunks to each workgroup (350 million parameters in chunks of 32768, 8192 and 4096: 1853, 1817 and 1827 us, with
// moments in 8 bits 1208, 1167 and 1172; as many workgroups as have the same number of chunks each: 1 to 8 % slower).
int chunk_of(const uint64_t elements)
{
    int c = 2048;
    while (c < 8192 && elements / c > 2 * MOST_BLOCKS) c *= 2;
    return c;
}

bool takes(const proteus_adamw_args& a, const int i, const int pt, const int gt, const bool master)
{
    return a.numel[i] > 0 && a.param_types[i] == pt && a.grad_types[i] == gt && (a.masters && a.masters[i]) == master;
}

// The tensors of one launch, from `i` on, which moves behind them; returns the chunks (0: none left).
template <bool EIGHT, bool MASTER>
uint32_t fill(Table<EIGHT, MASTER>& t, const proteus_adamw_args& a, const int pt, const int gt, int& i, bool& lines)
{
    using TABLE = Table<EIGHT, MASTER>;
    uint64_t elements = 0;
    for (int j = i, n = 0; j < a.count && n < TABLE::MOST; ++j) if (takes(a, j, pt, gt, MASTER)) { elements += a.numel[j]; ++n; }
    t.chunk = chunk_of(elements);
    t.count = 0;
    uint32_t chunks = 0;
    for (; i < a.count && t.count < TABLE::MOST; ++i) {
        if (!takes(a, i, pt, gt, MASTER)) continue;
        auto address = [](const void* x) { return (uint64_t)(uintptr_t)x; };
        const int64_t shift = EIGHT ? 0 : (int64_t)(address(a.params[i]) / size_of(pt) % 32), n = a.numel[i] + shift;
        const uint32_t k = (uint32_t)((n + t.chunk - 1) / t.chunk);
        auto from = [&](const void* x, const int size) {
            const uint64_t at = address(x) - (uint64_t)shift * size;
            lines = lines && at % 128 == 0;
            return at & ADDRESS;
        };
        t.p[t.count] = from(a.params[i], size_of(pt)) | (uint64_t)(n - (int64_t)(k - 1) * t.chunk - 1) << 48;
        t.g[t.count] = from(a.grads[i], size_of(gt)) | (uint64_t)shift << 48;
        t.m[t.count] = EIGHT ? address(a.states[i]) : from(a.exp_avgs[i], 4);
        if constexpr (EIGHT) t.tensor[t.count] = (uint32_t)i;
        else                 t.v[t.count] = from(a.exp_avg_sqs[i], 4);
        if constexpr (MASTER) t.w[t.count] = from(a.masters[i], 4);
        t.first[t.count++] = chunks;
        chunks += k;
    }
    t.first[t.count] = chunks;
    return chunks;
}

// The launch's own result: the thread's last error may be an earlier call's, and a step that went out is not one that failed.
template <typename A> int launch(void (*const kernel)(A), const unsigned blocks, const unsigned threads, hipStream_t st, const A& a)
{
    void* args[1] = {const_cast<A*>(&a)};
    return (int)hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(blocks), dim3(threads), args, 0, st);
}

template <typename P, typename G, bool MASTER, bool EIGHT>
int launches(const proteus_adamw_args& a, const Scalars& s, const int pt, const int gt, hipStream_t st)
{
    Table<EIGHT, MASTER> t = {};
    t.s = s;
    for (int i = 0;;) {
        bool lines = true;                          // all operands begin (chunk 0 of them) with a line
        const uint32_t chunks = fill(t, a, pt, gt, i, lines);
        if (!chunks) return 0;
        const unsigned blocks = chunks < (uint32_t)MOST_BLOCKS ? chunks : (uint32_t)MOST_BLOCKS;
        int rc;
        if constexpr (EIGHT) rc = lines ? launch(adamw8_kernel<P, G, MASTER, true>, blocks, THREADS, st, t) : launch(adamw8_kernel<P, G, MASTER, false>, blocks, THREADS, st, t);
        else                 rc = lines ? launch(adamw_kernel<P, G, MASTER, true>, blocks, THREADS, st, t) : launch(adamw_kernel<P, G, MASTER, false>, blocks, THREADS, st, t);
        if (rc) return rc;
    }
}

template <typename P, typename G> int go(const proteus_adamw_args& a, const Scalars& s, const int pt, const int gt, const bool master, hipStream_t st)
{
    if constexpr (sizeof(P) == 2) if (master) return a.states ? launches<P, G, true, true>(a, s, pt, gt, st) : launches<P, G, true, false>(a, s, pt, gt, st);
    return a.states ? launches<P, G, false, true>(a, s, pt, gt, st) : launches<P, G, false, false>(a, s, pt, gt, st);
}

bool known(const int type) { return type == PROTEUS_DTYPE_F32 || type == PROTEUS_DTYPE_BF16 || type == PROTEUS_DTYPE_F16; }

int check(const proteus_adamw_args* p)
{
    if (!p) return PROTEUS_ERR_NULL_POINTER;
    const proteus_adamw_args& a = *p;
    if (a.count < 0) return PROTEUS_ERR_BAD_SHAPE;
    if (a.count > 0 && (!a.params || !a.grads || !a.numel || !a.param_types || !a.grad_types || (a.states ? a.exp_avgs || a.exp_avg_sqs : !a.exp_avgs || !a.exp_avg_sqs))) return PROTEUS_ERR_NULL_POINTER;
    if (!(a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0 && a.eps >= 0.0 && a.weight_decay >= 0.0) || (!a.lr_gpu && !(a.lr >= 0.0)) || (!a.step_gpu && a.step < 1)
        || (a.norm && !(a.max_norm >= 0.0f))) return PROTEUS_ERR_BAD_SHAPE;
    uint64_t chunks = 0;
    for (int i = 0; i < a.count; ++i) {
        const int64_t n = a.numel[i];
        const int pt = a.param_types[i], gt = a.grad_types[i];
        if (n < 0 || n >= (1LL << 40)) return PROTEUS_ERR_BAD_SHAPE;
        if (!known(pt) || !known(gt) || (pt != PROTEUS_DTYPE_F32 && gt != pt && gt != PROTEUS_DTYPE_F32)) return PROTEUS_ERR_BAD_OPERAND_TYPE;
        if (a.masters && a.masters[i] && pt == PROTEUS_DTYPE_F32) return PROTEUS_ERR_BAD_OPERAND_TYPE;
        if (n == 0) continue;
        const void* const at[5] = {a.params[i], a.grads[i], a.states ? a.states[i] : a.exp_avgs[i], a.states ? a.states[i] : a.exp_avg_sqs[i], a.masters ? a.masters[i] : nullptr};
        const uint64_t by[5] = {(uint64_t)size_of(pt), (uint64_t)size_of(gt), a.states ? 16u : 4u, a.states ? 16u : 4u, 4u};
        for (int k = 0; k < 5; ++k) {
            const uint64_t x = (uint64_t)(uintptr_t)at[k];
            if (!x && k < 4) return PROTEUS_ERR_NULL_POINTER;
            if (x % by[k] || x + (uint64_t)n * 4 > ADDRESS) return PROTEUS_ERR_BAD_ALIGNMENT;
        }
        chunks += (uint64_t)n / 2048 + 1;
    }
    return chunks < 0x7fffffffull ? 0 : PROTEUS_ERR_TOO_LARGE;
}

}  // namespace

extern "C" size_t proteus_adamw_state_bytes(int64_t numel) { return numel > 0 && numel < (1LL << 40) ? (size_t)((numel + CODES - 1) / CODES) * ROW : 0; }

extern "C" int proteus_adamw_check(const proteus_adamw_args* args) { return check(args); }

extern "C" int proteus_adamw(const proteus_adamw_args* args, void* stream)
{
    if (const int rc = check(args)) return rc;
    const proteus_adamw_args& a = *args;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    Scalars s = {};
    s.lr = a.lr_gpu; s.step = a.step_gpu; s.norm = a.norm;
    s.lr_ = a.lr; s.decay = a.weight_decay; s.log_b1 = log(a.beta1); s.log_b2 = log(a.beta2);
    s.b1 = (float)a.beta1; s.b2 = (float)a.beta2; s.c1 = (float)(1.0 - a.beta1); s.c2 = (float)(1.0 - a.beta2); s.decays = (float)sqrt(a.beta2); s.eps = (float)a.eps; s.max_norm = a.max_norm;
    if (!a.lr_gpu && !a.step_gpu) {
        s.keep = (float)(1.0 - a.lr * a.weight_decay);
        s.size = (float)(a.lr / -expm1((double)a.step * s.log_b1));
        s.root = (float)(1.0 / sqrt(-expm1((double)a.step * s.log_b2)));
    }
    s.seed = a.seed; s.number = a.step;
    // tensors by kind: the parameter's type, the gradient's, whether there is a master weight
    bool present[3][3][2] = {};
    static_assert(PROTEUS_DTYPE_F32 >= 0 && PROTEUS_DTYPE_F32 < 3 && PROTEUS_DTYPE_BF16 >= 0 && PROTEUS_DTYPE_BF16 < 3 && PROTEUS_DTYPE_F16 >= 0 && PROTEUS_DTYPE_F16 < 3, "");
    for (int i = 0; i < a.count; ++i) if (a.numel[i] > 0) present[a.param_types[i]][a.grad_types[i]][a.masters && a.masters[i]] = true;
    for (const int pt : {PROTEUS_DTYPE_F32, PROTEUS_DTYPE_BF16, PROTEUS_DTYPE_F16})
        for (const int gt : {PROTEUS_DTYPE_F32, PROTEUS_DTYPE_BF16, PROTEUS_DTYPE_F16})
            for (const bool master : {false, true}) {
                if (!present[pt][gt][master]) continue;
                int rc;
                if (pt == PROTEUS_DTYPE_F32)
                    rc = gt == PROTEUS_DTYPE_F32 ? go<float, float>(a, s, pt, gt, master, st) : gt == PROTEUS_DTYPE_BF16 ? go<float, bf16_t>(a, s, pt, gt, master, st) : go<float, f16_t>(a, s, pt, gt, master, st);
                else if (pt == PROTEUS_DTYPE_BF16)
                    rc = gt == PROTEUS_DTYPE_F32 ? go<bf16_t, float>(a, s, pt, gt, master, st) : go<bf16_t, bf16_t>(a, s, pt, gt, master, st);
                else
                    rc = gt == PROTEUS_DTYPE_F32 ? go<f16_t, float>(a, s, pt, gt, master, st) : go<f16_t, f16_t>(a, s, pt, gt, master, st);
                if (rc) return rc;
            }
    return a.step_gpu ? launch(count_kernel, 1, 1, st, a.step_gpu) : 0;
}

// Matrix products of the gated feed-forward block in bf16: fp32 sums on the matrix cores, the block's element-wise parts as epilogues (gfx950).
//
// A workgroup of four waves makes a BM x BN tile of C and steps through K by 32.  Tiles of both operands travel global -> LDS directly (buffer_load ... lds, 16 bytes a
// lane), up to STAGES - 1 steps ahead, each stage an LDS object of its own (so that the compiler sees that a read of one does not wait for loads into another).  An operand
// whose rows run along k lies in LDS as rows of 64 bytes and is read 16 bytes a lane; one whose rows run across k lies as it is in memory, 32 rows of k, and
// is transposed as it is read (ds_read_b64_tr_b16).  16-byte chunks are XOR-swizzled in either, by the chunk that a lane asks memory for, so that reads touch all 64 banks.
//
// A step has two halves of 16 k, and the fragments of each are read under the products of the one before, across the barrier too: that stands between the halves, where the
// step's reads are over and the next step's data is waited for.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "gated_mlp_internal.h"

namespace {

using namespace proteus_gated;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float  f32x2  __attribute__((ext_vector_type(2)));
typedef float  f32x16 __attribute__((ext_vector_type(16)));
typedef short  s16x4  __attribute__((ext_vector_type(4)));

constexpr int HK = 32;                              // k of a step
constexpr uint32_t OUTSIDE = 0x80000000u;           // beyond any buffer here: reads as zeros
constexpr int64_t MOST_BYTES = 0x7ffffff0;          // of a buffer

#define GM_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))

struct Args {
    Product p;
    int tiles_m, tiles_n, tiles, per_xcd, group;    // tiles of all shares of K; tiles along m that go side by side
    int shares, steps;                              // shares of K, steps of each
};

__device__ __forceinline__ uint32_t pack2(const float a, const float b)
{
    const f32x2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}
__device__ __forceinline__ float low(const uint32_t w)  { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float high(const uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }

// One operand's tile of EXT rows (of C or of its transpose).  KC: rows along k.
template <bool KC, int EXT, int WAVES, bool PAIRED, int WAVE_EXT> struct Operand {
    static constexpr int BYTES = EXT * HK * 2, LOADS = BYTES / 1024 / WAVES, PITCH = EXT * 2;
    static_assert(BYTES % (1024 * WAVES) == 0, "whole loads");
    const uint16_t* base;                           // of the tile at k = 0
    int64_t ld;
    int K, cols;                                    // cols: of the matrix from the tile on (rows across k)
    uint32_t at[LOADS];
    int chunk_k;                                    // first k of the lane's chunk (rows along k)

    // PAIRED: each wave's WAVE_EXT rows are 32 gates and 32 values in turn; `second` rows lie between a gate and its value, and rows0 counts features
    __device__ __forceinline__ void begin(const uint16_t* X, const int64_t ld_, const int row0, const int rows, const int K_, const int wave, const int lane, const int second)
    {
        ld = ld_; K = K_;
        if (KC) {
            base = X + (PAIRED ? 0 : row0 * ld);
            chunk_k = 8 * ((lane & 3) ^ ((lane >> 4) & 3));
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = 16 * (i * WAVES + wave) + (lane >> 2);
                if (PAIRED) {
                    const int f = row0 + r / WAVE_EXT * (WAVE_EXT / 2) + r % WAVE_EXT / 64 * 32 + (r & 31);
                    at[i] = f < rows ? (uint32_t)(((f + (r & 32 ? second : 0)) * (int64_t)ld + chunk_k) * 2) : OUTSIDE;       // (the whole matrix below 2^31 bytes)
                } else
                    at[i] = row0 + r < rows ? (uint32_t)((r * ld + chunk_k) * 2) : OUTSIDE;
            }
        } else {
            base = X + row0;
            cols = rows - row0;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int byte = 1024 * (i * WAVES + wave) + 16 * lane, k = byte / PITCH, chunk = (byte % PITCH / 16) ^ swizzle(k);
                at[i] = 8 * chunk < cols ? (uint32_t)((k * ld + 8 * chunk) * 2) : OUTSIDE;
            }
        }
    }
    static __device__ __forceinline__ int swizzle(const int k) { return 2 * (k & 7); }

    __device__ __forceinline__ void issue(const int step, unsigned char* to, const int wave) const
    {
        const int k0 = step * HK, left = max(K - k0, 0);
        __amdgpu_buffer_rsrc_t r;
        if (KC) r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + k0), 0, (int)MOST_BYTES, 0x00020000);
        else {
            const int64_t bytes = left ? ((int64_t)(left - 1) * ld + cols) * 2 : 0;
            r = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)k0 * ld), 0, (int)(bytes < MOST_BYTES ? bytes : MOST_BYTES), 0x00020000);
        }
        const bool in = !KC || chunk_k < left;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, GM_LDS(void, to + 1024 * (i * WAVES + wave)), 16, in ? at[i] : OUTSIDE, 0, 0, 0);
    }
};

// Fragments of T tiles of 32 rows from row w0 of an operand's tile, 16 k.
template <bool KC, int EXT, int T> struct Reader {
    uint32_t at0[KC ? 2 : T], at1[KC ? 1 : T];
    __device__ __forceinline__ void begin(const int w0, const int lane)
    {
        const int half = lane >> 5, col = lane & 31;
        if (KC) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) at0[ks] = (w0 + col) * 64 + ((2 * ks + half) ^ ((col >> 2) & 3)) * 16;       // (32 rows further swizzle alike)
        } else {
            const int k = 8 * half + ((lane & 15) >> 2);
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const int n = w0 + 32 * i + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                at0[i] = k * (EXT * 2) + (((n >> 3) ^ (2 * (k & 7))) * 16) + 2 * (n & 7);
                at1[i] = (k + 4) * (EXT * 2) + (((n >> 3) ^ (2 * ((k + 4) & 7))) * 16) + 2 * (n & 7);
            }
        }
    }
    __device__ __forceinline__ void read(const unsigned char* from, const int ks, bf16x8* f) const
    {
#pragma unroll
        for (int i = 0; i < T; ++i) {
            if (KC) f[i] = *reinterpret_cast<const bf16x8*>(from + at0[ks] + i * 2048);
            else {
                const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(GM_LDS(s16x4, from + at0[i] + ks * 16 * EXT * 2));
                const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(GM_LDS(s16x4, from + at1[i] + ks * 16 * EXT * 2));
                const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
                f[i] = __builtin_bit_cast(bf16x8, make_uint4(x.x, x.y, y.x, y.y));
            }
        }
    }
};

template <bool AK, bool BK, int EPI, int BM, int BN, int WM, int WN, int STAGES, int BLOCKS>
__global__ __launch_bounds__(WM * WN * 64, BLOCKS)
void product_kernel(const Args g)
{
#ifdef __HIP_DEVICE_COMPILE__                       // (with the body in it, the host's pass leaves out the stubs of all instances but the first)
    constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;       // 32 x 32 tiles of a wave
    constexpr bool GATE = EPI == GATED || EPI == GATED_KEPT;
    constexpr int FEATURES = GATE ? BN / 2 : BN;                               // of a tile
    using OA = Operand<AK, BM, WAVES, false, 0>;
    using OB = Operand<BK, BN, WAVES, GATE, BN / WN>;
    constexpr int STAGE = OA::BYTES + OB::BYTES, LOADS = OA::LOADS + OB::LOADS;
    static_assert(WAVES == 4 && (STAGES == 3 || STAGES == 4) && (!GATE || TN % 2 == 0), "");
    __shared__ __align__(1024) unsigned char s0[STAGE];
    __shared__ __align__(1024) unsigned char s1[STAGE];
    __shared__ __align__(1024) unsigned char s2[STAGE];
    __shared__ __align__(1024) unsigned char s3[STAGES > 3 ? STAGE : 16];

    const Product& p = g.p;
    const int id = (blockIdx.x & 7) * g.per_xcd + (blockIdx.x >> 3);           // consecutive tiles on one XCD: `group` tiles along m by what follows along n
    if ((int)(blockIdx.x >> 3) >= g.per_xcd || id >= g.tiles) return;
    const int share = id / (g.tiles_m * g.tiles_n), tile = id - share * (g.tiles_m * g.tiles_n);
    const int band = tile / (g.group * g.tiles_n), in_band = tile - band * (g.group * g.tiles_n), high_ = min(g.group, g.tiles_m - band * g.group);
    const int m0 = (band * g.group + in_band % high_) * BM, n0 = in_band / high_ * FEATURES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5, col = lane & 31;
    const int first = share * g.steps, steps = min(g.steps, (p.K + HK - 1) / HK - first);

    OA a;
    OB b;
    a.begin(p.A, p.lda, m0, p.M, p.K, wave, lane, 0);
    b.begin(p.B, p.ldb, n0, p.N, p.K, wave, lane, p.N);
    const int wm = wave / WN * (TM * 32), wn = wave % WN * (TN * 32);
    Reader<AK, BM, TM> ra;
    Reader<BK, BN, TN> rb;
    ra.begin(wm, lane);
    rb.begin(wn, lane);
    auto issue = [&](const int step, unsigned char* to) {
        a.issue(first + step, to, wave);
        b.issue(first + step, to + OA::BYTES, wave);
    };
    bf16x8 fa[2][TM], fb[2][TN];
    f32x16 acc[TM][TN] = {};
    auto read = [&](const unsigned char* from, const int ks) { ra.read(from, ks, fa[ks]); rb.read(from + OA::BYTES, ks, fb[ks]); };
    auto multiply = [&](const int ks) {
        // rows of the accumulator are columns of C, so that a lane ends up with four of them side by side
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[ks][j], fa[ks][i], acc[i][j], 0, 0, 0);
    };
    // a half's products with the next half's reads between them
    auto spread = [&] {
        constexpr int READS = (AK ? TM : 2 * TM) + (BK ? TN : 2 * TN), PRODUCTS = TM * TN, PER = READS > PRODUCTS ? (READS + PRODUCTS - 1) / PRODUCTS : 1;
#pragma unroll
        for (int i = 0; i < PRODUCTS; ++i) {
            if (i * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto arrive = [&] {
        // the next stage's loads have landed for every wave, and everybody's reads of this one are over
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"((STAGES - 2) * LOADS) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto step = [&](const int s, unsigned char* mine, const unsigned char* next) {
        read(mine, 1);
        multiply(0);
        spread();
        arrive();
        issue(s + STAGES, mine);                                               // (past the end: zeros)
        read(next, 0);
        multiply(1);
        spread();
    };
    issue(0, s0);
    issue(1, s1);
    issue(2, s2);
    if (STAGES > 3) issue(3, s3);
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"((STAGES - 1) * LOADS) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(s0, 0);
    __builtin_amdgcn_sched_barrier(0);
    for (int s = 0;;) {
        step(s, s0, s1);
        if (++s >= steps) break;
        step(s, s1, s2);
        if (++s >= steps) break;
        if constexpr (STAGES == 3) step(s, s2, s0);
        else {
            step(s, s2, s3);
            if (++s >= steps) break;
            step(s, s3, s0);
        }
        if (++s >= steps) break;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");                // (zeros past the end still on their way)
    __syncthreads();

    // ---- epilogues: a wave's 32 rows through LDS, so that they leave in whole lines ----
    if (g.shares > 1) {
        // sums of a share of K: rows of the shares' own matrix [share][M][N]
        float* const to = p.part + (size_t)share * p.M * p.N;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = m0 + wm + 32 * i + col;
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int n = n0 + wn + 32 * j + 8 * q + 4 * half;
                    if (m < p.M && n < p.N) *reinterpret_cast<float4*>(to + (size_t)m * p.N + n) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                }
        }
        return;
    }
    auto own_rows = [&](const int bytes) -> unsigned char* {                   // (whole stages hold the blocks of all waves)
        const int per = STAGE / bytes, at = wave % per * bytes;
        return (wave / per == 0 ? s0 : wave / per == 1 ? s1 : wave / per == 2 ? s2 : s3) + at;
    };
    auto settled = [] {                                                        // the wave's own rows: no other wave reads them
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    auto four = [&](const uint16_t* v, const int n, const int end, float* to) {
        const uint2 w = v ? *reinterpret_cast<const uint2*>(v + min(n, end - 4)) : make_uint2(0u, 0u);
        to[0] = low(w.x); to[1] = high(w.x); to[2] = low(w.y); to[3] = high(w.y);
    };
    if constexpr (EPI == PLAIN) {
        constexpr int PITCH = TN * 64 + 16, CPR = TN * 4, RPI = 64 / CPR;      // bytes of a row; 16-byte chunks of it, rows an instruction
        static_assert(STAGE / (32 * PITCH) * (STAGES - 1) >= WAVES, "room");
        unsigned char* const own = own_rows(32 * PITCH);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[4];
                    four(p.bias, n0 + wn + 32 * j + 8 * q + 4 * half, p.N, v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += acc[i][j][4 * q + e];
                    *reinterpret_cast<uint2*>(own + col * PITCH + (32 * j + 8 * q + 4 * half) * 2) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
                }
            settled();
#pragma unroll
            for (int r = 0; r < 32; r += RPI) {
                const int row = r + lane / CPR, c = lane % CPR, m = m0 + wm + 32 * i + row, n = n0 + wn + 8 * c;
                const uint4 v = *reinterpret_cast<const uint4*>(own + row * PITCH + c * 16);
                if (m < p.M && n < p.N) *reinterpret_cast<uint4*>(p.C + (size_t)m * p.ldc + n) = v;
            }
            settled();
        }
    } else if constexpr (GATE) {
        constexpr int FEAT = TN / 2 * 32, OUTS = EPI == GATED_KEPT ? 3 : 1, PITCH = OUTS * FEAT * 2 + 16, CPR = FEAT / 8, RPI = 64 / CPR;
        static_assert(STAGE / (32 * PITCH) * (STAGES - 1) >= WAVES, "room");
        unsigned char* const own = own_rows(32 * PITCH);
        const int f0 = n0 + wn / 2;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; j += 2)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int f = 16 * j + 8 * q + 4 * half;
                    float gate[4], value[4], h[4];
                    four(p.bias, f0 + f, p.N, gate);
                    four(p.bias ? p.bias + p.N : nullptr, f0 + f, p.N, value);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float slope;
                        gate[e] += acc[i][j][4 * q + e];
                        value[e] += acc[i][j + 1][4 * q + e];
                        activate<false>(p.act, gate[e], h[e], slope);
                        h[e] *= value[e];
                    }
                    unsigned char* const to = own + col * PITCH + f * 2;
                    *reinterpret_cast<uint2*>(to) = make_uint2(pack2(h[0], h[1]), pack2(h[2], h[3]));
                    if (OUTS == 3) {
                        *reinterpret_cast<uint2*>(to + FEAT * 2) = make_uint2(pack2(gate[0], gate[1]), pack2(gate[2], gate[3]));
                        *reinterpret_cast<uint2*>(to + FEAT * 4) = make_uint2(pack2(value[0], value[1]), pack2(value[2], value[3]));
                    }
                }
            settled();
#pragma unroll
            for (int o = 0; o < OUTS; ++o)
#pragma unroll
                for (int r = 0; r < 32; r += RPI) {
                    const int row = r + lane / CPR, c = lane % CPR, m = m0 + wm + 32 * i + row, f = f0 + 8 * c;
                    const uint4 v = *reinterpret_cast<const uint4*>(own + row * PITCH + o * FEAT * 2 + c * 16);
                    if (m < p.M && f < p.N) *reinterpret_cast<uint4*>(o == 0 ? p.C + (size_t)m * p.ldc + f : p.z + (size_t)m * 2 * p.N + (o == 2 ? p.N : 0) + f) = v;
                }
            settled();
        }
    } else {
        constexpr int PITCH = TN * 128 + 16, CPR = TN * 4, RPI = 64 / CPR;     // fp32 here; chunks of eight columns
        static_assert(STAGE / (32 * PITCH) * STAGES >= WAVES, "room");
        unsigned char* const own = own_rows(32 * PITCH);
        float sums[16] = {};
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4*>(own + col * PITCH + (32 * j + 8 * q + 4 * half) * 4) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            settled();
#pragma unroll
            for (int r = 0; r < 32; r += RPI) {
                const int row = r + lane / CPR, c = lane % CPR, m = m0 + wm + 32 * i + row, n = n0 + wn + 8 * c;
                const float4 lo = *reinterpret_cast<const float4*>(own + row * PITCH + c * 32), hi = *reinterpret_cast<const float4*>(own + row * PITCH + c * 32 + 16);
                if (m >= p.M || n >= p.N) continue;
                const uint16_t* const z = p.z + (size_t)m * 2 * p.N + n;
                const uint4 gv = *reinterpret_cast<const uint4*>(z), vv = *reinterpret_cast<const uint4*>(z + p.N);
                const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w}, vw[4] = {vv.x, vv.y, vv.z, vv.w};
                const float dh[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                uint32_t og[4], ov[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float a0, s0_, a1, s1_;
                    activate<false>(p.act, low(gw[e]), a0, s0_);
                    activate<false>(p.act, high(gw[e]), a1, s1_);
                    const float g0 = dh[2 * e] * low(vw[e]) * s0_, g1 = dh[2 * e + 1] * high(vw[e]) * s1_, v0 = dh[2 * e] * a0, v1 = dh[2 * e + 1] * a1;
                    sums[2 * e] += g0; sums[2 * e + 1] += g1; sums[8 + 2 * e] += v0; sums[9 + 2 * e] += v1;
                    og[e] = pack2(g0, g1);
                    ov[e] = pack2(v0, v1);
                }
                uint16_t* const to = p.C + (size_t)m * 2 * p.N + n;
                *reinterpret_cast<uint4*>(to) = make_uint4(og[0], og[1], og[2], og[3]);
                *reinterpret_cast<uint4*>(to + p.N) = make_uint4(ov[0], ov[1], ov[2], ov[3]);
            }
            settled();
        }
        if (p.columns) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int o = CPR; o < 64; o <<= 1) sums[e] += __shfl_xor(sums[e], o);
            const int n = n0 + wn + 8 * lane;
            if (lane < CPR && n < p.N) {
                float* const to = p.columns + (size_t)(m0 / BM * WM + wave / WN) * 2 * p.N + n;
#pragma unroll
                for (int e = 0; e < 8; ++e) { to[e] = sums[e]; to[p.N + e] = sums[8 + e]; }
            }
        }
    }
#endif
}

// C = the shares' sums in their order.
__global__ __launch_bounds__(256)
void shares_kernel(const float* __restrict__ part, uint16_t* __restrict__ C, const int64_t n, const int shares, const int N, const int64_t ldc)
{
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 256 * 8) {
        float4 lo = *reinterpret_cast<const float4*>(part + i), hi = *reinterpret_cast<const float4*>(part + i + 4);
        for (int s = 1; s < shares; ++s) {
            const float4 a = *reinterpret_cast<const float4*>(part + s * n + i), b = *reinterpret_cast<const float4*>(part + s * n + i + 4);
            lo.x += a.x; lo.y += a.y; lo.z += a.z; lo.w += a.w;
            hi.x += b.x; hi.y += b.y; hi.z += b.z; hi.w += b.w;
        }
        *reinterpret_cast<uint4*>(C + i / N * ldc + i % N) = make_uint4(pack2(lo.x, lo.y), pack2(lo.z, lo.w), pack2(hi.x, hi.y), pack2(hi.z, hi.w));
    }
}

enum Tile { T256, T256x128, T128 };
int rows_of(const int t) { return t == T128 ? 128 : 256; }
int columns_of(const int t) { return t == T256 ? 256 : 128; }
int slots_of(const int t) { return t == T256 ? 256 : 512; }                    // workgroups that the chip holds at once
int64_t tiles_of(const int t, const int64_t M, const int64_t N) { return ((M + rows_of(t) - 1) / rows_of(t)) * ((N + columns_of(t) - 1) / columns_of(t)); }

struct Plan { int tile, shares, steps; };
// What a product takes, in clocks of a compute unit: rounds of workgroups by the time that a step's products or its LDS traffic take, whichever is longer.
double cost_of(const int t, const int64_t tiles, const int steps)
{
    static const double per_step[3] = {1150.0, 1250.0 / 2, 800.0 / 2}, fixed[3] = {9000.0, 8000.0 / 2, 5000.0 / 2};      // (of one workgroup where two share a unit)
    const int64_t slots = slots_of(t);
    const int64_t whole = tiles / slots, rest = tiles % slots;
    const double each = per_step[t] * steps + fixed[t], two = slots == 512 ? 2.0 : 1.0;
    return whole * two * each + (rest == 0 ? 0.0 : rest > 256 ? two * each : slots == 512 ? 1.3 * each : each);
}
Plan plan_of(const int form, const int M, const int N, const int K)
{
    const int steps = (K + HK - 1) / HK;
    Plan best = {T256, 1, steps};
    double least = 1e30;
    for (int t = T256; t <= T128; ++t)
        for (int s = 1; s <= (form == PROTEUS_GEMM_TN ? 16 : 1); s *= 2) {
            const int per = (steps + s - 1) / s;
            if (s > 1 && per < 16) break;
            // (the shares' sums written and read once each, at 2 KB a clock)
            const double c = cost_of(t, tiles_of(t, M, N) * s, per) + (s > 1 ? 6000.0 + (double)M * N * 4 * s * 2 / 2048.0 : 0.0);
            if (c < least) { least = c; best = {t, (steps + per - 1) / per, per}; }
        }
    return best;
}

template <bool AK, bool BK, int EPI, int BM, int BN, int STAGES, int BLOCKS>
int go(const Product& p, const Plan& plan, hipStream_t st)
{
    Args g = {};
    g.p = p;
    const int n = EPI == GATED || EPI == GATED_KEPT ? 2 * p.N : p.N;
    g.tiles_m = (p.M + BM - 1) / BM;
    g.tiles_n = (n + BN - 1) / BN;
    g.shares = plan.shares; g.steps = plan.steps;
    g.tiles = g.tiles_m * g.tiles_n * g.shares;
    g.per_xcd = (g.tiles + 7) / 8;
    g.group = 8;
    hipLaunchKernelGGL((product_kernel<AK, BK, EPI, BM, BN, 2, 2, STAGES, BLOCKS>), dim3((unsigned)g.per_xcd * 8), dim3(256), 0, st, g);
    return (int)hipGetLastError();
}
template <bool AK, bool BK, int EPI>
int go(const Product& p, const Plan& plan, hipStream_t st)
{
    switch (plan.tile) {
        case T256:     return go<AK, BK, EPI, 256, 256, 4, 1>(p, plan, st);
        case T256x128: return go<AK, BK, EPI, 256, 128, 3, 2>(p, plan, st);
        default:       return go<AK, BK, EPI, 128, 128, 4, 2>(p, plan, st);
    }
}

}  // namespace

size_t proteus_gated::product_bytes(const int form, const int M, const int N, const int K)
{
    const Plan plan = plan_of(form, M, N, K);
    return plan.shares > 1 ? (size_t)plan.shares * M * N * 4 : 0;
}

int proteus_gated::column_rows(const int M, const int N, const int K)
{
    const int rows = rows_of(plan_of(PROTEUS_GEMM_NN, M, N, K).tile);
    return (M + rows - 1) / rows * 2;
}

int proteus_gated::product(const Product& p, hipStream_t st)
{
    const bool gate = p.epilogue == GATED || p.epilogue == GATED_KEPT;
    const Plan plan = plan_of(p.form, p.M, gate ? 2 * p.N : p.N, p.K);
    if (p.form == PROTEUS_GEMM_NT) {
        if (p.epilogue == GATED)      return go<true, true, GATED>(p, plan, st);
        if (p.epilogue == GATED_KEPT) return go<true, true, GATED_KEPT>(p, plan, st);
        return go<true, true, PLAIN>(p, plan, st);
    }
    if (p.form == PROTEUS_GEMM_NN) {
        if (p.epilogue == GATED_GRAD) return go<true, false, GATED_GRAD>(p, plan, st);
        return go<true, false, PLAIN>(p, plan, st);
    }
    const int rc = go<false, false, PLAIN>(p, plan, st);
    if (rc || plan.shares == 1) return rc;
    const int64_t n = (int64_t)p.M * p.N, blocks = (n / 8 + 255) / 256;
    hipLaunchKernelGGL(shares_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, p.part, p.C, n, plan.shares, p.N, p.ldc);
    return (int)hipGetLastError();
}

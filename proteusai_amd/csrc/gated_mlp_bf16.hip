// Matrix products of the gated feed-forward block in bf16: fp32 sums on the matrix cores, the block's element-wise parts as epilogues (gfx950).
//
// A workgroup of four waves makes a tile of C and steps through K by 64.  Tiles of both operands travel global -> LDS directly (buffer_load ... lds, 16 bytes a lane) into one
// of two stages, each an LDS object of its own (so that the compiler sees that a read of one does not wait for loads into the other).  An operand whose rows run along k lies
// in LDS as rows of 128 bytes and is read 16 bytes a lane; one whose rows run across k lies as it is in memory, 64 rows of k, and is transposed as it is read
// (ds_read_b64_tr_b16).  16-byte chunks are XOR-swizzled in either, by the chunk that a lane asks memory for, so that reads touch all 64 banks.
//
// A step has four slices of 16 k.  The reads of a slice's fragments and the loads of a later step go out between the products of the slice before, in an order written
// out by hand, so that the matrix unit is not kept waiting; two barriers a step, one before a stage is written again and one before what was written is read.
//
// Tiles of 256 x 256, one workgroup to a compute unit, its accumulators in the accumulation registers: half the traffic into LDS for each product of 128 x 128, so that the
// matrix unit bounds a step (1.65 us where it could do 1.0 at its peak).  Nothing else runs on the unit under their epilogues, so a workgroup goes on with its next tile, whose first two
// steps it sends for before.  Tiles of 128 x 128, two workgroups to a unit, each under the other's epilogue: where there are too few of the others for the chip, and where the
// epilogue is the longest (the gradient's); of 64 x 128 where there are too few even of those.  Products of few tiles and many k (gradients of weights) are cut along k, and a second launch adds up the shares' fp32 sums.
//
// 32768 rows, d_model 1024, hidden 4096, us and TFLOP/s: x W^T with the gate and what is kept for the backward 575 and 956, without 483 and 1138; h Wo^T 218 and 1261; dy Wo with the gate's
// gradient 413 and 666; dz W 415 and 1325; dz^T x 430 and 1279; dy^T h 222 and 1238.  (A library product of 8192 x 8192 x 8192 runs at 1334.)
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include "gated_mlp_internal.h"
#include "mfma16.h"

namespace {

using namespace proteus_gated;
using namespace proteus_mfma16;

struct Args {
    Product p;
    int tiles_m, tiles_n, tiles, per_xcd, group;    // tiles of all shares of K; tiles along m that go side by side
    int shares, steps;                              // shares of K, steps of each
    int past;                                       // what is kept for the backward goes past the caches, both ways
};

__device__ __forceinline__ uint32_t pack2(const float a, const float b) { return pack_bf16(a, b); }

// Sums kept to 20 bits (1, 8 and 11: off by at most 2^-12): the upper 16 of two, and the four below of four gates and their values, a byte for each pair.
__device__ __forceinline__ uint32_t twenty(const float x) { return __builtin_bit_cast(uint32_t, x) + 0x800u; }      // (rounded; of a NaN from bf16 operands the lower bits are zeros)
__device__ __forceinline__ uint32_t upper2(const float a, const float b) { return __builtin_amdgcn_perm(twenty(b), twenty(a), 0x07060302u); }
__device__ __forceinline__ uint32_t second_bytes(const float* x)
{
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(twenty(x[3]), twenty(x[2]), 0x0c0c0501u), __builtin_amdgcn_perm(twenty(x[1]), twenty(x[0]), 0x0c0c0501u), 0x05040100u);
}
__device__ __forceinline__ uint32_t rest_of(const float* gate, const float* value) { return (second_bytes(value) & 0xf0f0f0f0u) | ((second_bytes(gate) >> 4) & 0x0f0f0f0fu); }
// element e of four: its upper bits in word e / 2 of `upper`, the next in byte e of `second` (the gates' or the values', in the bytes' upper halves)
template <int E> __device__ __forceinline__ float from20(const uint32_t upper, const uint32_t second)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_perm(upper, second, (E & 1 ? 0x07060000u : 0x05040000u) | (uint32_t)(E & 3) << 8 | 0x0cu));
}

constexpr int PAST = 2;                             // of a load or store: not to be kept in the caches
template <int AUX> __device__ __forceinline__ uint4 get_as(const __amdgpu_buffer_rsrc_t r, const uint32_t at)
{
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, AUX));
}
template <int AUX> __device__ __forceinline__ void put_as(const __amdgpu_buffer_rsrc_t r, const uint32_t at, const uint4 v)
{
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, at, 0, AUX);
}

// One operand's tile of EXT rows (of C or of its transpose).  KC: rows along k.
template <bool KC, int EXT, int WAVES, bool PAIRED, int WAVE_EXT> struct Operand {
    static constexpr int BYTES = EXT * HK * 2, LOADS = BYTES / 1024 / WAVES, PITCH = EXT * 2;
    static_assert(BYTES % (1024 * WAVES) == 0 && WAVES % 2 == 0, "whole loads");
    const uint16_t* base;                           // of the tile at k = 0
    int64_t ld;
    int K, cols;                                    // cols: of the matrix from the tile on (rows across k)
    uint32_t at[LOADS];
    int chunk_k;                                    // first k of the lane's chunk (rows along k)

    // PAIRED: each wave's WAVE_EXT rows are 32 gates and 32 values in turn; `second` rows lie between a gate and its value, and rows0 counts features
    __device__ __forceinline__ void begin(const uint16_t* X, const int64_t ld_, const int row0, const int rows, const int k0, const int K_, const int wave, const int lane, const int second)
    {
        ld = ld_; K = K_ - k0;
        if (KC) {
            base = X + (PAIRED ? 0 : row0 * ld) + k0;
            chunk_k = 8 * ((lane & 7) ^ ((4 * wave + (lane >> 4)) & 7));       // (its row's half, modulo 8: the same for all loads of a wave)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = 8 * (i * WAVES + wave) + (lane >> 3);
                if constexpr (PAIRED) {
                    const int f = row0 + r / WAVE_EXT * (WAVE_EXT / 2) + r % WAVE_EXT / 64 * 32 + (r & 31);
                    const uint32_t to = ((uint32_t)(f + (r & 32 ? second : 0)) * (uint32_t)ld + (uint32_t)chunk_k) * 2u;         // (the whole matrix below 2^31 bytes)
                    at[i] = f < rows ? to : OUTSIDE;
                } else {
                    const uint32_t to = ((uint32_t)r * (uint32_t)ld + (uint32_t)chunk_k) * 2u;
                    at[i] = row0 + r < rows ? to : OUTSIDE;
                }
            }
        } else {
            base = X + k0 * ld + row0;
            cols = rows - row0;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int byte = 1024 * (i * WAVES + wave) + 16 * lane, k = byte / PITCH, chunk = (byte % PITCH / 16) ^ swizzle(k);
                const uint32_t to = ((uint32_t)k * (uint32_t)ld + 8u * (uint32_t)chunk) * 2u;
                at[i] = 8 * chunk < cols ? to : OUTSIDE;
            }
        }
    }
    static __device__ __forceinline__ int swizzle(const int k) { return swizzle_of<EXT>(k); }

    // Where a step's loads read.
    struct From { __amdgpu_buffer_rsrc_t r; bool in; };
    __device__ __forceinline__ From from(const int step) const
    {
        const int k0 = step * HK, left = max(K - k0, 0);
        if (KC) return {__builtin_amdgcn_make_buffer_rsrc((void*)(base + k0), 0, (int)MOST_BYTES, 0x00020000), chunk_k < left};
        const int64_t bytes = left ? ((int64_t)(left - 1) * ld + cols) * 2 : 0;
        return {__builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)k0 * ld), 0, (int)(bytes < MOST_BYTES ? bytes : MOST_BYTES), 0x00020000), true};
    }
    __device__ __forceinline__ void issue(const From& f, const int i, unsigned char* to, const int wave) const
    {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(f.r, MFMA16_LDS(void, to + 1024 * (i * WAVES + wave)), 16, KC && !f.in ? OUTSIDE : at[i], 0, 0, 0);
    }
};

// fn with the activation as a constant
template <typename F> __device__ __forceinline__ void chosen(const int act, const F& fn)
{
    if (act == SILU)      fn(std::integral_constant<int, SILU>());
    else if (act == GELU) fn(std::integral_constant<int, GELU>());
    else if (act == RELU) fn(std::integral_constant<int, RELU>());
    else                  fn(std::integral_constant<int, SIGMOID>());
}

template <bool AK, bool BK, int EPI, int BM, int BN, int WM, int WN, int BLOCKS>
struct Workgroup {
    static constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;       // 32 x 32 tiles of a wave
    static constexpr bool GATE = EPI == GATED || EPI == GATED_KEPT;
    // One workgroup to a compute unit: nothing else runs under a tile's first loads and its epilogue, so that a workgroup goes on with its next tile's steps 0 and 1 as it
    // would with its own, and the epilogue, in LDS of its own, runs while they travel.  (Two: each runs under the other's.)
    static constexpr bool GOES_ON = BLOCKS == 1;
    static constexpr int FEATURES = GATE ? BN / 2 : BN;                        // of a tile
    using OA = Operand<AK, BM, WAVES, false, 0>;
    using OB = Operand<BK, BN, WAVES, GATE, BN / WN>;
    static constexpr int STAGE = OA::BYTES + OB::BYTES, LOADS = OA::LOADS + OB::LOADS;
    static_assert(WAVES == 4 && TN % 2 == 0, "");
    // a wave's 32 rows of 64 columns (GATED_GRAD: fp32 of all of its columns) on their way out
    static constexpr int OUT_PITCH = EPI == GATED_GRAD ? TN * 128 + 16 : GATE ? TN * 32 + 16 : 144, REST_PITCH = TN * 16 + 8,
                         OUT = 32 * (OUT_PITCH + (EPI == GATED_KEPT ? REST_PITCH : 0)), OUT_BYTES = GOES_ON ? WAVES * OUT : 16;
    static_assert(GOES_ON || STAGE / OUT * 2 >= WAVES, "room");

// Workgroup `block` of `blocks`; s0 and s1: the stages, out: OUT_BYTES.
static __device__ __forceinline__ void run(const Args& g, const int block, const int blocks, unsigned char* const s0, unsigned char* const s1, unsigned char* const out)
{
#ifdef __HIP_DEVICE_COMPILE__
    const Product& p = g.p;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = lane >> 5, col = lane & 31;
    // consecutive tiles on one XCD: `group` tiles along m by what follows along n; its workgroups take them in turn
    const int stop = min(g.tiles, ((block & 7) + 1) * g.per_xcd), stride = blocks >> 3;
    int id = (block & 7) * g.per_xcd + (block >> 3);
    if (id >= stop) return;

    OA a;
    OB b;
    int m0, n0, share, steps;
    // The loads from here on are tile `id`'s (past the last: zeros).
    auto aim = [&] {
        // (readfirstlane: divisions go through the vector unit, and a buffer's address has to be in scalar registers, or every load is a loop over the lanes' addresses)
        const int at = min(id, stop - 1);
        share = __builtin_amdgcn_readfirstlane(at / (g.tiles_m * g.tiles_n));
        const int tile = at - share * (g.tiles_m * g.tiles_n), band = __builtin_amdgcn_readfirstlane(tile / (g.group * g.tiles_n)), in_band = tile - band * (g.group * g.tiles_n);
        const int high_ = min(g.group, g.tiles_m - band * g.group), column = __builtin_amdgcn_readfirstlane(in_band / high_);
        m0 = (band * g.group + in_band - column * high_) * BM;
        n0 = column * FEATURES;
        const int first = share * g.steps * HK, end = min(p.K, first + g.steps * HK);
        steps = (end - first + HK - 1) / HK;
        a.begin(p.A, p.lda, m0, p.M, first, id < stop ? end : first, wave, lane, 0);
        b.begin(p.B, p.ldb, n0, p.N, first, id < stop ? end : first, wave, lane, p.N);
    };
    aim();
    const int wm = wave / WN * (TM * 32), wn = wave % WN * (TN * 32);
    Reader<AK, BM, TM> ra;
    Reader<BK, BN, TN> rb;
    ra.begin(wm, lane);
    rb.begin(wn, lane);
    bf16x8 fa[SLICES][TM], fb[SLICES][TN];
    constexpr int READS = TM + TN, PRODUCTS = TM * TN, HALF = LOADS / 2;
    // the r-th fragment of a slice in the order in which the products want them
    auto read = [&](const unsigned char* from, const int ks, const int r) {
        if (r == 0)       fa[ks][0] = ra.read(from, ks, 0);
        else if (r <= TN) fb[ks][r - 1] = rb.read(from + OA::BYTES, ks, r - 1);
        else              fa[ks][r - TN] = ra.read(from, ks, r - TN);
    };
    auto begin = [&](const int s, unsigned char* to) {
        const auto af = a.from(s);
        const auto bf = b.from(s);
#pragma unroll
        for (int i = 0; i < OA::LOADS; ++i) a.issue(af, i, to, wave);
#pragma unroll
        for (int i = 0; i < OB::LOADS; ++i) b.issue(bf, i, to + OA::BYTES, wave);
    };
    begin(0, s0);
    begin(1, s1);
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(LOADS) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < READS; ++r) read(s0, 0, r);
    __builtin_amdgcn_sched_barrier(0);
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  for (;;) {
    f32x16 acc[TM][TN] = {};
    // The products of a slice with reads of `count` slices from `ks1` on between them, early, and loads l0 to l1 - 1 of a step, spread evenly.  The order is kept as it is
    // written: a single wave to a SIMD has no other to fill the gaps that anything in a row between two products leaves.
    auto products = [&](const int ks, const unsigned char* from, const int ks1, const int count, const int l0, const int l1, const typename OA::From& af, const typename OB::From& bf,
                        unsigned char* to) {
        each<PRODUCTS>([&](const auto X) {
            constexpr int x = decltype(X)::value, i = x / TN, j = x % TN;
            // rows of the accumulator are columns of C, so that a lane ends up with four of them side by side
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[ks][j], fa[ks][i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            const int per = (count * READS + PRODUCTS - 1) / PRODUCTS, lx = (l1 - l0) * x / PRODUCTS, ly = (l1 - l0) * (x + 1) / PRODUCTS;
#pragma unroll
            for (int r = x * per; r < count * READS && r < (x + 1) * per; ++r) read(from, ks1 + r / READS, r % READS);
#pragma unroll
            for (int l = l0 + lx; l < l0 + ly; ++l) {
                if (l < OA::LOADS) a.issue(af, l, to, wave);
                else               b.issue(bf, l - OA::LOADS, to + OA::BYTES, wave);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // A step: its fragments are read under the first two slices' products; then its stage is everybody's to fill again, under the last two, and before the last the
    // next step's data is waited for.
    auto step = [&](unsigned char* mine, const unsigned char* next, const int load) {
        const auto af = a.from(load);                                          // (past the end: zeros)
        const auto bf = b.from(load);
        products(0, mine, 1, 2, 0, 0, af, bf, mine);
        products(1, mine, 3, 1, 0, 0, af, bf, mine);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        products(2, mine, 0, 0, 0, HALF, af, bf, mine);
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"(HALF) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        products(3, next, 0, 1, HALF, LOADS, af, bf, mine);
    };
    // (steps past the end multiply zeros: without branches the compiler's own waits stay exact)
    int s = 2;
    do {
        step(s0, s1, s);
        step(s1, s0, s + 1);
        s += 2;
    } while (s < (GOES_ON ? steps : steps + 2));
    const int done_m = m0, done_n = n0, done_share = share;
    if (GOES_ON) {                                                             // the last two, under which the next tile's first are sent for
        id += stride;
        aim();
        step(s0, s1, 0);
        step(s1, s0, 1);
    } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");            // (zeros past the end still on their way)
        __syncthreads();
    }
    [&](const int m0, const int n0, const int share) {
    // ---- epilogues: a wave's 32 rows through LDS, so that they leave in whole lines ----
    unsigned char* const own = GOES_ON ? out + wave * OUT : (wave / (STAGE / OUT) == 0 ? s0 : s1) + wave % (STAGE / OUT) * OUT;
    auto settled = [] {                                                        // the wave's own rows: no other wave reads them, and its LDS instructions are carried out in order
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);                                     // (or accumulators are fetched long before their turn, and spilt)
    };
    // rows of a matrix from the tile's first on: what lies outside is read as zeros and not written
    auto rows_from = [&](const uint16_t* X, const int64_t ld) {
        const int64_t bytes = (int64_t)min(BM, p.M - m0) * ld * 2;
        return __builtin_amdgcn_make_buffer_rsrc((void*)(X + m0 * ld), 0, (int)(bytes < MOST_BYTES ? bytes : MOST_BYTES), 0x00020000);
    };
    auto place = [&](const int row, const int n, const int64_t ld) {
        const uint32_t at = ((uint32_t)row * (uint32_t)ld + (uint32_t)n) * 2u;
        return ((m0 + row < p.M) & (n < p.N)) ? at : OUTSIDE;
    };
    auto put = [&](const __amdgpu_buffer_rsrc_t r, const uint32_t at, const uint4 v) { put_as<0>(r, at, v); };
    // (offsets in it are half of those in 16 bits: OUTSIDE / 2 is beyond it, too)
    auto rest = [&] { return __builtin_amdgcn_make_buffer_rsrc((void*)(p.rest + (int64_t)m0 * p.N), 0, min(BM, p.M - m0) * p.N, 0x00020000); };
    // An accumulator's element.  Where they fill the accumulation registers they are fetched one by one when their turn comes: left to itself the compiler fetches them all
    // at once and spills.  (It does not see that these wait for the products: the s_nop below does.)
    auto sum = [&](const float v) {
        if constexpr (!GOES_ON) return v;
        float r;
        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(r) : "a"(v));
        return r;
    };
    if constexpr (GOES_ON) asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (EPI == PLAIN) if (g.shares > 1) {
        // sums of a share of K: rows of the shares' own matrix [share][M][N]
        const int64_t rows = min(BM, p.M - m0);
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(p.part + ((int64_t)share * p.M + m0) * p.N), 0, (int)(rows * p.N * 4), 0x00020000);
        each<TM>([&](const auto I) {
            constexpr int i = decltype(I)::value;
            const int row = wm + 32 * i + col;
            each<TN * 4>([&](const auto J) {
                constexpr int j = decltype(J)::value / 4, q = decltype(J)::value % 4;
                const int n = n0 + wn + 32 * j + 8 * q + 4 * half;
                const float4 v = make_float4(sum(acc[i][j][4 * q]), sum(acc[i][j][4 * q + 1]), sum(acc[i][j][4 * q + 2]), sum(acc[i][j][4 * q + 3]));
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, ((row < rows) & (n < p.N)) ? ((uint32_t)row * (uint32_t)p.N + (uint32_t)n) * 4u : OUTSIDE, 0, 0);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        return;
    }
    // bias, zeros outside and where there is none
    const __amdgpu_buffer_rsrc_t bias = __builtin_amdgcn_make_buffer_rsrc((void*)p.bias, 0, p.bias ? (GATE ? 2 : 1) * p.N * 2 : 0, 0x00020000);
    auto four = [&](const int n) { return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(bias, n * 2, 0, 0)); };
    const __amdgpu_buffer_rsrc_t rc = rows_from(p.C, EPI == GATED_GRAD ? 2 * (int64_t)p.N : p.ldc);
    if constexpr (EPI == PLAIN) {
        uint2 bv[TN][4];
        each<TN * 4>([&](const auto I) { constexpr int j = decltype(I)::value / 4, q = decltype(I)::value % 4; bv[j][q] = four(n0 + wn + 32 * j + 8 * q + 4 * half); });
        each<TM * (TN / 2)>([&](const auto I) {                                // 32 rows of 64 columns
            constexpr int i = decltype(I)::value / (TN / 2), j0 = decltype(I)::value % (TN / 2) * 2;
            each<8>([&](const auto J) {
                constexpr int j = decltype(J)::value / 4, q = decltype(J)::value % 4;
                const uint2 b_ = bv[j0 + j][q];
                const f32x16& v = acc[i][j0 + j];
                *reinterpret_cast<uint2*>(own + col * OUT_PITCH + (32 * j + 8 * q + 4 * half) * 2) =
                    make_uint2(pack2(sum(v[4 * q]) + low(b_.x), sum(v[4 * q + 1]) + high(b_.x)), pack2(sum(v[4 * q + 2]) + low(b_.y), sum(v[4 * q + 3]) + high(b_.y)));
            });
            settled();
#pragma unroll
            for (int r = 0; r < 32; r += 8) {
                const int row = r + lane / 8, c = lane % 8;
                put(rc, place(wm + 32 * i + row, n0 + wn + 32 * j0 + 8 * c, p.ldc), *reinterpret_cast<const uint4*>(own + row * OUT_PITCH + c * 16));
            }
            settled();
        });
    } else if constexpr (GATE) {
        constexpr int FEAT = TN / 2 * 32, OUTS = EPI == GATED_KEPT ? 3 : 1, CPR = FEAT / 8, RPI = 64 / CPR;        // 16-byte chunks of a row, rows an instruction
        const int f0 = n0 + wn / 2;
        unsigned char* const rests = own + 32 * OUT_PITCH;
        const __amdgpu_buffer_rsrc_t rz = rows_from(OUTS == 3 ? p.z : p.C, 2 * (int64_t)p.N), rr = OUTS == 3 ? rest() : rz;
        uint2 bg[TN / 2][4], bu[TN / 2][4];
        each<TN * 2>([&](const auto I) {
            constexpr int j = decltype(I)::value / 4, q = decltype(I)::value % 4;
            const int f = f0 + 32 * j + 8 * q + 4 * half;
            bg[j][q] = four(f);
            bu[j][q] = four(p.N + f);
        });
        chosen(p.act, [&](const auto A) {
            constexpr int act = decltype(A)::value;
            each<TM>([&](const auto I) {
                constexpr int i = decltype(I)::value;
                uint2 words[OUTS][TN / 2][4];                                  // (h,) gates, values: 32 rows of each leave in turn
                each<TN * 2>([&](const auto J) {
                    constexpr int j = decltype(J)::value / 4, q = decltype(J)::value % 4;
                    uint2 g_ = bg[j][q], u_ = bu[j][q];
                    asm volatile("" : "+v"(g_.x), "+v"(g_.y), "+v"(u_.x), "+v"(u_.y));           // (or the biases are kept as floats from one 32 rows to the next, and spilt)
                    float gate[4] = {low(g_.x), high(g_.x), low(g_.y), high(g_.y)}, value[4] = {low(u_.x), high(u_.x), low(u_.y), high(u_.y)}, h[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float slope;
                        gate[e] += sum(acc[i][2 * j][4 * q + e]);
                        value[e] += sum(acc[i][2 * j + 1][4 * q + e]);
                        activate<false>(act, gate[e], h[e], slope);
                        h[e] *= value[e];
                    }
                    *reinterpret_cast<uint2*>(own + col * OUT_PITCH + (32 * j + 8 * q + 4 * half) * 2) = make_uint2(pack2(h[0], h[1]), pack2(h[2], h[3]));
                    if constexpr (OUTS == 3) {
                        words[1][j][q] = make_uint2(upper2(gate[0], gate[1]), upper2(gate[2], gate[3]));
                        words[2][j][q] = make_uint2(upper2(value[0], value[1]), upper2(value[2], value[3]));
                        *reinterpret_cast<uint32_t*>(rests + col * REST_PITCH + 32 * j + 8 * q + 4 * half) = rest_of(gate, value);
                    }
                });
                uint4 leaving[OUTS][32 / RPI];
                const int row = lane / CPR, c = lane % CPR;
                each<OUTS>([&](const auto O) {
                    constexpr int o = decltype(O)::value;
                    if constexpr (o > 0)
                        each<TN * 2>([&](const auto J) {
                            constexpr int j = decltype(J)::value / 4, q = decltype(J)::value % 4;
                            *reinterpret_cast<uint2*>(own + col * OUT_PITCH + (32 * j + 8 * q + 4 * half) * 2) = words[o][j][q];
                        });
                    settled();
#pragma unroll
                    for (int r = 0; r < 32 / RPI; ++r) leaving[o][r] = *reinterpret_cast<const uint4*>(own + (r * RPI + row) * OUT_PITCH + c * 16);
                    settled();
                });
                auto leave = [&](const auto X) {
                    constexpr int aux = decltype(X)::value;
                    each<OUTS>([&](const auto O) {
                        constexpr int o = decltype(O)::value;
#pragma unroll
                        for (int r = 0; r < 32 / RPI; ++r) {
                            const uint32_t at = place(wm + 32 * i + r * RPI + row, f0 + 8 * c, o ? 2 * (int64_t)p.N : p.ldc);
                            put_as<o ? aux : 0>(o ? rz : rc, o == 2 && at != OUTSIDE ? at + 2 * p.N : at, leaving[o][r]);
                        }
                    });
                    if constexpr (OUTS == 3)
#pragma unroll
                        for (int r = 0; r < 32 / RPI; ++r)
                            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, *reinterpret_cast<const uint2*>(rests + (r * RPI + row) * REST_PITCH + c * 8)), rr,
                                                                  place(wm + 32 * i + r * RPI + row, f0 + 8 * c, p.N) >> 1, 0, aux);
                };
                if (OUTS == 3 && g.past) leave(std::integral_constant<int, PAST>{});
                else leave(std::integral_constant<int, 0>{});
                settled();
            });
        });
    } else {
        constexpr int PITCH = OUT_PITCH, CPR = TN * 4, RPI = 64 / CPR, PIECES = 32 / RPI;         // fp32 here; chunks of eight columns
        const __amdgpu_buffer_rsrc_t rz = rows_from(p.z, 2 * (int64_t)p.N), rr = rest();
        const int n = n0 + wn + 8 * (lane % CPR);
        float sums[16] = {};
        // z of 32 rows is sent for at once (all of a tile's before its first step: no faster where another workgroup shares the unit, 429 / 419 us at 32768 x 4096 x 1024)
        uint4 zg[PIECES], zv[PIECES];
        uint2 zr[PIECES];
        auto fetch_as = [&](const int i, const auto X) {
            constexpr int aux = decltype(X)::value;
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
                const uint32_t at = place(wm + 32 * i + k * RPI + lane / CPR, n, 2 * (int64_t)p.N);
                zg[k] = get_as<aux>(rz, at);
                zv[k] = get_as<aux>(rz, at == OUTSIDE ? at : at + 2 * p.N);
                zr[k] = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rr, place(wm + 32 * i + k * RPI + lane / CPR, n, p.N) >> 1, 0, aux));
            }
        };
        auto fetch = [&](const int i) {
            if (g.past) fetch_as(i, std::integral_constant<int, PAST>{});
            else fetch_as(i, std::integral_constant<int, 0>{});
            __builtin_amdgcn_sched_barrier(0);
        };
        chosen(p.act, [&](const auto A) {
            constexpr int act = decltype(A)::value;
            each<TM>([&](const auto I) {
                constexpr int i = decltype(I)::value;
                fetch(i);
                each<TN * 4>([&](const auto J) {
                    constexpr int j = decltype(J)::value / 4, q = decltype(J)::value % 4;
                    *reinterpret_cast<float4*>(own + col * PITCH + (32 * j + 8 * q + 4 * half) * 4) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                });
                settled();
                each<PIECES>([&](const auto Q) {
                    constexpr int k = decltype(Q)::value;
                    const int row = k * RPI + lane / CPR, c = lane % CPR;
                    const float4 lo = *reinterpret_cast<const float4*>(own + row * PITCH + c * 32), hi = *reinterpret_cast<const float4*>(own + row * PITCH + c * 32 + 16);
                    const uint32_t gw[4] = {zg[k].x, zg[k].y, zg[k].z, zg[k].w}, vw[4] = {zv[k].x, zv[k].y, zv[k].z, zv[k].w};
                    // (zeros in rows past the last one, for the column sums: theirs of zeros are NaN beside a weight that is not finite)
                    const bool in = m0 + wm + 32 * i + row < p.M;
                    const float dh[8] = {in ? lo.x : 0.0f, in ? lo.y : 0.0f, in ? lo.z : 0.0f, in ? lo.w : 0.0f, in ? hi.x : 0.0f, in ? hi.y : 0.0f, in ? hi.z : 0.0f, in ? hi.w : 0.0f};
                    const uint32_t vr[2] = {zr[k].x & 0xf0f0f0f0u, zr[k].y & 0xf0f0f0f0u}, gr[2] = {zr[k].x << 4 & 0xf0f0f0f0u, zr[k].y << 4 & 0xf0f0f0f0u};
                    uint32_t og[4], ov[4];
                    each<4>([&](const auto E) {
                        constexpr int e = decltype(E)::value;
                        float a0, s0_, a1, s1_;
                        activate<false>(act, from20<2 * e>(gw[e], gr[e / 2]), a0, s0_);
                        activate<false>(act, from20<2 * e + 1>(gw[e], gr[e / 2]), a1, s1_);
                        const float g0 = dh[2 * e] * from20<2 * e>(vw[e], vr[e / 2]) * s0_, g1 = dh[2 * e + 1] * from20<2 * e + 1>(vw[e], vr[e / 2]) * s1_, v0 = dh[2 * e] * a0, v1 = dh[2 * e + 1] * a1;
                        sums[2 * e] += g0; sums[2 * e + 1] += g1; sums[8 + 2 * e] += v0; sums[9 + 2 * e] += v1;
                        og[e] = pack2(g0, g1);
                        ov[e] = pack2(v0, v1);
                    });
                    // (added up here, whether or not they are wanted: left to where they are, the compiler keeps every term until then)
#pragma unroll
                    for (int e = 0; e < 16; ++e) asm volatile("" : "+v"(sums[e]));
                    const uint32_t at = place(wm + 32 * i + row, n, 2 * (int64_t)p.N);
                    put(rc, at, make_uint4(og[0], og[1], og[2], og[3]));
                    put(rc, at == OUTSIDE ? at : at + 2 * p.N, make_uint4(ov[0], ov[1], ov[2], ov[3]));
                    __builtin_amdgcn_sched_barrier(0);
                });
                settled();
            });
        });
        if (p.columns) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int o = CPR; o < 64; o <<= 1) sums[e] += __shfl_xor(sums[e], o);
            if (lane < CPR && n < p.N) {
                float* const to = p.columns + (size_t)(m0 / BM * WM + wave / WN) * 2 * p.N + n;
#pragma unroll
                for (int e = 0; e < 8; ++e) { to[e] = sums[e]; to[p.N + e] = sums[8 + e]; }
            }
        }
    }
    }(done_m, done_n, done_share);
    if (!GOES_ON || id >= stop) break;
  }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                           // (nothing of a workgroup's may still be on its way into LDS when that is another's)
#endif
}
};

template <bool AK, bool BK, int EPI, int BM, int BN, int WM, int WN, int BLOCKS>
__global__ __launch_bounds__(WM * WN * 64, BLOCKS)
void product_kernel(const Args g)
{
#ifdef __HIP_DEVICE_COMPILE__                       // (with the body in it, the host's pass leaves out the stubs of all instances but the first)
    using T = Workgroup<AK, BK, EPI, BM, BN, WM, WN, BLOCKS>;
    __shared__ __align__(1024) unsigned char s0[T::STAGE];
    __shared__ __align__(1024) unsigned char s1[T::STAGE];
    __shared__ __align__(16) unsigned char out[T::OUT_BYTES];
    T::run(g, (int)blockIdx.x, (int)gridDim.x, s0, s1, out);
#endif
}

// Column sums of bf16 rows, `per` of them a share, workgroup `block` for 512 columns of share `share`, to part [share][C].  A thread has eight columns of every 4th row;
// s: 8 KB.
struct ColumnArgs { Columns c; int64_t per; int across, blocks; };
__device__ __forceinline__ void columns_run(const ColumnArgs& g, const int block, const int share, float (*const s)[64][8])
{
    const Columns& o = g.c;
    const int c = (block * 64 + (threadIdx.x & 63)) * 8, group = threadIdx.x >> 6;
    float v[8] = {};
    if (c < o.C) {
        const int64_t end = min(o.rows, (share + (int64_t)1) * g.per);
#pragma unroll 4
        for (int64_t r = share * g.per + group; r < end; r += 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(o.a + r * o.C + c);
            v[0] += low(w.x); v[1] += high(w.x); v[2] += low(w.y); v[3] += high(w.y); v[4] += low(w.z); v[5] += high(w.z); v[6] += low(w.w); v[7] += high(w.w);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[group][threadIdx.x & 63][e] = v[e];
    __syncthreads();
    if (group || c >= o.C) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.part[(int64_t)share * o.C + c + e] = s[0][threadIdx.x][e] + s[1][threadIdx.x][e] + s[2][threadIdx.x][e] + s[3][threadIdx.x][e];
}
__global__ __launch_bounds__(256)
void columns_kernel(const ColumnArgs g)
{
    __shared__ float s[4][64][8];
    columns_run(g, (int)blockIdx.x % g.across, (int)blockIdx.x / g.across, s);
}

// Up to three plain products, TN or NN, one behind the other in the grid, and column sums.
struct Together { Args product[3]; ColumnArgs columns; int first[5]; };
__global__ __launch_bounds__(256, 2)
void together_kernel(const Together t)
{
#ifdef __HIP_DEVICE_COMPILE__
    using TN_ = Workgroup<false, false, PLAIN, 128, 128, 2, 2, 2>;
    using NN_ = Workgroup<true, false, PLAIN, 128, 128, 2, 2, 2>;
    static_assert(TN_::STAGE == NN_::STAGE && TN_::OUT_BYTES == NN_::OUT_BYTES, "");
    __shared__ __align__(1024) unsigned char s0[TN_::STAGE];
    __shared__ __align__(1024) unsigned char s1[TN_::STAGE];
    __shared__ __align__(16) unsigned char out[TN_::OUT_BYTES];
    if ((int)blockIdx.x >= t.first[3]) {
        const int block = (int)blockIdx.x - t.first[3];
        columns_run(t.columns, block % t.columns.across, block / t.columns.across, reinterpret_cast<float (*)[64][8]>(s0));
        return;
    }
    const int job = (int)blockIdx.x >= t.first[2] ? 2 : (int)blockIdx.x >= t.first[1] ? 1 : 0, block = (int)blockIdx.x - t.first[job], blocks = t.first[job + 1] - t.first[job];
    const Args& g = t.product[job];
    if (g.p.form == PROTEUS_GEMM_TN) TN_::run(g, block, blocks, s0, s1, out);
    else                             NN_::run(g, block, blocks, s0, s1, out);
#endif
}

// Sums of shares (C = the shares' sums in their order, and the bias) and of columns (16 of them a workgroup, every 16th row a thread), one behind the other in the grid.
constexpr int END_COLUMNS = 16;
struct Grid { int first[6]; };                      // workgroups of each and the end: three products, two column sums
__global__ __launch_bounds__(256)
void ends_kernel(const Ends ends, const Grid grid)
{
    __shared__ float s[256 / END_COLUMNS][END_COLUMNS];
    int job = 0;
    while ((int)blockIdx.x >= grid.first[job + 1]) ++job;                      // (the last entry is gridDim.x)
    const int block = (int)blockIdx.x - grid.first[job], blocks = grid.first[job + 1] - grid.first[job];
    if (job >= 3) {
        const Ends::Columns c = ends.columns[job - 3];
        const int n = block * END_COLUMNS + (threadIdx.x & (END_COLUMNS - 1)), group = threadIdx.x / END_COLUMNS;
        float v = 0.0f;
        if (n < c.C)
#pragma unroll 8
            for (int r = group; r < c.rows; r += 256 / END_COLUMNS) v += c.part[(int64_t)r * c.C + n];
        s[group][threadIdx.x & (END_COLUMNS - 1)] = v;
        __syncthreads();
        if (group || n >= c.C) return;
        for (int k = 1; k < 256 / END_COLUMNS; ++k) v += s[k][threadIdx.x];
        c.out[n] = __builtin_bit_cast(uint16_t, (__bf16)v);
        return;
    }
    const Ends::Shares p = ends.shares[job];
    for (int64_t i = ((int64_t)block * 256 + threadIdx.x) * 8; i < p.n; i += (int64_t)blocks * 256 * 8) {
        float v[8] = {};
        for (int s_ = 0; s_ < p.shares; ++s_) {
            const float4 a = *reinterpret_cast<const float4*>(p.part + s_ * p.n + i), b = *reinterpret_cast<const float4*>(p.part + s_ * p.n + i + 4);
            v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w; v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
        }
        const int64_t row = i / p.N, column = i - row * p.N;
        if (p.bias) {
            const uint4 w = *reinterpret_cast<const uint4*>(p.bias + column);
            v[0] += low(w.x); v[1] += high(w.x); v[2] += low(w.y); v[3] += high(w.y); v[4] += low(w.z); v[5] += high(w.z); v[6] += low(w.w); v[7] += high(w.w);
        }
        *reinterpret_cast<uint4*>(p.C + row * p.ldc + column) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
    }
}

// Few rows (serving: single residues): what counts is to read the weights once, from everywhere at once.  A workgroup makes 16 columns of C (GATE: 16 features, from their gates' and
// their values' rows of B) for up to 16 MT rows; its waves take every WAVES-th 32 k of the weights straight into registers, as the matrix instruction's first operand, the
// rows of A being the second, and add up in LDS in their order.
template <int EPI, int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64)
void rows_kernel(const Product p)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr bool GATE = EPI != PLAIN;
    constexpr int SIDES = GATE ? 2 : 1, AHEAD = MT > 2 ? 2 : 4;                // steps whose loads are sent off together
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    __shared__ f32x4 sums[WAVES][MT][SIDES][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, row = lane & 15, k0 = 8 * (lane >> 4);
    const int steps = (p.K + 31) / 32;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)p.A, 0, (int)(((int64_t)(p.M - 1) * p.lda + p.K) * 2), 0x00020000);
    uint32_t at_a[MT], at_b[SIDES];
    __amdgpu_buffer_rsrc_t rb[SIDES];
#pragma unroll
    for (int s = 0; s < SIDES; ++s) {
        rb[s] = __builtin_amdgcn_make_buffer_rsrc((void*)(p.B + (s * (int64_t)p.N + n0) * p.ldb), 0, (int)(((int64_t)(min(16, p.N - n0) - 1) * p.ldb + p.K) * 2), 0x00020000);
        at_b[s] = n0 + row < p.N ? (uint32_t)((row * p.ldb + k0) * 2) : OUTSIDE;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) at_a[t] = 16 * t + row < p.M ? (uint32_t)(((16 * t + row) * p.lda + k0) * 2) : OUTSIDE;
    f32x4 acc[MT][SIDES] = {};
    auto get = [](const __amdgpu_buffer_rsrc_t r, const uint32_t at) { return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0)); };
    for (int s = wave; s < steps; s += WAVES * AHEAD) {
        bf16x8 a[AHEAD][MT], b[AHEAD][SIDES];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = (s + i * WAVES) * 32;
            const bool in = k + k0 < p.K;                                      // (K is a multiple of 8)
#pragma unroll
            for (int e = 0; e < SIDES; ++e) b[i][e] = get(rb[e], in ? at_b[e] + 2u * k : OUTSIDE);
#pragma unroll
            for (int t = 0; t < MT; ++t) a[i][t] = get(ra, in ? at_a[t] + 2u * k : OUTSIDE);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < SIDES; ++e) acc[t][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[i][e], a[i][t], acc[t][e], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < SIDES; ++e) sums[wave][t][e][lane] = acc[t][e];
    __syncthreads();
    if ((int)threadIdx.x >= 64 * MT) return;
    // four columns side by side of one row
    const int t = threadIdx.x >> 6, m = 16 * t + row, n = n0 + 4 * (lane >> 4);
    f32x4 v[SIDES];
#pragma unroll
    for (int e = 0; e < SIDES; ++e) {
        v[e] = sums[0][t][e][lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v[e] += sums[w][t][e][lane];
    }
    if (m >= p.M || n >= p.N) return;
    if (p.bias)
#pragma unroll
        for (int e = 0; e < SIDES; ++e) {
            const uint2 b = *reinterpret_cast<const uint2*>(p.bias + e * p.N + n);
            v[e] += f32x4{low(b.x), high(b.x), low(b.y), high(b.y)};
        }
    auto put = [](uint16_t* to, const f32x4 x) { *reinterpret_cast<uint2*>(to) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3])); };
    if constexpr (GATE) {
        if (EPI == GATED_KEPT) {
            const float gate[4] = {v[0][0], v[0][1], v[0][2], v[0][3]}, value[4] = {v[SIDES - 1][0], v[SIDES - 1][1], v[SIDES - 1][2], v[SIDES - 1][3]};
            uint16_t* const to = p.z + (size_t)m * 2 * p.N + n;
            *reinterpret_cast<uint2*>(to) = make_uint2(upper2(gate[0], gate[1]), upper2(gate[2], gate[3]));
            *reinterpret_cast<uint2*>(to + p.N) = make_uint2(upper2(value[0], value[1]), upper2(value[2], value[3]));
            *reinterpret_cast<uint32_t*>(p.rest + (size_t)m * p.N + n) = rest_of(gate, value);
        }
        f32x4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float slope, a;
            activate<false>(p.act, v[0][i], a, slope);
            h[i] = a * v[1][i];
        }
        put(p.C + (size_t)m * p.ldc + n, h);
    } else put(p.C + (size_t)m * p.ldc + n, v[0]);
#endif
}

template <int EPI> int go_rows(const Product& p, hipStream_t st)
{
    constexpr int WAVES = 8;
    const dim3 grid((unsigned)((p.N + 15) / 16)), block(WAVES * 64);
    if (p.M <= 16)      hipLaunchKernelGGL((rows_kernel<EPI, 1, WAVES>), grid, block, 0, st, p);
    else if (p.M <= 32) hipLaunchKernelGGL((rows_kernel<EPI, 2, WAVES>), grid, block, 0, st, p);
    else                hipLaunchKernelGGL((rows_kernel<EPI, 4, WAVES>), grid, block, 0, st, p);
    return (int)hipGetLastError();
}
// Us, by rows / in tiles (of 128 x 128; plain products of few tiles: gemm_bf16.hip's).  d_model 512, hidden 2048: the gate 8 rows 4.2 / 7.9, 64 5.5 / 7.6; down 8 4.7 / 8.0, 32 7.2 / 8.2,
// 33 8.4 / 8.1, 64 10.7 / 8.2.  1024 and 4096: 8 4.8 / 9.3 and 7.5 / 13.3, 32 6.6 / 9.4 and 12.3 / 13.4, 64 8.2 / 9.5 and 19.4 / 13.3.
bool by_rows(const int form, const int epilogue, const int M) { return form == PROTEUS_GEMM_NT && M <= (epilogue == PLAIN ? 32 : 64); }
// Plain products of at most one tile of 64 x 64 for every compute unit: 2048 x 512 x 2048 8.7 us there, 18.7 and in shares of K 13 here
bool by_small_tiles(const int form, const int epilogue, const int64_t M, const int64_t N)
{
    return form == PROTEUS_GEMM_NT && epilogue == PLAIN && ((M + 63) / 64) * ((N + 63) / 64) <= 256;
}

enum Tile { T256, T128, T64 };                      // T64: 64 x 128
int extent_of(const int t) { return t == T256 ? 256 : 128; }
int rows_of(const int t) { return t == T64 ? 64 : extent_of(t); }
int64_t tiles_of(const int t, const int64_t M, const int64_t N) { const int r = rows_of(t), c = extent_of(t); return ((M + r - 1) / r) * ((N + c - 1) / c); }

// What a product takes, us: rounds of workgroups by the time of one, measured (one tile of 256 x 256 to a compute unit; two of 128 x 128, or one where they are few).
double cost_of(const int t, const int epilogue, const int64_t tiles, const int steps)
{
    static const double gate256[4] = {5.5, 4.0, 8.5, 28.0}, gate128[4] = {1.5, 0.5, 2.4, 9.5};        // epilogues (and first loads) that nothing runs under, or another workgroup does
    if (t == T256) return 2.0 + (double)((tiles + 255) / 256) * ((tiles < 64 ? 1.1 : 1.65) * steps + gate256[epilogue]);
    const int64_t whole = tiles / 512, rest = tiles % 512;
    const double two = 1.02 * steps + gate128[epilogue], one = 0.55 * steps + gate128[epilogue];
    return 2.0 + whole * two + (rest == 0 ? 0.0 : rest > 256 ? two : one);
}
Plan plan_of(const int epilogue, const int M, const int N, const int K, double* const cost = nullptr)
{
    const int steps = (K + HK - 1) / HK;
    Plan best = {T128, 1, steps};
    double least = 1e30;
    // Tiles of 64 x 128 where there is a compute unit for each.  The gate with what is kept, 128 x 128 / 64 x 128, us: d_model 512, hidden 2048, 128 rows 8.0 / 6.4, 512 9.1 / 7.9,
    // 1000 (two to a unit) 11.2 / 11.7, 5003 37.9 / 39.5; 1024 and 4096, 256 rows 13.2 / 11.6, 512 15.2 / 16.0, 5003 96 / 117.  Its
    // gradient: 65 rows 10.4 / 8.1, 512 11.7 / 9.4, 1000 13.7 / 11.2; 1024 and 4096, 512 rows 15.8 / 13.7.
    if (epilogue != PLAIN && tiles_of(T64, M, N) <= 256) return {T64, 1, steps};
    // (GATED_GRAD in tiles of 256 x 256, whose epilogue nothing ran under: 32768 x 4096 x 1024 445 us, 128 x 128 419)
    for (int t = epilogue == GATED_GRAD ? T128 : T256; t <= T128; ++t)
        for (int s = 1; s <= (epilogue == PLAIN ? 16 : 1); ++s) {
            const int per = ((steps + s - 1) / s + 1) / 2 * 2;
            if (s > 1 && per < 4) break;
            // (the shares' sums written and read once each, and a launch)
            const double c = cost_of(t, epilogue, tiles_of(t, M, N) * s, per) + (s > 1 ? 2.5 + (double)M * N * 8 * s / 8e6 : 0.0);
            if (c < least) { least = c; best = {t, s == 1 ? 1 : (steps + per - 1) / per, s == 1 ? steps : per}; }
        }
    if (cost) *cost = least;
    return best;
}

Args args_of(const Product& p, const Plan& plan)
{
    Args g = {};
    g.p = p;
    const int n = p.epilogue == GATED || p.epilogue == GATED_KEPT ? 2 * p.N : p.N, extent = extent_of(plan.tile);
    g.tiles_m = (p.M + rows_of(plan.tile) - 1) / rows_of(plan.tile);
    g.tiles_n = (n + extent - 1) / extent;
    g.shares = plan.shares; g.steps = plan.steps;
    g.tiles = g.tiles_m * g.tiles_n * g.shares;
    g.per_xcd = (g.tiles + 7) / 8;
    g.group = 8;
    // Past the caches, where it would not be found in them (256 MB) any more: 32768 x 4096, 671 MB, written 609 / 575 us, read 436 / 415; 5003 x 1912, 48 MB, 53 / 62 and 43 / 47.
    g.past = (int64_t)p.M * p.N * 5 > (256 << 20);
    return g;
}

template <bool AK, bool BK, int EPI, int ROWS, int EXT, int BLOCKS>
int go(const Product& p, const Plan& plan, hipStream_t st)
{
    const Args g = args_of(p, plan);
    const int side_by_side = BLOCKS == 1 ? std::min(g.per_xcd, 32) : g.per_xcd;                        // (32 compute units of an XCD)
    hipLaunchKernelGGL((product_kernel<AK, BK, EPI, ROWS, EXT, 2, 2, BLOCKS>), dim3((unsigned)side_by_side * 8), dim3(256), 0, st, g);
    return (int)hipGetLastError();
}
template <bool AK, bool BK, int EPI>
int go(const Product& p, const Plan& plan, hipStream_t st)
{
    if constexpr (EPI != GATED_GRAD)
        if (plan.tile == T256) return go<AK, BK, EPI, 256, 256, 1>(p, plan, st);
    if constexpr (EPI != PLAIN)
        if (plan.tile == T64) return go<AK, BK, EPI, 64, 128, 3>(p, plan, st);
    return go<AK, BK, EPI, 128, 128, 2>(p, plan, st);
}
int go_plain(const Product& p, const Plan& plan, Ends& ends, hipStream_t st)
{
    if (ends.count == 3) if (const int rc = finish(ends, st)) return rc;
    const int rc = p.form == PROTEUS_GEMM_NT ? go<true, true, PLAIN>(p, plan, st) : p.form == PROTEUS_GEMM_NN ? go<true, false, PLAIN>(p, plan, st) : go<false, false, PLAIN>(p, plan, st);
    if (rc || plan.shares == 1) return rc;
    ends.shares[ends.count++] = {p.part, p.bias, p.C, (int64_t)p.M * p.N, p.ldc, plan.shares, p.N};
    return 0;
}

}  // namespace

size_t proteus_gated::product_bytes(const int form, const int M, const int N, const int K)
{
    if (by_rows(form, PLAIN, M) || by_small_tiles(form, PLAIN, M, N)) return 0;
    const Plan plan = plan_of(PLAIN, M, N, K);
    return plan.shares > 1 ? (size_t)plan.shares * M * N * 4 : 0;
}

int proteus_gated::column_rows(const int M, const int N, const int K)
{
    const int rows = rows_of(plan_of(GATED_GRAD, M, N, K).tile);
    return (M + rows - 1) / rows * 2;
}

int proteus_gated::product(const Product& p, Ends& ends, hipStream_t st)
{
    const bool gate = p.epilogue == GATED || p.epilogue == GATED_KEPT;
    if (by_rows(p.form, p.epilogue, p.M)) return p.epilogue == GATED ? go_rows<GATED>(p, st) : gate ? go_rows<GATED_KEPT>(p, st) : go_rows<PLAIN>(p, st);
    if (by_small_tiles(p.form, p.epilogue, p.M, p.N)) return proteus_gemm_bf16(p.A, p.B, p.bias, p.C, p.M, p.N, p.K, (int)p.lda, (int)p.ldb, (int)p.ldc, 0, st);
    const Plan plan = plan_of(p.epilogue, p.M, gate ? 2 * p.N : p.N, p.K);
    if (p.epilogue == GATED)      return go<true, true, GATED>(p, plan, st);
    if (p.epilogue == GATED_KEPT) return go<true, true, GATED_KEPT>(p, plan, st);
    if (p.epilogue == GATED_GRAD) return go<true, false, GATED_GRAD>(p, plan, st);
    return go_plain(p, plan, ends, st);
}

// What the three products take in one launch of 128 x 128, us, in these shares of K: the whole of their steps over all compute units, two workgroups each, or their longest.
// They are run so where that is less than one after the other: the tiles of each alone seldom fill the chip.  A training pass apart / together, us: d_model 512, hidden
// 2048, 40 rows 53 / 42, 300 66 / 52, 1000 81 / 61, 2048 108 / 91, 4096 164 / 144, 12000 369 / 324; 712 and 1912, 5003 rows 237 / 228; 1024 and 4096, 8192 rows 749 / 723.
Behind proteus_gated::behind(const int rows, const int D, const int F, const int O)
{
    const int sizes[3][3] = {{O, F, rows}, {2 * F, D, rows}, {rows, D, 2 * F}};
    Behind b;
    double apart = 0.0, least = 1e30;
    for (int i = 0; i < 3; ++i) {
        double c;
        b.plan[i] = plan_of(PLAIN, sizes[i][0], sizes[i][1], sizes[i][2], &c);
        apart += c;
    }
    Plan best[3];
    for (int most = 4; most <= 4096; most *= 2) {
        for (int i = 0; i < 2; ++i) {
            const int limit = most + i * most / 2;                             // steps of a share, at most
            double all = 0.0, longest = 0.0, sums = 0.0;
            Plan plan[3];
            for (int j = 0; j < 3; ++j) {
                const int steps = (sizes[j][2] + HK - 1) / HK, shares = std::min((steps + limit - 1) / limit, 16), per = shares == 1 ? steps : ((steps + shares - 1) / shares + 1) / 2 * 2;
                plan[j] = {T128, (steps + per - 1) / per, per};
                all += tiles_of(T128, sizes[j][0], sizes[j][1]) * plan[j].shares * (0.63 * per + 0.75) / 256;
                longest = std::max(longest, 1.2 * per + 1.5);
                if (plan[j].shares > 1) sums += (double)sizes[j][0] * sizes[j][1] * 8 * plan[j].shares / 8e6;
            }
            const double c = 2.0 + std::max(all, longest) + sums + (sums > 0.0 ? 2.5 : 0.0);
            if (c < least) { least = c; for (int j = 0; j < 3; ++j) best[j] = plan[j]; }
        }
    }
    b.together = least < apart;
    for (int i = 0; i < 3; ++i) {
        if (b.together) b.plan[i] = best[i];
        b.part[i] = b.plan[i].shares > 1 ? (size_t)b.plan[i].shares * sizes[i][0] * sizes[i][1] * 4 : 0;
    }
    return b;
}

namespace {
constexpr int COLUMN_SHARES = 256;                  // at most
int64_t rows_per_share(const int64_t rows)
{
    const int64_t per = (rows + COLUMN_SHARES - 1) / COLUMN_SHARES;
    return per < 64 ? 64 : per;
}
}  // namespace

int64_t proteus_gated::column_shares(const int64_t rows) { return (rows + rows_per_share(rows) - 1) / rows_per_share(rows); }

int proteus_gated::products_behind(const Behind& b, const Product (&p)[3], const Columns& columns, Ends& ends, hipStream_t st)
{
    ColumnArgs sums = {columns, rows_per_share(columns.rows), (columns.C / 8 + 63) / 64, 0};
    if (columns.a) {
        sums.blocks = sums.across * (int)column_shares(columns.rows);
        ends.columns[ends.column_count++] = {columns.part, columns.out, (int)column_shares(columns.rows), columns.C};
    }
    if (!b.together) {
        if (columns.a) {
            hipLaunchKernelGGL(columns_kernel, dim3((unsigned)sums.blocks), dim3(256), 0, st, sums);
            if (const int rc = (int)hipGetLastError()) return rc;
        }
        for (int i = 0; i < 3; ++i) if (p[i].C) if (const int rc = go_plain(p[i], b.plan[i], ends, st)) return rc;
        return 0;
    }
    // the longest first
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](const int x, const int y) { return b.plan[x].steps > b.plan[y].steps; });
    Together t = {};
    int n = 0;
    for (const int i : order) {
        if (!p[i].C) continue;
        t.product[n] = args_of(p[i], b.plan[i]);
        t.first[n + 1] = t.first[n] + t.product[n].per_xcd * 8;
        ++n;
        if (b.plan[i].shares > 1) ends.shares[ends.count++] = {p[i].part, p[i].bias, p[i].C, (int64_t)p[i].M * p[i].N, p[i].ldc, b.plan[i].shares, p[i].N};
    }
    for (int i = n; i < 3; ++i) t.first[i + 1] = t.first[n];
    t.columns = sums;
    t.first[4] = t.first[3] + sums.blocks;
    if (!t.first[4]) return 0;
    hipLaunchKernelGGL(together_kernel, dim3((unsigned)t.first[4]), dim3(256), 0, st, t);
    return (int)hipGetLastError();
}

int proteus_gated::finish(Ends& ends, hipStream_t st)
{
    Grid grid;
    int at = 0;
    for (int i = 0; i < 3; ++i) {
        grid.first[i] = at;
        if (i < ends.count) at += (int)std::min<int64_t>((ends.shares[i].n / 8 + 255) / 256, 4096);
    }
    for (int i = 0; i < 2; ++i) {
        grid.first[3 + i] = at;
        if (i < ends.column_count) at += (ends.columns[i].C + END_COLUMNS - 1) / END_COLUMNS;
    }
    grid.first[5] = at;
    const Ends all = ends;
    ends.count = ends.column_count = 0;
    if (!at) return 0;
    hipLaunchKernelGGL(ends_kernel, dim3((unsigned)at), dim3(256), 0, st, all, grid);
    return (int)hipGetLastError();
}

// What the 16-bit matrix products that step through K by 64 share (gated_mlp_bf16.hip, linear_ce_body.inc): constants, and fragments from the tiles that their stages hold in LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <utility>

namespace proteus_mfma16 {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float  f32x2  __attribute__((ext_vector_type(2)));
typedef float  f32x16 __attribute__((ext_vector_type(16)));
typedef short  s16x4  __attribute__((ext_vector_type(4)));

constexpr int HK = 64;                              // k of a step: rows along k are whole lines of 128 bytes
constexpr int SLICES = HK / 16;
constexpr uint32_t OUTSIDE = 0x80000000u;           // beyond any buffer here: reads as zeros
constexpr int64_t MOST_BYTES = 0x7ffffff0;          // of a buffer

#define MFMA16_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))

__device__ __forceinline__ uint32_t pack_bf16(const float a, const float b)
{
    const f32x2 f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}
__device__ __forceinline__ float low(const uint32_t w)  { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float high(const uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }

// fn(0), ... fn(N - 1) with constants: indexes of accumulators that have to be known whatever the size of the body
template <typename F, int... I> __device__ __forceinline__ void each(const F& fn, std::integer_sequence<int, I...>) { (fn(std::integral_constant<int, I>()), ...); }
template <int N, typename F> __device__ __forceinline__ void each(const F& fn) { each(fn, std::make_integer_sequence<int, N>()); }

// Chunks of 16 bytes of row k of a stage whose rows run across k are moved about by this: within the EXT / 8 that a row has.
template <int EXT> __device__ __forceinline__ int swizzle_of(const int k) { return 2 * (k & (EXT >= 128 ? 7 : 3)); }

// Fragments of T tiles of 32 rows from row w0 of an operand's tile, 16 k.
template <bool KC, int EXT, int T> struct Reader {
    uint32_t at0[KC ? SLICES : T], at1[KC ? 1 : T];
    __device__ __forceinline__ void begin(const int w0, const int lane)
    {
        const int half = lane >> 5, col = lane & 31;
        if (KC) {
#pragma unroll
            for (int ks = 0; ks < SLICES; ++ks) at0[ks] = (w0 + col) * 128 + ((2 * ks + half) ^ ((col >> 1) & 7)) * 16;      // (32 rows further swizzle alike)
        } else {
            const int k = 8 * half + ((lane & 15) >> 2);
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const int n = w0 + 32 * i + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                at0[i] = k * (EXT * 2) + (((n >> 3) ^ swizzle_of<EXT>(k)) * 16) + 2 * (n & 7);
                at1[i] = (k + 4) * (EXT * 2) + (((n >> 3) ^ swizzle_of<EXT>(k + 4)) * 16) + 2 * (n & 7);
            }
        }
    }
    __device__ __forceinline__ bf16x8 read(const unsigned char* from, const int ks, const int i) const
    {
        if (KC) return *reinterpret_cast<const bf16x8*>(from + at0[ks] + i * 4096);
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(MFMA16_LDS(s16x4, from + at0[i] + ks * 16 * EXT * 2));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(MFMA16_LDS(s16x4, from + at1[i] + ks * 16 * EXT * 2));
        const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
        return __builtin_bit_cast(bf16x8, make_uint4(x.x, x.y, y.x, y.y));
    }
};

}  // namespace proteus_mfma16

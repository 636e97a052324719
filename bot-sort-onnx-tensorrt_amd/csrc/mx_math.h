// mx_math.h -- the arithmetic of microscaled rows (quantisation, decoding, loads and stores of 8 consecutive elements), shared by
// the kernels of mx.hip.
//
// A row of d values is held as blocks of 32: one scale byte s per block, worth X = 2^(s - 127) (255: the block is NaN), and 32
// elements in E2M1 (4 bits: values 0 .5 1 1.5 2 3 4 6 and a sign; two a byte, the even one in the low nibble) or E4M3 (8 bits: up to
// 448, smallest step 2^-9).  X = 2^clamp(floor(log2(max |v|)) - emax, -127, 127) with emax = 2 or 8, the exponent of the format's
// largest power of two; elements are v / X rounded to nearest, ties to even, saturating (the conversion of the OCP microscaling
// formats).  A block that holds an infinity or a NaN is NaN as a whole.  Rows are padded with zeros to MX_ROW = 128 elements -- the
// depth of one matrix instruction -- so that no kernel has a tail along a row.
#pragma once

#include "bts_internal.h"

namespace mx {

constexpr int MX_ROW = 128, MX_BLOCK = 32;
constexpr int E2M1 = BTS_MX_E2M1, E4M3 = BTS_MX_E4M3;

__host__ __device__ inline long padded(int d) { return ((long)d + MX_ROW - 1) / MX_ROW * MX_ROW; }
__host__ __device__ inline long code_bytes(int fmt, int d) { return fmt == E2M1 ? padded(d) / 2 : padded(d); }
__host__ __device__ inline long scale_bytes(int d) { return padded(d) / MX_BLOCK; }

__device__ __forceinline__ float bits_f32(uint32_t b) { return __int_as_float((int)b); }
__device__ __forceinline__ uint32_t f32_bits(float f) { return (uint32_t)__float_as_int(f); }

// ---- element types of x / out: float, _Float16 and bfloat16 (held as its bits) ------------------------------------------------
struct bf16 { uint16_t bits; };
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(bf16 v) { return bits_f32((uint32_t)v.bits << 16); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 from_f32<_Float16>(float v) { return (_Float16)v; }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) {      // nearest, ties to even; a NaN stays one
    const uint32_t b = f32_bits(v);
    const uint32_t r = (b + 0x7fffu + ((b >> 16) & 1u)) >> 16;
    return bf16{(uint16_t)((b & 0x7fffffffu) > 0x7f800000u ? ((b >> 16) | 0x40u) : r)};
}

// ---- 8 consecutive elements of a row ------------------------------------------------------------------------------------------
// All 8 there: 16 bytes an access whatever the address is a multiple of (the part reads and writes unaligned; rows of odd width
// element by element took twice the time); otherwise element by element, zeros behind the end.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// two values as one word of a 16-bit type (one conversion instruction for two bfloat16)
template <class T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
#if !defined(BTS_HOST_EMU)
    if constexpr (__is_same(T, bf16)) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
    }
#endif
    return __builtin_bit_cast(uint16_t, from_f32<T>(a)) | (uint32_t)__builtin_bit_cast(uint16_t, from_f32<T>(b)) << 16;
}
// v rounded to T and back
template <class T> __device__ __forceinline__ void round8(float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w = pack2<T>(v[2 * k], v[2 * k + 1]);
            v[2 * k] = to_f32(__builtin_bit_cast(T, (uint16_t)w));
            v[2 * k + 1] = to_f32(__builtin_bit_cast(T, (uint16_t)(w >> 16)));
        }
    }
}
template <class T> __device__ __forceinline__ void load8(const T *p, int have, float (&v)[8]) {
    if (have >= 8) {
        const u32x4 a = *reinterpret_cast<const u32x4_any *>(p);
        if constexpr (sizeof(T) == 4) {
            const u32x4 b = *reinterpret_cast<const u32x4_any *>(p + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = bits_f32(a[k]); v[4 + k] = bits_f32(b[k]); }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[2 * k] = to_f32(__builtin_bit_cast(T, (uint16_t)a[k]));
                v[2 * k + 1] = to_f32(__builtin_bit_cast(T, (uint16_t)(a[k] >> 16)));
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k < have ? to_f32(p[k]) : 0.0f;
    }
}
// 8 elements as the words they are stored in (float: 8 words, 16-bit types: 4)
template <class T> struct Words { uint32_t w[2 * sizeof(T)]; };
template <class T> __device__ __forceinline__ Words<T> to_words(const float (&v)[8]) {
    Words<T> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 8; ++k) r.w[k] = f32_bits(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) r.w[k] = pack2<T>(v[2 * k], v[2 * k + 1]);
    }
    return r;
}
template <class T> __device__ __forceinline__ void store_words(T *p, int have, const Words<T> &x) {
    if (have >= 8) {
        *reinterpret_cast<u32x4_any *>(p) = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
        if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4_any *>(p + 4) = u32x4{x.w[4], x.w[5], x.w[6], x.w[7]};
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (k >= have) continue;
            if constexpr (sizeof(T) == 4) p[k] = bits_f32(x.w[k]);
            else p[k] = __builtin_bit_cast(T, (uint16_t)(x.w[k / 2] >> (16 * (k & 1))));
        }
    }
}
template <class T> __device__ __forceinline__ void store8(T *p, int have, const float (&v)[8]) { store_words<T>(p, have, to_words<T>(v)); }

// ---- quantisation -------------------------------------------------------------------------------------------------------------
// The scale byte of a block from the bits of its largest magnitude: floor(log2) is the exponent field (a subnormal's field, 0, and
// every field up to emax end at the clamp, byte 0); an infinity's or NaN's field makes the block NaN.
template <int FMT> __device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23), s = e - (FMT == E2M1 ? 2 : 8);
    return e == 255 ? 255 : s < 0 ? 0 : s;
}
// 1 / X, exact: byte 0 -> 2^127, byte 252 -> 2^-125; a NaN block's elements are multiplied by 0 (and its codes masked below)
__device__ __forceinline__ float scale_inverse(int s) { return bits_f32((uint32_t)(254 - s) << 23); }

// v[0..7] (already divided by X) -> packed codes: E2M1 in .x (8 nibbles), E4M3 in .x and .y.  The conversion instructions round to
// nearest even; E2M1 saturates by itself, E4M3 gives NaN above 464, so its operands are clamped first (448..464 rounds to 448 anyway).
template <int FMT> __device__ __forceinline__ uint2 encode8(const float (&v)[8]) {
    uint2 r;
    if (FMT == E2M1) {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.0f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.0f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.0f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.0f, 3);
        r.x = c; r.y = 0;
    } else {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_fmed3f(v[e], -448.0f, 448.0f);
        int a = 0, b = 0;
        a = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], a, false);
        a = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], a, true);
        b = __builtin_amdgcn_cvt_pk_fp8_f32(w[4], w[5], b, false);
        b = __builtin_amdgcn_cvt_pk_fp8_f32(w[6], w[7], b, true);
        r.x = (uint32_t)a; r.y = (uint32_t)b;
    }
    return r;
}

// Four consecutive lanes hold one block, 8 elements each: its scale byte (the same in all four) and this lane's packed codes.
template <int FMT> __device__ __forceinline__ uint2 encode_block(const float (&v)[8], int &sbyte) {
    uint32_t top = 0;                    // magnitudes compare like their bits; a NaN's are above an infinity's
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, f32_bits(v[e]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));      // lane ^ 1
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));      // lane ^ 2
    sbyte = scale_byte<FMT>(top);
    const float inv = scale_inverse(sbyte == 255 ? 254 : sbyte);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v[e] * inv;
    const uint2 c = encode8<FMT>(w);
    return uint2{sbyte == 255 ? 0u : c.x, sbyte == 255 ? 0u : c.y};
}

// ---- decoding -----------------------------------------------------------------------------------------------------------------
// 8 packed codes of one block -> the words they are stored as.  The conversion instructions multiply by the scale, whose byte they take
// from a float32's exponent field (byte 0 is 2^-127 to them and 255 a NaN, as in the format), and round once to the output's type.
template <class T, int FMT> __device__ __forceinline__ Words<T> decode8(uint2 c, int sbyte) {
    const float s = bits_f32((uint32_t)sbyte << 23);
    Words<T> r;
#define MX_PAIR(k, word, sel4, sel8)                                                                                                              \
    if constexpr (sizeof(T) == 4) {                                                                                                               \
        const f32x2 p = FMT == E2M1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, s, sel4) : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, s, sel8); \
        r.w[2 * k] = f32_bits(p[0]); r.w[2 * k + 1] = f32_bits(p[1]);                                                                              \
    } else if constexpr (__is_same(T, _Float16))                                                                                                   \
        r.w[k] = __builtin_bit_cast(uint32_t, FMT == E2M1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c.x, s, sel4) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, s, sel8)); \
    else                                                                                                                                          \
        r.w[k] = __builtin_bit_cast(uint32_t, FMT == E2M1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c.x, s, sel4) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, s, sel8));
    MX_PAIR(0, c.x, 0, false)
    MX_PAIR(1, c.x, 1, true)
    MX_PAIR(2, c.y, 2, false)
    MX_PAIR(3, c.y, 3, true)
#undef MX_PAIR
    return r;
}

}  // namespace mx

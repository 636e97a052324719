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
// VEC: the address is 16-byte aligned and all 8 exist (the caller's rule); otherwise element by element, zeros behind the end.
template <class T, bool VEC> __device__ __forceinline__ void load8(const T *p, int have, float (&v)[8]) {
    if (VEC) {
        struct alignas(16) Pack { T e[16 / sizeof(T)]; };
#pragma unroll
        for (int k = 0; k < (int)(8 * sizeof(T) / 16); ++k) {
            const Pack q = reinterpret_cast<const Pack *>(p)[k];
#pragma unroll
            for (int e = 0; e < (int)(16 / sizeof(T)); ++e) v[k * (int)(16 / sizeof(T)) + e] = to_f32(q.e[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < have ? to_f32(p[e]) : 0.0f;
    }
}
template <class T, bool VEC> __device__ __forceinline__ void store8(T *p, int have, const float (&v)[8]) {
    if (VEC) {
        struct alignas(16) Pack { T e[16 / sizeof(T)]; };
#pragma unroll
        for (int k = 0; k < (int)(8 * sizeof(T) / 16); ++k) {
            Pack q;
#pragma unroll
            for (int e = 0; e < (int)(16 / sizeof(T)); ++e) q.e[e] = from_f32<T>(v[k * (int)(16 / sizeof(T)) + e]);
            reinterpret_cast<Pack *>(p)[k] = q;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (e < have) p[e] = from_f32<T>(v[e]);
    }
}

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
        for (int e = 0; e < 8; ++e) w[e] = fminf(fmaxf(v[e], -448.0f), 448.0f);
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
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    sbyte = scale_byte<FMT>(top);
    const float inv = scale_inverse(sbyte == 255 ? 254 : sbyte);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = sbyte == 255 ? 0.0f : v[e] * inv;
    return encode8<FMT>(w);
}

// ---- decoding -----------------------------------------------------------------------------------------------------------------
// The code's exponent and fraction bits, put where a float32 has its own, are the value times 2^-126 (E2M1) or 2^-120 (E4M3),
// subnormal codes included; two exact products give the value.
template <int FMT> __device__ __forceinline__ float decode1(uint32_t c) {
    if (FMT == E2M1) return bits_f32(((c & 7u) << 22) | ((c & 8u) << 28)) * bits_f32((126u + 127u) << 23);
    const float v = bits_f32(((c & 127u) << 20) | ((c & 128u) << 24)) * bits_f32((120u + 127u) << 23);
    return (c & 127u) == 127u ? bits_f32(0x7fc00000u) : v;
}
__device__ __forceinline__ float scale_value(int s) { return s == 255 ? bits_f32(0x7fc00000u) : bits_f32(s == 0 ? 0x00400000u : (uint32_t)s << 23); }

}  // namespace mx

// mx.hip -- microscaled feature rows: quantisation to 4 or 8 bits with a scale per 32 elements, decoding, the root-mean-square norm
// (with the residual's addition) that writes such rows, and their product on the matrix cores.  mx_math.h holds the format.
#include "mx_math.h"

namespace {

using namespace mx;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// ---- quantisation: one thread per 8 elements, four lanes per block ------------------------------------------------------------
template <class T, int FMT, bool VEC>
__global__ __launch_bounds__(256) void k_mx_quantize(const T *__restrict__ x, long ldx, int n, int d, uint8_t *__restrict__ codes,
                                                     uint8_t *__restrict__ scales) {
    const int row8 = (int)(padded(d) / 8);                     // threads per row, a multiple of 16: a block's four lanes stay together
    const long total = (long)n * row8;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long)gridDim.x * 256) {
        const long i = t / row8;
        const int c = (int)(t - i * row8), k = c * 8;
        float v[8] = {};
        if (k < d) {
            if (VEC && k + 8 <= d) load8<T, true>(x + i * ldx + k, 8, v);
            else load8<T, false>(x + i * ldx + k, d - k, v);
        }
        int s;
        const uint2 q = encode_block<FMT>(v, s);
        if (FMT == E2M1) *reinterpret_cast<uint32_t *>(codes + t * 4) = q.x;
        else *reinterpret_cast<uint2 *>(codes + t * 8) = q;
        if ((c & 3) == 0) scales[t >> 2] = (uint8_t)s;
    }
}

template <class T, int FMT, bool VEC>
__global__ __launch_bounds__(256) void k_mx_dequantize(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, int n, int d,
                                                       T *__restrict__ out, long ldo) {
    const int row8 = (int)(padded(d) / 8);
    const long total = (long)n * row8;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long)gridDim.x * 256) {
        const long i = t / row8;
        const int c = (int)(t - i * row8), k = c * 8;
        if (k >= d) continue;
        const float s = scale_value(scales[t >> 2]);
        uint2 q;
        if (FMT == E2M1) q.x = *reinterpret_cast<const uint32_t *>(codes + t * 4);
        else q = *reinterpret_cast<const uint2 *>(codes + t * 8);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t code = FMT == E2M1 ? (q.x >> (4 * e)) & 15u : ((e < 4 ? q.x : q.y) >> (8 * (e & 3))) & 255u;
            v[e] = decode1<FMT>(code) * s;
        }
        if (VEC && k + 8 <= d) store8<T, true>(out + i * ldo + k, 8, v);
        else store8<T, false>(out + i * ldo + k, d - k, v);
    }
}

// ---- root-mean-square norm: one workgroup per row -----------------------------------------------------------------------------
template <class T> struct NormArgs {
    const T *x, *residual, *weight;
    T *sum, *y;
    long ldx, ldr, lds, ldy;
    int n, d;
    float eps;
    uint8_t *codes, *scales;
};

template <class T, bool VEC> __device__ __forceinline__ void norm_load(const NormArgs<T> &a, long i, int k, bool from_sum, float (&h)[8]) {
    const int have = a.d - k;
    const bool full = VEC && have >= 8;
    if (from_sum) {
        if (full) load8<T, true>(a.sum + i * a.lds + k, 8, h); else load8<T, false>(a.sum + i * a.lds + k, have, h);
        return;
    }
    if (full) load8<T, true>(a.x + i * a.ldx + k, 8, h); else load8<T, false>(a.x + i * a.ldx + k, have, h);
    if (!a.residual) return;
    float r[8];
    if (full) load8<T, true>(a.residual + i * a.ldr + k, 8, r); else load8<T, false>(a.residual + i * a.ldr + k, have, r);
    // the sum is rounded to its stored type first and normalised from there: whoever reads it back gets the same row
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = to_f32(from_f32<T>(h[e] + r[e]));
}

// FMT: E2M1, E4M3, or -1 (no quantised output)
template <class T, int FMT, bool VEC>
__global__ __launch_bounds__(256) void k_rms_norm(NormArgs<T> a) {
    __shared__ float part[4];
    const long i = blockIdx.x;
    const int width = (int)padded(a.d);
    float ss = 0.0f;
    for (int k = threadIdx.x * 8; k < a.d; k += 2048) {
        float h[8];
        norm_load<T, VEC>(a, i, k, false, h);
        if (a.sum) { if (VEC && k + 8 <= a.d) store8<T, true>(a.sum + i * a.lds + k, 8, h); else store8<T, false>(a.sum + i * a.lds + k, a.d - k, h); }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(h[e], h[e], ss);
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) ss += __shfl_xor(ss, m);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = (part[0] + part[1]) + (part[2] + part[3]);
    const float inv = 1.0f / sqrtf(ss / (float)a.d + a.eps);
    for (int k = threadIdx.x * 8; k < width; k += 2048) {
        float h[8] = {};
        if (k < a.d) {
            norm_load<T, VEC>(a, i, k, a.sum != nullptr, h);
            float w[8];
            if (a.weight) { if (VEC && k + 8 <= a.d) load8<T, true>(a.weight + k, 8, w); else load8<T, false>(a.weight + k, a.d - k, w); }
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = a.weight ? h[e] * inv * w[e] : h[e] * inv;
            if (!(VEC && k + 8 <= a.d)) {                       // behind the end: zeros, whatever inv is
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = k + e < a.d ? h[e] : 0.0f;
            }
            if (a.y) { if (VEC && k + 8 <= a.d) store8<T, true>(a.y + i * a.ldy + k, 8, h); else store8<T, false>(a.y + i * a.ldy + k, a.d - k, h); }
        }
        if (FMT >= 0) {
            int s;
            const uint2 q = encode_block<FMT == E2M1 ? E2M1 : E4M3>(h, s);
            const long t = (i * width + k) / 8;
            if (FMT == E2M1) *reinterpret_cast<uint32_t *>(a.codes + t * 4) = q.x;
            else *reinterpret_cast<uint2 *>(a.codes + t * 8) = q;
            if ((threadIdx.x & 3) == 0) a.scales[t >> 2] = (uint8_t)s;
        }
    }
}

// ---- product: out[i][j] = alpha * <A row i, B row j> --------------------------------------------------------------------------
// v_mfma_scale_f32_16x16x128_f8f6f4 takes the codes and the scale bytes as they are held.  Lane l supplies row l & 15; of the 128
// elements, an E2M1 operand's lane group g = l >> 4 holds elements 32 g .. 32 g + 31 (16 bytes), an E4M3 operand's holds elements
// 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15; the scale byte of lane group g is that of elements 32 g .. 32 g + 31 for both.
// B's rows go in as the instruction's first operand: a lane then receives four consecutive columns j of one row i.
struct ProductArgs {
    const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
    int n, m, steps;                     // steps of 128 elements
    float alpha;
    int floor_zero;
    void *out;
    int out_dtype;
    long ld;
    int out_vec;                         // 4 consecutive outputs may be stored as one vector (alignment of out and ld)
};

template <int FMT> __device__ __forceinline__ v8i load_fragment(const uint8_t *row, int step, int g) {
    v8i f = {};
    if (FMT == E2M1) {
        const v4i lo = *reinterpret_cast<const v4i *>(row + (long)step * 64 + g * 16);
        f[0] = lo[0]; f[1] = lo[1]; f[2] = lo[2]; f[3] = lo[3];
    } else {
        const v4i lo = *reinterpret_cast<const v4i *>(row + (long)step * 128 + g * 16);
        const v4i hi = *reinterpret_cast<const v4i *>(row + (long)step * 128 + 64 + g * 16);
        f[0] = lo[0]; f[1] = lo[1]; f[2] = lo[2]; f[3] = lo[3];
        f[4] = hi[0]; f[5] = hi[1]; f[6] = hi[2]; f[7] = hi[3];
    }
    return f;
}
template <int FMT> constexpr int mfma_code() { return FMT == E2M1 ? 4 : 0; }      // the instruction's format selectors

template <class T> __device__ __forceinline__ void store_out4(T *p, int have, bool vec, const float (&v)[4]) {
    if (vec && have >= 4) {
        struct alignas(sizeof(T) * 4) Pack { T e[4]; } q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q.e[e] = from_f32<T>(v[e]);
        *reinterpret_cast<Pack *>(p) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < have) p[e] = from_f32<T>(v[e]);
    }
}
// four consecutive columns j .. j + 3 of row i
__device__ __forceinline__ void epilogue4(const ProductArgs &p, long i, int j, v4f acc) {
    if (i >= p.n || j >= p.m) return;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = acc[e] * p.alpha;
        if (p.floor_zero) v[e] = v[e] < 0.0f ? 0.0f : v[e];       // (a NaN stays one)
    }
    const long at = i * p.ld + j;
    const int have = p.m - j;
    if (p.out_dtype == BTS_F32) store_out4(static_cast<float *>(p.out) + at, have, p.out_vec, v);
    else if (p.out_dtype == BTS_F16) store_out4(static_cast<_Float16 *>(p.out) + at, have, p.out_vec, v);
    else store_out4(static_cast<bf16 *>(p.out) + at, have, p.out_vec, v);
}

// A workgroup of KW wavefronts computes a (16 RT) x (16 CT) tile; each wavefront takes a contiguous part of the row, straight from
// memory to registers, and the parts are added through LDS in a fixed order.
template <int FA, int FB, int RT, int CT, int KW>
__global__ __launch_bounds__(64 * KW) void k_mx_direct(ProductArgs p) {
    __shared__ v4f part[KW > 1 ? KW - 1 : 1][RT * CT][64];
    const int tiles_n = (p.m + 16 * CT - 1) / (16 * CT);
    const int ti = (int)(blockIdx.x / (unsigned)tiles_n), tj = (int)(blockIdx.x % (unsigned)tiles_n);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const uint8_t *ac[RT], *as[RT], *bc[CT], *bs[CT];
    const long step_a = FA == E2M1 ? 64 : 128, step_b = FB == E2M1 ? 64 : 128;
#pragma unroll
    for (int u = 0; u < RT; ++u) {                                 // rows behind the last one read the last one; never stored
        const long i = min((long)ti * 16 * RT + 16 * u + r, (long)p.n - 1);
        ac[u] = p.a_codes + i * p.steps * step_a; as[u] = p.a_scales + i * p.steps * 4 + g;
    }
#pragma unroll
    for (int u = 0; u < CT; ++u) {
        const long j = min((long)tj * 16 * CT + 16 * u + r, (long)p.m - 1);
        bc[u] = p.b_codes + j * p.steps * step_b; bs[u] = p.b_scales + j * p.steps * 4 + g;
    }
    v4f acc[RT][CT];
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int w = 0; w < CT; ++w) acc[u][w] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int per = (p.steps + KW - 1) / KW, s0 = wave * per, s1 = min(p.steps, s0 + per);
    for (int s = s0; s < s1; ++s) {
        v8i fa[RT], fb[CT];
        int sa[RT], sb[CT];
#pragma unroll
        for (int u = 0; u < RT; ++u) { fa[u] = load_fragment<FA>(ac[u], s, g); sa[u] = as[u][(long)s * 4]; }
#pragma unroll
        for (int w = 0; w < CT; ++w) { fb[w] = load_fragment<FB>(bc[w], s, g); sb[w] = bs[w][(long)s * 4]; }
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
            for (int w = 0; w < CT; ++w)
                acc[u][w] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[w], fa[u], acc[u][w], mfma_code<FB>(), mfma_code<FA>(), 0, sb[w], 0, sa[u]);
    }
    if (KW > 1) {
        if (wave > 0) {
#pragma unroll
            for (int u = 0; u < RT; ++u)
#pragma unroll
                for (int w = 0; w < CT; ++w) part[wave - 1][u * CT + w][lane] = acc[u][w];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int q = 0; q < KW - 1; ++q)
#pragma unroll
            for (int u = 0; u < RT; ++u)
#pragma unroll
                for (int w = 0; w < CT; ++w) acc[u][w] += part[q][u * CT + w][lane];
    }
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int w = 0; w < CT; ++w) epilogue4(p, (long)ti * 16 * RT + 16 * u + r, tj * 16 * CT + 16 * w + 4 * g, acc[u][w]);
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
bool known_format(int f) { return f == BTS_MX_E2M1 || f == BTS_MX_E4M3; }
bool known_dtype(int t) { return t == BTS_F32 || t == BTS_F16 || t == BTS_BF16; }
size_t dtype_bytes(int t) { return t == BTS_F32 ? 4 : 2; }
bool aligned(const void *p, size_t to) { return (uintptr_t)p % to == 0; }
int row_grid(const bts_context *ctx, int n, int d) {           // workgroups of 256 threads, one thread per 8 elements
    const long blocks = ((long)n * (padded(d) / 8) + 255) / 256, most = (long)ctx->n_cu * 64;
    return (int)(blocks < most ? blocks : most);
}

template <class T> int quantize(bts_context *ctx, const T *x, int ldx, int n, int d, int format, uint8_t *codes, uint8_t *scales, hipStream_t st) {
    const bool vec = aligned(x, 16) && (size_t)ldx * sizeof(T) % 16 == 0;
    const dim3 grid(row_grid(ctx, n, d)), block(256);
    if (format == E2M1) {
        if (vec) hipLaunchKernelGGL((k_mx_quantize<T, E2M1, true>), grid, block, 0, st, x, (long)ldx, n, d, codes, scales);
        else hipLaunchKernelGGL((k_mx_quantize<T, E2M1, false>), grid, block, 0, st, x, (long)ldx, n, d, codes, scales);
    } else {
        if (vec) hipLaunchKernelGGL((k_mx_quantize<T, E4M3, true>), grid, block, 0, st, x, (long)ldx, n, d, codes, scales);
        else hipLaunchKernelGGL((k_mx_quantize<T, E4M3, false>), grid, block, 0, st, x, (long)ldx, n, d, codes, scales);
    }
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

template <class T> int dequantize(bts_context *ctx, const uint8_t *codes, const uint8_t *scales, int format, int n, int d, T *out, int ldo, hipStream_t st) {
    const bool vec = aligned(out, 16) && (size_t)ldo * sizeof(T) % 16 == 0;
    const dim3 grid(row_grid(ctx, n, d)), block(256);
    if (format == E2M1) {
        if (vec) hipLaunchKernelGGL((k_mx_dequantize<T, E2M1, true>), grid, block, 0, st, codes, scales, n, d, out, (long)ldo);
        else hipLaunchKernelGGL((k_mx_dequantize<T, E2M1, false>), grid, block, 0, st, codes, scales, n, d, out, (long)ldo);
    } else {
        if (vec) hipLaunchKernelGGL((k_mx_dequantize<T, E4M3, true>), grid, block, 0, st, codes, scales, n, d, out, (long)ldo);
        else hipLaunchKernelGGL((k_mx_dequantize<T, E4M3, false>), grid, block, 0, st, codes, scales, n, d, out, (long)ldo);
    }
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

template <class T, int FMT> void rms_norm_launch(const NormArgs<T> &a, bool vec, hipStream_t st) {
    if (vec) hipLaunchKernelGGL((k_rms_norm<T, FMT, true>), dim3(a.n), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_rms_norm<T, FMT, false>), dim3(a.n), dim3(256), 0, st, a);
}
template <class T> int rms_norm(const void *x, int ldx, const void *residual, int ldr, const void *weight, int n, int d, float eps,
                                void *sum, int lds, void *y, int ldy, int format, uint8_t *codes, uint8_t *scales, hipStream_t st) {
    NormArgs<T> a;
    a.x = static_cast<const T *>(x); a.residual = static_cast<const T *>(residual); a.weight = static_cast<const T *>(weight);
    a.sum = static_cast<T *>(sum); a.y = static_cast<T *>(y);
    a.ldx = ldx; a.ldr = ldr; a.lds = lds; a.ldy = ldy; a.n = n; a.d = d; a.eps = eps; a.codes = codes; a.scales = scales;
    const auto fits = [](const void *p, long ld) { return !p || (aligned(p, 16) && (size_t)ld * sizeof(T) % 16 == 0); };
    const bool vec = fits(x, ldx) && fits(residual, ldr) && fits(weight, 0) && fits(sum, lds) && fits(y, ldy);
    if (format == E2M1) rms_norm_launch<T, E2M1>(a, vec, st);
    else if (format == E4M3) rms_norm_launch<T, E4M3>(a, vec, st);
    else rms_norm_launch<T, -1>(a, vec, st);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

template <int FA, int FB> int product(bts_context *ctx, const ProductArgs &p, hipStream_t st) {
    const long tiles = (((long)p.n + 31) / 32) * (((long)p.m + 31) / 32);
    BTS_REQUIRE(tiles < (1L << 31), "n * m: too many tiles for one launch");
    hipLaunchKernelGGL((k_mx_direct<FA, FB, 2, 2, 4>), dim3((unsigned)tiles), dim3(256), 0, st, p);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

}  // namespace

extern "C" {

int bts_mx_row_bytes(int format, int d, int64_t *code_bytes, int64_t *scale_bytes) {
    BTS_REQUIRE(known_format(format), "unknown format");
    BTS_REQUIRE(d > 0 && code_bytes && scale_bytes, "d, code_bytes, scale_bytes");
    *code_bytes = mx::code_bytes(format, d);
    *scale_bytes = mx::scale_bytes(d);
    return BTS_OK;
}

int bts_mx_quantize(bts_context *ctx, const void *x, int x_dtype, int ldx, int n, int d, int format, uint8_t *codes, uint8_t *scales,
                    bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && d > 0 && ldx >= d, "ctx, n, d, ldx < d");
    BTS_REQUIRE(known_format(format) && known_dtype(x_dtype), "unknown format / type");
    BTS_ON_DEVICE(ctx);
    if (n == 0) return BTS_OK;
    BTS_REQUIRE(x && codes && scales, "null pointer");
    BTS_REQUIRE(aligned(x, dtype_bytes(x_dtype)) && aligned(codes, 16) && aligned(scales, 4), "x: element, codes: 16-byte, scales: 4-byte alignment");
    hipStream_t st = (hipStream_t)stream;
    if (x_dtype == BTS_F32) return quantize(ctx, static_cast<const float *>(x), ldx, n, d, format, codes, scales, st);
    if (x_dtype == BTS_F16) return quantize(ctx, static_cast<const _Float16 *>(x), ldx, n, d, format, codes, scales, st);
    return quantize(ctx, static_cast<const bf16 *>(x), ldx, n, d, format, codes, scales, st);
}

int bts_mx_dequantize(bts_context *ctx, const uint8_t *codes, const uint8_t *scales, int format, int n, int d, void *out, int out_dtype,
                      int ldo, bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && d > 0 && ldo >= d, "ctx, n, d, ldo < d");
    BTS_REQUIRE(known_format(format) && known_dtype(out_dtype), "unknown format / type");
    BTS_ON_DEVICE(ctx);
    if (n == 0) return BTS_OK;
    BTS_REQUIRE(out && codes && scales, "null pointer");
    BTS_REQUIRE(aligned(out, dtype_bytes(out_dtype)) && aligned(codes, 16) && aligned(scales, 4), "out: element, codes: 16-byte, scales: 4-byte alignment");
    hipStream_t st = (hipStream_t)stream;
    if (out_dtype == BTS_F32) return dequantize(ctx, codes, scales, format, n, d, static_cast<float *>(out), ldo, st);
    if (out_dtype == BTS_F16) return dequantize(ctx, codes, scales, format, n, d, static_cast<_Float16 *>(out), ldo, st);
    return dequantize(ctx, codes, scales, format, n, d, static_cast<bf16 *>(out), ldo, st);
}

int bts_rms_norm(bts_context *ctx, int dtype, const void *x, int ldx, const void *residual, int ldr, const void *weight, int n, int d,
                 double eps, void *sum, int lds, void *y, int ldy, int format, uint8_t *codes, uint8_t *scales, bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && d > 0 && ldx >= d, "ctx, n, d, ldx < d");
    BTS_REQUIRE(known_dtype(dtype), "unknown type");
    BTS_REQUIRE((float)eps > 0.0f && (float)eps <= 3.0e38f, "eps must be a positive finite float32");
    BTS_REQUIRE(!residual || ldr >= d, "ldr < d");
    BTS_REQUIRE(!sum || lds >= d, "lds < d");
    BTS_REQUIRE(!y || ldy >= d, "ldy < d");
    BTS_REQUIRE(!y || (y != sum && y != weight), "y may not be sum or weight");
    BTS_REQUIRE(!sum || sum != weight, "sum may not be weight");
    BTS_REQUIRE(!sum || ((sum != x || lds == ldx) && (sum != residual || lds == ldr)), "sum in the place of x / residual needs their row stride");
    BTS_REQUIRE(!y || ((y != x || ldy == ldx) && (y != residual || ldy == ldr)), "y in the place of x / residual needs their row stride");
    BTS_ON_DEVICE(ctx);
    if (n == 0) return BTS_OK;
    BTS_REQUIRE(x, "null pointer");
    BTS_REQUIRE(!codes == !scales, "codes and scales come together");
    BTS_REQUIRE(!codes || known_format(format), "unknown format");
    BTS_REQUIRE(codes || y, "nothing to write: codes and y are both null");
    const size_t b = dtype_bytes(dtype);
    BTS_REQUIRE(aligned(x, b) && aligned(residual, b) && aligned(weight, b) && aligned(sum, b) && aligned(y, b), "element alignment");
    BTS_REQUIRE(aligned(codes, 16) && aligned(scales, 4), "codes: 16-byte, scales: 4-byte alignment");
    hipStream_t st = (hipStream_t)stream;
    const int f = codes ? format : -1;
    if (dtype == BTS_F32) return rms_norm<float>(x, ldx, residual, ldr, weight, n, d, (float)eps, sum, lds, y, ldy, f, codes, scales, st);
    if (dtype == BTS_F16) return rms_norm<_Float16>(x, ldx, residual, ldr, weight, n, d, (float)eps, sum, lds, y, ldy, f, codes, scales, st);
    return rms_norm<bf16>(x, ldx, residual, ldr, weight, n, d, (float)eps, sum, lds, y, ldy, f, codes, scales, st);
}

int bts_mx_product(bts_context *ctx, const uint8_t *a_codes, const uint8_t *a_scales, int a_format, int n, const uint8_t *b_codes,
                   const uint8_t *b_scales, int b_format, int m, int d, double alpha, int floor_zero, void *out, int out_dtype, int ld,
                   bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && m >= 0 && d > 0 && ld >= m, "ctx, n, m, d, ld < m");
    BTS_REQUIRE(known_format(a_format) && known_format(b_format) && known_dtype(out_dtype), "unknown format / type");
    BTS_REQUIRE(out_dtype != BTS_F32 || (a_format == E2M1 && b_format == E2M1),
                "a float32 output needs two E2M1 operands (products with an E4M3 operand carry about 16 bits)");
    BTS_ON_DEVICE(ctx);
    if (n == 0 || m == 0) return BTS_OK;
    BTS_REQUIRE(a_codes && a_scales && b_codes && b_scales && out, "null pointer");
    BTS_REQUIRE(aligned(a_codes, 16) && aligned(b_codes, 16) && aligned(a_scales, 4) && aligned(b_scales, 4) && aligned(out, dtype_bytes(out_dtype)),
                "codes: 16-byte, scales: 4-byte, out: element alignment");
    const size_t b = dtype_bytes(out_dtype);
    ProductArgs p;
    p.a_codes = a_codes; p.a_scales = a_scales; p.b_codes = b_codes; p.b_scales = b_scales;
    p.n = n; p.m = m; p.steps = (int)(padded(d) / MX_ROW);
    p.alpha = (float)alpha; p.floor_zero = floor_zero != 0;
    p.out = out; p.out_dtype = out_dtype; p.ld = ld;
    p.out_vec = aligned(out, 4 * b) && ld % 4 == 0;
    hipStream_t st = (hipStream_t)stream;
    if (a_format == E2M1) return b_format == E2M1 ? product<E2M1, E2M1>(ctx, p, st) : product<E2M1, E4M3>(ctx, p, st);
    return b_format == E2M1 ? product<E4M3, E2M1>(ctx, p, st) : product<E4M3, E4M3>(ctx, p, st);
}

}  // extern "C"

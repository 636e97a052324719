// mx.hip -- microscaled feature rows: quantisation to 4 or 8 bits with a scale per 32 elements, decoding, the root-mean-square norm
// (with the residual's addition) that writes such rows, and their product on the matrix cores.  mx_math.h holds the format.
#include "mx_math.h"

#include <algorithm>

namespace {

using namespace mx;

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// ---- quantisation and back: one thread per 8 elements, four lanes per block, 16 lanes per 128 padded elements ------------------
// Groups of 16 lanes walk the 128-element pieces of all rows (their number fits 32 bits: the host's check).  Memory bounds both ways:
// 65536 x 2048 bfloat16 to E2M1, 340 MB, in 77 us (4.4 TB/s), back in 59 us (5.7 TB/s, the codes still in the last-level cache).
template <class T, int FMT>
__global__ __launch_bounds__(256) void k_mx_quantize(const T *__restrict__ x, long ldx, uint32_t pieces, uint32_t row_pieces, int d,
                                                     uint8_t *__restrict__ codes, uint8_t *__restrict__ scales) {
    const int lane16 = threadIdx.x & 15;
    for (uint32_t q = blockIdx.x * 16 + (threadIdx.x >> 4); q < pieces; q += gridDim.x * 16) {
        const uint32_t i = q / row_pieces;
        const int k = (int)(q - i * row_pieces) * 128 + lane16 * 8;
        float v[8] = {};
        if (k < d) load8(x + i * ldx + k, d - k, v);
        int s;
        const uint2 c = encode_block<FMT>(v, s);
        const size_t t = (size_t)q * 16 + lane16;
        if (FMT == E2M1) *reinterpret_cast<uint32_t *>(codes + t * 4) = c.x;
        else *reinterpret_cast<uint2 *>(codes + t * 8) = c;
        if ((lane16 & 3) == 0) scales[t >> 2] = (uint8_t)s;
    }
}

template <class T, int FMT>
__global__ __launch_bounds__(256) void k_mx_dequantize(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, uint32_t pieces,
                                                       uint32_t row_pieces, int d, T *__restrict__ out, long ldo) {
    const int lane16 = threadIdx.x & 15;
    for (uint32_t q = blockIdx.x * 16 + (threadIdx.x >> 4); q < pieces; q += gridDim.x * 16) {
        const uint32_t i = q / row_pieces;
        const int k = (int)(q - i * row_pieces) * 128 + lane16 * 8;
        if (k >= d) continue;
        const size_t t = (size_t)q * 16 + lane16;
        uint2 c = {0, 0};
        if (FMT == E2M1) c.x = *reinterpret_cast<const uint32_t *>(codes + t * 4);
        else c = *reinterpret_cast<const uint2 *>(codes + t * 8);
        store_words<T>(out + i * ldo + k, d - k, decode8<T, FMT>(c, scales[t >> 2]));
    }
}

// ---- root-mean-square norm -----------------------------------------------------------------------------------------------------
template <class T> struct NormArgs {
    const T *x, *residual, *weight;
    T *sum, *y;
    long ldx, ldr, lds, ldy;
    int n, d;
    long first;                          // the launch's first row
    double eps;
    int format;                          // -1: no quantised output
    uint8_t *codes, *scales;
};

// WHOLE: d is a multiple of 8, so every piece is (the tails' code, five times a piece, is most of the kernel otherwise)
template <class T, bool WHOLE> __device__ __forceinline__ void norm_load(const NormArgs<T> &a, long i, int k, float (&h)[8]) {
    const int have = WHOLE ? 8 : a.d - k;
    load8(a.x + i * a.ldx + k, have, h);
    if (!a.residual) return;
    float r[8];
    load8(a.residual + i * a.ldr + k, have, r);
    // the sum is rounded to its stored type first and normalised from there: whoever reads it back gets the same row
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] += r[e];
    round8<T>(h);
}
// 8 squares in float32 (each product of 16-bit values is exact), the row's sum in float64: the factor of a row is common to all of its
// elements, and a factor that is off by a few roundings turns that many codes at the borders between two values.  Squares that leave
// float32's range at either end are taken in float64.
__device__ __forceinline__ double squares(const float (&h)[8]) {
    const float s = ((h[0] * h[0] + h[1] * h[1]) + (h[2] * h[2] + h[3] * h[3])) + ((h[4] * h[4] + h[5] * h[5]) + (h[6] * h[6] + h[7] * h[7]));
    if (s > 1e-30f && s < 3e38f) return (double)s;
    double t = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) t += (double)h[e] * (double)h[e];
    return t;
}
// A row's factor as m * 2^e, m in [1, 2).  With a weight the elements are taken times 2^e first, so that their product with the weight is the
// result but for m: it leaves float32's range only where the result does, however far the row's norm and the weight lie from 1 (a row
// of 2^50 under a weight of 2^100).  Powers of two are exact, and for 16-bit types so is the product: one rounding follows that of the
// factor.  The multiplication hides behind memory: 32768 x 4096 bfloat16 with residual and weight 164 us with and without it, 32768 x
// 1111 float32 47.  Without a weight 2^e is apart only where the factor is subnormal.
struct Factor { float m, power; };
__device__ __forceinline__ Factor row_factor(double ss, int d, double eps, bool weight) {
    const double full = 1.0 / sqrt(ss / (double)d + eps);
    const float inv = (float)full;
    if (!weight && inv >= 0x1p-126f) return {inv, 1.0f};
    if (!(full >= 0x1p-130)) return {inv, inv};        // (a row with an infinity, 0, or a NaN)
    int e;
    const float m = (float)(2.0 * frexp(full, &e));    // (2 if it rounds up to that)
    return {m, ldexpf(1.0f, e - 1)};
}
// the normalised piece at column k: to y, and as codes (whole blocks: a block's four lanes come together)
template <class T, bool WHOLE> __device__ __forceinline__ void norm_emit(const NormArgs<T> &a, long i, int k, int width, Factor f, float (&h)[8]) {
    if (k < a.d) {
        const int have = WHOLE ? 8 : a.d - k;
        if (f.power != 1.0f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] *= f.power;
        }
        if (a.weight) {
            float w[8];
            load8(a.weight + k, have, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] *= w[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = WHOLE || e < have ? h[e] * f.m : 0.0f;
        if (a.y) store8(a.y + i * a.ldy + k, have, h);
    }
    if (a.format < 0) return;
    int s;
    const size_t t = ((size_t)i * width + k) / 8;
    if (a.format == E2M1) *reinterpret_cast<uint32_t *>(a.codes + t * 4) = encode_block<E2M1>(h, s).x;
    else *reinterpret_cast<uint2 *>(a.codes + t * 8) = encode_block<E4M3>(h, s);
    if ((threadIdx.x & 3) == 0) a.scales[t >> 2] = (uint8_t)s;
}

// TPR threads per row, CH pieces of 8 elements a thread: the row stays in registers between the sum and the output, so x and residual
// are read once.  CH = 0: rows beyond 8192 elements, in two passes; the second reads the stored sum, or x and residual again.
// One pass over memory bounds it: 32768 x 4096 bfloat16 with residual and weight, 0.94 GB in 164 us (5.7 TB/s; 178 between decodings).
template <class T, int TPR, int CH, bool WHOLE>
__global__ __launch_bounds__(256) void k_rms_norm(NormArgs<T> a) {
    __shared__ double part[4];
    const long i = a.first + (long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const int width = (int)padded(a.d), first = (threadIdx.x % TPR) * 8;
    if (TPR == 64 && i >= a.n) return;
    float h[CH > 0 ? CH : 1][8];
    double ss = 0.0;
    if (CH > 0) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = first + c * TPR * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[c][e] = 0.0f;
            if (k < a.d) norm_load<T, WHOLE>(a, i, k, h[c]);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = first + c * TPR * 8;
            if (a.sum && k < a.d) store8(a.sum + i * a.lds + k, WHOLE ? 8 : a.d - k, h[c]);
            ss += squares(h[c]);
        }
    } else {
        for (int k = first; k < a.d; k += TPR * 8) {
            norm_load<T, WHOLE>(a, i, k, h[0]);
            if (a.sum) store8(a.sum + i * a.lds + k, WHOLE ? 8 : a.d - k, h[0]);
            ss += squares(h[0]);
        }
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) ss += __shfl_xor(ss, m);
    if (TPR == 256) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = (part[0] + part[1]) + (part[2] + part[3]);
    }
    const Factor f = row_factor(ss, a.d, a.eps, a.weight != nullptr);
    if (CH > 0) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int k = first + c * TPR * 8;
            if (k < width) norm_emit<T, WHOLE>(a, i, k, width, f, h[c]);
        }
    } else {
        for (int k = first; k < width; k += TPR * 8) {
            if (k >= a.d) {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[0][e] = 0.0f;
            } else if (a.sum) load8(a.sum + i * a.lds + k, WHOLE ? 8 : a.d - k, h[0]);
            else norm_load<T, WHOLE>(a, i, k, h[0]);
            norm_emit<T, WHOLE>(a, i, k, width, f, h[0]);
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
    int first;                           // the launch's first tile
    float alpha;
    int floor_zero;
    void *out;
    int out_dtype;
    long ld;
    int out_vec;                         // rows may be stored 16 bytes at a time (alignment of out and ld)
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
template <int FMT> constexpr int MFMA_CODE = FMT == E2M1 ? 4 : 0;      // the instruction's format selectors

// acc += B fragment x A fragment, scale byte OB of sb and OA of sa
template <int FA, int FB, int OA, int OB> __device__ __forceinline__ v4f mma(v8i fb, v8i fa, v4f acc, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa, acc, (MFMA_CODE<FB>), (MFMA_CODE<FA>), OB, sb, OA, sa);
}
// (the byte selectors are immediates: the cases fold away in unrolled loops)
template <int FA, int FB, int OA> __device__ __forceinline__ v4f mma_b(v8i fb, v8i fa, v4f acc, int sb, int ob, int sa) {
    switch (ob & 3) {
        case 0: return mma<FA, FB, OA, 0>(fb, fa, acc, sb, sa);
        case 1: return mma<FA, FB, OA, 1>(fb, fa, acc, sb, sa);
        case 2: return mma<FA, FB, OA, 2>(fb, fa, acc, sb, sa);
        default: return mma<FA, FB, OA, 3>(fb, fa, acc, sb, sa);
    }
}
template <int FA, int FB> __device__ __forceinline__ v4f mma_bytes(v8i fb, v8i fa, v4f acc, int sb, int ob, int sa, int oa) {
    switch (oa & 3) {
        case 0: return mma_b<FA, FB, 0>(fb, fa, acc, sb, ob, sa);
        case 1: return mma_b<FA, FB, 1>(fb, fa, acc, sb, ob, sa);
        case 2: return mma_b<FA, FB, 2>(fb, fa, acc, sb, ob, sa);
        default: return mma_b<FA, FB, 3>(fb, fa, acc, sb, ob, sa);
    }
}

// the factor and the floor of N results (a NaN stays one)
template <int N> __device__ __forceinline__ void finish(const ProductArgs &p, float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] *= p.alpha;
    if (p.floor_zero) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = v[e] < 0.0f ? 0.0f : v[e];
    }
}
// four consecutive columns j .. j + 3 of row i, element by element
template <class T> __device__ __forceinline__ void epilogue4(const ProductArgs &p, long i, long j, v4f acc) {
    if (i >= p.n) return;
    float v[4] = {acc[0], acc[1], acc[2], acc[3]};
    finish(p, v);
    T *const to = static_cast<T *>(p.out) + i * p.ld + j;
#pragma unroll
    for (int e = 0; e < 4; ++e) if (j + e < p.m) to[e] = from_f32<T>(v[e]);
}

// A workgroup of 4 wavefronts computes one 16 x 16 tile straight from memory; each wavefront takes a quarter of the row, and the parts are
// added through LDS in a fixed order.  For few tiles, where the length of a row is what takes time (1 x 2000 x 2048: 3.4 us against 5.1
// with LDS tiles; 1 x 300 x 8192: 6.6 against 12.2), and for sizes beyond the tiles' 32-bit offsets.
template <int FA, int FB>
__global__ __launch_bounds__(256) void k_mx_direct(ProductArgs p) {
    __shared__ v4f part[3][64];
    const long tiles_n = ((long)p.m + 15) / 16, tile = (long)p.first + blockIdx.x, ti = tile / tiles_n, tj = tile % tiles_n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const long i = min(ti * 16 + r, (long)p.n - 1), j = min(tj * 16 + r, (long)p.m - 1);      // (rows behind the last one read it; never stored)
    const uint8_t *ac = p.a_codes + i * p.steps * (FA == E2M1 ? 64 : 128), *as = p.a_scales + i * p.steps * 4 + g;
    const uint8_t *bc = p.b_codes + j * p.steps * (FB == E2M1 ? 64 : 128), *bs = p.b_scales + j * p.steps * 4 + g;
    const int per = (p.steps + 3) / 4, s0 = wave * per, s1 = min(p.steps, s0 + per);
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = s0; s < s1; ++s)
        acc = mma<FA, FB, 0, 0>(load_fragment<FB>(bc, s, g), load_fragment<FA>(ac, s, g), acc, bs[(long)s * 4], as[(long)s * 4]);
    if (wave > 0) part[wave - 1][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    acc = ((acc + part[0][lane]) + part[1][lane]) + part[2][lane];
    if (p.out_dtype == BTS_F32) epilogue4<float>(p, ti * 16 + r, tj * 16 + 4 * g, acc);
    else if (p.out_dtype == BTS_F16) epilogue4<_Float16>(p, ti * 16 + r, tj * 16 + 4 * g, acc);
    else epilogue4<bf16>(p, ti * 16 + r, tj * 16 + 4 * g, acc);
}

// XCD-aware order of the tiles: the 8 XCDs have an L2 each and take workgroups in turn, so every XCD gets a contiguous run of tiles, and a
// run goes down groups of 8 tile rows, column by column: the tiles that are in flight together share their A and B rows.
__device__ __forceinline__ void tile_of(int bid, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int all = tiles_m * tiles_n, q = all / 8, rest = all % 8, xcd = bid % 8, slot = bid / 8;
    const int v = (xcd < rest ? xcd * (q + 1) : rest * (q + 1) + (xcd - rest) * q) + slot;
    const int group = v / (8 * tiles_n), first = group * 8, rows = min(8, tiles_m - first), in = v - group * 8 * tiles_n;
    tm = first + in % rows;
    tn = in / rows;
}

// The rows of one tile as a bounded buffer: what lies behind the last row reads as zeros, so no load needs a clamped address.
struct TileRows {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ TileRows(const uint8_t *base, int row, int rows, int tile, int stride) {
        rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base + (long)row * stride), 0, min(tile, rows - row) * stride, 0x00020000);
    }
    __device__ __forceinline__ v4i load16(int at) const { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0)); }
    static constexpr int BEHIND = 0x7ffffff0;
    __device__ __forceinline__ uint32_t load4(int at) const { return __builtin_amdgcn_raw_buffer_load_b32(rsrc, at, 0, 0); }
};

// Lane l has the four scale bytes of row l; after this it has byte l >> 4 of the rows l & 15, that + 16, + 32 and + 48: those of its elements
// in four fragments.  (A 4 x 4 transposition of bytes over lanes 16 apart, so that they go to LDS a word at a time instead of four bytes:
// 4 % of the time of 10000 x 2000 x 8192.)
__device__ __forceinline__ uint32_t transpose_bytes(uint32_t w, int lane) {
    const auto far = __builtin_amdgcn_permlane32_swap(w, w, false, false);        // [0]: the word of the lane's pair with bit 5 clear, [1]: set
    w = __builtin_amdgcn_perm(far[1], far[0], lane & 32 ? 0x07060302u : 0x05040100u);
    const auto near = __builtin_amdgcn_permlane16_swap(w, w, false, false);       // ... bit 4
    return __builtin_amdgcn_perm(near[1], near[0], lane & 16 ? 0x07030501u : 0x06020400u);
}

// One operand of a stage: ROWS rows of SK instruction depths, moved by THREADS threads.  A row of a stage is C 16-byte chunks; chunk c of
// row r lies at c ^ swizzle(r), so that the 16 lanes that an LDS read serves at a time -- 16 rows of one chunk, or 8 rows of each of two
// neighbouring chunks -- are in 16 different 16-byte bank groups (no bank conflict counted; 4 cycles a read with rows / 4 in the
// 64-byte rows' swizzle instead of its negative).
template <int FMT, int ROWS, int THREADS, int SK> struct Operand {
    static constexpr int S1 = FMT == E2M1 ? 64 : 128, S = SK * S1;                // bytes a row: an instruction depth, a stage
    static constexpr int C = S / 16, STEP = THREADS / C;                         // chunks a row; rows between a thread's chunks
    static constexpr int MOVES = ROWS * C < THREADS ? 1 : ROWS * C / THREADS;    // chunks a thread moves (at most, if there are fewer than threads)
    static constexpr int PERIOD = STEP % 16 == 0 ? 1 : 16 / STEP;                // moves after which the swizzle repeats
    static constexpr int BYTES = ROWS * S;
    static_assert((MOVES * THREADS == ROWS * C || MOVES == 1) && MOVES % PERIOD == 0, "even staging");
    static __device__ __forceinline__ int swizzle(int row) { return (C >= 16 ? row : C == 8 ? row / 2 : -(row / 4)) & (C >= 16 ? 15 : C - 1); }
    int from, depth, to[PERIOD], frag[SK][S1 / 64];
    struct Regs { v4i chunk[MOVES]; };
    __device__ __forceinline__ void init(int tid, int first_row, int r, int g, int stride) {
        const int row = tid / C, c = tid % C;
        from = row * stride + c * 16;
        depth = c / (S1 / 16);
#pragma unroll
        for (int q = 0; q < PERIOD; ++q) to[q] = (row + q * STEP) * S + (c ^ swizzle(row + q * STEP)) * 16;
#pragma unroll
        for (int k = 0; k < SK; ++k)
#pragma unroll
            for (int h = 0; h < S1 / 64; ++h) frag[k][h] = (first_row + r) * S + ((k * (S1 / 16) + 4 * h + g) ^ swizzle(r)) * 16;
    }
    // depths behind the row's end are zeros (the buffer goes on there with the next row)
    __device__ __forceinline__ void load(Regs &x, const TileRows &rows, int stage, int stride, int steps) const {
        const uint32_t at = stage * SK + depth >= steps ? TileRows::BEHIND : from + stage * S;
#pragma unroll
        for (int q = 0; q < MOVES; ++q) x.chunk[q] = rows.load16((int)(at + q * STEP * stride));
    }
    __device__ __forceinline__ void store(const Regs &x, uint8_t *image) const {
#pragma unroll
        for (int q = 0; q < MOVES; ++q)
            if (MOVES * THREADS == ROWS * C || to[0] < BYTES) *reinterpret_cast<v4i *>(image + to[q % PERIOD] + (q / PERIOD) * PERIOD * STEP * S) = x.chunk[q];
    }
    // the fragment of the 16 rows `u` times 16 behind the wavefront's first one, depth k of the stage
    __device__ __forceinline__ v8i fragment(const uint8_t *image, int u, int k) const {
        v8i f = {};
        const v4i lo = *reinterpret_cast<const v4i *>(image + frag[k][0] + u * S * 16);
        f[0] = lo[0]; f[1] = lo[1]; f[2] = lo[2]; f[3] = lo[3];
        if (S1 == 128) {
            const v4i hi = *reinterpret_cast<const v4i *>(image + frag[k][S1 / 64 - 1] + u * S * 16);
            f[4] = hi[0]; f[5] = hi[1]; f[6] = hi[2]; f[7] = hi[3];
        }
        return f;
    }
};

// A wavefront's (16 RT) x (16 CT) results leave through its own 2 KB of LDS, 16 rows of 128 bytes at a time, so that whole 128-byte lines are
// stored (16 rows of 8 or 16 bytes a lane straight from the accumulators cost 1.5 us more a round of 256 x 256 bfloat16 tiles).  Chunk c
// of row r lies at c ^ r.  Rows that cannot be stored 16 bytes at a time go element by element, neighbours in neighbouring lanes.
template <class T, int RT, int CT>
__device__ __forceinline__ void write_tile(const ProductArgs &p, const v4f (&acc)[RT][CT], uint8_t *room, int i0, int j0, int lane) {
    constexpr int FRAGS = 8 / (int)sizeof(T) < CT ? 8 / (int)sizeof(T) : CT, COLS = FRAGS * 16, ROWB = COLS * (int)sizeof(T), CHUNKS = ROWB / 16;
    constexpr int ACROSS = 64 / CHUNKS < 16 ? 64 / CHUNKS : 16;                    // rows a store
    static_assert(CT % FRAGS == 0, "whole passes");
    const int r = lane & 15, g = lane >> 4, rows = p.n - i0, cols = p.m - j0, ld = (int)(p.ld * (long)sizeof(T));   // (bytes; the host's check)
    uint8_t *out = reinterpret_cast<uint8_t *>(static_cast<T *>(p.out) + (i0 * p.ld + j0));                   // the same in all lanes
    const int row8 = lane / CHUNKS, at8 = row8 * ld + (lane % CHUNKS) * 16;
#pragma unroll
    for (int u = 0; u < RT; ++u, out += 16 * p.ld * (long)sizeof(T))
#pragma unroll
        for (int w0 = 0; w0 < CT; w0 += FRAGS) {
            float v[FRAGS * 4];
#pragma unroll
            for (int e = 0; e < FRAGS * 4; ++e) v[e] = acc[u][w0 + e / 4][e % 4];
            finish(p, v);
#pragma unroll
            for (int w = 0; w < FRAGS; ++w) {
                const int at = (w * 16 + 4 * g) * (int)sizeof(T);
                uint8_t *const to = room + r * ROWB + ((at / 16) ^ (r & (CHUNKS - 1))) * 16 + at % 16;
                if constexpr (sizeof(T) == 4) *reinterpret_cast<v4f *>(to) = v4f{v[4 * w], v[4 * w + 1], v[4 * w + 2], v[4 * w + 3]};
                else *reinterpret_cast<uint2 *>(to) = uint2{pack2<T>(v[4 * w], v[4 * w + 1]), pack2<T>(v[4 * w + 2], v[4 * w + 3])};
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (p.out_vec && w0 * 16 + COLS <= cols) {
#pragma unroll
                for (int q = 0; q < 16 / ACROSS; ++q) {
                    const int row = q * ACROSS + row8;
                    if (64 / CHUNKS > 16 && row >= 16) break;
                    const v4i x = *reinterpret_cast<const v4i *>(room + row * ROWB + ((lane % CHUNKS) ^ (row & (CHUNKS - 1))) * 16);
                    if (u * 16 + row < rows) *reinterpret_cast<v4i *>(out + (uint32_t)(at8 + q * ACROSS * ld + w0 * 16 * (int)sizeof(T))) = x;
                }
            } else {
#pragma unroll 4
                for (int q = 0; q < 16 * COLS / 64; ++q) {
                    const int row = q * (64 / COLS) + lane / COLS, col = lane % COLS, at = col * (int)sizeof(T);
                    const T x = *reinterpret_cast<const T *>(room + row * ROWB + ((at / 16) ^ (row & (CHUNKS - 1))) * 16 + at % 16);
                    if (u * 16 + row < rows && w0 * 16 + col < cols) *reinterpret_cast<T *>(out + (uint32_t)(row * ld + (w0 * 16 + col) * (int)sizeof(T))) = x;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
}

// A workgroup of WM x WN wavefronts computes a TM x TN tile in stages of SK instruction depths of 128 elements.  A stage's codes and scale
// bytes go from memory through registers to one of two LDS images while the other is multiplied; the loads of AHEAD stages are in flight.
// (Fragments straight from memory would be 16 rows x 64 bytes a load with the lanes of a row 16 apart: a quarter of the load path's rate.)
// With 8 wavefronts (two a SIMD) the second four run one phase behind the first: while one of a SIMD's two wavefronts multiplies, the
// other fetches its fragments, stores the next stage and issues the loads of the one after; barriers keep the two in step.  With 4
// wavefronts a stage has one barrier, a depth's fragments are read while the one before it is multiplied (a fifth faster at 1000 x 1000 x
// 1000 than both in turn: 5.4 us), and the workgroups of a CU overlap.
// What bounds it: waiting.  128 x 128, E2M1 x E2M1, 10240 x 2048 x 8192, 129 us: the matrix units are busy for 33 % of the cycles, the LDS for
// 38 %; without the loop's loads it takes 101 us, without its writes to LDS as well 76 (and 82 without the fragment reads as well: the
// parts overlap and do not add up).  Half of the requests that reach L2 are for scale bytes, a word a row and depth.  With an E4M3 operand
// (one depth a stage) 41 %; 256 x 256 tiles keep the matrix units busy for 74 to 77 % and take 415 us for E4M3 x E2M1, 16384 x 8192 x 4096
// (2.6 PFLOP/s; 367 with zeros in all codes, which power does not hold back).  A round of tiles computes and then stores together, so
// the output of 10000 x 2000 float32 (80 MB) comes on top of the loop.
template <int FA, int FB, int TM, int TN, int WM, int WN, int SK>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_mx_tile(ProductArgs p) {
    constexpr int THREADS = 64 * WM * WN, RT = TM / WM / 16, CT = TN / WN / 16;
    constexpr bool PHASED = WM * WN == 8;
    constexpr int AHEAD = PHASED ? 1 : 2;
    typedef Operand<FA, TM, THREADS, SK> OpA;
    typedef Operand<FB, TN, THREADS, SK> OpB;
    static_assert((RT % 4 == 0 || TM <= 64) && (CT % 4 == 0 || TN <= 64), "scale bytes come four fragments to a word");
    constexpr int GA = (TM + 63) / 64, GB = (TN + 63) / 64;  // groups of 64 rows = four fragments
    constexpr int SMOVES = (GA + GB + WM * WN - 1) / (WM * WN);      // groups whose scale bytes a wavefront moves
    constexpr int B_AT = 2 * OpA::BYTES, IMAGES = B_AT + 2 * OpB::BYTES, ROOM = WM * WN * 2048;      // A's two images, then B's
    __shared__ __attribute__((aligned(1024))) uint8_t image[IMAGES > ROOM ? IMAGES : ROOM];
    // scale bytes: lane l's word holds those of four fragments
    __shared__ uint32_t lscale[2][SK][GA + GB][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const int first_a = 8 * (wm * RT % 4), first_b = 8 * (wn * CT % 4);      // where a wavefront's fragments begin in their group's words
    int tm, tn;
    tile_of(p.first + (int)blockIdx.x, (p.n + TM - 1) / TM, (p.m + TN - 1) / TN, tm, tn);

    const int stride_a = p.steps * OpA::S1, stride_b = p.steps * OpB::S1, stride_s = p.steps * 4, stages = (p.steps + SK - 1) / SK;
    const TileRows ga(p.a_codes, tm * TM, p.n, TM, stride_a), gb(p.b_codes, tn * TN, p.m, TN, stride_b);
    const TileRows gsa(p.a_scales, tm * TM, p.n, TM, stride_s), gsb(p.b_scales, tn * TN, p.m, TN, stride_s);
    OpA a;
    OpB b;
    a.init(tid, wm * RT * 16, r, g, stride_a);
    b.init(tid, wn * CT * 16, r, g, stride_b);
    // (No branches around loads and stores: where the paths meet, the compiler would wait for all loads in flight.  Stages and depths behind
    // the row's end are zeros.)
    struct Stage { typename OpA::Regs a; typename OpB::Regs b; uint32_t scale[SMOVES][SK]; };
    const auto load = [&](Stage &st, int stage) {
        a.load(st.a, ga, stage, stride_a, p.steps);
        b.load(st.b, gb, stage, stride_b, p.steps);
        // a lane takes one row's scale bytes, a word a depth
#pragma unroll
        for (int q = 0; q < SMOVES; ++q) {
            const int group = wave + q * WM * WN, row = (group < GA ? group : group - GA) * 64 + lane;
            const uint32_t at = stage >= stages || group >= GA + GB ? TileRows::BEHIND : row * stride_s + stage * SK * 4;
            const TileRows &rows = group < GA ? gsa : gsb;
#pragma unroll
            for (int k = 0; k < SK; ++k) st.scale[q][k] = rows.load4((int)(at + 4 * k));
        }
    };
    const auto store = [&](const Stage &st, int stage) {
        const int buf = stage & 1;
        a.store(st.a, image + buf * OpA::BYTES);
        b.store(st.b, image + B_AT + buf * OpB::BYTES);
#pragma unroll
        for (int q = 0; q < SMOVES; ++q)
#pragma unroll
            for (int k = 0; k < SK; ++k) {
                const int group = wave + q * WM * WN;
                const uint32_t word = transpose_bytes(stage * SK + k < p.steps ? st.scale[q][k] : 0, lane);
                if ((GA + GB) % (WM * WN) == 0 || group < GA + GB) lscale[buf][k][group][lane] = word;
            }
    };
    v4f acc[RT][CT];
#pragma unroll
    for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int w = 0; w < CT; ++w) acc[u][w] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    struct Fragments { v8i a[RT], b[CT]; int sa[(RT + 3) / 4], sb[(CT + 3) / 4]; };
    const auto read = [&](Fragments &f, int t, int k) {      // depth k of stage t
        const int buf = t & 1;
#pragma unroll
        for (int u = 0; u < RT; ++u) f.a[u] = a.fragment(image + buf * OpA::BYTES, u, k);
#pragma unroll
        for (int w = 0; w < CT; ++w) f.b[w] = b.fragment(image + B_AT + buf * OpB::BYTES, w, k);
#pragma unroll
        for (int q = 0; q < (RT + 3) / 4; ++q) f.sa[q] = (int)(lscale[buf][k][wm * RT / 4 + q][lane] >> first_a);
#pragma unroll
        for (int q = 0; q < (CT + 3) / 4; ++q) f.sb[q] = (int)(lscale[buf][k][GA + wn * CT / 4 + q][lane] >> first_b);
    };
    const auto multiply = [&](const Fragments &f) {
#pragma unroll
        for (int w = 0; w < CT; ++w)
#pragma unroll
            for (int u = 0; u < RT; ++u) acc[u][w] = mma_bytes<FA, FB>(f.b[w], f.a[u], acc[u][w], f.sb[w / 4], w, f.sa[u / 4], u);
    };
    Stage odd, even;                                         // (PHASED: every stage goes through `odd`)
    load(odd, 0);
    if (!PHASED) load(even, 1);
    store(odd, 0);
    load(odd, AHEAD);
    __syncthreads();
    if constexpr (PHASED) {
        static_assert(SK == 1, "one depth a stage");
        constexpr int READS = RT * OpA::S1 / 64 + CT * OpB::S1 / 64 + RT / 4 + CT / 4, LOADS = OpA::MOVES + OpB::MOVES + SMOVES;
        if (wave >= 4) __syncthreads();
        for (int t = 0; t < stages; ++t) {
            store(odd, t + 1);
            __builtin_amdgcn_sched_barrier(0);
            Fragments f;
            read(f, t, 0);
            load(odd, t + 1 + AHEAD);
            // the load path and the LDS work side by side: a load after every few fragment reads
#pragma unroll
            for (int q = 0; q < LOADS; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x100, READS / LOADS, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            __builtin_amdgcn_s_setprio(1);
            multiply(f);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
        }
    } else {
        Fragments f[2];                                      // (the last read is of the stage behind the end; not multiplied)
        read(f[0], 0, 0);
        const auto step = [&](int t, Stage &next, int at) {  // `at`: which of f holds the stage's first depth
#pragma unroll
            for (int k = 0; k < SK; ++k) {
                if (k == SK - 1) {
                    store(next, t + 1);
                    load(next, t + 1 + AHEAD);
                    __syncthreads();
                }
                read(f[(at + k + 1) & 1], t + (k + 1) / SK, (k + 1) % SK);
                multiply(f[(at + k) & 1]);
            }
        };
        for (int t = 0; t + 1 < stages; t += 2) {
            step(t, even, 0);
            step(t + 1, odd, SK & 1);
        }
        if (stages & 1) step(stages - 1, even, 0);
    }
    if (PHASED && wave < 4) __syncthreads();
    uint8_t *room = image + wave * 2048;
    const int i0 = tm * TM + wm * RT * 16, j0 = tn * TN + wn * CT * 16;
    if (i0 >= p.n || j0 >= p.m) return;                      // (all of this wavefront's rows or columns lie behind the last one)
    if (p.out_dtype == BTS_F32) write_tile<float, RT, CT>(p, acc, room, i0, j0, lane);
    else if (p.out_dtype == BTS_F16) write_tile<_Float16, RT, CT>(p, acc, room, i0, j0, lane);
    else write_tile<bf16, RT, CT>(p, acc, room, i0, j0, lane);
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
bool known_format(int f) { return f == BTS_MX_E2M1 || f == BTS_MX_E4M3; }
bool known_dtype(int t) { return t == BTS_F32 || t == BTS_F16 || t == BTS_BF16; }
size_t dtype_bytes(int t) { return t == BTS_F32 ? 4 : 2; }
bool aligned(const void *p, size_t to) { return (uintptr_t)p % to == 0; }
constexpr int MOST_WIDE = 1 << 30;                             // a row's elements: its columns, padded and a stride further, are ints
constexpr long MOST_PIECES = 0xffffffffl - (1 << 24);          // 128-element pieces a call takes (the grid's stride is added in 32 bits)
long pieces(int n, int d) { return (long)n * (padded(d) / MX_ROW); }
dim3 piece_grid(const bts_context *ctx, long pieces) {
    const long blocks = (pieces + 15) / 16, most = (long)ctx->n_cu * 64;
    return dim3((unsigned)(blocks < most ? blocks : most));
}

// Rows of `bytes` bytes, `stride` bytes apart (null: none).  Whether two sets of them share a byte -- the kernels read and write rows in no
// order, so an output may not lie across an input; rows between another's rows are fine.
struct Rows {
    const void *p;
    long n, bytes, stride;
    bool same(const Rows &o) const { return p == o.p && stride == o.stride; }
};
Rows matrix(const void *p, long n, long d, long ld, int dtype) { return {p, n, d * (long)dtype_bytes(dtype), ld * (long)dtype_bytes(dtype)}; }
Rows block(const void *p, long bytes) { return {p, 1, bytes, bytes}; }
bool overlap(Rows a, Rows b) {
    if (!a.p || !b.p) return false;
    for (Rows *r : {&a, &b})
        if (r->n == 1 || r->bytes == r->stride) *r = block(r->p, r->n * r->bytes);
    const long at = (intptr_t)a.p, to = (intptr_t)b.p;
    if (at + (a.n - 1) * a.stride + a.bytes <= to || to + (b.n - 1) * b.stride + b.bytes <= at) return false;
    const auto floor_div = [](long v, long by) { return v / by - (v % by < 0); };
    if (a.n > 1 && a.stride == b.stride) {         // the first row distance at which b's row does not end before a's begins
        const long k = std::max(floor_div(at - to - b.bytes, a.stride) + 1, 1 - a.n);
        return k < b.n && to + k * a.stride < at + a.bytes;
    }
    if (a.n > b.n) return overlap(b, a);
    for (long i = 0; i < a.n; ++i) {
        const long from = at + i * a.stride, j = std::max(floor_div(from - to - b.bytes, b.stride) + 1, 0l);
        if (j < b.n && to + j * b.stride < from + a.bytes) return true;
    }
    return false;
}

template <class T> void quantize(bts_context *ctx, const void *x, int ldx, int n, int d, int format, uint8_t *codes, uint8_t *scales, hipStream_t st) {
    const uint32_t all = (uint32_t)pieces(n, d), row = (uint32_t)(padded(d) / MX_ROW);
    const T *const xs = static_cast<const T *>(x);
    if (format == E2M1) hipLaunchKernelGGL((k_mx_quantize<T, E2M1>), piece_grid(ctx, all), dim3(256), 0, st, xs, (long)ldx, all, row, d, codes, scales);
    else hipLaunchKernelGGL((k_mx_quantize<T, E4M3>), piece_grid(ctx, all), dim3(256), 0, st, xs, (long)ldx, all, row, d, codes, scales);
}
template <class T> void dequantize(bts_context *ctx, const uint8_t *codes, const uint8_t *scales, int format, int n, int d, void *out, int ldo, hipStream_t st) {
    const uint32_t all = (uint32_t)pieces(n, d), row = (uint32_t)(padded(d) / MX_ROW);
    T *const to = static_cast<T *>(out);
    if (format == E2M1) hipLaunchKernelGGL((k_mx_dequantize<T, E2M1>), piece_grid(ctx, all), dim3(256), 0, st, codes, scales, all, row, d, to, (long)ldo);
    else hipLaunchKernelGGL((k_mx_dequantize<T, E4M3>), piece_grid(ctx, all), dim3(256), 0, st, codes, scales, all, row, d, to, (long)ldo);
}

// A launch's threads have to number below 2^32: what takes more workgroups than this (a multiple of the 8 XCDs) goes out in several.
constexpr long RUN = 1L << 20;

template <class T, int TPR, int CH> void rms_norm_launch(NormArgs<T> a, hipStream_t st) {
    const int rows = 256 / TPR;
    for (a.first = 0; a.first < a.n; a.first += RUN * rows) {
        const long blocks = (a.n - a.first + rows - 1) / rows;
        const dim3 grid((unsigned)(blocks < RUN ? blocks : RUN));
        if (a.d % 8 == 0) hipLaunchKernelGGL((k_rms_norm<T, TPR, CH, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_rms_norm<T, TPR, CH, false>), grid, dim3(256), 0, st, a);
    }
}
template <class T> void rms_norm(const void *x, int ldx, const void *residual, int ldr, const void *weight, int n, int d, double eps,
                                 void *sum, int lds, void *y, int ldy, int format, uint8_t *codes, uint8_t *scales, hipStream_t st) {
    NormArgs<T> a;
    a.x = static_cast<const T *>(x); a.residual = static_cast<const T *>(residual); a.weight = static_cast<const T *>(weight);
    a.sum = static_cast<T *>(sum); a.y = static_cast<T *>(y);
    a.ldx = ldx; a.ldr = ldr; a.lds = lds; a.ldy = ldy; a.n = n; a.d = d; a.eps = eps; a.format = format; a.codes = codes; a.scales = scales;
    // a wavefront a row up to 1024 elements (32768 x 512 bfloat16: 21 us against 30 with a workgroup a row, x 1024: 37 against 44), a workgroup
    // beyond (32768 x 2048: 88 us against 95 with a wavefront a row; one row: 2.8 against 4.6)
    if (d <= 512) rms_norm_launch<T, 64, 1>(a, st);
    else if (d <= 1024) rms_norm_launch<T, 64, 2>(a, st);
    else if (d <= 2048) rms_norm_launch<T, 256, 1>(a, st);
    else if (d <= 4096) rms_norm_launch<T, 256, 2>(a, st);
    else if (d <= 8192) rms_norm_launch<T, 256, 4>(a, st);
    else rms_norm_launch<T, 256, 0>(a, st);
}

// launch(grid) of `tiles` workgroups
template <class Launch> void in_runs(ProductArgs &p, long tiles, Launch launch) {
    for (long first = 0; first < tiles; first += RUN) {
        p.first = (int)first;
        launch(dim3((unsigned)(tiles - first < RUN ? tiles - first : RUN)));
    }
}
template <int FA, int FB, int TM, int TN, int WM, int WN, int SK> void tile_launch(ProductArgs p, hipStream_t st) {
    in_runs(p, (((long)p.n + TM - 1) / TM) * (((long)p.m + TN - 1) / TN),
            [&](dim3 grid) { hipLaunchKernelGGL((k_mx_tile<FA, FB, TM, TN, WM, WN, SK>), grid, dim3(64 * WM * WN), 0, st, p); });
}
// Which kernel: by how many workgroups the sizes make of the chip, one border for all pairs of formats and all d.  Times in us of the kernel
// back to back; E4M3 x E2M1 and d = 2048 where nothing else is said.
//  - 256 x 256 tiles take a CU each, in whole rounds of the CUs, counted at 2/3 of the time per area of 128 x 128 ones (16384 x 8192 x 4096: 415
//    against 609; 6000 x 2000, one round: 27 against 34).  E2M1 x E2M1 gains less: 350 against 383, and 28 against 27.  10000 x 2000, 320
//    tiles in two rounds, goes to 128 x 128: 49 against 51, E2M1 x E4M3 49 against 53, E2M1 x E2M1 39 against 53 -- at d = 8192, 195 against
//    162, 192 against 160 and 125 against 155, so a border that knew the pair and d would give the first two of these to 256 x 256.
//    Two E4M3 operands: the fragments do not fit the registers (36 spilled): 16384 x 8192 x 4096 1131 against 712 with 128 x 128.
//  - 128 x 128 tiles from two a CU on (2000 x 2000 x 1024, one a CU: 12.1 against 11.4 with 64 x 64 ones).
//  - 64 x 64 tiles from one a CU on (48 x 65536: 18; 1000 x 1000 x 1000: 5.8), below that 16 x 64 ones (for these two 23 and 6.5; 200 x 2000 x
//    1024: 4.7 against 5.2), and these too where one side has up to 32 rows, lying along the other (1 x 65536: 12.4 against 17).
//  - 16 x 16 tiles with the row split where there are fewer of them than CUs (1 x 2000: 3.4 against 5.1; 16 x 3000 x 512: 2.9 against 3.4;
//    300 x 300 x 1000, one and a half a CU: 4.5 against 4.1; long rows do not move this border: 64 x 2000 x 8192 19.7 against 12.6).
template <int FA, int FB> int product(bts_context *ctx, ProductArgs p, hipStream_t st) {
    const auto tiles = [&](long a, long b) { return ((p.n + a - 1) / a) * ((p.m + b - 1) / b); };
    const long cus = ctx->n_cu, t256 = tiles(256, 256), t128 = tiles(128, 128), most = 1L << 31;
    BTS_REQUIRE(tiles(16, 16) < most, "n * m: too many tiles for one launch");
    constexpr int SK = FA == E2M1 && FB == E2M1 ? 2 : 1;      // 128 bytes a row and stage
    constexpr bool BIG = FA == E2M1 || FB == E2M1;
    // 32-bit offsets inside a tile: 256 rows of codes, 16 rows of the output (counted in 4-byte elements whatever the type)
    const bool fits = (long)p.steps * 128 * 256 < most && p.ld * 4 * 16 < most && p.n < most - 256 && p.m < most - 256;
    if (!fits || tiles(16, 16) < cus) {
        in_runs(p, tiles(16, 16), [&](dim3 grid) { hipLaunchKernelGGL((k_mx_direct<FA, FB>), grid, dim3(256), 0, st, p); });
        BTS_LAUNCH_CHECK();
        return BTS_OK;
    }
    if constexpr (BIG) {
        if ((t256 + cus - 1) / cus * cus * 4 * 2 <= t128 * 3) {
            tile_launch<FA, FB, 256, 256, FA == E2M1 ? 2 : 4, FA == E2M1 ? 4 : 2, 1>(p, st);
            BTS_LAUNCH_CHECK();
            return BTS_OK;
        }
    }
    if (p.n <= 32) tile_launch<FA, FB, 16, 64, 1, 4, 2>(p, st);
    else if (p.m <= 32) tile_launch<FA, FB, 64, 16, 4, 1, 2>(p, st);
    else if (t128 >= 2 * cus) tile_launch<FA, FB, 128, 128, 2, 2, SK>(p, st);
    else if (tiles(64, 64) >= cus) tile_launch<FA, FB, 64, 64, 1, 4, SK>(p, st);
    else tile_launch<FA, FB, 16, 64, 1, 4, 2>(p, st);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

}  // namespace

extern "C" {

int bts_mx_row_bytes(int format, int d, int64_t *code_bytes, int64_t *scale_bytes) {
    BTS_REQUIRE(known_format(format), "unknown format");
    BTS_REQUIRE(d > 0 && d <= MOST_WIDE && code_bytes && scale_bytes, "d (1 .. 2^30), code_bytes, scale_bytes");
    *code_bytes = mx::code_bytes(format, d);
    *scale_bytes = mx::scale_bytes(d);
    return BTS_OK;
}

int bts_mx_quantize(bts_context *ctx, const void *x, int x_dtype, int ldx, int n, int d, int format, uint8_t *codes, uint8_t *scales,
                    bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && d > 0 && d <= MOST_WIDE && ldx >= d, "ctx, n, d (1 .. 2^30), ldx < d");
    BTS_REQUIRE(known_format(format) && known_dtype(x_dtype), "unknown format / type");
    BTS_ON_DEVICE(ctx);
    if (n == 0) return BTS_OK;
    BTS_REQUIRE(x && codes && scales, "null pointer");
    BTS_REQUIRE(aligned(x, dtype_bytes(x_dtype)) && aligned(codes, 16) && aligned(scales, 4), "x: element, codes: 16-byte, scales: 4-byte alignment");
    hipStream_t st = (hipStream_t)stream;
    BTS_REQUIRE(pieces(n, d) <= MOST_PIECES, "n * d: too many elements for one call");
    const Rows xs = matrix(x, n, d, ldx, x_dtype), cs = block(codes, n * mx::code_bytes(format, d)), ss = block(scales, n * mx::scale_bytes(d));
    BTS_REQUIRE(!overlap(cs, ss) && !overlap(xs, cs) && !overlap(xs, ss), "x, codes and scales overlap");
    if (x_dtype == BTS_F32) quantize<float>(ctx, x, ldx, n, d, format, codes, scales, st);
    else if (x_dtype == BTS_F16) quantize<_Float16>(ctx, x, ldx, n, d, format, codes, scales, st);
    else quantize<bf16>(ctx, x, ldx, n, d, format, codes, scales, st);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

int bts_mx_dequantize(bts_context *ctx, const uint8_t *codes, const uint8_t *scales, int format, int n, int d, void *out, int out_dtype,
                      int ldo, bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && d > 0 && d <= MOST_WIDE && ldo >= d, "ctx, n, d (1 .. 2^30), ldo < d");
    BTS_REQUIRE(known_format(format) && known_dtype(out_dtype), "unknown format / type");
    BTS_ON_DEVICE(ctx);
    if (n == 0) return BTS_OK;
    BTS_REQUIRE(out && codes && scales, "null pointer");
    BTS_REQUIRE(aligned(out, dtype_bytes(out_dtype)) && aligned(codes, 16) && aligned(scales, 4), "out: element, codes: 16-byte, scales: 4-byte alignment");
    hipStream_t st = (hipStream_t)stream;
    BTS_REQUIRE(pieces(n, d) <= MOST_PIECES, "n * d: too many elements for one call");
    const Rows os = matrix(out, n, d, ldo, out_dtype);
    BTS_REQUIRE(!overlap(os, block(codes, n * mx::code_bytes(format, d))) && !overlap(os, block(scales, n * mx::scale_bytes(d))),
                "out overlaps codes or scales");
    if (out_dtype == BTS_F32) dequantize<float>(ctx, codes, scales, format, n, d, out, ldo, st);
    else if (out_dtype == BTS_F16) dequantize<_Float16>(ctx, codes, scales, format, n, d, out, ldo, st);
    else dequantize<bf16>(ctx, codes, scales, format, n, d, out, ldo, st);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

int bts_rms_norm(bts_context *ctx, int dtype, const void *x, int ldx, const void *residual, int ldr, const void *weight, int n, int d,
                 double eps, void *sum, int lds, void *y, int ldy, int format, uint8_t *codes, uint8_t *scales, bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && d > 0 && d <= MOST_WIDE && ldx >= d, "ctx, n, d (1 .. 2^30), ldx < d");
    BTS_REQUIRE(known_dtype(dtype), "unknown type");
    BTS_REQUIRE((float)eps > 0.0f && (float)eps <= 3.0e38f, "eps must be a positive finite float32");
    BTS_REQUIRE(!residual || ldr >= d, "ldr < d");
    BTS_REQUIRE(!sum || lds >= d, "lds < d");
    BTS_REQUIRE(!y || ldy >= d, "ldy < d");
    BTS_ON_DEVICE(ctx);
    if (n == 0) return BTS_OK;
    BTS_REQUIRE(x, "null pointer");
    BTS_REQUIRE(!codes == !scales, "codes and scales come together");
    BTS_REQUIRE(!codes || known_format(format), "unknown format");
    BTS_REQUIRE(codes || y, "nothing to write: codes and y are both null");
    const size_t b = dtype_bytes(dtype);
    BTS_REQUIRE(aligned(x, b) && aligned(residual, b) && aligned(weight, b) && aligned(sum, b) && aligned(y, b), "element alignment");
    BTS_REQUIRE(aligned(codes, 16) && aligned(scales, 4), "codes: 16-byte, scales: 4-byte alignment");
    const Rows xs = matrix(x, n, d, ldx, dtype), rs = matrix(residual, n, d, ldr, dtype), ws = matrix(weight, 1, d, d, dtype);
    const Rows hs = matrix(sum, n, d, lds, dtype), ys = matrix(y, n, d, ldy, dtype);
    const Rows cs = block(codes, codes ? n * mx::code_bytes(format, d) : 0), ss = block(scales, n * mx::scale_bytes(d));
    for (const Rows &to : {hs, ys})
        BTS_REQUIRE((to.same(xs) || !overlap(to, xs)) && (to.same(rs) || !overlap(to, rs)) && !overlap(to, ws),
                    "sum and y may take the place of x or residual (with its row stride), and may not overlap them or weight otherwise");
    BTS_REQUIRE(!overlap(hs, ys) && !overlap(cs, ss), "sum and y, or codes and scales, overlap");
    for (const Rows &to : {cs, ss})
        for (const Rows &of : {xs, rs, ws, hs, ys}) BTS_REQUIRE(!overlap(to, of), "codes or scales overlap a matrix");
    hipStream_t st = (hipStream_t)stream;
    const int f = codes ? format : -1;
    if (dtype == BTS_F32) rms_norm<float>(x, ldx, residual, ldr, weight, n, d, eps, sum, lds, y, ldy, f, codes, scales, st);
    else if (dtype == BTS_F16) rms_norm<_Float16>(x, ldx, residual, ldr, weight, n, d, eps, sum, lds, y, ldy, f, codes, scales, st);
    else rms_norm<bf16>(x, ldx, residual, ldr, weight, n, d, eps, sum, lds, y, ldy, f, codes, scales, st);
    BTS_LAUNCH_CHECK();
    return BTS_OK;
}

int bts_mx_product(bts_context *ctx, const uint8_t *a_codes, const uint8_t *a_scales, int a_format, int n, const uint8_t *b_codes,
                   const uint8_t *b_scales, int b_format, int m, int d, double alpha, int floor_zero, void *out, int out_dtype, int ld,
                   bts_stream stream) {
    BTS_REQUIRE(ctx && n >= 0 && m >= 0 && d > 0 && d <= MOST_WIDE && ld >= m, "ctx, n, m, d (1 .. 2^30), ld < m");
    BTS_REQUIRE(known_format(a_format) && known_format(b_format) && known_dtype(out_dtype), "unknown format / type");
    BTS_REQUIRE(out_dtype != BTS_F32 || (a_format == E2M1 && b_format == E2M1),
                "a float32 output needs two E2M1 operands (with an E4M3 operand, products are aligned to the largest with about 13 bits behind it)");
    BTS_REQUIRE(fabs(alpha) <= 3.4028234663852886e38 && ((float)alpha != 0.0f || alpha == 0.0), "alpha must be a float32: finite, and not too small for one");
    BTS_ON_DEVICE(ctx);
    if (n == 0 || m == 0) return BTS_OK;
    BTS_REQUIRE(a_codes && a_scales && b_codes && b_scales && out, "null pointer");
    BTS_REQUIRE(aligned(a_codes, 16) && aligned(b_codes, 16) && aligned(a_scales, 4) && aligned(b_scales, 4) && aligned(out, dtype_bytes(out_dtype)),
                "codes: 16-byte, scales: 4-byte, out: element alignment");
    const Rows os = matrix(out, n, m, ld, out_dtype);
    for (const Rows &of : {block(a_codes, n * mx::code_bytes(a_format, d)), block(a_scales, n * mx::scale_bytes(d)),
                           block(b_codes, m * mx::code_bytes(b_format, d)), block(b_scales, m * mx::scale_bytes(d))})
        BTS_REQUIRE(!overlap(os, of), "out overlaps an operand");
    const size_t b = dtype_bytes(out_dtype);
    ProductArgs p;
    p.a_codes = a_codes; p.a_scales = a_scales; p.b_codes = b_codes; p.b_scales = b_scales;
    p.n = n; p.m = m; p.steps = (int)(padded(d) / MX_ROW);
    p.alpha = (float)alpha; p.floor_zero = floor_zero != 0;
    p.out = out; p.out_dtype = out_dtype; p.ld = ld;
    p.out_vec = aligned(out, 16) && (size_t)ld * b % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
    if (a_format == E2M1) return b_format == E2M1 ? product<E2M1, E2M1>(ctx, p, st) : product<E2M1, E4M3>(ctx, p, st);
    return b_format == E2M1 ? product<E4M3, E2M1>(ctx, p, st) : product<E4M3, E4M3>(ctx, p, st);
}

}  // extern "C"

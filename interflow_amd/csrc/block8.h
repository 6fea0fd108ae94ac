// block8.h -- the 8-bit block format shared by block8.hip, matmul8.hip and wgrad8.hip.
//
// A row's values in blocks of 128 (the last may be shorter).  A block has one scale 2^e, stored as the E8M0 byte e + 127; its
// codes are OCP e4m3 or e5m2:
//     m = max finite |x|,   e = the smallest integer >= -126 with m <= F 2^e  (F = 448 = 1.75 2^8, or 57344 = 1.75 2^15),
//     code = x 2^-e rounded to nearest even.
// A power of two costs a floating code no precision, is exact to apply and to undo (a code times its scale is exact in bf16),
// makes codes independent of how they were computed, and is what the scaled matrix instructions take (one byte per row and
// 32 values).  |x| 2^-e <= F, so rounding never saturates; but next to float32's largest it rounds up to 2^128 (e4m3 from 0.96875 2^128 on,
// e5m2 from 0.9375 2^128), which is restored as infinity.  NaN has the code NaN; infinity keeps its sign in e5m2 and is NaN in
// e4m3, which has none; neither takes part in m, so the other values of the block are what they would be without it.
#pragma once
#include "ifl_common.h"

#define B8_BLK 128

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// element types at the boundary (IFL_T_*)
template <int T> struct B8Type;
template <> struct B8Type<IFL_T_F32> { typedef float type; };
template <> struct B8Type<IFL_T_BF16> { typedef __bf16 type; };
template <> struct B8Type<IFL_T_F16> { typedef _Float16 type; };
static inline int b8_size(int t) { return t == IFL_T_F32 ? 4 : 2; }

// N consecutive elements that need no alignment but their own: global loads and stores of 8 and 16 bytes take any address here, at
// full speed where it is aligned
template <class T, int N>
struct B8Vec { typedef T Aligned __attribute__((ext_vector_type(N))); typedef Aligned type __attribute__((aligned(alignof(T)))); };

// 8 consecutive elements as floats; `left` of them exist (the others are zeros)
template <class T>
__device__ __forceinline__ void b8_load8(const T* __restrict__ p, int left, float v[8]) {
    if (left >= 8) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 8 / V; ++h) {
            const typename B8Vec<T, V>::type a = ((const typename B8Vec<T, V>::type*)p)[h];
#pragma unroll
            for (int i = 0; i < V; ++i) v[h * V + i] = (float)a[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.f;
    }
}

template <class T>
__device__ __forceinline__ void b8_store8(T* __restrict__ p, int left, const float v[8]) {
    if (left >= 8) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int h = 0; h < 8 / V; ++h) {
            typename B8Vec<T, V>::Aligned a;
#pragma unroll
            for (int i = 0; i < V; ++i) a[i] = (T)v[h * V + i];
            ((typename B8Vec<T, V>::type*)p)[h] = a;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (i < left) p[i] = (T)v[i];
    }
}

__device__ __forceinline__ bool b8_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Largest magnitude of 8 values, as its bits (magnitudes order as unsigned integers; what is not finite is B8_INF or more), and
// the largest finite one.
constexpr uint32_t B8_INF = 0x7f800000u;
__device__ __forceinline__ uint32_t b8_max_bits(const float v[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ uint32_t b8_amax_bits(const float v[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(v[i]) & 0x7fffffffu;
        m = max(m, u < B8_INF ? u : 0u);
    }
    return m;
}

// maximum over groups of LANES neighbouring lanes (4, 8 or 16; `lanes` where that is not known before), in every lane: exchanges
// inside a row of 16 by DPP
template <int LANES>
__device__ __forceinline__ uint32_t b8_group_max(uint32_t m, int lanes = LANES) {
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));                        // lane ^ 1
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));                        // lane ^ 2
    if (lanes >= 8) m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));       // mirror within 8
    if (lanes >= 16) m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xf, 0xf, true));      // mirror within 16
    return m;
}

// E8M0 byte of a block whose largest magnitude has these bits: its exponent, one more where the mantissa is over 1.75
__device__ __forceinline__ int b8_scale_byte(uint32_t amax, int fmt) {
    const int e = (int)((amax + 0x1fffffu) >> 23) - (fmt == IFL_Q_E4M3 ? 8 : 15);
    return e < 1 ? 1 : e;
}
// 2^(127 - byte): what values are multiplied by before rounding (byte from b8_scale_byte: 1 .. 248)
__device__ __forceinline__ float b8_inv_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
// 2^(byte - 127) for any byte: 0 is 2^-127 (subnormal), 255 is NaN
__device__ __forceinline__ float b8_scale(int byte) {
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : (uint32_t)byte << 23);
}

// codes of 8 values already multiplied by 2^-e; odd: some of them may not be finite
__device__ __forceinline__ i32x2 b8_encode8(const float v[8], int fmt, bool odd) {
    i32x2 r = {0, 0};
    if (fmt == IFL_Q_E4M3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            r[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], r[h], false);
            r[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], r[h], true);
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            r[h] = __builtin_amdgcn_cvt_pk_bf8_f32(v[4 * h], v[4 * h + 1], r[h], false);
            r[h] = __builtin_amdgcn_cvt_pk_bf8_f32(v[4 * h + 2], v[4 * h + 3], r[h], true);
        }
    }
    if (odd) {                                      // (what the conversion makes of infinities depends on a mode bit: set here)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!b8_finite(v[i])) {
                const uint32_t u = __float_as_uint(v[i]);
                const uint32_t c = (u >> 24 & 0x80u) | ((fmt == IFL_Q_E4M3 || (u & 0x7fffffu)) ? 0x7fu : 0x7cu);
                r[i >> 2] = (int)(((uint32_t)r[i >> 2] & ~(0xffu << 8 * (i & 3))) | c << 8 * (i & 3));
            }
        }
    }
    return r;
}

// A block's scale byte and the codes of this lane's 8 values of it (LANES neighbouring lanes have the block).  What is not finite is
// looked at only where the block's maximum says that there is some (16384 x 2048 bf16: 25.0 us; looked at
// in every value 26.9).
template <int LANES>
__device__ __forceinline__ i32x2 b8_quantize8(const float x[8], int fmt, int& sb, int lanes = LANES) {
    uint32_t m = b8_group_max<LANES>(b8_max_bits(x), lanes);
    const bool odd = m >= B8_INF;
    if (odd) m = b8_group_max<LANES>(b8_amax_bits(x), lanes);                   // (all lanes of a block come here, or none)
    sb = b8_scale_byte(m, fmt);
    const float inv = b8_inv_scale(sb);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[i] * inv;
    return b8_encode8(v, fmt, odd);
}

__device__ __forceinline__ void b8_decode4(int w, int fmt, float* v) {
    const f32x2 a = fmt == IFL_Q_E4M3 ? __builtin_amdgcn_cvt_pk_f32_fp8(w, false) : __builtin_amdgcn_cvt_pk_f32_bf8(w, false);
    const f32x2 b = fmt == IFL_Q_E4M3 ? __builtin_amdgcn_cvt_pk_f32_fp8(w, true) : __builtin_amdgcn_cvt_pk_f32_bf8(w, true);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
}

// 8 codes, `left` of them exist (the others are zeros)
typedef i32x2 i32x2_any __attribute__((aligned(1)));
__device__ __forceinline__ i32x2 b8_load_codes(const uint8_t* __restrict__ p, int left) {
    if (left >= 8) return *(const i32x2_any*)p;
    i32x2 r = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < left) r[i >> 2] |= (int)((uint32_t)p[i] << 8 * (i & 3));
    return r;
}
__device__ __forceinline__ void b8_store_codes(uint8_t* __restrict__ p, int left, i32x2 w) {
    if (left >= 8) { *(i32x2_any*)p = w; return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) if (i < left) p[i] = (uint8_t)((uint32_t)w[i >> 2] >> 8 * (i & 3));
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 8 codes times their block's scale (a byte) as bf16: exact, as a code has at most 4 significant bits
template <int FMT>
__device__ __forceinline__ bf16x8 b8_bf16x8(int w0, int w1, int byte) {
    const float s = __uint_as_float(byte == 0 ? 0x00400000u : (uint32_t)byte << 23);
    if (byte == 255) w0 = w1 = 0x7f7f7f7f;                               // a scale that is NaN: codes that are
    bf16x2 p[4];
    if constexpr (FMT == IFL_Q_E4M3) {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false); p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false); p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
    } else {
        p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w0, s, false); p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w0, s, true);
        p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w1, s, false); p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w1, s, true);
    }
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) { r[2 * i] = p[i][0]; r[2 * i + 1] = p[i][1]; }
    return r;
}

// ------------------------------------------------------------------------------------------------ quantize, rows contiguous
// Group of LANES lanes = one block of a row; kg (a power of two) groups side by side along a row, the rest along rows.  Four
// rows per group are in flight at once: their loads are issued before the first is used.  Few, long rows: gy workgroups share
// one (4 x 1000000: 500 us with one each, 7.6 so).  16384 x 2048: bf16 19.4 us, 5.2 TB/s, float32 27.0 us, 6.2 TB/s.
struct B8Rows { const void* x; int64_t rs; uint8_t* codes; int64_t ldc; uint8_t* scales; int64_t lds; int64_t rows; int cols, pad, kg_log, fmt, gx, gy; };
template <class T, int LANES>
__device__ __forceinline__ void b8_quantize_rows(const B8Rows& q, int block) {
    constexpr int U = 4, GPB = 256 / LANES;
    const T* __restrict__ x = (const T*)q.x;
    const int by = block / q.gx, bx = block - by * q.gx;
    const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
    const int gk = grp & ((1 << q.kg_log) - 1), gr = grp >> q.kg_log, rpb = GPB >> q.kg_log;
    const int KB = (q.cols + B8_BLK - 1) / B8_BLK;
    const int64_t step = (int64_t)q.gx * rpb;
    for (int64_t r0 = (int64_t)bx * rpb + gr; r0 < q.rows; r0 += U * step) {
        for (int kb = gk + (by << q.kg_log); kb < KB; kb += q.gy << q.kg_log) {
            const int c = kb * B8_BLK + lane * 8;
            float v[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + u * step;
                b8_load8<T>(x + r * q.rs + c, r < q.rows ? q.cols - c : 0, v[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + u * step;
                if (r >= q.rows) break;                                  // (the same for all lanes of a group)
                int sb;
                const i32x2 w = b8_quantize8<LANES>(v[u], q.fmt, sb);
                b8_store_codes(q.codes + r * q.ldc + c, q.pad - c, w);
                if (lane == 0) q.scales[r * q.lds + kb] = (uint8_t)sb;
            }
        }
    }
}
// columns that rows of codes are filled up to (with zeros): whole 16 bytes, if the rows have them
static inline int b8_pad(int64_t cols, int64_t ldc) { const int64_t p = (cols + 15) / 16 * 16; return (int)(p < ldc ? p : ldc); }

// ------------------------------------------------------------------------------------------------ quantize, columns contiguous
// x[r][c] at x + r + c * cs (a transposed view).  Workgroup = 64 rows x one block of 128 columns: lanes run along the rows
// (contiguous in memory), a thread holds 32 columns of its row, the four threads of a row meet in LDS for the maximum and
// write 32 code bytes each.  Values of 16 bits come through LDS, 8 rows of a column in one load (16384 x 2048 bf16: 55 us with a
// load for each, 22.6 so; float32 28.0, without).
struct B8Cols { const void* x; int64_t cs; uint8_t* codes; int64_t ldc; uint8_t* scales; int64_t lds; int64_t rows; int cols, pad, fmt; };
constexpr int B8_PITCH = 72;                                             // rows of a column in LDS: 16-byte aligned, neighbours 36 banks apart
constexpr int B8_COLS_LDS = 4 * 64 * 4 + 128 * B8_PITCH * 2;             // bytes that a workgroup needs, 16-byte aligned
template <class T>
__device__ __forceinline__ void b8_quantize_cols(const B8Cols& q, void* sm, int64_t bx, int kb) {
    constexpr bool STAGE = sizeof(T) == 2;
    const T* __restrict__ x = (const T*)q.x;
    uint32_t (*red)[64] = (uint32_t(*)[64])sm;
    T* tile = (T*)((uint8_t*)sm + 4 * 64 * 4);
    const int lr = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int64_t first = bx * 64, r = first + lr;
    const int c0 = kb * B8_BLK + g * 32;
    const int64_t rc = r < q.rows ? r : q.rows - 1;
    float v[32];
    if constexpr (STAGE) {
        const int p = (threadIdx.x & 7) * 8, left = (int)min((int64_t)64, q.rows - first) - p;
        typedef typename B8Vec<T, 8>::type T8;
        T8 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = min(kb * B8_BLK + (int)(threadIdx.x >> 3) + 32 * i, q.cols - 1);
            const T* s = x + first + p + (int64_t)c * q.cs;
            if (left >= 8) w[i] = *(const T8*)s;
            else {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[i][e] = e < left ? s[e] : (T)0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) *(typename B8Vec<T, 8>::Aligned*)(tile + ((threadIdx.x >> 3) + 32 * i) * B8_PITCH + p) = w[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = c0 + i < q.cols ? (float)tile[(g * 32 + i) * B8_PITCH + lr] : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = c0 + i < q.cols ? (float)x[rc + (int64_t)(c0 + i) * q.cs] : 0.f;
    }
    uint32_t m = 0, any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) { m = max(m, b8_amax_bits(v + 8 * i)); any = max(any, b8_max_bits(v + 8 * i)); }
    red[g][lr] = m;
    __syncthreads();
    m = max(max(red[0][lr], red[1][lr]), max(red[2][lr], red[3][lr]));
    if (r >= q.rows) return;
    const int sb = b8_scale_byte(m, q.fmt);
    const float inv = b8_inv_scale(sb);
    typedef i32x4 i32x4_any __attribute__((aligned(1)));
    uint8_t* d = q.codes + r * q.ldc + c0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        i32x2 w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* u = v + 16 * j + 8 * h;
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] *= inv;
            w[h] = b8_encode8(u, q.fmt, any >= B8_INF);
        }
        if (c0 + 16 * j + 16 <= q.pad) *(i32x4_any*)(d + 16 * j) = i32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
        else { b8_store_codes(d + 16 * j, q.pad - (c0 + 16 * j), w[0]); b8_store_codes(d + 16 * j + 8, q.pad - (c0 + 16 * j + 8), w[1]); }
    }
    if (g == 0) q.scales[r * q.lds + kb] = (uint8_t)sb;
}

// dispatch on an element type: body sees `T`
#define B8_DISPATCH(type, ...) \
    do { if ((type) == IFL_T_F32) { typedef float T; __VA_ARGS__; } \
         else if ((type) == IFL_T_BF16) { typedef __bf16 T; __VA_ARGS__; } \
         else { typedef _Float16 T; __VA_ARGS__; } } while (0)

static inline bool b8_type_ok(int t) { return t == IFL_T_F32 || t == IFL_T_BF16 || t == IFL_T_F16; }
static inline bool b8_fmt_ok(int f) { return f == IFL_Q_E4M3 || f == IFL_Q_E5M2; }

// two matrices of K columns in e4m3, rows of codes and scales alike, in one launch; everything checked by the caller, M and N at least 1
int b8_quantize2(const void* x, int xtype, int64_t x_rs, const void* w, int wtype, int64_t w_rs, uint8_t* xc, uint8_t* xs, uint8_t* wc, uint8_t* ws,
                 int64_t ldc, int64_t lds, int64_t M, int64_t N, int64_t K, void* stream);

// whether a product of these sizes, M from 0 on, N and K from 1 on, fits a launch
bool b8_matmul_fits(int64_t M, int64_t N, int64_t K);

// ifl_block8_wgrad in two steps for the layer whose other product needs dy in 8-bit blocks, and its weights along their columns: 1
// prepares (and quantizes dy, if told where to, and w, if there is one), 2 multiplies and joins, 3 both.
struct B8Quant { uint8_t *codes, *scales; int64_t ldc, lds; int fmt; B8Cols w; int wtype; };
int b8_wgrad(int steps, const B8Quant* quant, const void* dy, int dytype, int64_t ldy, const uint8_t* codes, int64_t ldc, const uint8_t* scales,
             int64_t lds, int fmt, const float* chan, void* dw, int dwtype, int64_t ldw, void* db, int dbtype, float* scratch, int64_t M,
             int64_t N, int64_t K, void* stream);

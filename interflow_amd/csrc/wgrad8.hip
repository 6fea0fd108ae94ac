// wgrad8.hip -- the weight gradient of a product whose input was kept in 8-bit blocks (block8.h):
//     dw[n][k] = chan[k] sum_m dy[m][n] code[m][k] 2^e[m][k / 128],      db[n] = sum_m dy[m][n]
// The sum runs over the rows of both operands, whose scales change from row to row, so the 8-bit instructions cannot apply them;
// a code times its scale is exact in bf16.
#include "block8.h"

namespace {

template <class T, class TW>
__global__ __launch_bounds__(256)
void wgrad8_simple_kernel(const T* __restrict__ dy, int64_t ldy, const uint8_t* __restrict__ codes, int64_t ldc, const uint8_t* __restrict__ scales,
                          int64_t lds, int fmt, const float* __restrict__ chan, TW* __restrict__ dw, int64_t ldw, int64_t M, int N, int K)
{
    __shared__ float sy[16][64 + 4], sx[16][64 + 4];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int k0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
    float acc[4][4] = {};
    for (int64_t m0 = 0; m0 < M; m0 += 16) {
        for (int i = threadIdx.x; i < 16 * 64; i += 256) {
            const int r = i >> 6, c = i & 63;
            const int64_t m = m0 + r;
            sy[r][c] = m < M && n0 + c < N ? (float)dy[m * ldy + n0 + c] : 0.f;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (m < M && k0 + c < K) { b8_decode4(codes[m * ldc + k0 + c], fmt, v); v[0] *= b8_scale(scales[m * lds + (k0 + c) / B8_BLK]); }
            sx[r][c] = v[0];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sy[r][ty * 4 + i], sx[r][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + ty * 4 + i, k = k0 + tx * 4 + j;
            if (n < N && k < K) dw[(int64_t)n * ldw + k] = (TW)(chan ? acc[i][j] * chan[k] : acc[i][j]);
        }
}

// column sums: a workgroup takes 64 columns, its four waves every fourth row, joined in LDS
template <class T, class TW>
__global__ __launch_bounds__(256)
void colsum_kernel(const T* __restrict__ dy, int64_t ldy, TW* __restrict__ db, int64_t M, int N)
{
    __shared__ float red[4][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6, n = blockIdx.x * 64 + c;
    float t = 0.f;
    if (n < N) for (int64_t m = r; m < M; m += 4) t += (float)dy[m * ldy + n];
    red[r][c] = t;
    __syncthreads();
    if (r == 0 && n < N) db[n] = (TW)((red[0][c] + red[1][c]) + (red[2][c] + red[3][c]));
}

}  // namespace

extern "C" int64_t ifl_block8_wgrad_scratch_floats(int64_t M, int64_t N, int64_t K) { (void)M; (void)N; (void)K; return 0; }

extern "C" int ifl_block8_wgrad(const void* dy, int dytype, int64_t ldy, const uint8_t* codes, int64_t ldc, const uint8_t* scales,
                                int64_t lds, int fmt, const float* chan, void* dw, int dwtype, int64_t ldw, void* db, int dbtype,
                                float* scratch, int64_t M, int64_t N, int64_t K, void* stream)
{
    (void)scratch;
    IFL_CHECK_ARG(b8_fmt_ok(fmt) && b8_type_ok(dytype) && (!dw || b8_type_ok(dwtype)) && (!db || b8_type_ok(dbtype)), IFL_EINVAL, "block8_wgrad: types");
    IFL_CHECK_ARG(M >= 0 && N >= 1 && (K >= 1 || !dw) && N <= 0x3fffffff && K <= 0x3fffffff, IFL_EINVAL, "block8_wgrad: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG((dw || db) && (M == 0 || dy) && (M == 0 || !dw || (codes && scales)), IFL_EINVAL, "block8_wgrad: null pointer");
    IFL_CHECK_ARG(ldy >= N && (!dw || (ldc >= K && lds >= ifl_cdiv((int)K, B8_BLK) && ldw >= K)), IFL_EINVAL, "block8_wgrad: row strides");
    IFL_CHECK_ARG((N + 63) / 64 <= 65535, IFL_ENOTSUP, "block8_wgrad: N=%lld", (long long)N);
    hipStream_t st = (hipStream_t)stream;
#define WG8(TWCODE, ...) do { if ((TWCODE) == IFL_T_F32) { typedef float TW; __VA_ARGS__; } else if ((TWCODE) == IFL_T_BF16) { typedef __bf16 TW; __VA_ARGS__; } else { typedef _Float16 TW; __VA_ARGS__; } } while (0)
    if (dw) {
        B8_DISPATCH(dytype, WG8(dwtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_simple_kernel<T, TW>), dim3((unsigned)((K + 63) / 64), (unsigned)((N + 63) / 64)), dim3(256), 0, st,
                                                           (const T*)dy, ldy, codes, ldc, scales, lds, fmt, chan, (TW*)dw, ldw, M, (int)N, (int)K)));
        IFL_LAUNCH_CHECK();
    }
    if (db) {
        B8_DISPATCH(dytype, WG8(dbtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(colsum_kernel<T, TW>), dim3((unsigned)((N + 63) / 64)), dim3(256), 0, st, (const T*)dy, ldy, (TW*)db, M, (int)N)));
        IFL_LAUNCH_CHECK();
    }
    return 0;
}

// matmul8.hip -- C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]) over rows in 8-bit blocks (block8.h), on the scaled 8-bit matrix
// instructions of gfx950: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 codes and takes one E8M0 byte per row
// and 32 values.  A block of 128 is one instruction deep, so every scale is applied by the instruction, exactly, and sums are
// held in float32.
//
// Operands: the instruction's first is B (the n side) and its second A (the m side), so that a lane ends up with four
// neighbouring n of one m: a contiguous store.
//
// What the 8-bit instructions keep: within 8 products they drop what is below 2^-13 of the largest (measured), so a result is off
// by about 1.5e-5 of itself (2-norm; 1.7e-5 of sum |a b| at most in random data, 7 2^-13 of it at worst) -- a thirtieth of what
// rounding it to float16 costs and a hundredth of bfloat16's.  A float32 result would show it: for that the codes times their
// scales, exact in bf16, go through v_mfma_f32_16x16x32_bf16, which keeps 24 bits, at half the rate.
//  Lane l gives row l % 16 and 32 of the 128 values; which 32 is free as long
// as both operands agree (all of a block share a scale): 16 bytes from 16 (l / 16) and 16 from 64 + 16 (l / 16).
#include "block8.h"

namespace {

struct MM8 {
    const uint8_t *a, *b, *sa, *sb;
    int64_t lda, ldb, lsa, lsb;
    const void* bias; int btype;
    void* out; int64_t ldo;
    int64_t M, N; int K;
};

__device__ __forceinline__ float mm8_bias(const MM8& q, int64_t n) {
    return !q.bias ? 0.f : q.btype == IFL_T_F32 ? ((const float*)q.bias)[n] : q.btype == IFL_T_BF16 ? (float)((const __bf16*)q.bias)[n] : (float)((const _Float16*)q.bias)[n];
}

// 16 bytes of a row from k on, zero where k >= K
__device__ __forceinline__ i32x4 mm8_load16(const uint8_t* __restrict__ row, int k, int K) {
    if (k + 16 <= K) return *(const i32x4*)(row + k);
    i32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) if (k + i < K) r[i >> 2] |= (int)((uint32_t)row[k + i] << 8 * (i & 3));
    return r;
}

// c += 16 x 128 times 128 x 16.  EXACT: as bf16 operands (a code times its scale), four instructions.
template <int FA, int FB, bool EXACT>
__device__ __forceinline__ f32x4 mm8_mfma(i32x8 b, i32x8 a, f32x4 c, int sb, int sa) {
    if constexpr (!EXACT) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, FB, FA, 0, sb, 0, sa);
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b8_bf16x8<FB>(b[2 * i], b[2 * i + 1], sb), b8_bf16x8<FA>(a[2 * i], a[2 * i + 1], sa), c, 0, 0, 0);
        return c;
    }
}

// Wave = 32 n x 32 m, operands straight from memory.
template <int FA, int FB, class T>
__global__ __launch_bounds__(256)
void mm8_direct_kernel(MM8 q)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 64 + (wave & 1) * 32, m0 = (int64_t)blockIdx.y * 64 + (wave >> 1) * 32;
    const uint8_t *pb[2], *pa[2], *psb[2], *psa[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t n = min(n0 + 16 * i + r16, q.N - 1), m = min(m0 + 16 * i + r16, q.M - 1);
        pb[i] = q.b + n * q.ldb; psb[i] = q.sb + n * q.lsb;
        pa[i] = q.a + m * q.lda; psa[i] = q.sa + m * q.lsa;
    }
    f32x4 acc[2][2] = {};
    for (int k = 0, kb = 0; k < q.K; k += B8_BLK, ++kb) {
        i32x8 a[2], b[2];
        int sa[2], sb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const i32x4 a0 = mm8_load16(pa[i], k + 16 * g, q.K), a1 = mm8_load16(pa[i], k + 64 + 16 * g, q.K);
            const i32x4 b0 = mm8_load16(pb[i], k + 16 * g, q.K), b1 = mm8_load16(pb[i], k + 64 + 16 * g, q.K);
#pragma unroll
            for (int e = 0; e < 4; ++e) { a[i][e] = a0[e]; a[i][4 + e] = a1[e]; b[i][e] = b0[e]; b[i][4 + e] = b1[e]; }
            sa[i] = psa[i][kb]; sb[i] = psb[i][kb];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mm8_mfma<FA, FB, sizeof(T) == 4>(b[i], a[j], acc[i][j], sb[i], sa[j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t n = n0 + 16 * i + 4 * g + e, m = m0 + 16 * j + r16;
                if (n < q.N && m < q.M) ((T*)q.out)[m * q.ldo + n] = (T)(acc[i][j][e] + mm8_bias(q, n));
            }
}

}  // namespace

extern "C" int ifl_block8_matmul(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t lsa, int fa, const uint8_t* b, int64_t ldb,
                                 const uint8_t* sb, int64_t lsb, int fb, const void* bias, int btype, void* out, int otype, int64_t ldo,
                                 int64_t M, int64_t N, int64_t K, void* stream)
{
    IFL_CHECK_ARG(b8_fmt_ok(fa) && b8_fmt_ok(fb), IFL_EINVAL, "block8_matmul: formats %d, %d", fa, fb);
    IFL_CHECK_ARG(b8_type_ok(otype) && (!bias || b8_type_ok(btype)), IFL_EINVAL, "block8_matmul: element types");
    IFL_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && K <= 0x7ffffc00, IFL_EINVAL, "block8_matmul: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    if (M == 0) return 0;
    const int KB = ifl_cdiv((int)K, B8_BLK);
    IFL_CHECK_ARG(a && b && sa && sb && out, IFL_EINVAL, "block8_matmul: null pointer");
    IFL_CHECK_ARG(lda >= K && ldb >= K && lsa >= KB && lsb >= KB && ldo >= N, IFL_EINVAL, "block8_matmul: row strides");
    IFL_CHECK_ARG(lda % 16 == 0 && ldb % 16 == 0 && (uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0, IFL_EINVAL, "block8_matmul: codes in rows of whole, aligned 16 bytes");
    IFL_CHECK_ARG((M + 63) / 64 <= 65535 && (N + 63) / 64 <= 0x7fffffff, IFL_ENOTSUP, "block8_matmul: %lld x %lld", (long long)M, (long long)N);
    const MM8 q = {a, b, sa, sb, lda, ldb, lsa, lsb, bias, btype, out, ldo, M, N, (int)K};
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
#define MM8_GO(FA, FB) B8_DISPATCH(otype, hipLaunchKernelGGL(HIP_KERNEL_NAME(mm8_direct_kernel<FA, FB, T>), grid, dim3(256), 0, (hipStream_t)stream, q))
    if (fa == 0 && fb == 0) MM8_GO(0, 0); else if (fa == 0) MM8_GO(0, 1); else if (fb == 0) MM8_GO(1, 0); else MM8_GO(1, 1);
    IFL_LAUNCH_CHECK();
    return 0;
}

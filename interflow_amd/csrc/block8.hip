// block8.hip -- activations in 8-bit blocks: quantize, restore, and the coupling networks' ActNorm + ReLU whose backward pass
// reads an 8-bit checkpoint instead of two float32 tensors.  All of it is bound by memory traffic: one pass over the data, a
// block's maximum inside a group of 4, 8 or 16 lanes (8 values each), no LDS.
#include "block8.h"

namespace {

// ------------------------------------------------------------------------------------------------ quantize
template <class T, int LANES>
__global__ __launch_bounds__(256)
void quantize_kernel(B8Rows q) { b8_quantize_rows<T, LANES>(q, blockIdx.x); }

// two matrices with as many columns in one launch: a layer's input and its weights (16384 and 2048 rows of 2048 bf16: 30 us, 28 + 6
// one after the other)
template <class T, class T2, int LANES>
__global__ __launch_bounds__(256)
void quantize2_kernel(B8Rows q, B8Rows q2) {
    const int n = q.gx * q.gy;
    if ((int)blockIdx.x < n) b8_quantize_rows<T, LANES>(q, blockIdx.x);
    else b8_quantize_rows<T2, LANES>(q2, blockIdx.x - n);
}

template <class T>
__global__ __launch_bounds__(256)
void quantize_t_kernel(B8Cols q, int tiles) {
    __shared__ __attribute__((aligned(16))) uint8_t sm[B8_COLS_LDS];
    const int kb = blockIdx.x / tiles;
    b8_quantize_cols<T>(q, sm, blockIdx.x - kb * tiles, kb);
}

// ------------------------------------------------------------------------------------------------ restore
// out = code * 2^e (* chan[c]): a thread takes 8 columns, tpr (a power of two) threads along a row; four rows in flight; few, long
// rows are shared as above.  16384 x 2048: bf16 17.7 us, 5.7 TB/s, float32 29.9 us, 5.6 TB/s.
template <class T>
__global__ __launch_bounds__(256)
void dequantize_kernel(const uint8_t* __restrict__ codes, int64_t ldc, const uint8_t* __restrict__ scales, int64_t lds, int fmt,
                       const float* __restrict__ chan, T* __restrict__ out, int64_t ldo, int64_t rows, int cols, int tpr_log)
{
    constexpr int U = 4;
    const int rpb = 256 >> tpr_log;
    const int64_t step = (int64_t)gridDim.x * rpb;
    for (int64_t r0 = (int64_t)blockIdx.x * rpb + (threadIdx.x >> tpr_log); r0 < rows; r0 += U * step) {
        // (counted in groups of 8 columns: columns themselves, up to 2^31 of them, would wrap at the last step)
        for (int i8 = (threadIdx.x & ((1 << tpr_log) - 1)) + (blockIdx.y << tpr_log); i8 < (cols + 7) / 8; i8 += gridDim.y << tpr_log) {
            const int c = i8 * 8;
            i32x2 w[U];
            int sb[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + u * step;
                w[u] = b8_load_codes(codes + r * ldc + c, r < rows ? cols - c : 0);
                sb[u] = r < rows ? scales[r * lds + c / B8_BLK] : 0;
            }
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = chan && c + i < cols ? chan[c + i] : 1.f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + u * step;
                if (r >= rows) break;
                float v[8];
                b8_decode4(w[u][0], fmt, v);
                b8_decode4(w[u][1], fmt, v + 4);
                const float s = b8_scale(sb[u]);
#pragma unroll
                for (int i = 0; i < 8; ++i) { v[i] *= s; if (chan) v[i] *= f[i]; }
                b8_store8<T>(out + r * ldo + c, cols - c, v);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ ActNorm + ReLU, 8-bit checkpoint
// v = relu(x + bias), y = v exp(logs); the checkpoint is v in 8 bits, one scale per pixel and 128 channels.  v and not y: x +
// bias is one rounded addition whatever computes it, so the codes do not hang on an exp's last bit, and the backward pass and the
// next convolution's weight gradient multiply by exp(logs) in float32.  A positive v never gets the code 0 (the smallest
// subnormal instead): the code's zeros ARE the ReLU's mask.  Ring pixels of y and of the codes are written as zeros.  Bound by memory:
// 8 x 256 x 256 x 64 forward 57.6 us, 5.3 TB/s, backward 63, 4.9 (twice the blocks, or two pixels at a time: the same).
template <int LANES>
__global__ __launch_bounds__(256)
void an_relu8_fwd_kernel(const float* __restrict__ x, float* __restrict__ y, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                         const float* __restrict__ bias, const float* __restrict__ logs, uint32_t npx, int h2, int w2, int C, int kg)
{
    constexpr int GPB = 256 / LANES;
    const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
    const int KB = (C + B8_BLK - 1) / B8_BLK;
    const int gk = grp % kg, gr = grp / kg, ppb = GPB / kg;             // kg groups per pixel, ppb pixels per pass
    if (gr >= ppb) return;
    const int c = gk * B8_BLK + lane * 8;
    const bool here = c < C;                                             // (C is a multiple of 8)
    float b[8], s[8];
    b8_load8<float>(bias + (here ? c : 0), 8, b);
    b8_load8<float>(logs + (here ? c : 0), 8, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = expf(s[i]);
    for (uint32_t p = blockIdx.x * ppb + gr; p < npx; p += gridDim.x * ppb) {
        const uint32_t line = p / (uint32_t)w2, px = p - line * w2, py = line % (uint32_t)h2;
        const bool inside = px > 0 && px < (uint32_t)w2 - 1 && py > 0 && py < (uint32_t)h2 - 1;
        const int64_t o = (int64_t)p * C + c;
        float v[8];
        b8_load8<float>(x + o, here && inside ? 8 : 0, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = v[i] + b[i];
            v[i] = here && inside && !(t <= 0.f) ? t : 0.f;              // (NaN stays NaN, as torch's relu leaves it)
        }
        int sb;
        i32x2 w = b8_quantize8<LANES>(v, IFL_Q_E4M3, sb);
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = v[i] == 0.f ? 0.f : v[i] * s[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) if (v[i] > 0.f && ((uint32_t)w[i >> 2] >> 8 * (i & 3) & 0xffu) == 0u) w[i >> 2] |= 1 << 8 * (i & 3);
        if (here) {
            b8_store8<float>(y + o, 8, r);
            *(i32x2*)(codes + o) = w;
            if (lane == 0) scales[(int64_t)p * KB + gk] = (uint8_t)sb;
        }
    }
}

// dx = g s [code != 0];  part[blk][0:C] = sum g [..], part[blk][C:2C] = sum g v8 over the block's pixels (both still without
// the factor s, which the reduction applies).  A block walks a contiguous range of pixels; a thread keeps its 8 channels.
// Sums of 16 pixels are joined, then those sums, then the threads' in four rows: what is added up in one row stays short, and with it the
// rounding (700 x 700 x 1024: at most 47 2^-24 of the magnitudes' sum; in one row after the other 58 2^-24 were seen).
__global__ __launch_bounds__(256)
void an_relu8_bwd_kernel(const float* __restrict__ g, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                         const float* __restrict__ logs, float* __restrict__ dx, float* __restrict__ part, uint32_t npx,
                         uint32_t px_per_block, int h2, int w2, int C)
{
    extern __shared__ float sm[];                                        // [pixel lane][2][C]
    const int lpp = C / 8, ppb = 256 / lpp, KB = (C + B8_BLK - 1) / B8_BLK;
    const int pl = threadIdx.x / lpp, c = (threadIdx.x - pl * lpp) * 8;
    float sg[8], sv[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { sg[i] = sv[i] = 0.f; s[i] = expf(logs[c + i]); }
    const uint32_t end = min(npx, (blockIdx.x + 1) * px_per_block);
    if (pl < ppb) {
        float tg[8] = {}, tv[8] = {};
        int row = 0;
        for (uint32_t p = blockIdx.x * px_per_block + pl; p < end; p += ppb) {
            const uint32_t line = p / (uint32_t)w2, px = p - line * w2, py = line % (uint32_t)h2;
            const bool inside = px > 0 && px < (uint32_t)w2 - 1 && py > 0 && py < (uint32_t)h2 - 1;
            const int64_t o = (int64_t)p * C + c;
            float d[8], v[8], r[8];
            b8_load8<float>(g + o, inside ? 8 : 0, d);
            const i32x2 w = *(const i32x2*)(codes + o);
            const float sc = b8_scale(scales[(int64_t)p * KB + c / B8_BLK]);
            b8_decode4(w[0], IFL_Q_E4M3, v);
            b8_decode4(w[1], IFL_Q_E4M3, v + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = v[i] == 0.f ? 0.f : d[i];
                r[i] = e * s[i];
                tg[i] += e;
                tv[i] = fmaf(e, v[i] * sc, tv[i]);
            }
            b8_store8<float>(dx + o, 8, r);
            if (++row == 16) {
#pragma unroll
                for (int i = 0; i < 8; ++i) { sg[i] += tg[i]; sv[i] += tv[i]; tg[i] = tv[i] = 0.f; }
                row = 0;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) { sm[(pl * 2) * C + c + i] = sg[i] + tg[i]; sm[(pl * 2 + 1) * C + c + i] = sv[i] + tv[i]; }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * C; k += 256) {
        float t[4] = {};
        for (int i = 0; i < ppb; i += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) { const float v = sm[min(i + e, ppb - 1) * 2 * C + k]; t[e] += i + e < ppb ? v : 0.f; }
        part[(int64_t)blockIdx.x * 2 * C + k] = (t[0] + t[1]) + (t[2] + t[3]);
    }
}

constexpr int AN8_BLOCKS = 1024;                                         // most blocks (partial sums) of the backward pass

// out[k] = exp(logs[k mod C]) sum over blocks of part[blk][k].  Workgroup = 16 k, 64 threads to each, which take every 64th block and
// meet in LDS in a fixed order: a thread's loads are all under way together (979 blocks of 128: 3.9 to 4.7 us; a loop over them 4.8; a
// wave to each k, whose lanes read far apart, 7.0).
__global__ __launch_bounds__(1024)
void an_relu8_reduce_kernel(const float* __restrict__ part, int nblk, const float* __restrict__ logs, float* __restrict__ dbias,
                            float* __restrict__ dlogs, int C)
{
    __shared__ float red[64][17];
    const int i = threadIdx.x & 15, r = threadIdx.x >> 4, k = blockIdx.x * 16 + i;       // (2 C is a multiple of 16)
    float q[4] = {};
    if (nblk <= 64) q[0] = r < nblk ? part[(int64_t)r * 2 * C + k] : 0.f;
    else {
        float v[AN8_BLOCKS / 64];
#pragma unroll
        for (int e = 0; e < AN8_BLOCKS / 64; ++e) v[e] = part[(int64_t)min(r + 64 * e, nblk - 1) * 2 * C + k];
#pragma unroll
        for (int e = 0; e < AN8_BLOCKS / 64; ++e) q[e & 3] += r + 64 * e < nblk ? v[e] : 0.f;
    }
    float t = (q[0] + q[1]) + (q[2] + q[3]);
    auto pairs = [](const float (&u)[8]) { return ((u[0] + u[4]) + (u[2] + u[6])) + ((u[1] + u[5]) + (u[3] + u[7])); };
    red[r][i] = t;
    __syncthreads();
    if (r < 8) {
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = red[r + 8 * e][i];
        red[r][i] = pairs(u);
    }
    __syncthreads();
    if (r == 0) {
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = red[e][i];
        t = pairs(u);
        const int c = k < C ? k : k - C;
        (k < C ? dbias : dlogs)[c] = t * expf(logs[c]);
    }
}

int log2_up(int64_t n, int most) { int l = 0; while (l < most && (1 << l) < n) ++l; return l; }
bool aligned(const void* p, int64_t stride_bytes, int a) { return (uintptr_t)p % a == 0 && stride_bytes % a == 0; }

// how many workgroups share rows that are `passes` passes of a workgroup long: until there are 4096 of them
unsigned share_rows(int64_t grid, int64_t passes) {
    const int64_t n = grid >= 4096 ? 1 : 4096 / grid;
    return (unsigned)(n < passes ? n : passes);
}

int rows_lanes(int64_t cols) { return cols <= 32 ? 4 : cols <= 64 ? 8 : 16; }
B8Rows rows_job(const void* x, int64_t rs, uint8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, int64_t rows, int64_t cols, int fmt) {
    const int lanes = rows_lanes(cols), gpb_log = lanes == 4 ? 6 : lanes == 8 ? 5 : 4;
    const int64_t KB = (cols + B8_BLK - 1) / B8_BLK;
    const int kgl = log2_up(KB, gpb_log);
    const int64_t rpb = 1 << (gpb_log - kgl);
    int64_t grid = (rows + 4 * rpb - 1) / (4 * rpb);
    if (grid < 1024) grid = (rows + rpb - 1) / rpb < 1024 ? (rows + rpb - 1) / rpb : 1024;      // few rows: spread them before stacking them
    if (grid > 65536) grid = 65536;
    return {x, rs, codes, ldc, scales, lds, rows, (int)cols, b8_pad(cols, ldc), kgl, fmt, (int)grid, (int)share_rows(grid, (KB + (1 << kgl) - 1) >> kgl)};
}

}  // namespace

extern "C" int ifl_block8_quantize(const void* x, int xtype, int64_t row_stride, int64_t col_stride, uint8_t* codes, int64_t ldc,
                                   uint8_t* scales, int64_t lds, int64_t rows, int64_t cols, int fmt, void* stream)
{
    IFL_CHECK_ARG(b8_type_ok(xtype), IFL_EINVAL, "block8_quantize: element type %d", xtype);
    IFL_CHECK_ARG(b8_fmt_ok(fmt), IFL_EINVAL, "block8_quantize: format %d", fmt);
    IFL_CHECK_ARG(rows >= 0 && cols >= 1 && cols <= 0x7ffffc00, IFL_EINVAL, "block8_quantize: %lld x %lld", (long long)rows, (long long)cols);
    if (rows == 0) return 0;
    const int KB = ifl_cdiv((int)cols, B8_BLK);
    IFL_CHECK_ARG(x && codes && scales, IFL_EINVAL, "block8_quantize: null pointer");
    IFL_CHECK_ARG(ldc >= cols && lds >= KB, IFL_EINVAL, "block8_quantize: row strides %lld, %lld for %lld columns", (long long)ldc, (long long)lds, (long long)cols);
    IFL_CHECK_ARG(col_stride == 1 || row_stride == 1 || rows == 1, IFL_EINVAL, "block8_quantize: strides %lld, %lld: one of them has to be 1", (long long)row_stride, (long long)col_stride);
    hipStream_t st = (hipStream_t)stream;
    if (col_stride != 1) {
        const int64_t gx = (rows + 63) / 64;
        IFL_CHECK_ARG(gx < 1 << 24 && gx * KB < 1 << 24, IFL_ENOTSUP, "block8_quantize: transposed %lld x %lld", (long long)rows, (long long)cols);
        const B8Cols q = {x, col_stride, codes, ldc, scales, lds, rows, (int)cols, b8_pad(cols, ldc), fmt};
        B8_DISPATCH(xtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(quantize_t_kernel<T>), dim3((unsigned)(gx * KB)), dim3(256), 0, st, q, (int)gx));
        IFL_LAUNCH_CHECK();
        return 0;
    }
    const B8Rows q = rows_job(x, row_stride, codes, ldc, scales, lds, rows, cols, fmt);
    const int lanes = rows_lanes(cols);
#define Q8_GO(L) hipLaunchKernelGGL(HIP_KERNEL_NAME(quantize_kernel<T, L>), dim3(q.gx * q.gy), dim3(256), 0, st, q)
    B8_DISPATCH(xtype, if (lanes == 4) Q8_GO(4); else if (lanes == 8) Q8_GO(8); else Q8_GO(16));
    IFL_LAUNCH_CHECK();
    return 0;
}

int b8_quantize2(const void* x, int xtype, int64_t x_rs, const void* w, int wtype, int64_t w_rs, uint8_t* xc, uint8_t* xs, uint8_t* wc, uint8_t* ws,
                 int64_t ldc, int64_t lds, int64_t M, int64_t N, int64_t K, void* stream)
{
    const B8Rows a = rows_job(x, x_rs, xc, ldc, xs, lds, M, K, IFL_Q_E4M3), b = rows_job(w, w_rs, wc, ldc, ws, lds, N, K, IFL_Q_E4M3);
    const int lanes = rows_lanes(K);
#define Q8_GO2(L) hipLaunchKernelGGL(HIP_KERNEL_NAME(quantize2_kernel<TX, T, L>), dim3(a.gx * a.gy + b.gx * b.gy), dim3(256), 0, (hipStream_t)stream, a, b)
    B8_DISPATCH(xtype, typedef T TX; B8_DISPATCH(wtype, if (lanes == 4) Q8_GO2(4); else if (lanes == 8) Q8_GO2(8); else Q8_GO2(16)));
    IFL_LAUNCH_CHECK();
    return 0;
}

extern "C" int ifl_block8_dequantize(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, int fmt, const float* chan,
                                     void* out, int otype, int64_t ldo, int64_t rows, int64_t cols, void* stream)
{
    IFL_CHECK_ARG(b8_type_ok(otype), IFL_EINVAL, "block8_dequantize: element type %d", otype);
    IFL_CHECK_ARG(b8_fmt_ok(fmt), IFL_EINVAL, "block8_dequantize: format %d", fmt);
    IFL_CHECK_ARG(rows >= 0 && cols >= 1 && cols <= 0x7ffffc00, IFL_EINVAL, "block8_dequantize: %lld x %lld", (long long)rows, (long long)cols);
    if (rows == 0) return 0;
    IFL_CHECK_ARG(codes && scales && out, IFL_EINVAL, "block8_dequantize: null pointer");
    IFL_CHECK_ARG(ldc >= cols && ldo >= cols && lds >= ifl_cdiv((int)cols, B8_BLK), IFL_EINVAL, "block8_dequantize: row strides");
    const int tl = log2_up((cols + 7) / 8, 8);
    const int64_t rpb = 256 >> tl;
    int64_t grid = (rows + 4 * rpb - 1) / (4 * rpb);
    if (grid < 1024) grid = (rows + rpb - 1) / rpb < 1024 ? (rows + rpb - 1) / rpb : 1024;
    if (grid > 65536) grid = 65536;
    const dim3 g2((unsigned)grid, share_rows(grid, (cols + (8 << tl) - 1) >> (3 + tl)));
    B8_DISPATCH(otype, hipLaunchKernelGGL(HIP_KERNEL_NAME(dequantize_kernel<T>), g2, dim3(256), 0, (hipStream_t)stream, codes, ldc, scales, lds, fmt, chan, (T*)out, ldo, rows, (int)cols, tl));
    IFL_LAUNCH_CHECK();
    return 0;
}

static int an_relu8_check(const char* what, int B, int h, int w, int C)
{
    IFL_CHECK_ARG(B >= 1 && h >= 1 && w >= 1, IFL_EINVAL, "%s: bad shape %d x %d x %d", what, B, h, w);
    IFL_CHECK_ARG(C >= 32 && C % 32 == 0 && C <= 1024, IFL_ENOTSUP, "%s: C=%d (a multiple of 32, at most 1024)", what, C);
    IFL_CHECK_ARG((int64_t)B * (h + 2) * (w + 2) <= 0x7fffffff - 65536 * 64, IFL_ENOTSUP, "%s: more than 2^31 pixels", what);
    return 0;
}

extern "C" int ifl_an_relu8_fwd(const float* x, float* y, uint8_t* codes, uint8_t* scales, const float* bias, const float* logs, int B,
                                int h, int w, int C, void* stream)
{
    if (int rc = an_relu8_check("an_relu8_fwd", B, h, w, C)) return rc;
    IFL_CHECK_ARG(x && y && codes && scales && bias && logs, IFL_EINVAL, "an_relu8_fwd: null pointer");
    IFL_CHECK_ARG(aligned(x, 0, 16) && aligned(y, 0, 16) && aligned(codes, 0, 8), IFL_EINVAL, "an_relu8_fwd: alignment");
    const uint32_t npx = (uint32_t)B * (h + 2) * (w + 2);
    const int lanes = C <= 32 ? 4 : C <= 64 ? 8 : 16, kg = ifl_cdiv(C, B8_BLK), ppb = 256 / lanes / kg;
    uint32_t grid = (npx + ppb - 1) / ppb;
    if (grid > 8192) grid = 8192;
#define AN8_GO(L) hipLaunchKernelGGL(HIP_KERNEL_NAME(an_relu8_fwd_kernel<L>), dim3(grid), dim3(256), 0, (hipStream_t)stream, x, y, codes, scales, bias, logs, npx, h + 2, w + 2, C, kg)
    if (lanes == 4) AN8_GO(4); else if (lanes == 8) AN8_GO(8); else AN8_GO(16);
    IFL_LAUNCH_CHECK();
    return 0;
}

static uint32_t an_relu8_px_per_block(uint32_t npx, int C)
{
    const uint32_t ppb = 256 / (C / 8);
    const uint32_t p = (npx + AN8_BLOCKS - 1) / AN8_BLOCKS;
    return (p + ppb - 1) / ppb * ppb;
}

extern "C" int64_t ifl_an_relu8_blocks(int B, int h, int w, int C)
{
    if (an_relu8_check("an_relu8_blocks", B, h, w, C)) return 0;
    const uint32_t npx = (uint32_t)B * (h + 2) * (w + 2), p = an_relu8_px_per_block(npx, C);
    return (npx + p - 1) / p;
}

extern "C" int ifl_an_relu8_bwd(const float* dy, const uint8_t* codes, const uint8_t* scales, const float* logs, float* dx, float* dbias,
                                float* dlogs, float* partials, int B, int h, int w, int C, void* stream)
{
    if (int rc = an_relu8_check("an_relu8_bwd", B, h, w, C)) return rc;
    IFL_CHECK_ARG(dy && codes && scales && logs && dx && dbias && dlogs && partials, IFL_EINVAL, "an_relu8_bwd: null pointer");
    IFL_CHECK_ARG(aligned(dy, 0, 16) && aligned(dx, 0, 16) && aligned(codes, 0, 8), IFL_EINVAL, "an_relu8_bwd: alignment");
    const uint32_t npx = (uint32_t)B * (h + 2) * (w + 2), ppx = an_relu8_px_per_block(npx, C);
    const int nblk = (int)((npx + ppx - 1) / ppx);
    const int sm = 256 / (C / 8) * 2 * C * 4;
    hipLaunchKernelGGL(an_relu8_bwd_kernel, dim3(nblk), dim3(256), sm, (hipStream_t)stream, dy, codes, scales, logs, dx, partials, npx, ppx, h + 2, w + 2, C);
    IFL_LAUNCH_CHECK();
    hipLaunchKernelGGL(an_relu8_reduce_kernel, dim3(2 * C / 16), dim3(1024), 0, (hipStream_t)stream, partials, nblk, logs, dbias, dlogs, C);
    IFL_LAUNCH_CHECK();
    return 0;
}

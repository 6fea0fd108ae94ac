// wgrad8.hip -- the weight gradient of a product whose input was kept in 8-bit blocks (block8.h):
//     dw[n][k] = chan[k] sum_m dy[m][n] code[m][k] 2^e[m][k / 128],      db[n] = sum_m dy[m][n]
// The sum runs over the rows of both operands, whose scales change from row to row, so the 8-bit instructions cannot apply them.
// A code times its scale is exact in bf16, and so is a bf16 gradient; a float16 gradient is the sum of two bf16 terms and a
// float32 one of three (its 24 significant bits in pieces of 8).  So every product goes exactly through
// v_mfma_f32_16x16x32_bf16 (one, two or three of them), which keeps 24 bits of the sums.
#include "block8.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

template <bool V> struct Flag { static constexpr bool value = V; };

struct WG8 {
    const void* dy; int64_t ldy;
    const uint8_t* codes; int64_t ldc;
    const uint8_t* scales; int64_t lds;
    const float* chan;
    void* dw; int64_t ldw; int dwtype;
    float* part; int split, steps;       // float32 partial sums [split][N][K], steps of 64 rows per part
    int64_t M; int N, K;
    int tiles_n, tiles_k, per_xcd;
    int ywide;                           // whole 16-byte loads of dy
};

// One, two or three bf16 terms whose sum is the value, as floats with 16 low zero bits: its leading 8 significant bits, the next 8,
// the rest.  What is not finite is the first term alone.
template <int NP>
__device__ __forceinline__ void wg8_terms(float x, float t[NP]) {
    if constexpr (NP == 1) t[0] = x;                                     // (from bf16)
    else {
        x = __builtin_canonicalizef(x);                                  // (a NaN has a high bit set)
        t[0] = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
        float r = x - t[0];
        r = r == r ? r : 0.f;
#pragma unroll
        for (int i = 1; i < NP; ++i) {
            t[i] = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
            r -= t[i];
        }
    }
}

template <class TW>
__device__ __forceinline__ void wg8_store16(TW* d, int left, const float v[16]) {
    if (left >= 16 && (uintptr_t)d % 16 == 0) { b8_store8<TW, true>(d, 8, v); b8_store8<TW, true>(d + 8, 8, v + 8); }
    else { b8_store8<TW, false>(d, left, v); if (left > 8) b8_store8<TW, false>(d + 8, left - 8, v + 8); }
}

// Workgroup = TN x TK of dw over a range of rows, MS at a time through two LDS buffers (rows of dy and of the restored codes as they
// lie in memory); the fragments, which run along m, come out of LDS transposed (ds_read_b64_tr_b16: 16 lanes read 4 rows of
// 16 values and get columns).  The instruction's first operand is the k side: a lane ends up with 4 neighbouring k of one n.
//
// A fragment read touches, per group of 16 lanes, 4 rows and 4 pieces of 8 bytes of each.  n side: the four pieces are one granule
// of 32 bytes, granule i of row m at place i ^ (m & 7).  k side: piece f % 4 of four neighbouring granules, so that a lane's four
// fragments are 16 neighbouring k; piece j of granule i of row m at piece j ^ (m & 3) of place i ^ (m & 4).  Both: no bank conflicts.
//
// bf16 gradients go straight to LDS (DMA); others, and whatever is not aligned or is cut off, through registers, loaded one
// step ahead.
template <class T, int NP, int TN, int TK, int WN, int WK, int MS, int FMT, bool DMA>
__global__ __launch_bounds__(64 * WN * WK)
void wgrad8_kernel(WG8 q)
{
    constexpr int NT = 64 * WN * WK, NF = TN / WN / 16, KF = TK / WK / 16;
    constexpr int GR = KF * MS / 32, D = 2, R = 4;          // groups of a step, x fragments read ahead and held
    constexpr int YROW = TN * 2, XROW = TK * 2, YPL = MS * YROW;       // bytes
    constexpr int YP = MS * TN / 8 / NT, XP = MS * TK / 16 / NT;     // pieces (8 values of dy, 16 codes) per thread
    static_assert(YP * NT * 8 == MS * TN && XP * NT * 16 == MS * TK && NF == 4 && (KF == 4 || KF == 8) && GR % R == 0, "");
    __shared__ __attribute__((aligned(16))) uint8_t y0[NP * YPL], y1[NP * YPL], x0[MS * XROW], x1[MS * XROW];
    const int all = q.tiles_n * q.tiles_k * q.split;
    const int id = (blockIdx.x & 7) * q.per_xcd + (blockIdx.x >> 3);
    if (id >= all) return;
    const int part = id / (q.tiles_n * q.tiles_k), tile = id - part * (q.tiles_n * q.tiles_k);
    const int tn = tile / q.tiles_k, tk = tile - tn * q.tiles_k;
    const int n0 = tn * TN, k0 = tk * TK;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int wk = wave % WK, wn = wave / WK;
    const int64_t mb = (int64_t)part * q.steps * MS, me = min(q.M, mb + (int64_t)q.steps * MS);
    const int steps = (int)((me - mb + MS - 1) / MS);

    // ---- staging: registers of the step that is on its way
    float yr[DMA ? 1 : YP][8];
    i32x4 xr[XP];
    int xs[XP];
    const T* dy = (const T*)q.dy;
    // (what is cut off is loaded from a place that exists and made zero when it is stored: a load that is used or branched around at
    // once would be waited for at once)
    auto y_load = [&](int64_t m0) {
        if constexpr (!DMA) {
            const T* base = dy + m0 * q.ldy;
            const int rows = (int)min((int64_t)MS, me - m0) - 1;
#pragma unroll
            for (int i = 0; i < YP; ++i) {
                const int p = i * NT + tid, n = n0 + p % (TN / 8) * 8;
                const uint32_t at = (uint32_t)(min(p / (TN / 8), rows) * (int)q.ldy);
                if (q.ywide) b8_load8<T, true>(base + (at + (n < q.N ? n : 0)), 8, yr[i]);
                else b8_load8<T, false>(base + (at + n), q.N - n, yr[i]);
            }
        }
    };
    // (fresh: an address or offset that is made again at its use instead of being held in registers of its own)
    auto fresh = [](auto x) { asm volatile("" : "+v"(x)); return x; };
    uint32_t ycol = 0;
    if constexpr (DMA) {
        const int r = tid / (TN / 8), c = tid % (TN / 8), s = ((c >> 1) ^ (r & 7)) * 2 + (c & 1);
        ycol = n0 + s * 8 < q.N ? s * 16 : 0;                            // (columns past the end: any, their results are not stored)
    }
    auto y_dma = [&](uint8_t* buf, int64_t m0) {
        if constexpr (DMA) {
            const uint8_t* base = (const uint8_t*)(dy + m0 * q.ldy + n0);
            const int rows = (int)min((int64_t)MS, me - m0) - 1;
#pragma unroll
            for (int i = 0; i < YP; ++i) {
                // a thread's pieces lie NT / (TN / 8) rows, a multiple of 8, apart: the same column in all of them
                static_assert(NT / (TN / 8) % 8 == 0, "");
                const uint32_t o = fresh(ycol) + (uint32_t)(min(fresh(tid) / (TN / 8) + i * (NT / (TN / 8)), rows) * 2 * (int)q.ldy);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + o),
                                                 (__attribute__((address_space(3))) void*)(buf + (i * NT + wave * 64) * 16), 16, 0, 0);
            }
        }
    };
    auto y_store = [&](uint8_t* buf, int64_t m0) {
        if constexpr (!DMA) {
#pragma unroll
            for (int i = 0; i < YP; ++i) {
                const int p = i * NT + tid, r = p / (TN / 8), c = p % (TN / 8);
                float t[8][NP];
                const bool in = m0 + r < me && n0 + c * 8 < q.N;
#pragma unroll
                for (int e = 0; e < 8; ++e) wg8_terms<NP>(in ? yr[i][e] : 0.f, t[e]);
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    i32x4 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (int)__builtin_amdgcn_perm(__float_as_uint(t[2 * e + 1][k]), __float_as_uint(t[2 * e][k]), 0x07060302u);   // the high halves
                    *(i32x4*)(buf + k * YPL + r * YROW + ((c >> 1) ^ (r & 7)) * 32 + (c & 1) * 16) = w;
                }
            }
        }
    };
    auto x_load = [&](int64_t m0) {
        const uint8_t *base = q.codes + m0 * q.ldc, *sbase = q.scales + m0 * q.lds;
        const int rows = (int)min((int64_t)MS, me - m0) - 1;
#pragma unroll
        for (int i = 0; i < XP; ++i) {
            const int p = i * NT + tid, k = k0 + p % (TK / 16) * 16;
            const int r = min(p / (TK / 16), rows), kc = k < q.K ? k : 0;
            xr[i] = *(const i32x4*)(base + (uint32_t)(r * (int)q.ldc + kc));
            xs[i] = sbase[(uint32_t)(r * (int)q.lds + kc / B8_BLK)];
        }
    };
    auto x_store = [&](uint8_t* buf, int64_t m0, int i) {
        {
            const int p = i * NT + tid, r = p / (TK / 16), c = p % (TK / 16);
            const int left = m0 + r < me ? q.K - k0 - c * 16 : 0;
            if (left < 16) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int l = left - 4 * e;
                    xr[i][e] = l >= 4 ? xr[i][e] : l <= 0 ? 0 : (int)((uint32_t)xr[i][e] & ((1u << 8 * l) - 1));
                }
                if (left <= 0) xs[i] = 127;
            }
            const bf16x8 lo = b8_bf16x8<FMT>(xr[i][0], xr[i][1], xs[i]), hi = b8_bf16x8<FMT>(xr[i][2], xr[i][3], xs[i]);
            const i32x4 a = __builtin_bit_cast(i32x4, lo), b = __builtin_bit_cast(i32x4, hi);
            const bool odd = r & 1;                                      // piece j at j ^ (r & 3): first within 16 bytes, then the halves
            const i32x4 u = {odd ? a[2] : a[0], odd ? a[3] : a[1], odd ? a[0] : a[2], odd ? a[1] : a[3]};
            const i32x4 v = {odd ? b[2] : b[0], odd ? b[3] : b[1], odd ? b[0] : b[2], odd ? b[1] : b[3]};
            uint8_t* d = buf + r * XROW + (c ^ (r & 4)) * 32;
            *(i32x4*)(d + (r & 2 ? 16 : 0)) = u;
            *(i32x4*)(d + (r & 2 ? 0 : 16)) = v;
        }
    };

    // ---- fragments
    const int mrow = 4 * g + (r16 >> 2), q4 = r16 & 3;
    // (places are XORs of a lane's own and of a fragment's constants)
    const int ya = mrow * YROW + ((wn * NF) ^ (mrow & 7)) * 32 + q4 * 8;
    const int xa = mrow * XROW + ((wk * KF + q4) ^ (mrow & 4)) * 32 + (mrow & 3) * 8;
    auto tr8 = [&](const uint8_t* a, int rows16) {
        const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + rows16));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto y_frag = [&](const uint8_t* buf, int pl, int f, int h) { return tr8(buf + (fresh(ya) ^ f << 5) + (pl * YPL + 32 * h * YROW), 16 * YROW); };
    auto x_frag = [&](const uint8_t* buf, int f, int h) { return tr8(buf + (fresh(xa) ^ ((f & 3) << 3 | (f >> 2) << 7)) + 32 * h * XROW, 16 * XROW); };
    // One step: GR groups (an x fragment with all y fragments of its 32 rows), x fragments read D groups ahead, y fragments 32 rows
    // ahead.  The next step's rows that come through registers are stored before group GR - D; those registers are then loaded
    // for the step after it.  At group GR - D everything of this step is in registers, and what goes straight to LDS has had the
    // time since the step's start: there the workgroup meets and goes on reading in the next step's buffer.
    f32x4 acc[KF][NF] = {};
    bf16x8 y[2][NF][NP], x[R];
    auto read_y = [&](const uint8_t* yb, int h, int o) {
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int k = 0; k < NP; ++k) y[o][f][k] = y_frag(yb, k, f, h);
    };
    auto products = [&](int i, int o) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int k = 0; k < NP; ++k)
                acc[i % KF][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i % R], y[o][f][k], acc[i % KF][f], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // (not __syncthreads: that would also wait for the loads on their way to registers)
    auto turn = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto landed = [&]() { if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
    const int64_t mlast = mb + (int64_t)(steps - 1) * MS;                // (behind the last step it is loaded again, unused)
    // behind a load that goes straight to LDS: rows past the end, made zero where this thread has just put them
    auto y_cut = [&](uint8_t* buf, int64_t m0) {
        if constexpr (DMA) {
            if (m0 + MS > me) {
#pragma unroll
                for (int i = 0; i < YP; ++i)
                    if (m0 + (i * NT + tid) / (TN / 8) >= me) *(i32x4*)(buf + (i * NT + tid) * 16) = i32x4{0, 0, 0, 0};
            }
        }
    };
    // (CHECK: the next step may be cut off.  In the others no branches: the compiler would move products past them.)
    auto step = [&](auto CHECK, auto ODD, uint8_t* yc, uint8_t* xc, uint8_t* yn, uint8_t* xn, int64_t m) {
        constexpr int H = MS / 32;
        const int64_t m1 = min(m + MS, mlast), m2 = min(m + 2 * MS, mlast);
        y_dma(yn, m1);
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            const int h = i / KF, o = (h + (H & 1) * ODD.value) & 1;
            constexpr int S = GR - D - 1;                                // the last group before the meeting
            if (i + D < GR) x[(i + D) % R] = x_frag(xc, (i + D) % KF, (i + D) / KF);
#pragma unroll
            for (int e = 0; e < XP; ++e) if (i == S - 2 * (XP - 1 - e)) x_store(xn, m1, e);
            if (i == S) {
                y_store(yn, m1);
                landed();
                if constexpr (CHECK.value) y_cut(yn, m1);
                x_load(m2);
                y_load(m2);
            }
            if (i == GR - D) {
                turn();
                read_y(yn, 0, o ^ 1);
            }
            if (i + D >= GR) x[(i + D) % R] = x_frag(xn, i + D - GR, 0);
            if (i % KF == KF - 4 && h + 1 < H) read_y(yc, h + 1, o ^ 1);
            products(i, o);
        }
    };

    x_load(mb);
    y_load(mb);
    y_dma(y0, mb);
    y_store(y0, mb);
#pragma unroll
    for (int e = 0; e < XP; ++e) x_store(x0, mb, e);
    landed();
    y_cut(y0, mb);
    x_load(min(mb + MS, mlast));
    y_load(min(mb + MS, mlast));
    turn();
    read_y(y0, 0, 0);
#pragma unroll
    for (int e = 0; e < D; ++e) x[e] = x_frag(x0, e, 0);
    int64_t m = mb;
    int s = 0;
    for (; s + 3 < steps; s += 2, m += 2 * MS) {
        step(Flag<false>(), Flag<false>(), y0, x0, y1, x1, m);
        step(Flag<false>(), Flag<true>(), y1, x1, y0, x0, m + MS);
    }
    step(Flag<true>(), Flag<false>(), y0, x0, y1, x1, m);
    if (s + 1 < steps) step(Flag<true>(), Flag<true>(), y1, x1, y0, x0, m + MS);
    if (s + 2 < steps) step(Flag<true>(), Flag<false>(), y0, x0, y1, x1, m + 2 * MS);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    const int kw = k0 + wk * KF * 16 + 16 * g, nw = n0 + wn * NF * 16 + r16;
#pragma unroll
    for (int h = 0; h < KF / 4; ++h) {
        const int k = kw + 64 * h;
        float ch[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) ch[e] = q.chan && k + e < q.K && q.split == 1 ? q.chan[k + e] : 1.f;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int n = nw + 16 * f;
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = acc[4 * h + e / 4][f][e % 4] * ch[e];
            if (n < q.N && k < q.K) {
                if (q.split > 1) {
                    float* d = q.part + ((int64_t)part * q.N + n) * q.K + k;
                    wg8_store16(d, q.K - k, v);
                } else {
                    const int64_t at = (int64_t)n * q.ldw + k;
                    if (q.dwtype == IFL_T_F32) wg8_store16((float*)q.dw + at, q.K - k, v);
                    else if (q.dwtype == IFL_T_BF16) wg8_store16((__bf16*)q.dw + at, q.K - k, v);
                    else wg8_store16((_Float16*)q.dw + at, q.K - k, v);
                }
            }
        }
    }
}

// dw = chan * sum of the parts, in order: four parts' values are on their way at a time
template <class TW, int V>
__global__ __launch_bounds__(256)
void wgrad8_join_kernel(WG8 q)
{
    typedef float FV __attribute__((ext_vector_type(V)));
    const int64_t nk = (int64_t)q.N * q.K;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < nk; i += (int64_t)gridDim.x * 256 * V) {
        FV t = 0.f;
        int s = 0;
        for (; s + 4 <= q.split; s += 4) {
            FV u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = *(const FV*)(q.part + (s + e) * nk + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) t += u[e];
        }
        for (; s < q.split; ++s) t += *(const FV*)(q.part + s * nk + i);
        const int n = (int)(i / q.K), k = (int)(i - (int64_t)n * q.K);
        TW* d = (TW*)q.dw + (int64_t)n * q.ldw + k;
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] = (TW)(q.chan ? t[e] * q.chan[k + e] : t[e]);
    }
}

template <class TW>
__global__ void fill_zero_kernel(TW* p, int64_t ld, int rows, int cols)
{
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)rows * cols; i += (int64_t)gridDim.x * blockDim.x) p[i / cols * ld + i % cols] = (TW)0.f;
}

// Column sums, first pass: a workgroup takes 64 columns of a range of rows, its four waves every fourth row.  part[blk][N]
template <class T>
__global__ __launch_bounds__(256)
void colsum_kernel(const T* __restrict__ dy, int64_t ldy, float* __restrict__ part, int64_t M, int N, int64_t rows_per)
{
    __shared__ float red[4][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6, n = blockIdx.x * 64 + c;
    const int64_t end = min(M, (int64_t)(blockIdx.y + 1) * rows_per);
    float t = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int64_t m = (int64_t)blockIdx.y * rows_per + r; m < end; m += 4) t += (float)dy[m * ldy + n];
    }
    red[r][c] = t;
    __syncthreads();
    if (r == 0 && n < N) part[(int64_t)blockIdx.y * N + n] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
}
// second pass: a workgroup takes 16 columns, 16 threads of each every 16th part, joined in LDS in a fixed order
template <class TW>
__global__ __launch_bounds__(256)
void colsum_join_kernel(const float* __restrict__ part, TW* __restrict__ db, int N, int parts)
{
    __shared__ float red[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
    float t = 0.f;
    if (n < N) {
#pragma unroll 4
        for (int s = r; s < parts; s += 16) t += part[(int64_t)s * N + n];
    }
    red[r][c] = t;
    __syncthreads();
    if (r == 0 && n < N) {
#pragma unroll
        for (int i = 1; i < 16; ++i) t += red[i][c];
        db[n] = (TW)t;
    }
}

// bf16 gradients: tiles of 256 x 256 for large layers if they can go straight to LDS, else 128 x 128; gradients of two or three terms,
// which take that much more LDS: 128 x 256.  The rows are split until about 256 workgroups are at work, each with two steps at
// least.
struct WPlan { int tn, tk, ms, split, steps, cs_parts; int64_t cs_rows; };
WPlan wg8_plan(int64_t M, int64_t N, int64_t K, int dytype, bool dma)
{
    WPlan p = {128, 128, 64, 1, 0, 1, 0};
    auto tiles = [&](int64_t a, int64_t b) { return ((N + a - 1) / a) * ((K + b - 1) / b); };
    if (dytype != IFL_T_BF16) { p.tk = 256; p.ms = 32; }
    else if (dma && tiles(256, 256) >= 32) p.tn = p.tk = 256;
    const int64_t steps = (M + p.ms - 1) / p.ms, n = tiles(p.tn, p.tk);
    int64_t s = n >= 192 ? 1 : 256 / n;
    if (s > steps / 2) s = steps / 2;
    if (s > 64) s = 64;
    if (s < 1) s = 1;
    p.steps = (int)((steps + s - 1) / s);
    p.split = p.steps ? (int)((steps + p.steps - 1) / p.steps) : 1;
    const int64_t cols = (N + 63) / 64;
    int64_t c = 512 / cols;
    if (c > M / 32) c = M / 32;
    if (c > 256) c = 256;
    if (c < 1) c = 1;
    p.cs_rows = (M + c - 1) / c;
    p.cs_parts = p.cs_rows ? (int)((M + p.cs_rows - 1) / p.cs_rows) : 1;
    return p;
}

}  // namespace

extern "C" int64_t ifl_block8_wgrad_scratch_floats(int64_t M, int64_t N, int64_t K, int dytype)
{
    if (M < 1 || N < 1 || K < 0) return 0;
    const WPlan p = wg8_plan(M, N, K > 0 ? K : 1, dytype, false), d = wg8_plan(M, N, K > 0 ? K : 1, dytype, true);
    const int64_t s = p.split > d.split ? p.split : d.split;
    return (K > 0 && s > 1 ? s * N * K : 0) + (int64_t)p.cs_parts * N;
}

extern "C" int ifl_block8_wgrad(const void* dy, int dytype, int64_t ldy, const uint8_t* codes, int64_t ldc, const uint8_t* scales,
                                int64_t lds, int fmt, const float* chan, void* dw, int dwtype, int64_t ldw, void* db, int dbtype,
                                float* scratch, int64_t M, int64_t N, int64_t K, void* stream)
{
    IFL_CHECK_ARG(b8_fmt_ok(fmt) && b8_type_ok(dytype) && (!dw || b8_type_ok(dwtype)) && (!db || b8_type_ok(dbtype)), IFL_EINVAL, "block8_wgrad: types");
    IFL_CHECK_ARG(M >= 0 && N >= 1 && (K >= 1 || !dw), IFL_EINVAL, "block8_wgrad: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG(N <= 0x3fffff && K <= 0x3fffff && M < ((int64_t)1 << 40), IFL_ENOTSUP, "block8_wgrad: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG((dw || db) && (M == 0 || (dy && scratch)) && (M == 0 || !dw || (codes && scales)), IFL_EINVAL, "block8_wgrad: null pointer");
    IFL_CHECK_ARG((M <= 1 || ldy >= N) && (!dw || ((M <= 1 || (ldc >= K && lds >= ifl_cdiv((int)K, B8_BLK))) && ldw >= K)), IFL_EINVAL, "block8_wgrad: row strides");
    IFL_CHECK_ARG(!dw || M == 0 || ((uintptr_t)codes % 16 == 0 && (M == 1 || ldc % 16 == 0)), IFL_EINVAL, "block8_wgrad: codes in rows of whole, aligned 16 bytes");
    IFL_CHECK_ARG(ldy < (1 << 23) && ldc < (1 << 23) && lds < (1 << 23), IFL_ENOTSUP, "block8_wgrad: rows of %lld gradients, %lld codes", (long long)ldy, (long long)ldc);
    hipStream_t st = (hipStream_t)stream;
    if (M == 0) {
        if (dw) { B8_DISPATCH(dwtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(fill_zero_kernel<T>), dim3(256), dim3(256), 0, st, (T*)dw, ldw, (int)N, (int)K)); IFL_LAUNCH_CHECK(); }
        if (db) { B8_DISPATCH(dbtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(fill_zero_kernel<T>), dim3(16), dim3(256), 0, st, (T*)db, N, 1, (int)N)); IFL_LAUNCH_CHECK(); }
        return 0;
    }
    const bool ywide = (uintptr_t)dy % 16 == 0 && (M == 1 || ldy * b8_size(dytype) % 16 == 0) && N % 8 == 0;
    const bool dma = dytype == IFL_T_BF16 && ywide;
    const WPlan p = wg8_plan(M, N, K > 0 ? K : 1, dytype, dma);
    if (dw) {
        WG8 q = {};
        q.dy = dy; q.ldy = ldy; q.codes = codes; q.ldc = ldc; q.scales = scales; q.lds = lds; q.chan = chan; q.dw = dw; q.ldw = ldw;
        q.dwtype = dwtype; q.part = scratch; q.split = p.split; q.steps = p.steps; q.M = M; q.N = (int)N; q.K = (int)K;
        q.tiles_n = (int)((N + p.tn - 1) / p.tn); q.tiles_k = (int)((K + p.tk - 1) / p.tk);
        q.per_xcd = (q.tiles_n * q.tiles_k * p.split + 7) / 8;
        q.ywide = ywide;
        const dim3 grid(8 * q.per_xcd);
#define WG8_K(T, NP, TN, TK, WN, WK, MS, F, D) hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_kernel<T, NP, TN, TK, WN, WK, MS, F, D>), grid, dim3(64 * WN * WK), 0, st, q)
#define WG8_F(F) do { \
            if (dytype == IFL_T_F32) WG8_K(float, 3, 128, 256, 2, 4, 32, F, false); \
            else if (dytype == IFL_T_F16) WG8_K(_Float16, 2, 128, 256, 2, 4, 32, F, false); \
            else if (p.tn == 256) WG8_K(__bf16, 1, 256, 256, 4, 2, 64, F, true); \
            else { if (dma) WG8_K(__bf16, 1, 128, 128, 2, 2, 64, F, true); else WG8_K(__bf16, 1, 128, 128, 2, 2, 64, F, false); } } while (0)
        if (fmt == IFL_Q_E4M3) WG8_F(0); else WG8_F(1);
        IFL_LAUNCH_CHECK();
        if (p.split > 1) {
            // four values per thread where the parts are large, else one: the parts' loads are what it waits for
            const bool v4 = K % 4 == 0 && N * K >= 1 << 18;
            const int64_t jobs = (v4 ? N * K / 4 : N * K) / 256 + 1;
            const unsigned jg = (unsigned)(jobs < 4096 ? jobs : 4096);
            B8_DISPATCH(dwtype, if (v4) hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_join_kernel<T, 4>), dim3(jg), dim3(256), 0, st, q);
                        else hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_join_kernel<T, 1>), dim3(jg), dim3(256), 0, st, q));
            IFL_LAUNCH_CHECK();
        }
    }
    if (db) {
        float* part = scratch + (dw && p.split > 1 ? (int64_t)p.split * N * K : 0);
        const unsigned cols = (unsigned)((N + 63) / 64);
        B8_DISPATCH(dytype, hipLaunchKernelGGL(HIP_KERNEL_NAME(colsum_kernel<T>), dim3(cols, p.cs_parts), dim3(256), 0, st, (const T*)dy, ldy, part, M, (int)N, p.cs_rows));
        IFL_LAUNCH_CHECK();
        B8_DISPATCH(dbtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(colsum_join_kernel<T>), dim3((unsigned)((N + 15) / 16)), dim3(256), 0, st, part, (T*)db, (int)N, p.cs_parts));
        IFL_LAUNCH_CHECK();
    }
    return 0;
}

// wgrad8.hip -- the weight gradient of a product whose input was kept in 8-bit blocks (block8.h):
//     dw[n][k] = chan[k] sum_m dy[m][n] code[m][k] 2^e[m][k / 128],      db[n] = sum_m dy[m][n]
// The sum runs over the rows of both operands, whose scales change from row to row, so the 8-bit instructions cannot apply them.
// A code times its scale is exact in bf16, and so is a bf16 gradient; a float16 gradient is the sum of two bf16 terms and a
// float32 one of three (its 24 significant bits in pieces of 8).  So every product goes exactly through
// v_mfma_f32_16x16x32_bf16 (one, two or three of them), which keeps 24 bits of the sums.
//
// Three launches: codes restored to bf16 and gradients split into their terms, with dy's column sums (memory-bound, one pass); the
// product; the parts of a split sum joined.  Restoring and splitting inside the product, where every workgroup of a row of
// tiles repeats it, was the slower way: its arithmetic does not fit beside the matrix instructions (2048 x 2048 over 65536 rows,
// bf16: 615 us with it, 390 without; float32: 1644 and 841).
#include "block8.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

struct WG8 {
    // the caller's
    const void* dy; int64_t ldy;
    const uint8_t* codes; int64_t ldc;
    const uint8_t* scales; int64_t lds;
    const float* chan;
    void* dw; int64_t ldw; int dwtype;
    void* db; int dbtype;
    int64_t M; int N, K, fmt;
    int want_x;                          // 0: column sums alone
    uint8_t *gc, *gs; int64_t ldgc, ldgs; int gfmt;  // where dy's own 8-bit blocks go, if they are wanted
    // scratch
    uint16_t* xb; int64_t kp;            // restored codes [rows up to a multiple of 32][kp], zeros behind row M
    uint16_t* yb; int64_t np, yplane;    // terms of dy [NP][rows up to a multiple of 32][np]; of bf16 read in place: its last M % 32 rows
    int in_place;
    float* part; int split, steps;       // float32 partial sums [split][N][K], steps of 32 rows per part
    float* cs; int cs_parts; int64_t cs_rows, y_row0;        // partial column sums [cs_parts][N], of cs_rows rows from y_row0 on
    int tiles_n, tiles_k, per_xcd;
    int x_blocks, x_tpr_log, y_cols, y_tpr_log;      // first launch: workgroups that restore codes, threads along a row; ranges of columns of dy, threads along a row
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
__device__ __forceinline__ void wg8_store4(TW* d, int left, const float v[4]) {
    typedef TW TW4 __attribute__((ext_vector_type(4)));
    if (left >= 4 && (uintptr_t)d % sizeof(TW4) == 0) {
        TW4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (TW)v[e];
        *(TW4*)d = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < left) d[e] = (TW)v[e];
    }
}

constexpr int MS = 32;                                                  // rows per step: the depth of one product

// ------------------------------------------------------------------------------------------------ first launch
// Workgroups 0 .. x_blocks - 1 restore codes, 8 a thread.  The others take up to 256 columns (8 a thread) of cs_rows rows of dy, with
// column sums on the way that are joined in LDS in a fixed order.  QUANT: they also put dy into 8-bit blocks (for the layer's
// other product), which saves a pass over it (16384 x 2048, both operands, bf16: 46 us instead of 25 + 33).
template <class T, int NP, bool VEC, bool QUANT>
__global__ __launch_bounds__(256)
void wgrad8_prepare_kernel(WG8 q)
{
    const int64_t mp = (q.M + MS - 1) / MS * MS;
    if ((int)blockIdx.x < q.x_blocks) {
        const int rpb = 256 >> q.x_tpr_log;
        const int64_t step = (int64_t)q.x_blocks * rpb;
        constexpr int U = 4;
        for (int64_t r0 = (int64_t)blockIdx.x * rpb + (threadIdx.x >> q.x_tpr_log); r0 < mp; r0 += U * step) {
            for (int c = (threadIdx.x & ((1 << q.x_tpr_log) - 1)) * 8; c < q.kp; c += 8 << q.x_tpr_log) {
                i32x2 w[U];
                int sb[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t r = r0 + u * step;
                    const bool in = r < q.M && c < q.K;                  // (rows are whole 16 bytes)
                    w[u] = in ? *(const i32x2*)(q.codes + r * q.ldc + c) : i32x2{0, 0};
                    sb[u] = in ? q.scales[r * q.lds + c / B8_BLK] : 127;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t r = r0 + u * step;
                    if (r < mp) *(bf16x8*)(q.xb + r * q.kp + c) = q.fmt == IFL_Q_E4M3 ? b8_bf16x8<IFL_Q_E4M3>(w[u][0], w[u][1], sb[u]) : b8_bf16x8<IFL_Q_E5M2>(w[u][0], w[u][1], sb[u]);
                }
            }
        }
        return;
    }
    __shared__ float red[256 * 8 + 256];
    const int b = blockIdx.x - q.x_blocks, part = b / q.y_cols, cb = b - part * q.y_cols;
    const int tpr = 1 << q.y_tpr_log, rpp = 256 >> q.y_tpr_log, rl = threadIdx.x >> q.y_tpr_log;
    const int c0 = cb * 8 * tpr, c = c0 + (threadIdx.x & (tpr - 1)) * 8;
    const int64_t first = q.y_row0 + (int64_t)part * q.cs_rows, last = min(mp, first + q.cs_rows);
    const int64_t m32 = q.M / MS * MS;
    const T* dy = (const T*)q.dy;
    float sum[8] = {};
    for (int64_t r0 = first + rl; r0 < last; r0 += 4 * rpp) {
        float v[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = r0 + u * rpp;
            b8_load8<T, VEC>(dy + (r < q.M ? r : 0) * q.ldy + c, r < q.M && r < last ? q.N - c : 0, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = r0 + u * rpp;
            if (r >= last) break;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v[u][i];
            if constexpr (QUANT) {
                int sb;                                                  // (of a block: 16 threads, or the 4 or 8 of a short row)
                const i32x2 w = b8_quantize8<16>(v[u], q.gfmt, sb, tpr);
                if (r < q.M) {
                    if (c < q.ldgc) *(i32x2*)(q.gc + r * q.ldgc + c) = w;
                    if (c < q.N && (c & (B8_BLK - 1)) == 0) q.gs[r * q.ldgs + c / B8_BLK] = (uint8_t)sb;
                }
            }
            // terms of what is not read in place: everything, or the rows behind the last 32 whole ones
            if (q.want_x && c < q.np && (!q.in_place || r >= m32)) {
                float t[8][NP];
#pragma unroll
                for (int i = 0; i < 8; ++i) wg8_terms<NP>(v[u][i], t[i]);
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    i32x4 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (int)__builtin_amdgcn_perm(__float_as_uint(t[2 * e + 1][k]), __float_as_uint(t[2 * e][k]), 0x07060302u);   // the high halves
                    *(i32x4*)(q.yb + k * q.yplane + (q.in_place ? r - m32 : r) * q.np + c) = w;
                }
            }
        }
    }
    if (!q.db) return;
    const int pitch = 8 * tpr + 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) red[rl * pitch + (threadIdx.x & (tpr - 1)) * 8 + i] = sum[i];
    __syncthreads();
    if ((int)threadIdx.x < 8 * tpr && c0 + (int)threadIdx.x < q.N) {
        float t = red[threadIdx.x];
        for (int i = 1; i < rpp; ++i) t += red[i * pitch + threadIdx.x];
        q.cs[(int64_t)part * q.N + c0 + threadIdx.x] = t;
    }
}

// ------------------------------------------------------------------------------------------------ the product
// Workgroup = TN x TK of dw over a range of rows, 32 at a time.  Rows of both operands lie in LDS as they do in memory; the fragments,
// which run along m, come out of LDS transposed (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 values and get columns).  The
// instruction's first operand is the k side: a lane ends up with 4 neighbouring k of one n.
//
// A fragment read touches, per group of 16 lanes, 4 rows and 4 pieces of 8 bytes of each: one granule of 32 bytes, granule i of row m at
// place i ^ (m & 7), which leaves no bank conflicts.  Loads go straight to LDS in lane order, so it is the source that is permuted.
//
// A step is a term of dy with 32 rows (the terms of the same rows follow one another and share the k side's fragments).  It has two
// phases.  MEM: the loads of the step three ahead are issued (rings of four), this step's fragments are read.  COMPUTE: its
// products, nothing else.  With 8 waves the second four run one phase behind the first, so that of the two waves on a SIMD one
// multiplies while the other one reads: the workgroup meets after every phase.  Three steps are about 1.5 us, what rows that
// all workgroups ask for at the same time take to come from memory.
template <int V> struct Int { static constexpr int value = V; };

template <int NP, int TN, int TK, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK)
void wgrad8_kernel(WG8 q)
{
    constexpr int NW = WN * WK, NT = 64 * NW, NF = TN / WN / 16, KF = TK / WK / 16;
    constexpr bool TURNS = NW == 8;
    constexpr int YROW = TN * 2, XROW = TK * 2, YB = MS * YROW, XB = MS * XROW;          // bytes
    constexpr int YP = YB / 16 / NT, XP = XB / 16 / NT;                  // 16-byte pieces per thread
    static_assert(YP == 2 && XP == 2 && NF == 4 && (KF == 4 || KF == 8), "");
    __shared__ __attribute__((aligned(16))) uint8_t ys[4 * YB], xs[4 * XB];
    const int all = q.tiles_n * q.tiles_k * q.split;
    const int id = (blockIdx.x & 7) * q.per_xcd + (blockIdx.x >> 3);
    if (id >= all) return;
    const int part = __builtin_amdgcn_readfirstlane(id / (q.tiles_n * q.tiles_k)), tile = id - part * (q.tiles_n * q.tiles_k);
    const int tn = __builtin_amdgcn_readfirstlane(tile / q.tiles_k), tk = tile - tn * q.tiles_k;
    const int n0 = tn * TN, k0 = tk * TK;
    const uint32_t tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int wk = wave % WK, wn = wave / WK;
    const int s0 = part * q.steps, rows_steps = (int)((q.M + MS - 1) / MS), steps = (min(rows_steps, s0 + q.steps) - s0) * NP;
    // (fresh: an address or offset that is made again at its use instead of being held in registers of its own)
    auto fresh = [](auto x) { asm volatile("" : "+v"(x)); return x; };

    // ---- loads: 64 lanes' 16 bytes each, from base + their offsets, to LDS in lane order.  By hand: the compiler waits for all loads
    // wherever it thinks that one might have written what is read.  (The instruction reads M0 one wait state after it is written.)
    auto to_lds = [&](const void* base, uint32_t o, const uint8_t* to) {
        const uint32_t at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)to;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(at), "v"(o), "s"(base) : "memory", "m0");
    };
    // a thread's pieces: a column (past the end: any, its results are not stored), rows that lie a multiple of 8 apart
    constexpr int YSTEP = NT / (TN / 8), XSTEP = NT / (TK / 8);
    static_assert(YSTEP % 8 == 0 && XSTEP % 8 == 0, "");
    const int64_t ldy = q.in_place ? q.ldy : q.np;
    uint32_t yo, xo;
    {
        const int r = tid / (TN / 8), c = ((tid % (TN / 8) >> 1) ^ (r & 7)) * 2 + (tid & 1);
        yo = (n0 + c * 8 < q.np ? n0 * 2 + c * 16 : 0) + (uint32_t)(r * 2 * (int)ldy);
        const int rx = tid / (TK / 8), cx = ((tid % (TK / 8) >> 1) ^ (rx & 7)) * 2 + (tid & 1);
        xo = (k0 + cx * 8 < q.kp ? k0 * 2 + cx * 16 : 0) + (uint32_t)(rx * 2 * (int)q.kp);
    }
    const int m32 = (int)(q.M / MS);
    // step t: term PL of rows 32 (s0 + t / NP) on; behind the last step it is loaded again, unused
    auto load = [&](auto PL, int t, int ry, int rx) {
        const int s = s0 + min(t, steps - 1) / NP;
        // of rows read in place the last ones, which do not fill a step, were copied to a place with zeros behind them: np apart there
        const uint16_t* y = q.in_place ? (const uint16_t*)q.dy + (int64_t)s * MS * ldy : q.yb + PL.value * q.yplane + (int64_t)s * MS * ldy;
        const bool cut = q.in_place && s >= m32;
        y = cut ? q.yb : y;
        const int dl = cut ? (int)(q.np - ldy) * 2 : 0;                  // (rows of the copy are closer together)
#pragma unroll
        for (int i = 0; i < YP; ++i)
            to_lds(y, fresh(yo) + (uint32_t)(((int)(fresh(tid) / (TN / 8)) + i * YSTEP) * dl + i * YSTEP * 2 * (int)ldy), ys + ry * YB + (i * NT + wave * 64) * 16);
        if constexpr (PL.value == 0) {
            const uint16_t* x = q.xb + (int64_t)s * MS * q.kp;
#pragma unroll
            for (int i = 0; i < XP; ++i) to_lds(x, fresh(xo) + (uint32_t)(i * XSTEP * 2 * (int)q.kp), xs + rx * XB + (i * NT + wave * 64) * 16);
        }
    };

    // ---- fragments (places are XORs of a lane's own and of a fragment's constants)
    const int mrow = 4 * g + (r16 >> 2), q4 = r16 & 3;
    const int ya = mrow * YROW + ((wn * NF) ^ (mrow & 7)) * 32 + q4 * 8, xa = mrow * XROW + ((wk * KF) ^ (mrow & 7)) * 32 + q4 * 8;
    auto tr8 = [&](const uint8_t* a, int rows16) {
        const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + rows16));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    f32x4 acc[KF][NF] = {};
    bf16x8 y[NF], x[KF];
    // (not __syncthreads: that would also wait for the loads that are on their way)
    auto meet = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // one step: term PL of step t; ry, rx its places in the rings.  No branches inside: the compiler would move products past them.
    auto step = [&](auto PL, int t, int ry, int rx) {
        constexpr int P3 = (PL.value + 3) % NP;
        constexpr int AHEAD = (PL.value + 3) / NP;                       // row steps that term lies ahead
        load(Int<P3>(), t + 3, (ry + 3) & 3, (rx + AHEAD) & 3);
#pragma unroll
        for (int f = 0; f < NF; ++f) y[f] = tr8(ys + ry * YB + (fresh(ya) ^ f << 5), 16 * YROW);
        if constexpr (PL.value == 0) {
#pragma unroll
            for (int f = 0; f < KF; ++f) x[f] = tr8(xs + rx * XB + (fresh(xa) ^ f << 5), 16 * XROW);
        }
        // the next step's loads have come: those of the two behind it are newer
        constexpr int NEWER = YP * 2 + XP * (((PL.value + 2) % NP == 0) + (P3 == 0));
        if constexpr (NEWER == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else if constexpr (NEWER == 6) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
        else { static_assert(NEWER == 4, ""); asm volatile("s_waitcnt vmcnt(4)" ::: "memory"); }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        meet();
#pragma unroll
        for (int i = 0; i < KF; ++i)
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[i], y[f], acc[i][f], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (TURNS) meet();
    };

    load(Int<0>(), 0, 0, 0);
    load(Int<1 % NP>(), 1, 1, 1 / NP);
    load(Int<2 % NP>(), 2, 2, 2 / NP);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    meet();
    if (TURNS && wave >= NW / 2) meet();
    for (int t = 0, r = 0; t < steps; t += NP, ++r) {
        step(Int<0>(), t, t & 3, r & 3);
        if constexpr (NP > 1) step(Int<1>(), t + 1, (t + 1) & 3, r & 3);
        if constexpr (NP > 2) step(Int<2>(), t + 2, (t + 2) & 3, r & 3);
    }
    if (TURNS && wave < NW / 2) meet();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    const int kw = k0 + wk * KF * 16 + 4 * g, nw = n0 + wn * NF * 16 + r16;
#pragma unroll
    for (int i = 0; i < KF; ++i) {
        const int k = kw + 16 * i;
        float ch[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ch[e] = q.chan && k + e < q.K && q.split == 1 ? q.chan[k + e] : 1.f;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int n = nw + 16 * f;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][f][e] * ch[e];
            if (n < q.N && k < q.K) {
                if (q.split > 1) wg8_store4(q.part + ((int64_t)part * q.N + n) * q.K + k, q.K - k, v);
                else {
                    const int64_t at = (int64_t)n * q.ldw + k;
                    if (q.dwtype == IFL_T_F32) wg8_store4((float*)q.dw + at, q.K - k, v);
                    else if (q.dwtype == IFL_T_BF16) wg8_store4((__bf16*)q.dw + at, q.K - k, v);
                    else wg8_store4((_Float16*)q.dw + at, q.K - k, v);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ last launch
// Workgroups 0 .. join_blocks - 1: dw = chan * sum of the parts, V values a thread, four parts' values on their way at a time.  A small dw
// has few threads: then 16 of them share a value's parts (ACROSS), each takes every 16th, and the sums meet in LDS.  The
// others: db, 16 columns each, shared in the same way.  All orders are fixed.
template <class TW, class TB, int V, bool ACROSS>
__global__ __launch_bounds__(256)
void wgrad8_finish_kernel(WG8 q, int join_blocks)
{
    typedef float FV __attribute__((ext_vector_type(V)));
    __shared__ FV red[ACROSS ? 16 * 17 : 1];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    if ((int)blockIdx.x < join_blocks) {
        const int64_t nk = (int64_t)q.N * q.K;
        const int first = ACROSS ? r : 0, by = ACROSS ? 16 : 1;
        const int64_t stride = (int64_t)join_blocks * (ACROSS ? 16 : 256) * V;
        for (int64_t i0 = (int64_t)blockIdx.x * (ACROSS ? 16 : 256) * V; i0 < nk; i0 += stride) {
            const int64_t i = i0 + (ACROSS ? c : (int)threadIdx.x) * V;
            FV t = 0.f;
            if (i < nk) {
                int s = first;
                for (; s + 3 * by < q.split; s += 4 * by) {
                    FV u[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] = *(const FV*)(q.part + (s + e * by) * nk + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) t += u[e];
                }
                for (; s < q.split; s += by) t += *(const FV*)(q.part + s * nk + i);
            }
            if constexpr (ACROSS) {
                __syncthreads();
                red[r * 17 + c] = t;
                __syncthreads();
                if (r) continue;
#pragma unroll
                for (int e = 1; e < 16; ++e) t += red[e * 17 + c];
            }
            if (i >= nk) continue;
            const int n = (int)(i / q.K), k = (int)(i - (int64_t)n * q.K);
            TW* d = (TW*)q.dw + (int64_t)n * q.ldw + k;
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = (TW)(q.chan ? t[e] * q.chan[k + e] : t[e]);
        }
        return;
    }
    __shared__ float cred[16][17];
    const int n = ((int)blockIdx.x - join_blocks) * 16 + c;
    float t = 0.f;
    if (n < q.N) {
#pragma unroll 4
        for (int s = r; s < q.cs_parts; s += 16) t += q.cs[(int64_t)s * q.N + n];
    }
    cred[r][c] = t;
    __syncthreads();
    if (r == 0 && n < q.N) {
#pragma unroll
        for (int i = 1; i < 16; ++i) t += cred[i][c];
        ((TB*)q.db)[n] = (TB)t;
    }
}

template <class TW>
__global__ void fill_zero_kernel(TW* p, int64_t ld, int rows, int cols)
{
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)rows * cols; i += (int64_t)gridDim.x * blockDim.x) p[i / cols * ld + i % cols] = (TW)0.f;
}

// Tiles of 256 x 256 for large layers, else 128 x 128.  The rows are split until the card is full (one workgroup on a CU of the
// large tiles, two of the small ones), each with four steps at least.
struct WPlan { int tile, split, steps, cs_parts, y_tpr_log; int64_t cs_rows, kp, np, x_floats, y_floats, part_floats, cs_floats; bool in_place; };
WPlan wg8_plan(int64_t M, int64_t N, int64_t K, int dytype, bool aligned)
{
    WPlan p = {};
    auto tiles = [&](int64_t t) { return ((N + t - 1) / t) * ((K + t - 1) / t); };
    const int terms = dytype == IFL_T_F32 ? 3 : dytype == IFL_T_F16 ? 2 : 1;
    p.tile = tiles(256) >= 32 ? 256 : 128;
    const int64_t steps = (M + MS - 1) / MS, n = K > 0 ? tiles(p.tile) : 1;
    const int64_t full = p.tile == 256 ? 256 : 512;
    int64_t s = 4 * n >= 3 * full ? 1 : full / n;
    if (s > steps * terms / 4) s = steps * terms / 4;
    if (s > 256) s = 256;
    if (s < 1) s = 1;
    p.steps = (int)((steps + s - 1) / s);
    p.split = (int)((steps + p.steps - 1) / p.steps);
    // column sums (and terms): about 1024 workgroups, 32 rows each at least
    p.y_tpr_log = 2;
    while (p.y_tpr_log < 5 && (8 << p.y_tpr_log) < N) ++p.y_tpr_log;
    const int64_t cols = (N + (8 << p.y_tpr_log) - 1) / (8 << p.y_tpr_log);
    int64_t c = 1024 / cols;
    if (c > steps) c = steps;
    if (c > 512) c = 512;
    if (c < 1) c = 1;
    p.cs_rows = (steps + c - 1) / c * MS;
    p.cs_parts = (int)((steps * MS + p.cs_rows - 1) / p.cs_rows);
    p.in_place = dytype == IFL_T_BF16 && aligned;
    p.kp = (K + 7) / 8 * 8;
    p.np = (N + 7) / 8 * 8;
    auto up = [](int64_t floats) { return (floats + 3) / 4 * 4; };
    p.x_floats = K > 0 ? up(steps * MS * p.kp / 2) : 0;
    p.y_floats = K > 0 ? up((p.in_place ? MS : terms * steps * MS) * p.np / 2) : 0;
    p.part_floats = K > 0 && p.split > 1 ? up(p.split * N * K) : 0;
    p.cs_floats = up(p.cs_parts * N);
    return p;
}

}  // namespace

extern "C" int64_t ifl_block8_wgrad_scratch_floats(int64_t M, int64_t N, int64_t K, int dytype)
{
    if (M < 1 || N < 1 || K < 0 || !b8_type_ok(dytype)) return 0;
    const WPlan p = wg8_plan(M, N, K, dytype, false);
    return p.x_floats + p.y_floats + p.part_floats + p.cs_floats;
}

extern "C" int ifl_block8_wgrad(const void* dy, int dytype, int64_t ldy, const uint8_t* codes, int64_t ldc, const uint8_t* scales,
                                int64_t lds, int fmt, const float* chan, void* dw, int dwtype, int64_t ldw, void* db, int dbtype,
                                float* scratch, int64_t M, int64_t N, int64_t K, void* stream)
{
    return b8_wgrad(3, nullptr, dy, dytype, ldy, codes, ldc, scales, lds, fmt, chan, dw, dwtype, ldw, db, dbtype, scratch, M, N, K, stream);
}

int b8_wgrad(int todo, const B8Quant* quant, const void* dy, int dytype, int64_t ldy, const uint8_t* codes, int64_t ldc, const uint8_t* scales,
             int64_t lds, int fmt, const float* chan, void* dw, int dwtype, int64_t ldw, void* db, int dbtype, float* scratch, int64_t M,
             int64_t N, int64_t K, void* stream)
{
    IFL_CHECK_ARG(b8_fmt_ok(fmt) && b8_type_ok(dytype) && (!dw || b8_type_ok(dwtype)) && (!db || b8_type_ok(dbtype)), IFL_EINVAL, "block8_wgrad: types");
    IFL_CHECK_ARG(M >= 0 && N >= 1 && (K >= 1 || !dw), IFL_EINVAL, "block8_wgrad: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG(N <= 0x3fffff && K <= 0x3fffff && M < ((int64_t)1 << 36), IFL_ENOTSUP, "block8_wgrad: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG((dw || db) && (M == 0 || (dy && scratch)) && (M == 0 || !dw || (codes && scales)), IFL_EINVAL, "block8_wgrad: null pointer");
    IFL_CHECK_ARG((M <= 1 || ldy >= N) && (!dw || ((M <= 1 || (ldc >= K && lds >= ifl_cdiv((int)K, B8_BLK))) && ldw >= K)), IFL_EINVAL, "block8_wgrad: row strides");
    IFL_CHECK_ARG(!dw || M == 0 || ((uintptr_t)codes % 16 == 0 && (M == 1 || ldc % 16 == 0)), IFL_EINVAL, "block8_wgrad: codes in rows of whole, aligned 16 bytes");
    IFL_CHECK_ARG(M == 0 || (uintptr_t)scratch % 16 == 0, IFL_EINVAL, "block8_wgrad: scratch");
    IFL_CHECK_ARG(ldy < (1 << 23), IFL_ENOTSUP, "block8_wgrad: rows of %lld gradients", (long long)ldy);
    hipStream_t st = (hipStream_t)stream;
    if (M == 0) {
        if (!(todo & 2)) return 0;
        if (dw) { B8_DISPATCH(dwtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(fill_zero_kernel<T>), dim3(256), dim3(256), 0, st, (T*)dw, ldw, (int)N, (int)K)); IFL_LAUNCH_CHECK(); }
        if (db) { B8_DISPATCH(dbtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(fill_zero_kernel<T>), dim3(16), dim3(256), 0, st, (T*)db, N, 1, (int)N)); IFL_LAUNCH_CHECK(); }
        return 0;
    }
    const int es = b8_size(dytype);
    const bool wide = (uintptr_t)dy % 16 == 0 && (M == 1 || ldy * es % 16 == 0);
    const WPlan p = wg8_plan(M, N, dw ? K : 0, dytype, wide && N % 8 == 0);
    WG8 q = {};
    q.dy = dy; q.ldy = ldy; q.codes = codes; q.ldc = ldc; q.scales = scales; q.lds = lds; q.chan = chan; q.dw = dw; q.ldw = ldw;
    q.dwtype = dwtype; q.db = db; q.dbtype = dbtype; q.M = M; q.N = (int)N; q.K = (int)K; q.fmt = fmt; q.want_x = dw != nullptr;
    q.kp = p.kp; q.np = p.np; q.yplane = (M + MS - 1) / MS * MS * p.np; q.in_place = p.in_place;
    q.xb = (uint16_t*)scratch;
    q.yb = (uint16_t*)(scratch + p.x_floats);
    q.part = scratch + p.x_floats + p.y_floats;
    q.cs = q.part + p.part_floats;
    q.split = p.split; q.steps = p.steps; q.cs_parts = p.cs_parts; q.cs_rows = p.cs_rows;

    const int64_t mp = (M + MS - 1) / MS * MS;
    if (todo & 1) {
        if (dw) {
            while (q.x_tpr_log < 8 && (8 << q.x_tpr_log) < p.kp) ++q.x_tpr_log;
            const int64_t rows = (mp + (256 >> q.x_tpr_log) - 1) / (256 >> q.x_tpr_log);           // in turns of one workgroup
            const int64_t four = (rows + 3) / 4;
            q.x_blocks = (int)(four >= 16384 ? 16384 : four >= 512 ? four : rows < 512 ? rows : 512);
        }
        q.y_tpr_log = p.y_tpr_log;
        q.y_cols = (int)((N + (8 << p.y_tpr_log) - 1) / (8 << p.y_tpr_log));
        // of gradients that are read in place and of which nothing else is wanted only the last rows are looked at, if they do not
        // fill a step
        int64_t y_blocks = (int64_t)p.cs_parts * q.y_cols;
        if (p.in_place && !db && !quant) {
            q.y_row0 = M / MS * MS;
            q.cs_rows = MS;
            y_blocks = M % MS ? q.y_cols : 0;
        }
        if (quant) { q.gc = quant->codes; q.gs = quant->scales; q.ldgc = quant->ldc; q.ldgs = quant->lds; q.gfmt = quant->fmt; }
        const dim3 pg((unsigned)(q.x_blocks + y_blocks));
#define WG8_P2(T, NP, V, Q) hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_prepare_kernel<T, NP, V, Q>), pg, dim3(256), 0, st, q)
#define WG8_P(T, NP) do { \
            if (wide && quant) WG8_P2(T, NP, true, true); else if (wide) WG8_P2(T, NP, true, false); \
            else if (quant) WG8_P2(T, NP, false, true); else WG8_P2(T, NP, false, false); \
        } while (0)
        if (dytype == IFL_T_F32) WG8_P(float, 3); else if (dytype == IFL_T_F16) WG8_P(_Float16, 2); else WG8_P(__bf16, 1);
        IFL_LAUNCH_CHECK();
    }
    if (!(todo & 2)) return 0;
    if (dw) {
        q.tiles_n = (int)((N + p.tile - 1) / p.tile);
        q.tiles_k = (int)((K + p.tile - 1) / p.tile);
        q.per_xcd = (q.tiles_n * q.tiles_k * p.split + 7) / 8;
        const dim3 grid(8 * q.per_xcd);
#define WG8_K(NP) do { \
        if (p.tile == 256) hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_kernel<NP, 256, 256, 4, 2>), grid, dim3(512), 0, st, q); \
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_kernel<NP, 128, 128, 2, 2>), grid, dim3(256), 0, st, q); \
    } while (0)
        if (dytype == IFL_T_F32) WG8_K(3); else if (dytype == IFL_T_F16) WG8_K(2); else WG8_K(1);
        IFL_LAUNCH_CHECK();
    }
    int64_t jobs = 0;
    const bool v4 = K % 4 == 0, across = (v4 ? N * K / 4 : N * K) < 1 << 16;
    if (dw && p.split > 1) {
        jobs = ((v4 ? N * K / 4 : N * K) + (across ? 15 : 255)) / (across ? 16 : 256);
        if (jobs > 4096) jobs = 4096;
    }
    if (jobs || db) {
        const dim3 fg((unsigned)(jobs + (db ? (N + 15) / 16 : 0)));
#define WG8_E2(TW, TB, V, A) hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_finish_kernel<TW, TB, V, A>), fg, dim3(256), 0, st, q, (int)jobs)
#define WG8_E(TW, TB) do { \
        if (v4 && across) WG8_E2(TW, TB, 4, true); else if (v4) WG8_E2(TW, TB, 4, false); \
        else if (across) WG8_E2(TW, TB, 1, true); else WG8_E2(TW, TB, 1, false); \
    } while (0)
        const int wt = dw ? dwtype : IFL_T_F32, bt = db ? dbtype : wt;
        B8_DISPATCH(wt, typedef T TW; B8_DISPATCH(bt, WG8_E(TW, T)));
        IFL_LAUNCH_CHECK();
    }
    return 0;
}

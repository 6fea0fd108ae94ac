// wgrad8.hip -- the weight gradient of a product whose input was kept in 8-bit blocks (block8.h):
//     dw[n][k] = chan[k] sum_m dy[m][n] code[m][k] 2^e[m][k / 128],      db[n] = sum_m dy[m][n]
// The sum runs over the rows of both operands, whose scales change from row to row, so the 8-bit instructions cannot apply them.
// A code times its scale is exact in bf16, and so is a bf16 gradient; a float16 gradient is the sum of two bf16 terms and a
// float32 one of three (its 24 significant bits in pieces of 8).  So every product goes exactly through
// v_mfma_f32_16x16x32_bf16 (one, two or three of them), which keeps 24 bits of the sums.  (Below 2^-109 a float32's last piece, and in a block
// of values that small a code, falls under bf16's smallest step, 2^-133, and is lost.)
//
// Three launches: codes restored to bf16 and gradients split into their terms, with dy's column sums (memory-bound, one pass, 4.9 TB/s); the
// product (2048 x 2048 over 65536 rows: bf16 1.25 PFLOP/s, the three terms of float32 together 1.6; a large library product in bf16 1.34);
// the parts of a split sum joined.  Restoring and splitting inside the product, where every workgroup of a row of
// tiles repeats it, was the slower way: its arithmetic does not fit beside the matrix instructions (2048 x 2048 over 65536 rows,
// bf16: 615 us with it, 390 without; float32: 1644 and 841).
#include "block8.h"
#include <math.h>

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
    B8Cols w; int w_blocks, w_tiles;                 // and the layer's weights, to be quantized along their columns: workgroups, those of a block of columns
    // scratch
    uint16_t* xb;                        // restored codes, rows up to a multiple of 64 (zeros)
    uint16_t* yb; int64_t yplane;        // terms of dy in the same way, yplane apart; or of bf16 read in place the last M % 64 rows
    int in_place;
    float* part; int split, steps;       // float32 partial sums [split][N][K], steps of 32 rows per part
    float* cs; int cs_parts; int64_t cs_rows, y_row0;        // partial column sums [cs_parts][N], of cs_rows rows from y_row0 on
    int tiles_n, tiles_k, per_xcd;
    int x_blocks, x_tpr_log, y_cols, y_tpr_log;      // first launch: workgroups that restore codes, threads along a row; ranges of columns of dy, threads along a row
};

// The next of the bf16 terms whose sum is a value, as a float with 16 low zero bits: its leading 8 significant bits; x becomes what is
// left.  What is not finite is the first term alone.  (FIRST; of bf16 the first term is the value.)
template <bool FIRST, class T>
__device__ __forceinline__ uint32_t wg8_term(float& x) {
    if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16)) return __float_as_uint(x);
    if (FIRST) x = __builtin_canonicalizef(x);                           // (a NaN has a high bit set)
    const uint32_t t = __float_as_uint(x) & 0xffff0000u;
    x -= __uint_as_float(t);
    if (FIRST) x = x == x ? x : 0.f;
    return t;
}

// Two bf16 values, the largest finite one in place of infinities.  An infinity of a checkpoint meets the first term of a gradient only: the
// others may be zero, and infinity times zero is NaN; what they give instead has the first one's sign.  (As unsigned numbers negative
// infinities are above all else but NaN, as signed ones positive ones are.)
__device__ __forceinline__ uint32_t wg8_finite2(uint32_t w) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
    const u16x2 u = __builtin_elementwise_min(__builtin_bit_cast(u16x2, w), (u16x2)(uint16_t)0xff7f);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(i16x2, u), (i16x2)(int16_t)0x7f7f));
}

template <class TW>
__device__ __forceinline__ void wg8_store4(TW* d, int left, const float v[4]) {
    if (left >= 4) {
        typename B8Vec<TW, 4>::Aligned w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (TW)v[e];
        *(typename B8Vec<TW, 4>::type*)d = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (e < left) d[e] = (TW)v[e];
    }
}

constexpr int MS = 32;                                                  // rows per step: the depth of one product
constexpr int MP = 2 * MS;                                              // what rows are padded to with zeros
__host__ __device__ inline int64_t wg8_rows(int64_t M) { return (M + MP - 1) / MP * MP; }

// ------------------------------------------------------------------------------------------------ first launch
// The product's fragments are 8 rows of a column; of 32 rows lane group g = 0 .. 3 has 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3
// (what two transposing reads give it).  So that they can be read from LDS 16 bytes at a time, what this launch writes is ordered
// [32 rows][g][column][8 rows].
//
// A thread has the 8 rows of one g and 8 columns; 16 bytes per column.  They meet in LDS so that the stores are whole lines (slot
// i of the workgroup's at i ^ (i / 16 & 7): no bank conflicts on either side).
__device__ __forceinline__ void wg8_put(i32x4* lds, const i32x4 w[8], uint16_t* out, int64_t row0, int64_t rows, int64_t cols, int c0, int tpr_log) {
    int j = threadIdx.x;
    asm volatile("" : "+v"(j));                                          // (places are made here, not kept)
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) { const int at = j * 8 + i; lds[at ^ (at >> 4 & 7)] = w[i]; }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const int at = n * 256 + j, gg = at >> (3 + tpr_log), c = c0 + (at & ((8 << tpr_log) - 1));
        const int64_t r = row0 + 8 * gg;                                 // (counted in groups of 8 rows that follow one another)
        if (c < cols && r < rows) *(i32x4*)(out + (r / 8 * cols + c) * 8) = lds[at ^ (at >> 4 & 7)];
    }
}
// row e of group gg (from a multiple of 32 on)
__device__ __forceinline__ int wg8_row(int gg, int e) { return (gg >> 2) * 32 + 4 * (gg & 3) + (e & 3) + 16 * (e >> 2); }

// QUANT, for a layer's other product: the first w_blocks workgroups quantize its weights, tiles of 64 x 128, and those of dy put it into
// 8-bit blocks as well.  The next x_blocks restore codes.  The others take up to 256 columns of cs_rows rows of dy, with column
// sums on the way that are joined in LDS in a fixed order, and dy's terms, if the product does not read it in place.  (16384 x 2048,
// both operands, bf16: 30 us; with dy's blocks 43, 25 more on its own; with 2048 x 2048 weights 47, 19 more on their own.)
template <class T, int NP, bool QUANT, class TW>
__global__ __launch_bounds__(256, NP > 1 ? 2 : 3)
void wgrad8_prepare_kernel(WG8 q)
{
    __shared__ __attribute__((aligned(16))) i32x4 stage[2048];
    static_assert(sizeof(stage) >= B8_COLS_LDS, "");
    if (QUANT && (int)blockIdx.x < q.w_blocks) {
        const int kb = blockIdx.x / q.w_tiles;
        b8_quantize_cols<TW>(q.w, stage, blockIdx.x - kb * q.w_tiles, kb);
        return;
    }
    const int64_t mp = wg8_rows(q.M);
    const int bid = blockIdx.x - (QUANT ? q.w_blocks : 0);
    if (bid < q.x_blocks) {
        const int tpr = 1 << q.x_tpr_log, gg = threadIdx.x >> q.x_tpr_log, rpp = 8 * (256 >> q.x_tpr_log);
        const int cols = (q.K + 8 * tpr - 1) / (8 * tpr);
        const int64_t jobs = (mp + rpp - 1) / rpp * cols;
        for (int64_t job = bid; job < jobs; job += q.x_blocks) {
            const int64_t row0 = job / cols * rpp;
            const int c0 = (int)(job % cols) * 8 * tpr, c = c0 + (threadIdx.x & (tpr - 1)) * 8;
            i32x2 w[8];
            int sb[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t r = row0 + wg8_row(gg, e);
                const bool in = r < q.M && c < q.K;                      // (rows are whole 16 bytes)
                w[e] = in ? *(const i32x2*)(q.codes + r * q.ldc + c) : i32x2{0, 0};
                sb[e] = in ? q.scales[r * q.lds + c / B8_BLK] : 127;
            }
            i32x4 v[8], t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(i32x4, q.fmt == IFL_Q_E4M3 ? b8_bf16x8<IFL_Q_E4M3>(w[e][0], w[e][1], sb[e]) : b8_bf16x8<IFL_Q_E5M2>(w[e][0], w[e][1], sb[e]));
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    t[i][e] = (int)__builtin_amdgcn_perm((uint32_t)v[2 * e + 1][i / 2], (uint32_t)v[2 * e][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
            wg8_put(stage, t, q.xb, row0, mp, q.K, c0, q.x_tpr_log);
        }
        return;
    }
    __shared__ float red[256 * 8 + 256];
    const int b = bid - q.x_blocks, part = b / q.y_cols, cb = b - part * q.y_cols;
    const int tpr = 1 << q.y_tpr_log, rpp = 256 >> q.y_tpr_log, rl = threadIdx.x >> q.y_tpr_log;
    const int c0 = cb * 8 * tpr, c = c0 + (threadIdx.x & (tpr - 1)) * 8;
    const int64_t first = q.y_row0 + (int64_t)part * q.cs_rows, last = min(mp, first + q.cs_rows);
    const int64_t whole = q.M / MP * MP;
    const T* dy = (const T*)q.dy;
    float sum[8] = {};
    for (int64_t row0 = first; row0 < last; row0 += 8 * rpp) {
        // rows and columns past the end: the last one's values, then zeros
        float v[8][8];
        const T* rows = dy + row0 * q.ldy;
        const int left = (int)(min(q.M, last) - row0);                   // (negative: all of them are zeros, read from row M - 1)
        int row = wg8_row(rl, 0), cc = c;
        asm volatile("" : "+v"(row), "+v"(cc));                          // (addresses are made here, not kept)
        auto at = [&](int e) { return rows + (int64_t)min(row + (e & 3) + 16 * (e >> 2), left > 0 ? left - 1 : (int)(q.M - 1 - row0)) * q.ldy; };
        if (cc + 8 <= q.N) {
#pragma unroll
            for (int e = 0; e < 8; ++e) b8_load8<T>(at(e) + cc, 8, v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) { const float t = (float)at(e)[min(cc + i, q.N - 1)]; v[e][i] = cc + i < q.N ? t : 0.f; }
        }
        if (left < 8 * rpp) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[e][i] = row + (e & 3) + 16 * (e >> 2) < left ? v[e][i] : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);                               // (here and below: the compiler would otherwise do it all side by side, in 300 registers)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int r = row + (e & 3) + 16 * (e >> 2);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v[e][i];
            if constexpr (QUANT) {
                int sb;                                                  // (of a block: 16 threads, or the 4 or 8 of a short row)
                const i32x2 w = b8_quantize8<16>(v[e], q.gfmt, sb, tpr);
                if (r < left) {
                    if (cc < q.ldgc) *(i32x2*)(q.gc + (row0 + r) * q.ldgc + cc) = w;
                    if (cc < q.N && (cc & (B8_BLK - 1)) == 0) q.gs[(row0 + r) * q.ldgs + cc / B8_BLK] = (uint8_t)sb;
                }
            }
            if constexpr (NP == 1) {
                if (q.want_x && q.in_place && cc < q.N && row0 + r >= whole && row0 + r < last) {        // the last rows, as they are
                    i32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = (int)__builtin_amdgcn_perm(__float_as_uint(v[e][2 * i + 1]), __float_as_uint(v[e][2 * i]), 0x07060302u);    // the high halves
                    *(i32x4*)(q.yb + (row0 + r - whole) * q.N + cc) = w;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (q.want_x && !q.in_place) {
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                i32x4 t[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t lo = k ? wg8_term<false, T>(v[2 * e][i]) : wg8_term<true, T>(v[2 * e][i]);
                        const uint32_t hi = k ? wg8_term<false, T>(v[2 * e + 1][i]) : wg8_term<true, T>(v[2 * e + 1][i]);
                        t[i][e] = (int)__builtin_amdgcn_perm(hi, lo, 0x07060302u);       // the high halves
                        __builtin_amdgcn_sched_barrier(0);
                    }
                wg8_put(stage, t, q.yb + k * q.yplane, row0, last, q.N, c0, q.y_tpr_log);
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
// Workgroup = TN x TK of dw over a range of rows, 32 at a time.  The instruction's first operand is the k side: a lane ends up with 4
// neighbouring k of one n.
//
// The k side, and dy's terms, lie in LDS as they do in memory, [g][column][8 rows]: a fragment is 16 bytes a lane, 16 lanes 256 bytes in a
// row.  bf16 gradients are read in place (TR): their rows lie in LDS as in memory, and fragments come out transposed
// (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 values and get columns), at half the rate.  Such a read touches, per group of 16
// lanes, 4 rows and 4 pieces of 8 bytes of each: one granule of 32 bytes, granule i of row m at place i ^ (m & 7), which leaves no
// bank conflicts.  Loads go straight to LDS in lane order, so it is the source that is permuted.
//
// A step is a term of dy with 32 rows (the terms of the same rows follow one another and share the k side's fragments).  It has two
// phases.  MEM: the loads of the step three ahead are issued (rings of four), this step's fragments are read.  COMPUTE: its
// products, nothing else.  With 8 waves the second four run one phase behind the first, so that of the two waves on a SIMD one
// multiplies while the other one reads: the workgroup meets after every phase.  Three steps are about 1.5 us, what rows that
// all workgroups ask for at the same time take to come from memory.
template <int V> struct Int { static constexpr int value = V; };

template <int NP, bool TR, bool INF, int TN, int TK, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK)
void wgrad8_kernel(WG8 q)
{
    constexpr int NW = WN * WK, NT = 64 * NW, NF = TN / WN / 16, KF = TK / WK / 16;
    constexpr bool TURNS = NW == 8;
    constexpr int YROW = TN * 2, YB = MS * YROW, XB = MS * TK * 2;         // bytes
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
    const int s0 = part * q.steps, rows_steps = (int)(wg8_rows(q.M) / MS), steps = (min(rows_steps, s0 + q.steps) - s0) * NP;
    // (fresh: an address or offset that is made again at its use instead of being held in registers of its own)
    auto fresh = [](auto x) { asm volatile("" : "+v"(x)); return x; };

    // ---- loads: 64 lanes' 16 bytes each, from base + their offsets, to LDS in lane order.  By hand: the compiler waits for all loads
    // wherever it thinks that one might have written what is read.  (The instruction reads M0 one wait state after it is written.)
    auto to_lds = [&](const void* base, uint32_t o, const uint8_t* to) {
        const uint32_t at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)to;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(at), "v"(o), "s"(base) : "memory", "m0");
    };
    // a thread's pieces: a column (past the end: any, its results are not stored), and rows (TR) or groups of 8 that lie apart
    constexpr int YSTEP = TR ? NT / (TN / 8) : NT / TN, XSTEP = NT / TK;
    static_assert(YSTEP >= 1 && XSTEP >= 1 && (!TR || YSTEP % 8 == 0), "");
    const int yr = TR ? tid / (TN / 8) : tid / TN, xr = tid / TK;
    const int yn = n0 + (TR ? (((tid % (TN / 8) >> 1) ^ (yr & 7)) * 2 + (tid & 1)) * 8 : tid % TN), xk = k0 + tid % TK;
    const uint32_t yc = yn < q.N ? (uint32_t)yn * (TR ? 2 : 16) : 0, xc = xk < q.K ? (uint32_t)xk * 16 : 0;
    const int whole = TR ? (int)(q.M / MP) * 2 : 0;                      // steps read in place
    // step t: term PL of rows 32 (s0 + t / NP) on; behind the last step it is loaded again, unused
    auto load = [&](auto PL, int t, int ry, int rx) __attribute__((always_inline)) {
        const int s = s0 + min(t, steps - 1) / NP;
        const uint8_t* y;
        uint32_t yl;                                                     // bytes from row to row, or group to group
        if constexpr (TR) {                                              // the last rows were copied to a place with zeros behind them
            const bool cut = s >= whole;
            y = cut ? (const uint8_t*)q.yb : (const uint8_t*)q.dy;
            yl = (uint32_t)(cut ? q.N : (int)q.ldy) * 2;
            y += (int64_t)(cut ? s - whole : s) * (MS * yl);
        } else {
            yl = (uint32_t)q.N * 16;
            y = (const uint8_t*)(q.yb + PL.value * q.yplane) + (int64_t)s * 4 * yl;
        }
        const uint32_t xl = (uint32_t)q.K * 16;
#pragma unroll
        for (int i = 0; i < YP; ++i) to_lds(y, (uint32_t)(fresh(yr) + i * YSTEP) * yl + yc, ys + ry * YB + (i * NT + wave * 64) * 16);
        if constexpr (PL.value == 0) {
            const uint8_t* x = (const uint8_t*)q.xb + (int64_t)s * 4 * xl;
#pragma unroll
            for (int i = 0; i < XP; ++i) to_lds(x, (uint32_t)(fresh(xr) + i * XSTEP) * xl + xc, xs + rx * XB + (i * NT + wave * 64) * 16);
        }
    };

    // ---- fragments (TR: places are XORs of a lane's own and of a fragment's constants)
    const int mrow = 4 * g + (r16 >> 2), q4 = r16 & 3;
    const int ya = TR ? mrow * YROW + ((wn * NF) ^ (mrow & 7)) * 32 + q4 * 8 : (g * TN + wn * NF * 16 + r16) * 16;
    const int xa = (g * TK + wk * KF * 16 + r16) * 16;
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
    auto step = [&](auto PL, int t, int ry, int rx) __attribute__((always_inline)) {
        constexpr int P3 = (PL.value + 3) % NP;
        constexpr int AHEAD = (PL.value + 3) / NP;                       // row steps that term lies ahead
        load(Int<P3>(), t + 3, (ry + 3) & 3, (rx + AHEAD) & 3);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            if constexpr (TR) y[f] = tr8(ys + ry * YB + (fresh(ya) ^ f << 5), 16 * YROW);
            else y[f] = *(const bf16x8*)(ys + ry * YB + ya + f * 256);
        }
        if constexpr (PL.value == 0) {
#pragma unroll
            for (int f = 0; f < KF; ++f) x[f] = *(const bf16x8*)(xs + rx * XB + xa + f * 256);
        }
        if constexpr (INF && PL.value == 1) {                            // (the terms after the first share what this leaves)
#pragma unroll
            for (int f = 0; f < KF; ++f) {
                i32x4 w = __builtin_bit_cast(i32x4, x[f]);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (int)wg8_finite2((uint32_t)w[e]);
                x[f] = __builtin_bit_cast(bf16x8, w);
            }
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

// Tiles of 128 x 128, or 256 x 256 where there are 32 of them, an eighth of them at most lies past the edge, and a workgroup gets 48 steps.
// Measured (bf16; 128 / 256): 1024 x 2048 x 2048 33.0 / 40.3 us, 4096 x 2048 x 2048 56.7 / 59.5, 16384 x 2048 x 2048 156 / 141, 2048 x
// 4096 x 4096 90.2 / 71.9, 16384 x 1024 x 1024 60.8 / 64.0, 16384 x 64 x 2048 42.5 / 50.0.  The rows are split until the card is full
// (one workgroup on a CU of the large tiles, two of the small ones), each with four steps at least, but not further than pays: a part
// costs 1.6 us for each million of dw's values (written and read), a step 0.4 us (512 x 2048 x 2048: 32.3 us in two parts, 21.0 in
// one; 256 x 1024 x 1024: 19.4 in two, 15.1 in one).
struct WPlan { int tile, split, steps, cs_parts, y_tpr_log; int64_t cs_rows, x_floats, y_floats, part_floats, cs_floats; bool in_place; };
WPlan wg8_plan(int64_t M, int64_t N, int64_t K, int dytype, bool aligned)
{
    WPlan p = {};
    auto tiles = [&](int64_t t) { return ((N + t - 1) / t) * ((K + t - 1) / t); };
    const int terms = dytype == IFL_T_F32 ? 3 : dytype == IFL_T_F16 ? 2 : 1;
    const int64_t steps = wg8_rows(M) / MS;
    p.tile = tiles(256) >= 32 && 32 * tiles(256) <= 9 * tiles(128) && steps * terms * tiles(256) >= 48 * 256 ? 256 : 128;
    const int64_t n = K > 0 ? tiles(p.tile) : 1;
    const int64_t full = p.tile == 256 ? 256 : 512;
    int64_t s = 4 * n >= 3 * full ? 1 : full / n;
    if (s > steps * terms / 4) s = steps * terms / 4;
    const double best = sqrt(0.4 * (double)(steps * terms) / (1.6e-6 * (double)N * (double)(K > 0 ? K : 1)));
    if ((double)s > best + 0.5) s = (int64_t)(best + 0.5);
    if (s > 256) s = 256;
    if (s < 1) s = 1;
    p.steps = (int)((steps + s - 1) / s);
    p.split = (int)((steps + p.steps - 1) / p.steps);
    // column sums (and terms): about as many workgroups as run at a time (bf16: 3 on a CU) or two such rounds (the terms' kernels: 512
    // instead of 1024 took 87 us instead of 80 at 16384 x 2048), each with the rows of one pass at least
    p.y_tpr_log = 2;
    while (p.y_tpr_log < 5 && (8 << p.y_tpr_log) < N) ++p.y_tpr_log;
    const int64_t cols = (N + (8 << p.y_tpr_log) - 1) / (8 << p.y_tpr_log), pass = 8 * (256 >> p.y_tpr_log);
    int64_t c = (terms > 1 ? 1024 : 768) / cols;
    if (c > (M + pass - 1) / pass) c = (M + pass - 1) / pass;
    if (c < 1) c = 1;
    p.cs_rows = ((steps + c - 1) / c + 1) / 2 * MP;
    p.cs_parts = (int)((steps * MS + p.cs_rows - 1) / p.cs_rows);
    p.in_place = dytype == IFL_T_BF16 && aligned;
    auto up = [](int64_t floats) { return (floats + 3) / 4 * 4; };
    p.x_floats = K > 0 ? up(steps * MS * K / 2) : 0;
    p.y_floats = K > 0 ? up((p.in_place ? MP : terms * steps * MS) * N / 2) : 0;
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

extern "C" int ifl_block8_wgrad_plan(int64_t M, int64_t N, int64_t K, int dytype)
{
    if (M < 1 || N < 1 || K < 1 || !b8_type_ok(dytype)) return 0;
    const WPlan p = wg8_plan(M, N, K, dytype, false);
    return p.tile | p.split << 16;
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
    q.yplane = wg8_rows(M) * N; q.in_place = p.in_place;
    q.xb = (uint16_t*)scratch;
    q.yb = (uint16_t*)(scratch + p.x_floats);
    q.part = scratch + p.x_floats + p.y_floats;
    q.cs = q.part + p.part_floats;
    q.split = p.split; q.steps = p.steps; q.cs_parts = p.cs_parts; q.cs_rows = p.cs_rows;

    if (todo & 1) {
        if (dw) {
            while (q.x_tpr_log < 5 && (8 << q.x_tpr_log) < K) ++q.x_tpr_log;
            const int64_t rpp = 8 * (256 >> q.x_tpr_log), jobs = (wg8_rows(M) + rpp - 1) / rpp * ((K + (8 << q.x_tpr_log) - 1) / (8 << q.x_tpr_log));
            q.x_blocks = (int)(jobs < 16384 ? jobs : 16384);
        }
        q.y_tpr_log = p.y_tpr_log;
        q.y_cols = (int)((N + (8 << p.y_tpr_log) - 1) / (8 << p.y_tpr_log));
        // of gradients that are read in place and of which nothing else is wanted only the last rows are looked at, if they do not
        // fill a step
        int64_t y_blocks = (int64_t)p.cs_parts * q.y_cols;
        if (p.in_place && !db && !quant) {
            q.y_row0 = M / MP * MP;
            q.cs_rows = MP;
            y_blocks = M % MP ? q.y_cols : 0;
        }
        if (quant) {
            q.gc = quant->codes; q.gs = quant->scales; q.ldgc = quant->ldc; q.ldgs = quant->lds; q.gfmt = quant->fmt;
            if (quant->w.x) {
                q.w = quant->w;
                q.w_tiles = (int)((q.w.rows + 63) / 64);
                q.w_blocks = q.w_tiles * ((q.w.cols + B8_BLK - 1) / B8_BLK);
            }
        }
        const dim3 pg((unsigned)(q.w_blocks + q.x_blocks + y_blocks));
#define WG8_P(TY, NP) do { \
            if (!quant) hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_prepare_kernel<TY, NP, false, float>), pg, dim3(256), 0, st, q); \
            else B8_DISPATCH(quant->wtype, hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_prepare_kernel<TY, NP, true, T>), pg, dim3(256), 0, st, q)); \
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
        const bool inf = fmt == IFL_Q_E5M2;                                // (only that format has infinities)
#define WG8_L(NP, TR, INF, T, WN, WK) hipLaunchKernelGGL(HIP_KERNEL_NAME(wgrad8_kernel<NP, TR, INF, T, T, WN, WK>), grid, dim3(64 * WN * WK), 0, st, q)
#define WG8_K(NP, TR) do { \
        if (p.tile == 256) { if (inf) WG8_L(NP, TR, (NP > 1), 256, 4, 2); else WG8_L(NP, TR, false, 256, 4, 2); } \
        else if (inf) WG8_L(NP, TR, (NP > 1), 128, 2, 2); else WG8_L(NP, TR, false, 128, 2, 2); \
    } while (0)
        if (dytype == IFL_T_F32) WG8_K(3, false); else if (dytype == IFL_T_F16) WG8_K(2, false);
        else if (p.in_place) WG8_K(1, true); else WG8_K(1, false);
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

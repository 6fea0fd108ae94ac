// matmul8.hip -- C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]) over rows in 8-bit blocks (block8.h), in one of two ways:
//
// Exact (the default, and all float32 results): the codes times their scales, exact in bf16 (what is below its smallest step, 2^-133,
// aside), go through v_mfma_f32_16x16x32_bf16, which keeps 24 bits.
//
// By the scaled 8-bit instructions, where the caller allows a 16-bit result that (IFL_P_8BIT): v_mfma_scale_f32_16x16x128_f8f6f4
// multiplies 16 x 128 by 128 x 16 codes and takes one E8M0 byte per row and 32 values.  A block of 128 is one instruction deep, so
// every scale is applied by the instruction, exactly, and what it returns is summed in float32.  But within 8 products it drops what is
// below 2^-13 of the largest (measured): a result is off by up to 7 2^-13 of sum |a b|, and in the 2-norm by 4.1e-5 of itself for
// activations with outliers and spread, 1.5e-5 for normal values (K = 4096).  Rounding to float16 adds 2.1e-4, to bfloat16 1.7e-3; but
// where large products cancel, what they leave is lost.  Twice the rate: 8192 x 8192 x 4096 bf16 237 us, exact 444 (1.24 PFLOP/s; a large
// bf16 library product on this card 1.34); 16384 x 2048 x 2048 67 and 121, 512 x 2048 x 2048 7.0 and 11.8, 1 x 4096 x 4096 4.9 and 5.1.  Times
// quoted below are of the 8-bit instructions unless they say exact or float32: what they compare is the same for both.
//
// Operands: the instruction's first is B (the n side) and its second A (the m side), so that a lane ends up with four
// neighbouring n of one m: a contiguous store.
//
// Lane l gives row l % 16 and 32 of the 128 values; which 32 is free as long
// as both operands agree (all of a block share a scale): 16 bytes from 16 (l / 16) and 16 from 64 + 16 (l / 16).
#include "block8.h"

namespace {

struct MM8 {
    const uint8_t *a, *b, *sa, *sb;
    int64_t lda, ldb, lsa, lsb;
    const void* bias; int btype;
    void* out; int otype; int64_t ldo;
    int64_t M, N; int K;
    const void* x; int64_t ldx;          // skinny kernel with its own quantization: the m side as it is
    float* part; int split, ksteps;      // float32 partial sums [split][M][N], K steps of 128 per part
    int tiles_m, tiles_n, per_xcd;
};

__device__ __forceinline__ float mm8_bias(const MM8& q, int64_t n) {
    return !q.bias ? 0.f : q.btype == IFL_T_F32 ? ((const float*)q.bias)[n] : q.btype == IFL_T_BF16 ? (float)((const __bf16*)q.bias)[n] : (float)((const _Float16*)q.bias)[n];
}

// 16 bytes of a row from k on (rows are whole 16 bytes in memory), and zeros in them where k >= K
__device__ __forceinline__ i32x4 mm8_load16(const uint8_t* __restrict__ row, int k, int K) { return *(const i32x4*)(row + (k < K ? k : 0)); }
__device__ __forceinline__ i32x4 mm8_cut16(i32x4 r, int k, int K) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = K - k - 4 * i;
        r[i] = left >= 4 ? r[i] : left <= 0 ? 0 : (int)((uint32_t)r[i] & ((1u << 8 * left) - 1));
    }
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

__device__ __forceinline__ i32x8 mm8_join(i32x4 a, i32x4 b) {
    i32x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) { r[i] = a[i]; r[4 + i] = b[i]; }
    return r;
}

// A wave's results: m0 the lane's first row, nw its first column, bias its columns' (in LDS).
template <class T, int NF, int MF, int G>
__device__ __forceinline__ void mm8_results(const MM8& q, const f32x4 (&acc)[NF][MF], int64_t m0, int64_t nw, const float* bias) {
    constexpr int V = 4 * G * sizeof(T) >= 16 ? 16 / sizeof(T) : 4 * G;
    T* p = (T*)q.out + m0 * q.ldo + nw;
    int rows = (int)(q.M - m0), cols = (int)(q.N - nw);
#pragma unroll
    for (int j = 0; j < MF; ++j) {
#pragma unroll
        for (int h = 0; h < NF / G; ++h) {
            float v[4 * G];
#pragma unroll
            for (int i = 0; i < 4 * G; ++i) v[i] = acc[h * G + i / 4][j][i % 4] + bias[16 * G * h + i];
            asm volatile("" : "+v"(cols));                               // (compared here: there are no registers for what is made ahead)
            if (16 * j < rows && 16 * G * h + 4 * G <= cols) {
#pragma unroll
                for (int i = 0; i < 4 * G / V; ++i) {
                    typename B8Vec<T, V>::Aligned t;
#pragma unroll
                    for (int e = 0; e < V; ++e) t[e] = (T)v[i * V + e];
                    *(typename B8Vec<T, V>::type*)(p + 16 * G * h + V * i) = t;
                }
            } else if (16 * j < rows) {
#pragma unroll
                for (int i = 0; i < 4 * G; ++i) if (16 * G * h + i < cols) p[16 * G * h + i] = (T)v[i];
            }
            __builtin_amdgcn_sched_barrier(0);                           // (one at a time, for the same reason)
        }
        p += 16 * q.ldo;
    }
}
template <int NF, int MF, int G>
__device__ __forceinline__ void mm8_part(const MM8& q, const f32x4 (&acc)[NF][MF], int64_t m0, int64_t nw) {
    float* out = q.part + (int64_t)blockIdx.y * q.M * q.N;
#pragma unroll
    for (int j = 0; j < MF; ++j) {
        const int64_t m = m0 + 16 * j;
        if (m < q.M) {
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                const int64_t n = nw + 16 * G * (i / G) + 4 * (i % G);
                if (n + 4 <= q.N) *(B8Vec<float, 4>::type*)(out + m * q.N + n) = acc[i][j];
                else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (n + e < q.N) out[m * q.N + n + e] = acc[i][j][e];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ tiles
// Workgroup = TN x TM of the result, K in steps of 128 bytes through two LDS buffers: while one is multiplied, the other is
// filled by loads that go straight to LDS (16 bytes a lane, no registers).  Those write LDS in lane order, so rows lie 128 bytes
// apart and it is the SOURCE that is permuted: position p of row r holds the 16 bytes p ^ s(r).  s takes 8 different values in the
// rows that 8 neighbouring lanes read, so no fragment read has bank conflicts, and the same value in all fragments of a
// lane, so that their addresses differ by constants.  Rows past the end repeat the last one (their results are not
// stored); a last step that K does not fill goes through registers with zeros behind K.
//
// Waves WN x WM; a wave has NF x MF fragments of 16 x 16.  Row r of n-fragment f is row 16 G (f / G) + 4 G (r / 4) + 4 (f % G) +
// r % 4 of the wave's: so the four values a lane gets from each of G fragments are 4 G neighbours of one output row, and 16 bytes
// (G = 2 for 16-bit results, 1 for float32): four lanes' stores fill 64 bytes of a row.  With twice as many neighbours to a lane each
// store left gaps for the next (16384 x 2048 x 2048: 69.3 us instead of 67.3, float32 in tiles of 128 169 instead of 144).
//
// Workgroups go to the 8 XCDs in turn; an XCD takes a contiguous run of tiles, in groups of 8 along m, so that the 32 tiles
// it works on at a time share rows of both operands in its own L2.
template <int TN, int TM, int WN, int WM, int FA, int FB, bool EXACT, bool SPLIT, int G>
__global__ __launch_bounds__(64 * WN * WM, 1)
void mm8_tile_kernel(MM8 q)
{
    constexpr int NW = WN * WM, NF = TN / WN / 16, MF = TM / WM / 16;
    constexpr int CH = (TN + TM) * 8, PER = CH / (64 * NW);              // 16-byte pieces of a step, per thread
    constexpr int D = 1, R = 2 * D;                                          // n-fragments read ahead, and the registers they rotate through
    static_assert(NF % R == 0 && D < R, "");
    __shared__ __attribute__((aligned(16))) uint8_t buf0[(TN + TM) * 128];
    __shared__ __attribute__((aligned(16))) uint8_t buf1[(TN + TM) * 128];
    constexpr int SR = (TN + TM + 64 * NW - 1) / (64 * NW);              // rows of scales per thread
    __shared__ uint32_t sc[2][SR * 64 * NW];                             // scale bytes of four steps, per row
    __shared__ __attribute__((aligned(16))) float bias[TN];
    static_assert(TN <= 64 * NW, "");
    const int tiles = q.tiles_m * q.tiles_n;
    const int t = (blockIdx.x & 7) * q.per_xcd + (blockIdx.x >> 3);
    if (t >= tiles) return;
    const int gsz = 8 * q.tiles_n, grp = t / gsz, rest = t - grp * gsz;
    const int gm = min(8, q.tiles_m - grp * 8);
    const int tm = __builtin_amdgcn_readfirstlane(grp * 8 + rest % gm), tn = __builtin_amdgcn_readfirstlane(rest / gm);
    const int64_t n0 = (int64_t)tn * TN, m0 = (int64_t)tm * TM;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
    const int wn = wave % WN, wm = wave / WN;

    // s(r): n side its bits 0, 1 and the one that r16's bit 2 goes to; m side bits 0 .. 2
    auto swz = [&](int row, bool nside) { return nside ? (row & 3) | (row / (4 * G) & 1) << 2 : row & 7; };
    // where this thread's pieces come from: 32-bit offsets from the tile's first rows
    auto piece = [&](int i, bool nside, int& ch) {
        const int p = (i * NW + wave) * 64 + lane, row = p >> 3, r = nside ? row : row - TN;
        ch = (p & 7) ^ swz(r, nside);
        const int64_t left = nside ? q.N - 1 - n0 : q.M - 1 - m0;
        return (uint32_t)((int64_t)(r < left ? r : (int)left) * (nside ? q.ldb : q.lda));
    };
    uint32_t off[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        int ch;
        off[i] = piece(i, (i * NW * 64) >> 3 < TN, ch);
        off[i] += ch * 16;
    }
    const uint8_t* bb = q.b + n0 * q.ldb;
    const uint8_t* ab = q.a + m0 * q.lda;
    const int k_first = SPLIT ? blockIdx.y * q.ksteps : 0;
    const int all = (q.K + B8_BLK - 1) / B8_BLK, k_end = SPLIT ? min(all, k_first + q.ksteps) : all;

    const int whole = min(k_end, q.K / B8_BLK);                          // steps that K fills
    auto fill = [&](uint8_t* buf, int ks) {
        int k0 = __builtin_amdgcn_readfirstlane(ks) * B8_BLK;
        asm volatile("" : "+s"(k0));                                     // (a scalar offset at every step: sums per lane would be kept in registers)
        const uint8_t *bk = bb + k0, *ak = ab + k0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint8_t* src = (i * NW * 64) >> 3 < TN ? bk : ak;      // (a piece's side is the same for all waves)
            const uint32_t at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)(buf + (i * NW + wave) * 1024);
            // By hand: the compiler waits for all loads wherever it thinks that one might have written what is read, here once in two steps
            // (8192 x 8192 x 4096 behind the quantization of its input: 285 us, so 252).  M0 is read one wait state after it is written.
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(at), "v"(off[i]), "s"(src) : "memory", "m0");
        }
    };
    auto fill_last = [&](uint8_t* buf, int ks) {
#pragma unroll 1
        for (int i = 0; i < PER; ++i) {
            const bool nside = (i * NW * 64) >> 3 < TN;
            int ch;
            const uint32_t o = piece(i, nside, ch);
            const int k = ks * B8_BLK + ch * 16;
            *(i32x4*)(buf + ((i * NW + wave) * 64 + lane) * 16) = mm8_cut16(mm8_load16((nside ? bb : ab) + o, k, q.K), k, q.K);
        }
    };

    // fragment addresses of this lane in LDS, but for constants: its two 16-byte pieces of fragment 0 of either side
    const int nrow0 = wn * NF * 16 + 4 * G * (r16 >> 2) + (r16 & 3), mrow0 = wm * MF * 16 + r16;
    const int nat[2] = {nrow0 * 128 + (g ^ swz(nrow0, true)) * 16, nrow0 * 128 + ((g + 4) ^ swz(nrow0, true)) * 16};
    const int mat[2] = {(TN + mrow0) * 128 + (g ^ swz(mrow0, false)) * 16, (TN + mrow0) * 128 + ((g + 4) ^ swz(mrow0, false)) * 16};
    auto nrow = [](int f) { return 16 * G * (f / G) + 4 * (f % G); };

    // a thread's rows of the scales (threads past the tile's rows repeat one): n side first
    const uint8_t *sp[SR], *sb = q.sb, *sa = q.sa;
    int64_t lsb = q.lsb, lsa = q.lsa;
    asm volatile("" : "+s"(sb), "+s"(sa), "+s"(lsb), "+s"(lsa));         // (arguments chosen between per lane would be loaded per lane)
#pragma unroll
    for (int i = 0; i < SR; ++i) {
        const int r = i * 64 * NW + threadIdx.x;
        sp[i] = r < TN ? sb + min(n0 + r, q.N - 1) * lsb : sa + min(m0 + (r - TN), q.M - 1) * lsa;
    }
    uint32_t snext[SR];

    f32x4 acc[NF][MF] = {};
    i32x8 a[1][MF], b[R];
    int ca[1][MF], cb[R];
    // (Addresses are made anew for each fragment: the second buffer's are out of an instruction's offset range, and the compiler
    // would keep one register for each of them.)
    auto fresh = [](int x) { asm volatile("" : "+v"(x)); return x; };
    auto read_a = [&](const uint8_t* buf, int ks, int o) {
        const uint8_t* s = (const uint8_t*)sc[(ks >> 2) & 1] + (ks & 3);
#pragma unroll
        for (int j = 0; j < MF; ++j) {
            a[o][j] = mm8_join(*(const i32x4*)(buf + fresh(mat[0]) + 2048 * j), *(const i32x4*)(buf + fresh(mat[1]) + 2048 * j));
            ca[o][j] = s[4 * (TN + mrow0 + 16 * j)];
        }
    };
    auto read_b = [&](const uint8_t* buf, int ks, int i) {
        const uint8_t* s = (const uint8_t*)sc[(ks >> 2) & 1] + (ks & 3);
        b[i % R] = mm8_join(*(const i32x4*)(buf + fresh(nat[0]) + 128 * nrow(i)), *(const i32x4*)(buf + fresh(nat[1]) + 128 * nrow(i)));
        cb[i % R] = s[4 * (nrow0 + nrow(i))];
    };
    auto turn = [&]() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // One step: NF groups of MF products.  Fragments of the n side are read D groups ahead.  Before the last D groups everything
    // this step needs is in registers, and the next step's bytes have had the time of NF - D groups to arrive: there the
    // workgroup meets, this step's buffer is handed to the step after the next, and the next step's first fragments are read
    // while the last D groups run.
    // (No branches inside, the compiler would move products past them: behind the last steps it is the last whole step that is
    // loaded again, unused.)
    const int last = (k_end - 1) >> 2;
    auto ask = [&](int grp) {
#pragma unroll
        for (int i = 0; i < SR; ++i) snext[i] = ((const uint32_t*)sp[i])[min(grp, last)];
    };
    auto put = [&](int grp) {
#pragma unroll
        for (int i = 0; i < SR; ++i) sc[grp & 1][i * 64 * NW + threadIdx.x] = snext[i];
    };
    auto step = [&](uint8_t* cur, const uint8_t* nxt, int ks, bool first) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            if (i + D < NF) read_b(cur, ks, i + D);
            if (i == NF - D) {
                turn();
                if (first) put((ks >> 2) + 1);
                fill(cur, min(ks + 2, whole - 1));
            }
            if (i >= NF - D) read_b(nxt, ks + 1, i + D - NF);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < MF; ++j) acc[i][j] = mm8_mfma<FA, FB, EXACT>(b[i % R], a[0][j], acc[i][j], cb[i % R], ca[0][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        read_a(nxt, ks + 1, 0);
    };

    // the first step's codes, the first scales and the bias are asked for together: one wait for all of them
    int ks = k_first;
    if (ks < whole) fill(buf0, ks);
    ask(k_first >> 2);                                                   // (k_first is a multiple of 4)
    if (!SPLIT && (int)threadIdx.x < TN) bias[threadIdx.x] = n0 + threadIdx.x < q.N ? mm8_bias(q, n0 + threadIdx.x) : 0.f;
    put(k_first >> 2);
    if (ks < whole) {
        turn();
        fill(buf1, min(ks + 1, whole - 1));
        read_a(buf0, ks, 0);
#pragma unroll
        for (int e = 0; e < D; ++e) read_b(buf0, ks, e);
        // Scales of the next four steps are asked for and put into LDS in every pair of steps, needed or not: no branch.  (Put where the
        // workgroup has just waited for its loads, and before it asks for more: anywhere else the compiler waits for those too.)
        for (; ks + 1 < whole; ks += 2) {
            ask((ks >> 2) + 1);
            step(buf0, buf1, ks, true);
            step(buf1, buf0, ks + 1, false);
        }
        if (ks < whole) step(buf0, buf1, ks, false);
    }
    if (k_end > whole) {                                                 // a last step that K does not fill
        turn();
        fill_last(buf0, whole);
        turn();
        read_a(buf0, whole, 0);
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            read_b(buf0, whole, i);
#pragma unroll
            for (int j = 0; j < MF; ++j) acc[i][j] = mm8_mfma<FA, FB, EXACT>(b[i % R], a[0][j], acc[i][j], cb[i % R], ca[0][j]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     // (no load into LDS outlives the workgroup)

    const int64_t mw = m0 + wm * MF * 16 + r16, nw = n0 + wn * NF * 16 + 4 * G * g;
    if constexpr (SPLIT) mm8_part<NF, MF, G>(q, acc, mw, nw);
    else {
        const float* bs = bias + wn * NF * 16 + 4 * G * g;
        if constexpr (G == 1) mm8_results<float, NF, MF, G>(q, acc, mw, nw, bs);
        else if (q.otype == IFL_T_BF16) mm8_results<__bf16, NF, MF, G>(q, acc, mw, nw, bs);
        else mm8_results<_Float16, NF, MF, G>(q, acc, mw, nw, bs);
    }
}

// out = sum of the parts, in order, + bias
template <class T>
__global__ __launch_bounds__(256)
void mm8_join_kernel(MM8 q)
{
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
    if (n >= q.N) return;
    const float* p = q.part + m * q.N + n;
    float t = p[0];
    for (int s = 1; s < q.split; ++s) t += p[(int64_t)s * q.M * q.N];
    ((T*)q.out)[m * q.ldo + n] = (T)(t + mm8_bias(q, n));
}

// ------------------------------------------------------------------------------------------------ few rows
// M <= 16 MF: bound by reading B once, so nothing is staged.  Workgroup = 16 n; its 16 waves take every sixteenth step of K (8 waves were
// 5 to 10% slower), four (M > 16: two) of their steps' loads in flight at a time, and meet in LDS.  OWN: the m side is not quantized yet: each
// workgroup quantizes all of it (M K values) into LDS, which saves a launch.
constexpr int SK_WAVES = 16;

template <int MF, int FA, int FB, bool EXACT, bool OWN, class TX>
__global__ __launch_bounds__(64 * SK_WAVES)
void mm8_skinny_kernel(MM8 q)
{
    __shared__ float red[SK_WAVES][16 * 16 * MF];
    extern __shared__ __attribute__((aligned(16))) uint8_t own[];        // [M][KP] codes, then [M][KB] scale bytes
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
    const int KB = (q.K + B8_BLK - 1) / B8_BLK, KP = KB * B8_BLK;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int64_t n = min(n0 + r16, q.N - 1);
    const uint8_t *pb = q.b + n * q.ldb, *psb = q.sb + n * q.lsb;
    // what this lane multiplies of the m side (OWN: of its copy in LDS)
    const uint8_t *pa[MF], *psa[MF];
#pragma unroll
    for (int j = 0; j < MF; ++j) {
        const int m = min(16 * j + r16, (int)q.M - 1);
        pa[j] = OWN ? own + m * KP : q.a + m * q.lda;
        psa[j] = OWN ? own + (int)q.M * KP + m * KB : q.sa + m * q.lsa;
    }
    constexpr int U = OWN || MF == 1 ? 4 : 2;
    // Of a step's 128 bytes a lane takes 16 from 16 g and 16 from 64 + 16 g; in odd rows the second ones first.  With the same half of
    // every row in one load they kept each other waiting (1 x 8192 x 2048: 8.2 us, so 6.8; 32 x 4096 x 4096: 10.5 and 7.9).
    const int odd = (r16 & 1) * 64;
    i32x4 b[U][2], a[U][MF][2];
    int cb[U], ca[U][MF];
    auto load = [&](int ks0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ks = ks0 + u * SK_WAVES, k = ks * B8_BLK + 16 * g;
            if (ks >= KB) break;
            b[u][0] = mm8_load16(pb, k + odd, q.K);
            b[u][1] = mm8_load16(pb, k + (odd ^ 64), q.K);
            cb[u] = psb[ks];
            if constexpr (!OWN) {
#pragma unroll
                for (int j = 0; j < MF; ++j) {
                    a[u][j][0] = mm8_load16(pa[j], k + odd, q.K);
                    a[u][j][1] = mm8_load16(pa[j], k + (odd ^ 64), q.K);
                    ca[u][j] = psa[j][ks];
                }
            }
        }
    };
    load(wave);                                                          // (the first loads run while the m side is quantized)
    if constexpr (OWN) {
        const int l16 = threadIdx.x & 15;
        for (int i = threadIdx.x >> 4; i < (int)q.M * KB; i += 64 * SK_WAVES / 16) {
            const int m = i / KB, kb = i - m * KB, c = kb * B8_BLK + l16 * 8;
            float v[8];
            b8_load8<TX>((const TX*)q.x + m * q.ldx + c, q.K - c, v);
            int s;
            *(i32x2*)(own + m * KP + c) = b8_quantize8<16>(v, IFL_Q_E4M3, s);
            if (l16 == 0) own[(int)q.M * KP + i] = (uint8_t)s;
        }
        __syncthreads();
    }
    f32x4 acc[MF] = {};
    for (int ks0 = wave; ks0 < KB; ks0 += U * SK_WAVES) {
        if (ks0 != wave) load(ks0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ks = ks0 + u * SK_WAVES, k = ks * B8_BLK + 16 * g;
            if (ks >= KB) break;
            const bool cut = (ks + 1) * B8_BLK > q.K;                    // a step that K does not fill
            auto order = [&](i32x4 (&w)[2]) { const i32x4 t = odd ? w[1] : w[0]; w[1] = odd ? w[0] : w[1]; w[0] = t; };
            order(b[u]);
            if (cut) { b[u][0] = mm8_cut16(b[u][0], k, q.K); b[u][1] = mm8_cut16(b[u][1], k + 64, q.K); }
#pragma unroll
            for (int j = 0; j < MF; ++j) {
                if constexpr (OWN) {
                    a[u][j][0] = *(const i32x4*)(pa[j] + k);
                    a[u][j][1] = *(const i32x4*)(pa[j] + k + 64);
                    ca[u][j] = psa[j][ks];
                } else order(a[u][j]);
                if (!OWN && cut) { a[u][j][0] = mm8_cut16(a[u][j][0], k, q.K); a[u][j][1] = mm8_cut16(a[u][j][1], k + 64, q.K); }
                acc[j] = mm8_mfma<FA, FB, EXACT>(mm8_join(b[u][0], b[u][1]), mm8_join(a[u][j][0], a[u][j][1]), acc[j], cb[u], ca[u][j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[wave][(16 * j + r16) * 16 + 4 * g + e] = acc[j][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 16 * MF; i += 64 * SK_WAVES) {
        const int m = i >> 4;
        const int64_t nn = n0 + (i & 15);
        float t = red[0][i];
#pragma unroll
        for (int w = 1; w < SK_WAVES; ++w) t += red[w][i];
        if (m < q.M && nn < q.N) {
            t += mm8_bias(q, nn);
            if (q.otype == IFL_T_F32) ((float*)q.out)[m * q.ldo + nn] = t;
            else if (q.otype == IFL_T_BF16) ((__bf16*)q.out)[m * q.ldo + nn] = (__bf16)t;
            else ((_Float16*)q.out)[m * q.ldo + nn] = (_Float16)t;
        }
    }
}

// ------------------------------------------------------------------------------------------------ which of them
// Few rows: the skinny kernel.  Else the tile that costs least.  With n tiles on a CU, halfway between the busiest one's and the mean, a
// product takes in us at K = 2048 about 2 + 4.4 n in tiles of 64 x 64, 7 + 10.5 n of 128 x 128, 4 + 34 n of 256 x 256 by the 8-bit instructions;
// the second terms grow with K, and are all about 1.6 times that where products are exact: one rule serves both.  Measured, 64 / 128 / 256,
// exact, bf16: 1024 x 2048 18.1 / 25.9 / 55.7, 2048 x 2048 31.0 / 27.4 / 57.3, 16384 x 512 51.4 / 38.4 / 59.1, 3584 x 3584 78.7 / 68.8 / 60.2, 8192 x
// 2048 98.2 / 70.9 / 61.9, 5000 x 1000 35.2 / 37.1; by the 8-bit instructions 1024 x 2048 10.7 / 16.2 /
// 30.7, 2048 x 2048 18.5 / 18.4 / 33, 16384 x 512 35.6 / 25.5 / 33.8, 3584 x 3584 52.8 / 43.4 / 36.3, 8192 x 2048 69.2 / 47.7 / 39.0, 5000 x 1000
// 24.9 / 22.6, and at K = 4096 48.1 / 37.7.  A product of few tiles and a long K is split along K.
// The skinny kernel quantizes the m side itself where that is at most 32768 values: then it is the faster way, in a graph (1 x 2048 x
// 2048: 3.5 us, 6.9 with a launch for it; 16 x 2048 x 2048: 5.8 and 7.3, exact too) and out of one (9 and 13.6).
bool mm8_own(int64_t M, int64_t K) { return M <= 16 && M * K <= 32768; }
struct Plan { int kind, tile, split, ksteps; };
Plan mm8_plan(int64_t M, int64_t N, int64_t K)
{
    Plan p = {0, 0, 1, 0};
    if (M <= 32) { p.kind = M <= 16 ? 1 : 2; return p; }
    auto tiles = [&](int t) { return ((M + t - 1) / t) * ((N + t - 1) / t); };
    auto cost = [&](int t, double fixed, double each) {
        const double mean = tiles(t) / 256.0, busiest = (double)((tiles(t) + 255) / 256);
        return fixed + each * (busiest <= 1 ? 1 : (mean + busiest) / 2) * (double)K / 2048;
    };
    const double c64 = cost(64, 2, 4.4), c128 = cost(128, 7, 10.5), c256 = cost(256, 4, 34);
    p.tile = c64 <= c128 ? 64 : 128;
    if (c256 < c64 && c256 < c128) p.tile = 256;
    const int64_t n = tiles(p.tile), steps = (K + B8_BLK - 1) / B8_BLK;
    if (p.tile == 64 && n <= 128 && steps >= 8) {
        int64_t s = 256 / n;
        if (s > steps / 4) s = steps / 4;
        if (s > 16) s = 16;
        if (s > 1) { p.ksteps = (int)(((steps + s - 1) / s + 3) / 4 * 4); p.split = (int)((steps + p.ksteps - 1) / p.ksteps); }
    }
    if (p.split <= 1) { p.split = 1; p.ksteps = (int)steps; }
    return p;
}

// whether a result of this type, perhaps with IFL_P_8BIT, gets exact products
bool mm8_exact(int otype) { return otype != (IFL_T_BF16 | IFL_P_8BIT) && otype != (IFL_T_F16 | IFL_P_8BIT); }

template <int FA, int FB>
int mm8_launch(MM8 q, const Plan& p, bool exact, hipStream_t st)
{
    const bool f32 = q.otype == IFL_T_F32;
    if (p.kind) {
        const dim3 grid((unsigned)((q.N + 15) / 16)), block(64 * SK_WAVES);
#define MM8_SK(MF, EX) hipLaunchKernelGGL(HIP_KERNEL_NAME(mm8_skinny_kernel<MF, FA, FB, EX, false, float>), grid, block, 0, st, q)
        if (p.kind == 1) { if (exact) MM8_SK(1, true); else MM8_SK(1, false); }
        else { if (exact) MM8_SK(2, true); else MM8_SK(2, false); }
        IFL_LAUNCH_CHECK();
        return 0;
    }
    q.tiles_m = (int)((q.M + p.tile - 1) / p.tile);
    q.tiles_n = (int)((q.N + p.tile - 1) / p.tile);
    q.per_xcd = (q.tiles_m * q.tiles_n + 7) / 8;
    q.split = p.split; q.ksteps = p.ksteps;
    const dim3 grid(8 * q.per_xcd, p.split);
#define MM8_TILE(T, WN, WM, EX, SP, G) hipLaunchKernelGGL(HIP_KERNEL_NAME(mm8_tile_kernel<T, T, WN, WM, FA, FB, EX, SP, G>), grid, dim3(64 * WN * WM), 0, st, q)
    if (p.tile == 256) { if (f32) MM8_TILE(256, 2, 4, true, false, 1); else if (exact) MM8_TILE(256, 2, 4, true, false, 2); else MM8_TILE(256, 2, 4, false, false, 2); }
    else if (p.tile == 128) { if (f32) MM8_TILE(128, 2, 2, true, false, 1); else if (exact) MM8_TILE(128, 2, 2, true, false, 2); else MM8_TILE(128, 2, 2, false, false, 2); }
    else if (p.split == 1) { if (f32) MM8_TILE(64, 2, 2, true, false, 1); else if (exact) MM8_TILE(64, 2, 2, true, false, 2); else MM8_TILE(64, 2, 2, false, false, 2); }
    else { if (exact) MM8_TILE(64, 2, 2, true, true, 1); else MM8_TILE(64, 2, 2, false, true, 2); }
    IFL_LAUNCH_CHECK();
    if (p.split > 1) {
        const dim3 jg((unsigned)((q.N + 255) / 256), (unsigned)q.M);
        B8_DISPATCH(q.otype, hipLaunchKernelGGL(HIP_KERNEL_NAME(mm8_join_kernel<T>), jg, dim3(256), 0, st, q));
        IFL_LAUNCH_CHECK();
    }
    return 0;
}

// a launch has fewer than 2^32 threads
bool mm8_fits(int64_t M, int64_t N, int64_t K)
{
    if (M < 1) return true;
    const Plan p = mm8_plan(M, N, K);
    const int64_t blocks = p.kind ? (N + 15) / 16 : ((M + p.tile - 1) / p.tile) * ((N + p.tile - 1) / p.tile) + 7;
    return blocks < (int64_t)1 << (p.kind ? 22 : p.tile == 256 ? 23 : 24);
}

int mm8_check(int64_t M, int64_t N, int64_t K, const uint8_t* b, int64_t ldb, const uint8_t* sb, int64_t lsb, const void* bias, int btype,
              const void* out, int otype, int64_t ldo)
{
    IFL_CHECK_ARG(b8_type_ok(otype) && (!bias || b8_type_ok(btype)), IFL_EINVAL, "block8 product: element types");
    IFL_CHECK_ARG(M >= 0 && N >= 1 && K >= 1, IFL_EINVAL, "block8 product: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG(K <= 0x7ffffc00 && M <= 0x3fffffff && N <= 0x3fffffff && mm8_fits(M, N, K), IFL_ENOTSUP, "block8 product: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    if (M == 0) return 0;
    const int KB = ifl_cdiv((int)K, B8_BLK);
    IFL_CHECK_ARG(b && sb && out, IFL_EINVAL, "block8 product: null pointer");
    IFL_CHECK_ARG(ldb >= K && lsb >= KB && ldo >= N, IFL_EINVAL, "block8 product: row strides");
    IFL_CHECK_ARG(ldb % 16 == 0 && (uintptr_t)b % 16 == 0 && lsb % 4 == 0 && (uintptr_t)sb % 4 == 0, IFL_EINVAL,
                  "block8 product: codes in rows of whole, aligned 16 bytes, scales of whole, aligned 4");
    IFL_CHECK_ARG(ldb < (1 << 23), IFL_ENOTSUP, "block8 product: rows of %lld bytes", (long long)ldb);
    return 0;
}

}  // namespace

bool b8_matmul_fits(int64_t M, int64_t N, int64_t K) { return mm8_fits(M, N, K); }

extern "C" int64_t ifl_block8_matmul_scratch_floats(int64_t M, int64_t N, int64_t K, int)
{
    if (M < 1 || N < 1 || K < 1) return 0;
    const Plan p = mm8_plan(M, N, K);
    return p.split > 1 ? p.split * M * N : 0;
}

extern "C" int ifl_block8_matmul_plan(int64_t M, int64_t N, int64_t K)
{
    if (M < 1 || N < 1 || K < 1) return 0;
    const Plan p = mm8_plan(M, N, K);
    return (p.kind ? 16 * p.kind : p.tile) | p.split << 16;
}

extern "C" int ifl_block8_matmul(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t lsa, int fa, const uint8_t* b, int64_t ldb,
                                 const uint8_t* sb, int64_t lsb, int fb, const void* bias, int btype, void* out, int otype, int64_t ldo,
                                 float* scratch, int64_t M, int64_t N, int64_t K, void* stream)
{
    const bool exact = mm8_exact(otype);
    otype &= ~IFL_P_8BIT;
    IFL_CHECK_ARG(b8_fmt_ok(fa) && b8_fmt_ok(fb), IFL_EINVAL, "block8_matmul: formats %d, %d", fa, fb);
    if (int rc = mm8_check(M, N, K, b, ldb, sb, lsb, bias, btype, out, otype, ldo)) return rc;
    if (M == 0) return 0;
    IFL_CHECK_ARG(a && sa, IFL_EINVAL, "block8_matmul: null pointer");
    IFL_CHECK_ARG(lda >= K && lsa >= ifl_cdiv((int)K, B8_BLK), IFL_EINVAL, "block8_matmul: row strides");
    IFL_CHECK_ARG(lda % 16 == 0 && (uintptr_t)a % 16 == 0 && lsa % 4 == 0 && (uintptr_t)sa % 4 == 0, IFL_EINVAL,
                  "block8_matmul: codes in rows of whole, aligned 16 bytes, scales of whole, aligned 4");
    IFL_CHECK_ARG(lda < (1 << 23), IFL_ENOTSUP, "block8_matmul: rows of %lld bytes", (long long)lda);
    const Plan p = mm8_plan(M, N, K);
    IFL_CHECK_ARG(p.split == 1 || scratch, IFL_EINVAL, "block8_matmul: no scratch");
    MM8 q = {};
    q.a = a; q.b = b; q.sa = sa; q.sb = sb; q.lda = lda; q.ldb = ldb; q.lsa = lsa; q.lsb = lsb; q.bias = bias; q.btype = btype;
    q.out = out; q.otype = otype; q.ldo = ldo; q.M = M; q.N = N; q.K = (int)K; q.part = scratch;
    hipStream_t st = (hipStream_t)stream;
    if (fa == 0 && fb == 0) return mm8_launch<0, 0>(q, p, exact, st);
    if (fa == 0) return mm8_launch<0, 1>(q, p, exact, st);
    if (fb == 0) return mm8_launch<1, 0>(q, p, exact, st);
    return mm8_launch<1, 1>(q, p, exact, st);
}

extern "C" int64_t ifl_block8_linear_scratch_bytes(int64_t M, int64_t N, int64_t K, int otype)
{
    if (M < 1 || N < 1 || K < 1) return 0;
    if (mm8_own(M, K)) return 0;
    return M * ((K + 15) / 16 * 16) + M * ((K + 511) / 512 * 4) + 4 * ifl_block8_matmul_scratch_floats(M, N, K, otype) + 16;
}

extern "C" int ifl_block8_linear(const void* x, int xtype, int64_t ldx, const uint8_t* b, int64_t ldb, const uint8_t* sb, int64_t lsb, int fb,
                                 const void* bias, int btype, void* out, int64_t ldo, void* scratch, int64_t M, int64_t N, int64_t K,
                                 void* stream)
{
    const bool exact = mm8_exact(xtype);
    const int otype = xtype;
    xtype &= ~IFL_P_8BIT;
    IFL_CHECK_ARG(b8_fmt_ok(fb) && b8_type_ok(xtype), IFL_EINVAL, "block8_linear: types");
    if (int rc = mm8_check(M, N, K, b, ldb, sb, lsb, bias, btype, out, xtype, ldo)) return rc;
    if (M == 0) return 0;
    IFL_CHECK_ARG(x && (M == 1 || ldx >= K), IFL_EINVAL, "block8_linear: x");
    hipStream_t st = (hipStream_t)stream;
    if (mm8_own(M, K)) {
        MM8 q = {};
        q.b = b; q.sb = sb; q.ldb = ldb; q.lsb = lsb; q.bias = bias; q.btype = btype; q.out = out; q.otype = xtype; q.ldo = ldo;
        q.M = M; q.N = N; q.K = (int)K; q.x = x; q.ldx = ldx;
        const int KB = ifl_cdiv((int)K, B8_BLK), sm = (int)M * KB * B8_BLK + (int)M * KB;
        const dim3 grid((unsigned)((N + 15) / 16)), block(64 * SK_WAVES);
#define MM8_OWN2(FB, EX, TX) hipLaunchKernelGGL(HIP_KERNEL_NAME(mm8_skinny_kernel<1, 0, FB, EX, true, TX>), grid, block, sm, st, q)
#define MM8_OWN(FB) do { \
            if (xtype == IFL_T_F32) MM8_OWN2(FB, true, float); \
            else if (xtype == IFL_T_BF16) { if (exact) MM8_OWN2(FB, true, __bf16); else MM8_OWN2(FB, false, __bf16); } \
            else if (exact) MM8_OWN2(FB, true, _Float16); else MM8_OWN2(FB, false, _Float16); } while (0)
        if (fb == 0) MM8_OWN(0); else MM8_OWN(1);
        IFL_LAUNCH_CHECK();
        return 0;
    }
    IFL_CHECK_ARG(scratch && (uintptr_t)scratch % 16 == 0, IFL_EINVAL, "block8_linear: scratch");
    const int64_t lda = (K + 15) / 16 * 16, lsa = (K + 511) / 512 * 4;
    uint8_t* codes = (uint8_t*)scratch;
    uint8_t* scales = codes + M * lda;
    float* part = (float*)(scales + M * lsa);                            // (both sizes are multiples of 4)
    if (int rc = ifl_block8_quantize(x, xtype, ldx, 1, codes, lda, scales, lsa, M, K, IFL_Q_E4M3, stream)) return rc;
    return ifl_block8_matmul(codes, lda, scales, lsa, IFL_Q_E4M3, b, ldb, sb, lsb, fb, bias, btype, out, otype, ldo, part, M, N, K, stream);
}

// linear8.hip -- the 8-bit linear layer's forward and backward pass, one call each: what to quantize, which products, and where
// their scratch lies.  The kernels are block8.hip's, matmul8.hip's and wgrad8.hip's.
#include "block8.h"

namespace {

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t code_ld(int64_t cols) { return up16(cols); }
int64_t scale_ld(int64_t cols) { return (cols + 511) / 512 * 4; }
int64_t block_bytes(int64_t rows, int64_t cols) { return up16(rows * code_ld(cols)) + up16(rows * scale_ld(cols)); }
// what the products and the weight gradient take: looked at before anything is launched
constexpr int64_t PRODUCT_ROWS = 0x3fffffff, PRODUCT_LD = 1 << 23, WGRAD_COLS = 0x3fffff;
bool sizes_ok(int64_t M, int64_t N, int64_t K) { return M >= 0 && N >= 1 && K >= 1 && M < ((int64_t)1 << 40) && N < ((int64_t)1 << 30) && K < ((int64_t)1 << 30); }

}  // namespace

extern "C" int64_t ifl_linear8_fwd_scratch_bytes(int64_t M, int64_t N, int64_t K, int xtype)
{
    if (!sizes_ok(M, N, K)) return 0;
    return block_bytes(N, K) + 4 * ifl_block8_matmul_scratch_floats(M, N, K, xtype);
}

extern "C" int ifl_linear8_fwd(const void* x, int xtype, int64_t x_rs, int64_t x_cs, const void* w, int wtype, int64_t w_rs, int64_t w_cs,
                               const void* bias, int btype, uint8_t* codes, uint8_t* scales, void* y, void* scratch, int64_t M, int64_t N,
                               int64_t K, void* stream)
{
    const int otype = xtype;
    xtype &= ~IFL_P_8BIT;
    IFL_CHECK_ARG(sizes_ok(M, N, K), IFL_EINVAL, "linear8_fwd: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG(b8_type_ok(xtype) && b8_type_ok(wtype) && (!bias || b8_type_ok(btype)), IFL_EINVAL, "linear8_fwd: element types");
    IFL_CHECK_ARG(M <= PRODUCT_ROWS && N <= PRODUCT_ROWS && code_ld(K) < PRODUCT_LD && b8_matmul_fits(M, N, K), IFL_ENOTSUP, "linear8_fwd: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    if (M == 0) return 0;
    IFL_CHECK_ARG(x && w && codes && scales && y, IFL_EINVAL, "linear8_fwd: null pointer");
    IFL_CHECK_ARG(w_rs == 1 || w_cs == 1 || N == 1, IFL_EINVAL, "linear8_fwd: strides of w");
    IFL_CHECK_ARG(scratch && (uintptr_t)scratch % 16 == 0 && (uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 4 == 0, IFL_EINVAL, "linear8_fwd: alignment of scratch, codes or scales");
    uint8_t* wc = (uint8_t*)scratch;
    uint8_t* ws = wc + up16(N * code_ld(K));
    float* part = (float*)(wc + block_bytes(N, K));
    if (x_cs == 1 && w_cs == 1) {
        if (int rc = b8_quantize2(x, xtype, x_rs, w, wtype, w_rs, codes, scales, wc, ws, code_ld(K), scale_ld(K), M, N, K, stream)) return rc;
    } else {
        if (int rc = ifl_block8_quantize(x, xtype, x_rs, x_cs, codes, code_ld(K), scales, scale_ld(K), M, K, IFL_Q_E4M3, stream)) return rc;
        if (int rc = ifl_block8_quantize(w, wtype, w_rs, w_cs, wc, code_ld(K), ws, scale_ld(K), N, K, IFL_Q_E4M3, stream)) return rc;
    }
    return ifl_block8_matmul(codes, code_ld(K), scales, scale_ld(K), IFL_Q_E4M3, wc, code_ld(K), ws, scale_ld(K), IFL_Q_E4M3, bias, btype, y, otype, N, part,
                             M, N, K, stream);
}

extern "C" int64_t ifl_linear8_bwd_scratch_bytes(int64_t M, int64_t N, int64_t K, int xtype, int need_dx, int need_dw)
{
    if (!sizes_ok(M, N, K)) return 0;
    const int64_t a = need_dx ? block_bytes(M, N) + block_bytes(K, N) + up16(4 * ifl_block8_matmul_scratch_floats(M, K, N, xtype)) : 0;
    return a + 4 * ifl_block8_wgrad_scratch_floats(M, N, need_dw ? K : 0, xtype & ~IFL_P_8BIT) + 16;
}

extern "C" int ifl_linear8_bwd(const void* dy, int xtype, int64_t ldy, const uint8_t* codes, const uint8_t* scales, const void* w, int wtype,
                               int64_t w_rs, int64_t w_cs, int gfmt, void* dx, void* dw, void* db, int dbtype, void* scratch, int64_t M,
                               int64_t N, int64_t K, void* stream)
{
    const int otype = xtype;
    xtype &= ~IFL_P_8BIT;
    IFL_CHECK_ARG(sizes_ok(M, N, K), IFL_EINVAL, "linear8_bwd: %lld x %lld x %lld", (long long)M, (long long)N, (long long)K);
    IFL_CHECK_ARG(b8_type_ok(xtype) && b8_type_ok(wtype) && b8_fmt_ok(gfmt) && (!db || b8_type_ok(dbtype)), IFL_EINVAL, "linear8_bwd: types");
    IFL_CHECK_ARG(M <= PRODUCT_ROWS && (!dx || (K <= PRODUCT_ROWS && code_ld(N) < PRODUCT_LD && b8_matmul_fits(M, K, N))) && (!(dw || db) || (N <= WGRAD_COLS && ldy < PRODUCT_LD)) && (!dw || K <= WGRAD_COLS),
                  IFL_ENOTSUP, "linear8_bwd: %lld x %lld x %lld, rows of dy %lld apart", (long long)M, (long long)N, (long long)K, (long long)ldy);
    IFL_CHECK_ARG(M == 0 || (dy && (w || !dx) && ((codes && scales) || !dw)), IFL_EINVAL, "linear8_bwd: null pointer");
    IFL_CHECK_ARG(M <= 1 || ldy >= N, IFL_EINVAL, "linear8_bwd: rows of dy %lld apart", (long long)ldy);
    IFL_CHECK_ARG(!dx || w_rs == 1 || w_cs == 1 || K == 1, IFL_EINVAL, "linear8_bwd: strides of w");
    IFL_CHECK_ARG(scratch && (uintptr_t)scratch % 16 == 0, IFL_EINVAL, "linear8_bwd: scratch");
    uint8_t* at = (uint8_t*)scratch;
    const bool sums = dw || db;
    uint8_t *gc = at, *gs = gc + up16(M * code_ld(N)), *wc = gc + block_bytes(M, N), *ws = wc + up16(K * code_ld(N));
    float* part = (float*)(wc + block_bytes(K, N));
    if (dx) at = (uint8_t*)part + up16(4 * ifl_block8_matmul_scratch_floats(M, K, N, otype));
    // (w^T has rows of w's columns: next to each other in memory as a rule)
    const bool together = dx && sums && w_cs == 1;
    const B8Quant quant = {gc, gs, code_ld(N), scale_ld(N), gfmt,
                           {together ? w : nullptr, w_rs, wc, code_ld(N), ws, scale_ld(N), K, (int)N, b8_pad(N, code_ld(N)), IFL_Q_E4M3}, wtype};
    auto gradients = [&](int steps) {
        return b8_wgrad(steps, dx ? &quant : nullptr, dy, xtype, ldy, codes, code_ld(K), scales, scale_ld(K), IFL_Q_E4M3, nullptr, dw, wtype, K, db, dbtype, (float*)at, M, N, dw ? K : 0, stream);
    };
    if (dx && M > 0) {
        if (int rc = sums ? gradients(1) : ifl_block8_quantize(dy, xtype, ldy, 1, gc, code_ld(N), gs, scale_ld(N), M, N, gfmt, stream)) return rc;
        if (!together)
            if (int rc = ifl_block8_quantize(w, wtype, w_cs, w_rs, wc, code_ld(N), ws, scale_ld(N), K, N, IFL_Q_E4M3, stream)) return rc;
        if (int rc = ifl_block8_matmul(gc, code_ld(N), gs, scale_ld(N), gfmt, wc, code_ld(N), ws, scale_ld(N), IFL_Q_E4M3, nullptr, 0, dx, otype, K, part, M, K, N, stream)) return rc;
    }
    return sums ? gradients(dx ? 2 : 3) : 0;
}

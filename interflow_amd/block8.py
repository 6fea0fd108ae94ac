"""Values in 8-bit blocks: what an activation checkpoint keeps, and what the 8-bit matrix product multiplies.

Format (csrc/block8.h): a row's values in blocks of 128 (the last may be shorter).  A block has one power-of-two scale 2^e, e the
smallest integer >= -126 with max |x| <= F 2^e (F = 448 for e4m3, 57344 for e5m2), and its codes are x 2^-e rounded to nearest
even.  A value is off by at most 2^-4 of itself (e5m2: 2^-3), or by 2^-10 2^e (2^-17 2^e) where it is that small beside its
block's largest; from 0.97 2^128 on (e5m2: 0.94 2^128) it rounds up to 2^128, which is infinity.  NaN stays NaN; infinity stays infinity in e5m2 and becomes NaN in e4m3; neither changes the other values.

* `quantize` / `dequantize`  -- to and from 8-bit blocks
* `matmul`                   -- A B^T of two such matrices on the matrix cores
* `linear`                   -- a layer whose weights are kept in 8-bit blocks (serving); `train_ops.linear8` is its training form
* `weight_grad`              -- dy^T A (and dy's column sums) from a checkpoint A

What a product keeps: the codes times their scales are multiplied exactly and summed in float32, like the other matrix products here.
With `exact=False` a bfloat16 or float16 result comes from the scaled 8-bit matrix instructions instead, which are up to twice as fast
on large products and keep less: among 8 products they drop what is below 2^-13 of the largest.  A result is then off by 4e-5
of itself in the 2-norm for activations with outliers (rounding to float16 adds 2e-4, to bfloat16 1.7e-3), by up to 7 2^-13 of the
sum of its products' magnitudes, and where large products cancel, what they leave is lost.  float32 results are always exact.

Everything runs on the current stream of the tensors' device; nothing synchronises, and calls may be captured into a graph.
There is no CPU fallback."""
from __future__ import annotations

import torch

from . import hip

BLOCK = 128
_FMT = {"e4m3": 0, "e5m2": 1}
_FMT_OF = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_8BIT = 0x100                                           # or-ed to a result's type: products by the 8-bit instructions
_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _on_gpu(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise hip.InterflowHipError(f"{name}: tensor is on {t.device}; the HIP path needs a GPU tensor (no CPU fallback)")
    return t


def _real(t, name):
    """The element type's code."""
    code = _TYPE.get(t.dtype) if isinstance(t, torch.Tensor) and t.is_cuda else None
    if code is None:
        _on_gpu(t, name)
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return code


def _dtype(dtype, what):
    code = _TYPE.get(dtype)
    if code is None:
        raise TypeError(f"{what}: dtype has to be float32, bfloat16 or float16, got {dtype}")
    return code


def _format(fmt, what):
    code = _FMT.get(fmt)
    if code is None:
        raise ValueError(f"{what}: the format has to be 'e4m3' or 'e5m2', got {fmt!r}")
    return code


def _same_device(dev, *ts):
    for t in ts:
        assert t is None or t.get_device() == dev, f"tensors on cuda:{dev} and {t.device}"


_fns = {}
_raw_stream = _get_device = None                        # torch's own, bound at the first call: a build of torch without a GPU lacks them


def _bind():
    global _raw_stream, _get_device                     # (a current_stream() object costs a small call more than its launch)
    _raw_stream, _get_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _call(what, dev, *args):
    """One library call on the current stream of device number `dev`."""
    fn = _fns.get(what)
    if fn is None:
        fn = _fns[what] = getattr(hip.lib(), what)
    if _get_device is None:
        _bind()
    if _get_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        hip.check(rc, what)


def _size(what, *args):
    """A size that the library names; what it refuses raises."""
    fn = _fns.get(what)
    if fn is None:
        fn = _fns[what] = getattr(hip.lib(), what)
    return fn(*args)


def _scratch(n, like):
    """n bytes beside the tensor `like`, or nothing."""
    return like.new_empty((n,), dtype=torch.uint8) if n else None


def _rows_apart(t):
    """Columns contiguous and rows that do not overlap, as far as there are several."""
    return (t.shape[1] == 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])


def _rows_of(t, rows, cols):
    """(t or a contiguous copy, distance of its rows) for a t whose columns may not be contiguous."""
    rs, cs = t.stride()
    if (cs == 1 or cols == 1) and (rows <= 1 or rs >= cols):
        return t, rs if rows > 1 else cols
    return t.contiguous(), cols


_FAR = 1 << 23                                          # elements between rows that the products do not reach across


def _near_rows(t):
    """t, or a copy whose rows follow one another: for what the products read."""
    return t if _rows_apart(t) and (t.shape[0] <= 1 or t.stride(0) < _FAR) else t.contiguous()


def _ld(t):
    """Distance of rows in elements; of a single row, the columns it has."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class Block8:
    """A matrix in 8-bit blocks: `codes` [rows, cols] (torch.float8_e4m3fn or float8_e5m2) and `scales` [rows, ceil(cols / 128)]
    (torch.float8_e8m0fnu), columns contiguous, rows any distance apart.  Made by `quantize`, or from tensors of that form, which
    every call reads as they then are."""
    __slots__ = ("rows", "cols", "_f", "_dev", "_raw", "_codes", "_scales", "_cp", "_ldc", "_sp", "_lds")

    def __init__(self, codes, scales):
        _on_gpu(codes, "Block8 codes")
        _on_gpu(scales, "Block8 scales")
        f = _FMT_OF.get(codes.dtype)
        if f is None or scales.dtype != torch.float8_e8m0fnu:
            raise TypeError(f"Block8: codes in float8_e4m3fn or float8_e5m2 and scales in float8_e8m0fnu, got {codes.dtype} and {scales.dtype}")
        shape, blocks = codes.shape, scales.shape
        assert len(shape) == 2 and len(blocks) == 2 and shape[1] >= 1, (tuple(shape), tuple(blocks))
        rows, cols = shape
        assert blocks[0] == rows and blocks[1] == (cols + 127) // 128, (tuple(shape), tuple(blocks))
        self._dev = dev = codes.get_device()
        if scales.get_device() != dev:
            _same_device(dev, scales)
        self._codes, self._scales = codes, scales
        self.rows, self.cols, self._f, self._raw = rows, cols, f, None

    @classmethod
    def _new(cls, rows, cols, f, like):
        """Room for rows x cols beside the tensor `like`: one allocation, codes in rows of whole 16 bytes and behind them scales in rows
        of whole 4, which is what the product's wide loads want."""
        q = cls.__new__(cls)
        ldc, lds = (cols + 15) // 16 * 16, (cols + 511) // 512 * 4
        q._raw = raw = like.new_empty((rows * (ldc + lds),), dtype=torch.uint8)
        q.rows, q.cols, q._f, q._dev, q._codes, q._scales = rows, cols, f, raw.get_device(), None, None
        q._cp = p = raw.data_ptr()
        q._ldc, q._lds, q._sp = ldc, lds, p + rows * ldc
        return q

    @property
    def codes(self):
        if self._codes is None:
            c = self._raw[:self.rows * self._ldc].view(self.rows, self._ldc)
            self._codes = c.view(torch.float8_e5m2 if self._f else torch.float8_e4m3fn)[:, :self.cols]
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            s = self._raw[self.rows * self._ldc:].view(self.rows, self._lds)
            self._scales = s.view(torch.float8_e8m0fnu)[:, :(self.cols + 127) // 128]
        return self._scales

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def device(self):
        return torch.device("cuda", self._dev)

    @property
    def fmt(self):
        return "e5m2" if self._f else "e4m3"

    def _like(self):
        """A tensor on its device."""
        return self._codes if self._raw is None else self._raw

    def _now(self):
        """Itself, with the addresses and strides that its tensors have now (their owner may have given them other memory); or a
        copy, if their columns are not contiguous."""
        if self._raw is not None:
            return self
        codes, scales, rows, cols = self._codes, self._scales, self.rows, self.cols
        blocks = (cols + 127) // 128
        dev, (cr, cc), (sr, sc) = self._dev, codes.stride(), scales.stride()
        if codes.shape != (rows, cols) or scales.shape != (rows, blocks) or codes.get_device() != dev or scales.get_device() != dev \
                or _FMT_OF.get(codes.dtype) != self._f or scales.dtype != torch.float8_e8m0fnu:
            raise RuntimeError(f"{self}: its tensors were given another shape, type or device: {tuple(codes.shape)} {codes.dtype} on {codes.device}, "
                               f"{tuple(scales.shape)} {scales.dtype} on {scales.device}")
        if cc != 1 and cols > 1 or sc != 1 and blocks > 1:
            return self._copy()
        if rows <= 1:
            cr, sr = cols, blocks
        elif cr < cols or sr < blocks:
            return self._copy()
        self._cp, self._ldc, self._sp, self._lds = codes.data_ptr(), cr, scales.data_ptr(), sr
        return self

    def _copy(self):
        """The same in memory of its own, rows whole 16 and 4 bytes."""
        q = Block8._new(self.rows, self.cols, self._f, self._like())
        q.codes.view(torch.uint8).copy_(self.codes.view(torch.uint8))
        q.scales.view(torch.uint8).copy_(self.scales.view(torch.uint8))
        return q

    def __repr__(self):
        return f"Block8({self.rows} x {self.cols}, {self.fmt}, {self.device})"

    def aligned(self):
        """Itself, or a copy whose rows are whole, aligned 16 and 4 bytes, as `quantize` makes them (a single row's length does not
        matter).  `matmul`, `linear` and `weight_grad` make such a copy in every call that needs one: of weights built from tensors of
        other layouts (scales of 5 bytes a row, say) keep this one instead."""
        self = self._now()
        one = self.rows <= 1
        if self._cp % 16 == 0 and self._sp % 4 == 0 and (one or (self._ldc % 16 == 0 and self._lds % 4 == 0 and self._ldc < _FAR)):
            return self
        return self._copy()


def _b8(q, name):
    if not isinstance(q, Block8):
        raise TypeError(f"{name}: expected a Block8")
    return q


def _up(n, k):
    return (n + k - 1) // k * k


def _matrix(x, rows, cols):
    """(x, row stride, column stride) of x [rows, cols] as the library reads it: one of the strides is 1."""
    rs, cs = x.stride()
    if cs == 1 or cols == 1:
        return x, rs, 1
    if cs and (rs == 1 or rows == 1):
        return x, 1, cs
    return x.contiguous(), cols, 1


def quantize(x, fmt: str = "e4m3") -> Block8:
    """x [rows, cols] (float32, bfloat16 or float16, any strides; a transposed view is read as it is) in 8-bit blocks."""
    t = _real(x, "quantize input")
    f = _format(fmt, "quantize")
    assert x.dim() == 2 and x.shape[1] >= 1, tuple(x.shape)
    rows, cols = x.shape
    x, rs, cs = _matrix(x, rows, cols)
    q = Block8._new(rows, cols, f, x)
    _call("ifl_block8_quantize", q._dev, x.data_ptr(), t, rs, cs, q._cp, q._ldc, q._sp, q._lds, rows, cols, f)
    return q


def dequantize(q: Block8, dtype=torch.float32) -> torch.Tensor:
    """The values [rows, cols] that `q` stands for, rounded once to `dtype` (float16 overflows to infinity above 65504)."""
    q = _b8(q, "dequantize")._now()
    t = _dtype(dtype, "dequantize")
    out = q._like().new_empty((q.rows, q.cols), dtype=dtype)
    _call("ifl_block8_dequantize", q._dev, q._cp, q._ldc, q._sp, q._lds, q._f, None, out.data_ptr(), t, q.cols, q.rows, q.cols)
    return out


def _bias(bias, n, dev):
    """(bias, its address, its type)"""
    if bias is None:
        return None, None, 0
    t = _real(bias, "bias")
    assert bias.shape == (n,), (tuple(bias.shape), n)
    _same_device(dev, bias)
    bias = bias.contiguous()
    return bias, bias.data_ptr(), t


def matmul(a: Block8, b: Block8, bias=None, dtype=torch.bfloat16, exact: bool = True) -> torch.Tensor:
    """a [M, K] times b [N, K]^T (+ bias [N]) -> [M, N] of `dtype`.  Formats may differ.  Products are exact (operands' bits below
    2^-133 aside) and sums float32, rounded once; `exact=False` allows a 16-bit result the 8-bit instructions, which keep less (above)."""
    a, b = _b8(a, "matmul a").aligned(), _b8(b, "matmul b").aligned()
    M, K, N, dev = a.rows, a.cols, b.rows, a._dev
    assert b.cols == K and N >= 1, (tuple(a.shape), tuple(b.shape))
    assert b._dev == dev, f"{a} and {b}"
    bias, bp, bt = _bias(bias, N, dev)
    t = _dtype(dtype, "matmul")
    p = t if exact else t | _8BIT
    out = a._like().new_empty((M, N), dtype=dtype)
    scratch = _scratch(4 * _size("ifl_block8_matmul_scratch_floats", M, N, K, p), out)
    _call("ifl_block8_matmul", dev, a._cp, _up(a._ldc, 16), a._sp, _up(a._lds, 4), a._f, b._cp, _up(b._ldc, 16), b._sp, _up(b._lds, 4), b._f, bp, bt,
          out.data_ptr(), p, N, scratch.data_ptr() if scratch is not None else None, M, N, K)
    return out


def linear(x, w: Block8, bias=None, exact: bool = True) -> torch.Tensor:
    """x [..., K] (float32, bfloat16 or float16) through a layer whose weights w [N, K] are kept in 8-bit blocks: x is quantized
    along its last dimension (e4m3) and multiplied as in `matmul` (`exact` too) -> [..., N] of x's type."""
    t = _real(x, "linear input")
    if not exact:
        t |= _8BIT
    w = _b8(w, "linear weights").aligned()
    shape, K, N = x.shape, w.cols, w.rows
    assert len(shape) >= 1 and shape[-1] == K and N >= 1, (tuple(shape), tuple(w.shape))
    dev = x.get_device()
    assert w._dev == dev, f"x on cuda:{dev}, weights {w}"
    bias, bp, bt = _bias(bias, N, dev) if bias is not None else (None, None, 0)
    x2, ldx = _rows_of(x if len(shape) == 2 else x.reshape(-1, K), x.numel() // K, K)
    M = x2.shape[0]
    out = x.new_empty((M, N) if len(shape) == 2 else (*shape[:-1], N))
    scratch = _scratch(_size("ifl_block8_linear_scratch_bytes", M, N, K, t), x)
    _call("ifl_block8_linear", dev, x2.data_ptr(), t, ldx, w._cp, _up(w._ldc, 16), w._sp, _up(w._lds, 4), w._f, bp, bt, out.data_ptr(), N,
          scratch.data_ptr() if scratch is not None else None, M, N, K)
    return out


def weight_grad(dy, q: Block8, dtype=torch.float32, bias_dtype=None, weight: bool = True):
    """(dw, db): dy [M, N]^T times the checkpoint q [M, K] -> dw [N, K] of `dtype` (None unless `weight`), and dy's column sums
    [N] of `bias_dtype` (None without one).  Products are exact (operands' bits below 2^-133 aside) and sums float32, in an order
    that depends on the sizes only; an infinity of an e5m2 checkpoint gives infinities of its and the gradients' sign.  Both operands pass through scratch as bfloat16 terms: 2 bytes per code, 2 to 6 per gradient."""
    _real(dy, "weight_grad dy")
    _b8(q, "weight_grad checkpoint")
    assert dy.dim() == 2 and dy.shape[0] == q.rows and dy.shape[1] >= 1, (tuple(dy.shape), tuple(q.shape))
    _same_device(q._dev, dy)
    dy = _near_rows(dy)
    if weight:
        _dtype(dtype, "weight_grad")
    if bias_dtype is not None:
        _dtype(bias_dtype, "weight_grad")
    if not weight and bias_dtype is None:
        return None, None
    if not weight:
        return _wgrad(dy, None, 0, None, 0, 0, 0, None, None, bias_dtype)
    q = q.aligned()
    return _wgrad(dy, q._cp, _up(q._ldc, 16), q._sp, q._lds, q._f, q.cols, None, dtype, bias_dtype)


def _wgrad(dy, cp, ldc, sp, lds, f, K, chan, dtype, bias_dtype):
    """dy [M, N], contiguous columns; codes [M, K] and scales by their addresses and row strides; chan float32 [K] or None."""
    M, N = dy.shape
    dev = dy.get_device()
    dw = dy.new_empty((N, K), dtype=dtype) if dtype is not None else None
    db = dy.new_empty((N,), dtype=bias_dtype) if bias_dtype is not None else None
    scratch = _scratch(4 * _size("ifl_block8_wgrad_scratch_floats", M, N, K if dw is not None else 0, _TYPE[dy.dtype]), dy)
    _call("ifl_block8_wgrad", dev, dy.data_ptr(), _TYPE[dy.dtype], _ld(dy), cp, ldc, sp, lds, f, chan.data_ptr() if chan is not None else None,
          dw.data_ptr() if dw is not None else None, _TYPE[dtype] if dw is not None else 0, K, db.data_ptr() if db is not None else None,
          _TYPE[bias_dtype] if db is not None else 0, scratch.data_ptr() if scratch is not None else None, M, N, K if dw is not None else 0)
    return dw, db


# ------------------------------------------------------------------------------------------------ the layer in training
def _linear_fwd(x2, w, bias, keep: bool, exact: bool):
    """(y [M, N], x's 8-bit blocks as one tensor, if they are to be kept): quantize x and w along K and multiply."""
    M, K = x2.shape
    N = w.shape[0]
    t, wt, dev = _TYPE[x2.dtype], _TYPE[w.dtype], x2.get_device()
    if not exact:
        t |= _8BIT
    x2, rs, cs = _matrix(x2, M, K)
    w, wrs, wcs = _matrix(w, N, K)
    bias, bp, bt = _bias(bias, N, dev) if bias is not None else (None, None, 0)
    y = x2.new_empty((M, N))
    codes, scales = M * ((K + 15) // 16 * 16), M * ((K + 511) // 512 * 4)
    raw = x2.new_empty((codes + scales,), dtype=torch.uint8)
    scratch = x2.new_empty((_size("ifl_linear8_fwd_scratch_bytes", M, N, K, t),), dtype=torch.uint8)
    cp = raw.data_ptr()
    _call("ifl_linear8_fwd", dev, x2.data_ptr(), t, rs, cs, w.data_ptr(), wt, wrs, wcs, bp, bt, cp, cp + codes, y.data_ptr(),
          scratch.data_ptr(), M, N, K)
    return y, raw if keep else None


def _backward_reaches(N, K, need_x, need_w, need_b):
    """Refuses a layer that the forward pass takes and the backward pass does not, before either."""
    if need_x and N > (1 << 23) - 16 or (need_w or need_b) and N > 0x3fffff or need_w and K > 0x3fffff:
        raise NotImplementedError(f"linear8: gradients of a weight of {N} x {K}")


def _linear_bwd(g, raw, w, need_x, need_w, bias_dtype, f, exact: bool):
    """(dx, dw, db) of `_linear_fwd`; g [M, N] contiguous columns, raw the kept blocks of x."""
    M, N = g.shape
    K = w.shape[1]
    t, wt = _TYPE[g.dtype], _TYPE[w.dtype]
    if not exact:
        t |= _8BIT
    w, wrs, wcs = _matrix(w, N, K)
    dx = dw = db = dxp = dwp = dbp = cp = sp = None
    if need_x:
        dx = g.new_empty((M, K))
        dxp = dx.data_ptr()
    if need_w:
        dw = w.new_empty((N, K))
        dwp, cp = dw.data_ptr(), raw.data_ptr()
        sp = cp + M * ((K + 15) // 16 * 16)
    if bias_dtype is not None:
        db = g.new_empty((N,), dtype=bias_dtype)
        dbp = db.data_ptr()
    scratch = g.new_empty((_size("ifl_linear8_bwd_scratch_bytes", M, N, K, t, int(need_x), int(need_w)),), dtype=torch.uint8)
    _call("ifl_linear8_bwd", g.get_device(), g.data_ptr(), t, _ld(g), cp, sp, w.data_ptr(), wt, wrs, wcs, f, dxp, dwp, dbp,
          _TYPE[bias_dtype] if bias_dtype is not None else 0, scratch.data_ptr(), M, N, K)
    return dx, dw, db

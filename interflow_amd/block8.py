"""Values in 8-bit blocks: what an activation checkpoint keeps, and what the 8-bit matrix product multiplies.

Format (csrc/block8.h): a row's values in blocks of 128 (the last may be shorter).  A block has one power-of-two scale 2^e, e the
smallest integer >= -126 with max |x| <= F 2^e (F = 448 for e4m3, 57344 for e5m2), and its codes are x 2^-e rounded to nearest
even.  A value is off by at most 2^-4 of itself (e5m2: 2^-3), or by 2^-10 2^e (2^-17 2^e) where it is that small beside its
block's largest.  NaN stays NaN; infinity stays infinity in e5m2 and becomes NaN in e4m3; neither changes the other values.

* `quantize` / `dequantize`  -- to and from 8-bit blocks
* `matmul`                   -- A B^T of two such matrices on the scaled 8-bit matrix instructions, sums in float32
* `linear`                   -- a layer whose weights are kept in 8-bit blocks (serving); `train_ops.linear8` is its training form
* `weight_grad`              -- dy^T A (and dy's column sums) from a checkpoint A

Everything runs on the current stream of the tensors' device; nothing synchronises, and calls may be captured into a graph.
There is no CPU fallback."""
from __future__ import annotations

import torch

from . import hip

BLOCK = 128
_FMT = {"e4m3": (0, torch.float8_e4m3fn), "e5m2": (1, torch.float8_e5m2)}
_FMT_OF = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _on_gpu(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise hip.InterflowHipError(f"{name}: tensor is on {t.device}; the HIP path needs a GPU tensor (no CPU fallback)")
    return t


def _real(t, name):
    _on_gpu(t, name)
    if t.dtype not in _TYPE:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return t


def _dtype(dtype, what):
    if dtype not in _TYPE:
        raise TypeError(f"{what}: dtype has to be float32, bfloat16 or float16, got {dtype}")
    return dtype


def _same_device(dev, *ts):
    for t in ts:
        if t is not None:
            assert t.device == dev, f"tensors on {dev} and {t.device}"


def _call(what, dev, *args):
    """One library call on the current stream of `dev`."""
    fn = getattr(hip.lib(), what)
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    if rc:
        hip.check(rc, what)


class Block8:
    """A matrix in 8-bit blocks: `codes` [rows, cols] (torch.float8_e4m3fn or float8_e5m2) and `scales` [rows, ceil(cols / 128)]
    (torch.float8_e8m0fnu), columns contiguous, rows any distance apart.  Made by `quantize`, or from tensors of that form."""
    __slots__ = ("codes", "scales")

    def __init__(self, codes, scales):
        _on_gpu(codes, "Block8 codes")
        _on_gpu(scales, "Block8 scales")
        if codes.dtype not in _FMT_OF or scales.dtype != torch.float8_e8m0fnu:
            raise TypeError(f"Block8: codes in float8_e4m3fn or float8_e5m2 and scales in float8_e8m0fnu, got {codes.dtype} and {scales.dtype}")
        assert codes.dim() == 2 and scales.dim() == 2 and codes.shape[1] >= 1, (tuple(codes.shape), tuple(scales.shape))
        assert scales.shape == (codes.shape[0], -(-codes.shape[1] // BLOCK)), (tuple(codes.shape), tuple(scales.shape))
        _same_device(codes.device, scales)
        self.codes = codes if _rows_apart(codes) else codes.contiguous()
        self.scales = scales if _rows_apart(scales) else scales.contiguous()

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    @property
    def fmt(self):
        return "e4m3" if self.codes.dtype == torch.float8_e4m3fn else "e5m2"

    def __repr__(self):
        return f"Block8({self.codes.shape[0]} x {self.codes.shape[1]}, {self.fmt}, {self.device})"


def _rows_apart(t):
    """Columns contiguous and rows that do not overlap, as far as there are several."""
    return (t.shape[1] == 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])


def _ld(t):
    """Distance of rows in elements; of a single row, the columns it has."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _alloc(rows, cols, fmt, dev):
    """Codes in rows of whole 16 bytes, scales in rows of whole 4: what the product's wide loads want."""
    codes = torch.empty((rows, (cols + 15) // 16 * 16), dtype=_FMT[fmt][1], device=dev)
    scales = torch.empty((rows, (cols + 511) // 512 * 4), dtype=torch.float8_e8m0fnu, device=dev)
    q = Block8.__new__(Block8)
    q.codes, q.scales = codes[:, :cols], scales[:, :(cols + 127) // 128]
    return q


def quantize(x, fmt: str = "e4m3") -> Block8:
    """x [rows, cols] (float32, bfloat16 or float16, any strides; a transposed view is read as it is) in 8-bit blocks."""
    _real(x, "quantize input")
    if fmt not in _FMT:
        raise ValueError(f"quantize: fmt has to be 'e4m3' or 'e5m2', got {fmt!r}")
    assert x.dim() == 2 and x.shape[1] >= 1, tuple(x.shape)
    rows, cols = x.shape
    rs, cs = x.stride()
    if cs == 1 or cols == 1:
        cs = 1
    elif rs != 1 and rows > 1 or cs == 0:
        x = x.contiguous()
        rs, cs = cols, 1
    elif rows == 1:
        rs = 1
    q = _alloc(rows, cols, fmt, x.device)
    _call("ifl_block8_quantize", x.device, x.data_ptr(), _TYPE[x.dtype], rs, cs, q.codes.data_ptr(), _ld(q.codes), q.scales.data_ptr(),
          _ld(q.scales), rows, cols, _FMT[fmt][0])
    return q


def dequantize(q: Block8, dtype=torch.float32) -> torch.Tensor:
    """The values [rows, cols] that `q` stands for, rounded once to `dtype` (float16 overflows to infinity above 65504)."""
    if not isinstance(q, Block8):
        raise TypeError("dequantize: expected a Block8")
    out = torch.empty(q.shape, dtype=_dtype(dtype, "dequantize"), device=q.device)
    _call("ifl_block8_dequantize", q.device, q.codes.data_ptr(), _ld(q.codes), q.scales.data_ptr(), _ld(q.scales), _FMT_OF[q.codes.dtype], None,
          out.data_ptr(), _TYPE[dtype], out.shape[1], out.shape[0], out.shape[1])
    return out


def _operand(q, name):
    """(codes, scales) as the product reads them: aligned rows of whole 16 and 4 bytes; copies where they are not."""
    if not isinstance(q, Block8):
        raise TypeError(f"{name}: expected a Block8")
    codes, scales = q.codes, q.scales
    if _ld(codes) % 16 or codes.data_ptr() % 16:
        if codes.shape[0] != 1 or codes.data_ptr() % 16:
            codes = torch.empty((codes.shape[0], (codes.shape[1] + 15) // 16 * 16), dtype=codes.dtype, device=codes.device)[:, :codes.shape[1]]
            codes.view(torch.uint8).copy_(q.codes.view(torch.uint8))
    if _ld(scales) % 4 or scales.data_ptr() % 4:
        scales = torch.empty((scales.shape[0], (scales.shape[1] + 3) // 4 * 4), dtype=scales.dtype, device=scales.device)[:, :scales.shape[1]]
        scales.view(torch.uint8).copy_(q.scales.view(torch.uint8))
    return codes, scales


def _up(n, k):
    return (n + k - 1) // k * k


def _bias(bias, n, dev):
    if bias is None:
        return None, 0
    _real(bias, "bias")
    assert bias.shape == (n,), (tuple(bias.shape), n)
    _same_device(dev, bias)
    return bias.contiguous(), _TYPE[bias.dtype]


def matmul(a: Block8, b: Block8, bias=None, dtype=torch.bfloat16) -> torch.Tensor:
    """a [M, K] times b [N, K]^T (+ bias [N]) -> [M, N] of `dtype`.  Formats may differ.  Sums are float32, rounded once."""
    a_c, a_s = _operand(a, "a")
    b_c, b_s = _operand(b, "b")
    M, K = a_c.shape
    N = b_c.shape[0]
    assert b_c.shape[1] == K and N >= 1, (tuple(a.shape), tuple(b.shape))
    _same_device(a_c.device, b_c)
    bias, bt = _bias(bias, N, a_c.device)
    out = torch.empty((M, N), dtype=_dtype(dtype, "matmul"), device=a_c.device)
    n = hip.lib().ifl_block8_matmul_scratch_floats(M, N, K, _TYPE[dtype])
    scratch = torch.empty((n,), dtype=torch.float32, device=out.device) if n else None
    _call("ifl_block8_matmul", a_c.device, a_c.data_ptr(), _up(_ld(a_c), 16), a_s.data_ptr(), _up(_ld(a_s), 4), _FMT_OF[a_c.dtype], b_c.data_ptr(),
          _up(_ld(b_c), 16), b_s.data_ptr(), _up(_ld(b_s), 4), _FMT_OF[b_c.dtype], bias.data_ptr() if bias is not None else None, bt,
          out.data_ptr(), _TYPE[dtype], N, scratch.data_ptr() if n else None, M, N, K)
    return out


def linear(x, w: Block8, bias=None) -> torch.Tensor:
    """x [..., K] (float32, bfloat16 or float16) through a layer whose weights w [N, K] are kept in 8-bit blocks: x is quantized
    along its last dimension (e4m3) and multiplied -> [..., N] of x's type."""
    _real(x, "linear input")
    if not isinstance(w, Block8):
        raise TypeError("linear: the weights have to be a Block8 (block8.quantize)")
    assert x.dim() >= 1 and x.shape[-1] == w.shape[1], (tuple(x.shape), tuple(w.shape))
    _same_device(x.device, w)
    K, N = x.shape[-1], w.shape[0]
    b_c, b_s = _operand(w, "weights")
    bias, bt = _bias(bias, N, x.device)
    x2 = x.reshape(-1, K)
    if not _rows_apart(x2):
        x2 = x2.contiguous()
    M = x2.shape[0]
    out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
    t = _TYPE[x.dtype]
    n = hip.lib().ifl_block8_linear_scratch_bytes(M, N, K, t)
    scratch = torch.empty((n,), dtype=torch.uint8, device=x.device) if n else None
    _call("ifl_block8_linear", x.device, x2.data_ptr(), t, _ld(x2), b_c.data_ptr(), _up(_ld(b_c), 16), b_s.data_ptr(), _up(_ld(b_s), 4),
          _FMT_OF[b_c.dtype], bias.data_ptr() if bias is not None else None, bt, out.data_ptr(), N, scratch.data_ptr() if n else None, M, N, K)
    return out


def weight_grad(dy, q: Block8, dtype=torch.float32, bias_dtype=None, weight: bool = True):
    """(dw, db): dy [M, N]^T times the checkpoint q [M, K] -> dw [N, K] of `dtype` (None unless `weight`), and dy's column sums
    [N] of `bias_dtype` (None without one).  Products are exact and sums float32, in an order that depends on the sizes only."""
    _real(dy, "weight_grad dy")
    if not isinstance(q, Block8):
        raise TypeError("weight_grad: expected a Block8")
    assert dy.dim() == 2 and dy.shape[0] == q.shape[0] and dy.shape[1] >= 1, (tuple(dy.shape), tuple(q.shape))
    _same_device(dy.device, q)
    if not _rows_apart(dy):
        dy = dy.contiguous()
    codes, scales = _operand(q, "checkpoint") if weight else (None, None)
    return _wgrad(dy, codes, scales, None, _dtype(dtype, "weight_grad") if weight else None,
                  _dtype(bias_dtype, "weight_grad") if bias_dtype is not None else None)


def _wgrad(dy, codes, scales, chan, dtype, bias_dtype):
    """dy [M, N], codes [M, K], scales [M, ceil(K / 128)] with contiguous columns, chan float32 [K] or None; without `dtype` the
    column sums alone (no codes)."""
    M, N = dy.shape
    dev = dy.device
    if dtype is None:
        if bias_dtype is None:
            return None, None
        db = torch.empty((N,), dtype=bias_dtype, device=dev)
        n = hip.lib().ifl_block8_wgrad_scratch_floats(M, N, 0, _TYPE[dy.dtype])
        scratch = torch.empty((n,), dtype=torch.float32, device=dev) if n else None
        _call("ifl_block8_wgrad", dev, dy.data_ptr(), _TYPE[dy.dtype], _ld(dy), None, 0, None, 0, 0, None, None, 0, 0, db.data_ptr(), _TYPE[bias_dtype],
              scratch.data_ptr() if n else None, M, N, 0)
        return None, db
    K = codes.shape[1]
    dw = torch.empty((N, K), dtype=dtype, device=dev)
    db = torch.empty((N,), dtype=bias_dtype, device=dev) if bias_dtype is not None else None
    n = hip.lib().ifl_block8_wgrad_scratch_floats(M, N, K, _TYPE[dy.dtype])
    scratch = torch.empty((n,), dtype=torch.float32, device=dev) if n else None
    _call("ifl_block8_wgrad", dev, dy.data_ptr(), _TYPE[dy.dtype], _ld(dy), codes.data_ptr(), _ld(codes), scales.data_ptr(), _ld(scales),
          _FMT_OF[codes.dtype], chan.data_ptr() if chan is not None else None, dw.data_ptr(), _TYPE[dtype], K,
          db.data_ptr() if db is not None else None, _TYPE[bias_dtype] if db is not None else 0,
          scratch.data_ptr() if n else None, M, N, K)
    return dw, db

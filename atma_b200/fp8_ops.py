"""Rows and weights in 8 bits (libatma_decoder.so): what a layer multiplies, in e4m3 with fp32 scales.

A row has a scale for every block of 128 channels: s = max(max |x| / 448, 2^-126), values = e4m3(x / s), the quotient rounded once.
A weight has one for every block of 128 rows and 128 columns.  A NaN or an infinity in a row makes the row's results NaN, and no
other's.  Everything launches on the current CUDA stream, allocates only its results and never synchronises.
"""

import ctypes

import torch

from . import _lib
from .decoder_ops import _check
from .inference_ops import _overlap

_new, _device, _stream = torch.empty_strided, torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream

BLOCK = 128                           # channels that share a scale
TOP, LEAST = 448.0, 2.0 ** -126       # the largest e4m3 value, the smallest scale
E4M3 = torch.float8_e4m3fn
_TYPES = (torch.bfloat16, torch.float32)


def blocks(n):
    return -(-n // BLOCK)


def _here(*tensors):
    """All of them on the current CUDA device (its number), to whose current stream launches go."""
    here = _device()
    for t in tensors:
        if t is not None and t.get_device() != here:
            if t.get_device() < 0:
                raise RuntimeError("operations in 8 bits require CUDA tensors (atma_b200 has no CPU path)")
            raise ValueError(f"a tensor on {t.device}, the current device is cuda:{here}")
    return here


def _apart(out, *inputs):
    """Refuses results over what is read: other CTAs read on while the first ones write."""
    for t in inputs:
        if t is not None and _overlap(out, t):
            raise ValueError("results must not overlap what is read")


def _own(out):
    """Refuses results into a copy: the memory that the caller named would keep what it has."""
    if out.copied:
        raise ValueError("out must be rows that start on 16-byte boundaries with scales that lie block by block; these were copied")


def _stride(width):
    """Bytes between rows that start on 16-byte boundaries."""
    return width + -width % 16


def _storage(shape, width, device):
    """Values whose rows lie dense on 16-byte boundaries."""
    strides = [_stride(width), 1]
    for n in reversed(shape[1:]):
        strides.insert(0, strides[0] * n)
    return torch.empty_strided((*shape, width), strides, device=device, dtype=E4M3)


def _row_stride(values):
    """Bytes between the rows of (..., rows, width) if they lie dense behind one another on 16-byte boundaries, else None."""
    shape, strides = values.shape, values.stride()
    width = shape[-1]
    if strides[-1] != 1 and width > 1 or values.data_ptr() % 16:
        return None
    if values.numel() == width:                                                    # one row: its stride is not used
        return _stride(width)
    step = rs = strides[-2]
    if step % 16 or step < width:
        return None
    for d in range(len(shape) - 3, -1, -1):
        step *= shape[d + 1]
        if shape[d] > 1 and strides[d] != step:
            return None
    return rs


class Fp8Rows:
    """Rows in 8 bits: ``values`` (rows, width) float8_e4m3fn, ``scales`` (rows, blocks) float32.  Rows that do not start on 16-byte
    boundaries and scales that do not lie block by block (stride 1 along the rows) are copied, and such rows take no results."""

    __slots__ = ("values", "scales", "row_stride", "scale_stride", "copied")

    def __init__(self, values, scales):
        shape = values.shape
        if len(shape) != 2 or values.dtype is not E4M3 or scales.dtype is not torch.float32 or scales.shape != (shape[0], -(-shape[1] // BLOCK)):
            raise ValueError("rows in 8 bits are (rows, width) float8_e4m3fn values and (rows, blocks of 128) float32 scales")
        if scales.get_device() != values.get_device():
            raise ValueError("values and scales must be on one device")
        (rows, width), (step, unit) = shape, values.stride()
        self.copied = False
        if rows < 2 or unit != 1 or step < width or step % 16 or values.data_ptr() % 16:
            step = _row_stride(values)
            if step is None:
                values = _storage(shape[:1], width, values.device).copy_(values)
                step, self.copied = _stride(width), rows > 0
        self.row_stride = step
        along, step = scales.stride()
        if width <= BLOCK:                       # one block: its stride is not used
            step = rows
        if rows > 1 and along != 1 or step < rows:
            scales, step, self.copied = scales.t().contiguous().t(), rows, True
        self.values, self.scales, self.scale_stride = values, scales, step if step > 0 else 1      # words between neighbouring blocks' scales

    @property
    def shape(self):
        return self.values.shape

    def __getitem__(self, rows):
        """Some of the rows (a slice)."""
        return Fp8Rows(self.values[rows], self.scales[rows])

    def columns(self, start, stop, used=None):
        """Columns start .. stop - 1, whole blocks, as rows of their own in the same memory; ``used``: only so many of them, the rest of the
        last block is left."""
        if start % BLOCK or not 0 <= start < stop <= self.shape[1] or stop % BLOCK and stop != self.shape[1]:
            raise ValueError(f"columns {start} to {stop} of {self.shape[1]} are not whole blocks of {BLOCK}")
        if used is not None:
            if not 0 < used <= stop - start or blocks(used) != blocks(stop - start):
                raise ValueError(f"{used} columns do not reach the last of the blocks of {stop - start}")
            stop = start + used
        return Fp8Rows(self.values[:, start:stop], self.scales[:, start // BLOCK:blocks(stop)])

    def wide(self):
        """What the rows stand for, in fp32."""
        return self.values.float() * self.scales.repeat_interleave(BLOCK, 1)[:, :self.shape[1]]


class Fp8Weight:
    """A weight in 8 bits: ``values`` (..., N, K) float8_e4m3fn, ``scales`` (..., blocks of N, blocks of K) float32.  Leading dimensions
    hold matrices of one shape: an expert's, or the gate and the up projection of a feed-forward (2, N, K)."""

    __slots__ = ("values", "scales", "row_stride")

    def __init__(self, values, scales):
        shape = values.shape
        if len(shape) < 2 or values.dtype is not E4M3 or scales.dtype is not torch.float32 or \
                scales.shape != (*shape[:-2], -(-shape[-2] // BLOCK), -(-shape[-1] // BLOCK)):
            raise ValueError("a weight in 8 bits is (..., N, K) float8_e4m3fn values and (..., N / 128, K / 128) float32 scales")
        if scales.get_device() != values.get_device():
            raise ValueError("values and scales must be on one device")
        rs = shape[-1] if shape[-1] % 16 == 0 and values.is_contiguous() and values.data_ptr() % 16 == 0 else _row_stride(values)
        if rs is None:
            values = _storage(values.shape[:-1], values.shape[-1], values.device).copy_(values)
            rs = _stride(values.shape[-1])
        self.values, self.scales, self.row_stride = values, scales if scales.is_contiguous() else scales.contiguous(), rs

    @classmethod
    def of(cls, weight):
        """A weight (..., N, K) in 8 bits (once, when a model is loaded)."""
        *lead, n, k = weight.shape
        flat = weight.reshape(-1, n, k)
        values = _storage((flat.shape[0], n), k, weight.device)
        scales = torch.empty((flat.shape[0], blocks(n), blocks(k)), device=weight.device)
        for i, w in enumerate(flat):                                               # one matrix at a time: fp64 copies are large
            full = torch.zeros((blocks(n) * BLOCK, blocks(k) * BLOCK), device=w.device, dtype=torch.float64)
            full[:n, :k] = w
            cells = full.view(blocks(n), BLOCK, blocks(k), BLOCK)
            s = (cells.abs().amax((1, 3)) / TOP).clamp_min(LEAST).float()
            q = cells / s[:, None, :, None].double()
            step = torch.ldexp(torch.ones_like(q), torch.frexp(q).exponent.clamp_min(-5) - 4)     # a conversion would round to fp32 in between
            values[i].copy_((torch.round(q / step) * step).view_as(full)[:n, :k].to(E4M3))
            scales[i] = s
        return cls(values.view(*lead, n, k) if values.is_contiguous() else values.unflatten(0, lead) if lead else values[0], scales.view(*lead, blocks(n), blocks(k)))

    @property
    def shape(self):
        return self.values.shape

    def nbytes(self):
        return self.values.numel() + 4 * self.scales.numel()

    def wide(self):
        """What the weight stands for, in fp32."""
        n, k = self.shape[-2:]
        return self.values.float() * self.scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def empty_rows(rows, width, device):
    """Fp8Rows (rows, width) in new memory, not filled."""
    r = Fp8Rows.__new__(Fp8Rows)
    r.copied = False
    r.row_stride, r.scale_stride = rs, bs = width + -width % 16, rows if rows else 1
    r.values = _new((rows, width), (rs, 1), device=device, dtype=E4M3)
    r.scales = _new((rows, -(-width // BLOCK)), (1, bs), device=device, dtype=torch.float32)
    return r


def quantize_rows(x, out=None):
    """Rows (rows, width) of bfloat16 or float32 in 8 bits.  ``out``: Fp8Rows of that shape, such as some columns of wider ones (from a
    multiple of 128 on)."""
    here = _here(x, None if out is None else out.values)
    if x.ndim != 2 or x.dtype not in _TYPES or x.shape[1] == 0:
        raise ValueError("quantize_rows takes a (rows, width) matrix of bfloat16 or float32")
    if out is not None:
        if out.shape != x.shape:
            raise ValueError(f"out has the shape {tuple(out.shape)}, x {tuple(x.shape)}")
        _own(out)
        _apart(out.values, x), _apart(out.scales, x)
    if x.stride(1) != 1 and x.shape[1] > 1:
        x = x.contiguous()
    n, width = x.shape
    r = empty_rows(n, width, x.device) if out is None else out
    rc = _lib.load_decoder().atma_quantize_rows(x.data_ptr(), x.stride(0), r.values.data_ptr(), r.row_stride, r.scales.data_ptr(), r.scale_stride, n,
                                                width, _lib.DTYPE_CODE[x.dtype], _stream(here))
    if rc:
        _check(rc)
    return r


def residual_norms_fp8(x, y, weights, eps, offset=1.0, out=None, plain=False):
    """``decoder_ops.residual_norms`` with results in 8 bits: x + y (x (rows, width) float32; y in the weights' type, or None) goes to
    ``out`` (None: to x itself); for every weight of ``weights`` (one or two, None = skipped) the normalised row times (offset + weight).
    Returns [(Fp8Rows, None)], and with ``plain`` the last norm in the weights' type beside its rows in 8 bits."""
    first, second = (*weights, None)[:2] if 0 < len(weights) <= 2 else (None, None)
    some = first if first is not None else second
    if some is None:
        raise ValueError("one or two norms")
    here = _here(x, y, out, first, second)
    dtype, shape = some.dtype, x.shape
    if x.dtype is not torch.float32 or len(shape) != 2 or shape[1] == 0 or not x.is_contiguous():
        raise ValueError("x must be a contiguous float32 matrix")
    n, D = shape
    for w in weights:
        if w is not None and (w.dtype is not dtype or w.shape != (D,) or not w.is_contiguous()) or dtype not in _TYPES:
            raise ValueError(f"weights must have {D} values each and one type, bfloat16 or float32")
    if y is not None and (y.shape != shape or y.dtype is not dtype or not y.is_contiguous()):
        raise ValueError("y must be contiguous, of x's shape and of the weights' type")
    if out is not None:
        if out.shape != shape or out.dtype is not torch.float32 or not out.is_contiguous():
            raise ValueError("out must be contiguous, of x's shape and float32")
        at, nbytes = out.data_ptr(), 4 * n * D
        if at != x.data_ptr() and abs(at - x.data_ptr()) < nbytes or y is not None and -n * D * y.element_size() < y.data_ptr() - at < nbytes:
            raise ValueError("out may be x, and must not overlap x or y otherwise")
    dev, last = x.device, len(weights) - 1
    to = x if out is None else out
    h = _new((n, D), (D, 1), device=dev, dtype=dtype) if plain and weights[last] is not None else None
    parts, results = [], []
    for i, w in enumerate(weights):
        if w is None:
            parts += _NO_NORM
            results.append((None, None))
        else:
            r, beside = empty_rows(n, D, dev), h if i == last else None
            parts += (w.data_ptr(), r.values.data_ptr(), r.scales.data_ptr(), None if beside is None else beside.data_ptr())
            results.append((r, beside))
    if last == 0:
        parts += _NO_NORM
    rc = _lib.load_decoder().atma_residual_norms_fp8(x.data_ptr(), None if y is None else y.data_ptr(), None if y is None and out is None else to.data_ptr(),
                                                     *parts, n, D, D + -D % 16, n if n else 1, eps, offset, _lib.DTYPE_CODE[dtype], _stream(here))
    if rc:
        _check(rc)
    return results


_NO_NORM = (None, None, None, None)


def _product(x, w, out, here):
    """x w^T into ``out``: a matrix, or Fp8Rows for the gelu-gated form."""
    (m, n), k, v = out.shape, x.values.shape[1], w.values
    if isinstance(out, Fp8Rows):
        to = (out.values.data_ptr(), out.row_stride, out.scales.data_ptr(), out.scale_stride)
        sizes = (m, 2 * n, k, 1, 1, 0)
    else:
        to = (out.data_ptr(), out.stride(0) if m > 1 else n, None, 0)
        sizes = (m, n, k, 1, 0, _lib.DTYPE_CODE[out.dtype])
    a = _lib.Fp8Args(x.values.data_ptr(), x.row_stride, x.scales.data_ptr(), x.scale_stride, v.data_ptr(), w.row_stride, w.scales.data_ptr(), *to, None, *sizes)
    rc = _lib.load_decoder().atma_linear_fp8(ctypes.byref(a), _stream(here))
    if rc:
        _check(rc)
    return out


def linear_fp8(x, weight, out=None, dtype=torch.bfloat16):
    """x @ weight.T of rows (rows, K) and a weight (N, K) in 8 bits, in ``dtype`` (bfloat16 or float32) or ``out``'s type: sums in fp32,
    rounded once.  ``out``: (rows, N) with contiguous rows, any row stride."""
    if not isinstance(x, Fp8Rows) or not isinstance(weight, Fp8Weight) or weight.values.ndim != 2:
        raise ValueError("linear_fp8 takes Fp8Rows (rows, K) and an Fp8Weight (N, K)")
    (n, K), (N, columns) = x.values.shape, weight.values.shape
    if columns != K or N == 0 or K == 0:
        raise ValueError(f"rows of {K} do not fit a weight ({N}, {columns})")
    here = _here(x.values, weight.values, out)
    if out is None:
        if dtype not in _TYPES:
            raise ValueError(f"unsupported dtype {dtype}; expected float32 or bfloat16")
        out = _new((n, N), (N, 1), device=x.values.device, dtype=dtype)
    else:
        if out.shape != (n, N) or out.dtype not in _TYPES or out.stride(1) != 1 and N > 1 or out.stride(0) < N and n > 1:
            raise ValueError("out must have the result's shape, contiguous rows and type bfloat16 or float32")
        _apart(out, x.values, x.scales, weight.values, weight.scales)
    return _product(x, weight, out, here)


def gelu_gated_linear_fp8(x, weight, out=None):
    """gelu_tanh(x @ weight[0].T) * (x @ weight[1].T) of rows (rows, K) and a weight (2, N, K) in 8 bits, back in 8 bits: Fp8Rows
    (rows, N), ``out`` as for ``quantize_rows``.  Everything between is fp32."""
    if not isinstance(x, Fp8Rows) or not isinstance(weight, Fp8Weight) or weight.values.ndim != 3 or weight.shape[0] != 2 or \
            weight.shape[2] != x.shape[1] or 0 in weight.shape:
        raise ValueError("gelu_gated_linear_fp8 takes Fp8Rows (rows, K) and an Fp8Weight (2, N, K)")
    here = _here(x.values, weight.values, None if out is None else out.values)
    if out is not None:
        if out.shape != (x.shape[0], weight.shape[1]):
            raise ValueError(f"out has the shape {tuple(out.shape)}, the result {(x.shape[0], weight.shape[1])}")
        _own(out)
        for t in (out.values, out.scales):
            _apart(t, x.values, x.scales, weight.values, weight.scales)
    return _product(x, weight, empty_rows(x.shape[0], weight.shape[1], x.values.device) if out is None else out, here)

"""8-bit dense layers for the towers at inference (uniter_model/model/layer.py:53-170 in e4m3 with scales).

A value stands for code * scale; scale = largest magnitude of its block / 448 in fp32.  Activations have one scale for each row and 128
columns, weights one for each block of 128 x 128:

    w8, ws = quantize_weight(weight)                                     # once per model
    x8, xs = quantize_rows(x)
    h = linear(x8, xs, w8, ws, bias, gelu=True)                          # act(x w^T + b)
    y, y8, ys = add_layer_norm(h, residual, ln.weight, ln.bias, ln.eps)  # the next layer's input, in both forms

HIP kernels of csrc/fp8.hip and csrc/fp8_linear.hip; no gradients, no CPU fallback: tensors that need a gradient or
carry a forward-mode tangent, traces and CPU tensors raise."""
from typing import Optional, Tuple

import torch
from torch import Tensor as T

from . import _lib as L

BLOCK = 128
MAX_NORM_WIDTH = 16384
_CODES = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}


def _check(name: str, t: T, what: str, device=None):
    if not isinstance(t, T) or t.dim() != 2:
        raise ValueError(f'{name} is a tensor {what}')
    if not t.is_cuda:
        raise L.LdotError(-2, f'{name}: the 8-bit kernels need CUDA(HIP) tensors: there is no CPU fallback')
    if device is not None and t.device != device:
        raise ValueError(f'{name} is on {t.device}, not on {device}')


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError('the 8-bit layers have no gradients: call them under torch.no_grad()')


def _vector(name: str, t: Optional[T], n: int, device) -> Optional[T]:
    if t is None:
        return None
    if not isinstance(t, T) or t.shape != (n,) or t.device != device or t.dtype not in _CODES:
        raise ValueError(f'{name} is a vector of {n} elements on {device}')
    t = t if t.dtype is torch.float32 and t.is_contiguous() else t.detach().float().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.detach().clone()


def _rows(t: T) -> T:
    """t with rows of consecutive elements; rows of whole groups of 8 begin on 16 bytes (others are read element by element)"""
    row, one = t.stride()
    m, k = t.shape
    if one == 1 and row >= k and (k % 8 or not (t.data_ptr() | (row * t.element_size() if m > 1 else 0)) & 15):
        return t
    t = t.contiguous()
    return t.clone() if k % 8 == 0 and t.data_ptr() & 15 else t


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _quantize(x: T, rows: int) -> Tuple[T, T]:
    L.values_only('quantize_rows' if rows == 1 else 'quantize_weight', x)
    _check('x', x, '[rows, columns]')
    if rows == 1:
        _no_grad(x)
    if x.dtype not in _CODES:
        raise ValueError(f'float32, bfloat16 or float16, not {x.dtype}')
    m, k = x.shape
    if k < 1 or (rows == 1 and k > MAX_NORM_WIDTH):
        raise ValueError(f'rows of {k} elements: 1 to {MAX_NORM_WIDTH} are supported')
    lib = L.load_library()
    x = _rows(x.detach())
    codes = x.new_empty((m, k), dtype=torch.float8_e4m3fn)
    scales = x.new_empty((-(-m // rows), _blocks(k)), dtype=torch.float32)
    if m:
        L.launch(lib.ldot_quantize_e4m3, x.device, x.data_ptr(), _CODES[x.dtype], m, k, max(x.stride(0), k), rows, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def quantize_rows(x: T) -> Tuple[T, T]:
    """x [rows, columns] -> (codes float8_e4m3fn [rows, columns], scales fp32 [rows, ceil(columns / 128)]).  A block of zeros has scale 1;
    a NaN stays a NaN, a block that holds an infinity has an infinite scale."""
    return _quantize(x, 1)


def quantize_weight(w: T) -> Tuple[T, T]:
    """w [out, in] -> (codes float8_e4m3fn [out, in], scales fp32 [ceil(out / 128), ceil(in / 128)])"""
    return _quantize(w, BLOCK)


def linear(x8: T, x_scale: T, w8: T, w_scale: T, bias: Optional[T] = None, gelu: bool = False, out_dtype: torch.dtype = torch.bfloat16) -> T:
    """act(x w^T + bias) -> [rows, out] of ``out_dtype``: x8 [rows, in] and w8 [out, in] codes with their scales (quantize_rows,
    add_layer_norm, quantize_weight); ``gelu``: the towers' erf-GELU.  ``in`` is a multiple of 16.  Products are exact, the
    scales are applied to every block's sum in fp32, the result is rounded once.  For 16-bit results the 8-bit matrix unit adds the
    products; it drops what lies 2^-13 below the largest of 8 neighbouring ones (2.5e-5 of a typical result, 1/60 of the rounding to
    bfloat16); for float32 results all sums are held in fp32, at half the rate."""
    L.values_only('linear', x8, x_scale, w8, w_scale, bias)
    _check('x8', x8, '[rows, in]')
    device = x8.device
    _check('w8', w8, '[out, in]', device)
    if x8.dtype != torch.float8_e4m3fn or w8.dtype != torch.float8_e4m3fn:
        raise ValueError('x8 and w8 hold float8_e4m3fn codes')
    m, k = x8.shape
    n = w8.shape[0]
    if w8.shape[1] != k or k < 16 or k % 16 or n < 1:
        raise ValueError(f'x8 {tuple(x8.shape)} and w8 {tuple(w8.shape)}: rows of the same length, a multiple of 16, are needed')
    if k > 1 << 20 or n > 1 << 24:
        raise ValueError(f'a layer of {n} x {k} is too large')
    if out_dtype not in _CODES:
        raise ValueError(f'float32, bfloat16 or float16, not {out_dtype}')
    for name, s, shape in (('x_scale', x_scale, (m, _blocks(k))), ('w_scale', w_scale, (_blocks(n), _blocks(k)))):
        if not isinstance(s, T) or s.shape != shape or s.dtype != torch.float32 or s.device != device:
            raise ValueError(f'{name} is an fp32 tensor {shape} on {device}')
    _no_grad(x8, w8, x_scale, w_scale, bias)
    bias = _vector('bias', bias, n, device)
    lib = L.load_library()
    row, one = x8.stride()
    if one != 1 or row % 16 or not k <= row <= 1 << 22 or x8.data_ptr() % 16:
        x8 = x8.clone(memory_format=torch.contiguous_format)
    w8 = w8 if w8.is_contiguous() and w8.data_ptr() % 16 == 0 else w8.clone(memory_format=torch.contiguous_format)
    out = x8.new_empty((m, n), dtype=out_dtype)
    if m:
        x_scale, w_scale = x_scale.contiguous(), w_scale.contiguous()
        L.launch(lib.ldot_linear_e4m3, device, x8.data_ptr(), x_scale.data_ptr(), x8.stride(0) if m > 1 else k, w8.data_ptr(), w_scale.data_ptr(),
                 bias.data_ptr() if bias is not None else None, int(bool(gelu)), m, n, k, out.data_ptr(), _CODES[out_dtype])
    return out


def add_layer_norm(x: T, residual: Optional[T], weight: T, bias: T, eps: float = 1e-12) -> Tuple[T, T, T]:
    """y = LayerNorm(x + residual) * weight + bias over rows -> (y in x's type, codes, scales): computed in 64 bits, and each of the three
    rounded from there (a 16-bit y by way of 32 bits; the codes are not made from the rounded y).  Rows of 1 to 16384 elements; ``residual`` (x's shape and type) may be
    None."""
    L.values_only('add_layer_norm', x, residual, weight, bias)
    _check('x', x, '[rows, width]')
    if x.dtype not in _CODES:
        raise ValueError(f'float32, bfloat16 or float16, not {x.dtype}')
    m, k = x.shape
    device = x.device
    if not 1 <= k <= MAX_NORM_WIDTH:
        raise ValueError(f'rows of {k} elements: 1 to {MAX_NORM_WIDTH} are supported')
    if residual is not None and (not isinstance(residual, T) or residual.shape != x.shape or residual.dtype != x.dtype or residual.device != device):
        raise ValueError('residual has the shape, type and device of x')
    eps = float(eps)
    if not eps >= 0:
        raise ValueError('eps has to be >= 0')
    if weight is None or bias is None:
        raise ValueError('weight and bias are vectors of the rows\' width')
    _no_grad(x, residual, weight, bias)
    weight, bias = _vector('weight', weight, k, device), _vector('bias', bias, k, device)
    lib = L.load_library()
    x = _rows(x)
    residual = _rows(residual) if residual is not None else None
    y, codes = x.new_empty((m, k)), x.new_empty((m, k), dtype=torch.float8_e4m3fn)
    scales = x.new_empty((m, _blocks(k)), dtype=torch.float32)
    if m:
        L.launch(lib.ldot_add_layer_norm_e4m3, device, x.data_ptr(), max(x.stride(0), k), residual.data_ptr() if residual is not None else None,
                 max(residual.stride(0), k) if residual is not None else 0, _CODES[x.dtype], m, k, weight.data_ptr(), bias.data_ptr(), eps,
                 y.data_ptr(), codes.data_ptr(), scales.data_ptr())
    return y, codes, scales

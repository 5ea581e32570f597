"""Global gradient norm and clipping — torch.nn.utils.clip_grad_norm_ of train_itm.py:262 on the MI355X (csrc/grad_clip.hip).

    clip_grad_norm_(parameters, max_norm)        in place on the parameters' gradients, as torch's function is called
    clip_gradients(gradients, max_norm, out=...) the same on a list of tensors, in place or into another list
    global_grad_norm(gradients)                  the norm alone

Two passes over the gradients and no host synchronisation (error_if_nonfinite needs one).  The norm is summed in fp64, in an order that the
tensors' sizes and types and where they begin within 16 bytes decide: no atomics, the same list gives the same bits.  No CPU fallback here: train.py keeps torch's own function for parameters on the CPU."""
import ctypes
import math
from array import array
from operator import attrgetter, eq
from typing import Iterable, List, Optional, Sequence, Union

import numpy as np
import torch
from torch import Tensor as T

from . import _lib as L

_CODES = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
_PLAIN = {T, torch.nn.Parameter}


# (hundreds of tensors per call: lists of them are walked by built-in functions, and no list of objects that the garbage collector counts
# is made: a collection of everything costs 35 ms)
_SHAPE = attrgetter('shape')


def _int64(values, n: int):
    return (ctypes.c_int64 * n).from_buffer(array('q', values))


def _run(src: List[T], dst: Optional[List[T]], codes: List[int], max_norm: float, inf: bool, device) -> T:
    lib = L.load_library()
    n = len(src)
    sp = _int64(map(T.data_ptr, src), n)
    dp = None if dst is None else sp if dst is src else _int64(map(T.data_ptr, dst), n)
    sizes, codes = _int64(map(T.numel, src), n), (ctypes.c_int * n).from_buffer(array('i', codes))
    partial = torch.empty(lib.ldot_clip_grad_partials(sizes, n), dtype=torch.float64, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    L.launch(lib.ldot_clip_grad, device, sp, dp, sizes, codes, n, max_norm, int(inf), partial.data_ptr(), norm.data_ptr())
    if dst is not None:
        torch.autograd.graph.increment_version(dst)
    return norm


def _check(tensors: List[T], name: str) -> List[int]:
    """the codes of the tensors' types"""
    if not set(map(type, tensors)) <= _PLAIN and not all(isinstance(t, T) for t in tensors):
        raise ValueError(f'{name} are tensors')
    if len(set(map(T.get_device, tensors))) != 1:
        raise ValueError(f'{name} are on one device')
    L.values_only(name, *tensors)
    if not tensors[0].is_cuda:
        raise L.LdotError(-2, f'{name}: the clipping kernels need CUDA(HIP) tensors: there is no CPU fallback')
    if set(map(attrgetter('layout'), tensors)) != {torch.strided}:
        raise ValueError(f'{name} are dense tensors')
    try:
        return list(map(_CODES.__getitem__, map(attrgetter('dtype'), tensors)))
    except KeyError as e:
        raise ValueError(f'float32, bfloat16 or float16, not {e.args[0]}') from None


def _bytes(t: T) -> int:
    """from the first to the last byte of t"""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else 0


def separate(tensors: Sequence[T]) -> bool:
    """no two of the tensors lie, from their first to their last byte, over each other"""
    tensors = [t for t in tensors if t.numel()]
    n = len(tensors)
    size = np.fromiter(map(T.numel, tensors), np.int64, n) * np.fromiter(map(T.element_size, tensors), np.int64, n) \
        if all(map(T.is_contiguous, tensors)) else np.fromiter(map(_bytes, tensors), np.int64, n)
    first = np.fromiter(map(T.data_ptr, tensors), np.int64, n)
    order = np.argsort(first, kind='stable')
    first, size = first[order], size[order]
    return bool((first[1:] >= (first + size)[:-1]).all())


class _Places:
    """where a tensor's elements lie, for numpy's exact overlap test: no memory is read"""

    def __init__(self, t: T):
        e = t.element_size()
        self.__array_interface__ = dict(data=(t.data_ptr(), False), shape=tuple(t.shape), strides=tuple(s * e for s in t.stride()), typestr=f'|V{e}', version=3)


def _share_memory(a: T, b: T) -> bool:
    try:
        return np.shares_memory(np.asarray(_Places(a)), np.asarray(_Places(b)), max_work=100000)
    except np.exceptions.TooHardError:
        return True


def _check_places(src: List[T], dst: List[T]):
    """for tensors whose elements do not lie one behind the other, before anything is written: a destination overlaps neither itself nor
    anything but its own source (dense ones are checked by the C entry)"""
    for d in dst:
        reach = 0                          # of the dimensions with smaller strides: the next one has to step over it
        for s, n in sorted((s, n) for n, s in zip(d.shape, d.stride()) if n > 1) if d.numel() else ():
            if s <= reach:
                raise L.LdotError(-1, 'a destination has several elements in one place')
            reach += (n - 1) * s
    if separate(dst if dst is src else [*src, *dst]):
        return
    every = [(t.data_ptr(), i, True, t) for i, t in enumerate(dst) if t.numel()]
    if dst is not src:
        every += [(t.data_ptr(), i, False, t) for i, t in enumerate(src) if t.numel()]
    every.sort(key=lambda e: e[:3])
    for at, (a, i, i_written, t) in enumerate(every):
        end = a + _bytes(t)
        for b, j, j_written, other in every[at + 1:]:
            if b >= end:
                break
            own = i == j and a == b and t.stride() == other.stride()
            if (i_written or j_written) and not own and _share_memory(t, other):
                raise L.LdotError(-1, 'a destination overlaps another tensor of the list')


def _norm_type(norm_type) -> bool:
    norm_type = float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f'norm_type {norm_type}: 2 and inf are supported')
    return math.isinf(norm_type)


def clip_gradients(gradients: Sequence[T], max_norm: float, norm_type: float = 2.0, out: Optional[Sequence[T]] = None) -> T:
    """Scales ``gradients`` by min(1, max_norm / (norm + 1e-6)), norm over all of them, in place or into ``out`` (tensors of the same
    shapes and types that overlap nothing else) and returns the norm (fp32, 0-dim, on the GPU; it is not read by the host).  Tensors of
    different sizes and of types float32, bfloat16, float16 may be mixed; a tensor that is in the list twice is refused."""
    gradients = list(gradients)
    inf, max_norm = _norm_type(norm_type), float(max_norm)
    if not max_norm >= 0:
        raise ValueError('max_norm has to be >= 0')
    if not gradients:
        if out:
            raise ValueError('out does not fit the gradients')
        return torch.tensor(0.0)
    codes = _check(gradients, 'gradients')
    device = gradients[0].device
    src = dst = gradients
    if out is not None:
        dst = list(out)
        if len(dst) != len(src):
            raise ValueError('out does not fit the gradients')
        if _check(dst, 'out') != codes or not all(map(eq, map(_SHAPE, src), map(_SHAPE, dst))) or dst[0].device != device:
            raise ValueError('out does not fit the gradients')
    # (a tensor whose elements do not lie one behind the other is worked on in a copy)
    if all(map(T.is_contiguous, src)) and (dst is src or all(map(T.is_contiguous, dst))):
        return _run(src, dst, codes, max_norm, inf, device)
    _check_places(src, dst)
    flat = [t.detach().contiguous() for t in src]
    to = [t if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=device) for t in dst]
    norm = _run(flat, to, codes, max_norm, inf, device)
    for t, d in zip(to, dst):
        if t is not d:
            d.detach().copy_(t)
    return norm


def global_grad_norm(gradients: Sequence[T], norm_type: float = 2.0) -> T:
    """The norm over all gradients (fp32, 0-dim, on the GPU)."""
    gradients = list(gradients)
    inf = _norm_type(norm_type)
    if not gradients:
        return torch.tensor(0.0)
    codes = _check(gradients, 'gradients')
    return _run([t.detach().contiguous() for t in gradients], None, codes, 0.0, inf, gradients[0].device)


def clip_grad_norm_(parameters: Union[T, Iterable[T]], max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> T:
    """torch.nn.utils.clip_grad_norm_ for parameters on the GPU: parameters without a gradient are left out, the norm is returned.  With
    ``error_if_nonfinite`` the norm is read by the host and the gradients stay as they are if it is infinite or NaN."""
    parameters = [parameters] if isinstance(parameters, T) else list(parameters)
    gradients = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and gradients:
        norm = global_grad_norm(gradients, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f'The total norm of order {float(norm_type)} for gradients from `parameters` is non-finite, so it cannot be clipped.')
    return clip_gradients(gradients, max_norm, norm_type)

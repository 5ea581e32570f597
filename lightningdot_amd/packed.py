"""Attention over a packed batch — the towers' self attention (uniter_model/model/layer.py:53-101) without padding.

The tokens of all documents (captions, images' regions) lie one behind the other in one tensor; a token sees the tokens of its own
document, and the documents' lengths are the mask.

    plan = DocumentPlan.from_lengths([12, 31, 7], device='cuda')        # once per batch, for all layers and directions
    out = document_attention(q, k, v, plan)                             # q [tokens, heads, dim], k / v [tokens, kv_heads, dim]

Differentiable in q, k and v (first derivatives in reverse mode; forward-mode tangents raise, and traces of calls without gradients); HIP
kernels of csrc/packed_attention.h, no CPU fallback: CPU tensors raise.  Both directions can be captured into a graph; as with every operator of autograd, capture a backward pass that accumulates into leaves only
while no eager graph of the same leaves is alive (it would wait for their stream)."""
import ctypes
import math
from typing import Optional, Sequence

import torch
from torch import Tensor as T

from . import _lib as L

_CODES = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}


class DocumentPlan:
    """Where the documents of a packed batch lie: document i holds the tokens [offsets[i], offsets[i + 1]).

    ``offsets``: int32 or int64 tensor [documents + 1] on the GPU, not decreasing; ``total``: the rows of the tensors that the plan is
    used with (>= offsets[-1]; rows that no document holds come out as zeros).  The offsets are not read by the host: a plan can be made
    while a graph is captured, and a replay follows the offsets then in the tensor (a plan made before is read by the replays as it is:
    keep it as long as the graph).  Wrong offsets (decreasing, outside [0, total]) are clamped on the device, they never lead outside the
    tensors."""

    def __init__(self, offsets: T, total: int, _lengths: Optional[Sequence[int]] = None):
        if not isinstance(offsets, T) or offsets.dim() != 1 or offsets.numel() < 1 or offsets.dtype not in (torch.int32, torch.int64):
            raise ValueError('offsets is a one-dimensional int32 or int64 tensor with one element more than there are documents')
        self.documents, self.total = offsets.numel() - 1, int(total)
        if self.total < 0 or self.total >= 1 << 31:
            raise ValueError('a packed batch holds 0 to 2^31 - 1 tokens')
        if not offsets.is_cuda:
            raise L.LdotError(-2, 'DocumentPlan needs its offsets on the GPU: there is no CPU fallback')
        lib = L.load_library()
        offsets = offsets.contiguous()
        self.device = offsets.device
        self.stream = L._raw_stream(self.device.index)
        self.data = torch.empty(lib.ldot_packed_plan_ints(self.documents, self.total), dtype=torch.int32, device=self.device)
        L.launch(lib.ldot_packed_plan, self.device, offsets.data_ptr(), int(offsets.dtype == torch.int64), self.documents, self.total,
                 self.data.data_ptr())
        # which kinds of documents there are comes to the host by itself: once it is there (no call waits for it), nothing is launched for
        # the others.  A plan made while a graph is captured follows its offsets on replay and is not read.
        self._absent, self._kinds, self._here = 0, None, None
        if _lengths is not None:
            self._absent = 7 & ~sum({1 if n <= 64 else 2 if n <= 128 else 4 for n in _lengths if n > 0})
        elif self.total > 64 and not torch.cuda.is_current_stream_capturing():
            with torch.cuda.device(self.device):
                self._kinds = torch.empty(3, dtype=torch.int32, pin_memory=True).copy_(self.data[:3], non_blocking=True)
                self._here = torch.cuda.Event()
                self._here.record()

    def absent(self) -> int:
        """bits of the kinds of documents that the batch does not hold (0: not known yet)"""
        here = self._here
        if here is not None and not torch.cuda.is_current_stream_capturing() and here.query():
            self._absent = sum(1 << i for i, n in enumerate(self._kinds.tolist()) if n == 0)
            self._here = None
        return self._absent

    @classmethod
    def from_lengths(cls, lengths: Sequence[int], device, total: Optional[int] = None) -> 'DocumentPlan':
        """The plan of documents of these lengths (host numbers; 0 is an empty document), one behind the other from token 0 on."""
        offsets = [0]
        for n in lengths:
            if int(n) < 0:
                raise ValueError(f'a document of {n} tokens')
            offsets.append(offsets[-1] + int(n))
        total = offsets[-1] if total is None else int(total)
        if total < offsets[-1]:
            raise ValueError(f'the documents hold {offsets[-1]} tokens, the batch {total}')
        if total >= 1 << 31:
            raise ValueError('a packed batch holds 0 to 2^31 - 1 tokens')
        sizes = [b - a for a, b in zip(offsets[:-1], offsets[1:])] + [total - offsets[-1]]
        return cls(torch.tensor(offsets, dtype=torch.int32).to(device), total, _lengths=sizes)


def _operand(t: T) -> T:
    """t with rows of consecutive elements, and an address and strides that are multiples of 16 bytes"""
    st, sh, se = t.stride()
    if se == 1 and not (t.data_ptr() | st * (e := t.element_size()) | sh * e) & 15:
        return t
    return t.clone(memory_format=torch.contiguous_format)      # (contiguous() leaves the strides of dimensions of one element as they are)


def _plan_data(plan) -> int:
    """the plan's address; on another stream than the one it was made on, its memory is kept until that stream is done with it too"""
    if L._raw_stream(plan.device.index) != plan.stream:
        plan.data.record_stream(torch.cuda.current_stream(plan.device))
    return plan.data.data_ptr()


def _args(q, k, v, out, lse, plan, scale, dropout_p, seed):
    tokens, heads, dim = q.shape
    (a, b, _), (c, d, _), (e, f, _) = q.stride(), k.stride(), v.stride()
    return L.PackedAttn(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), None, None, None, None, lse.data_ptr() if lse is not None else None,
                        None, _plan_data(plan), seed.data_ptr() if seed is not None else None, a, b, c, d, e, f, 0, 0, plan.documents, tokens,
                        dropout_p, scale, _CODES[q.dtype], heads, k.shape[1], dim, plan.absent())


def _forward(q, k, v, plan, scale, dropout_p, seed, want_lse):
    out = q.new_empty(q.shape)
    lse = q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32) if want_lse else None
    if q.shape[0]:
        L.launch(L.load_library().ldot_packed_attn_fwd, q.device, ctypes.byref(_args(q, k, v, out, lse, plan, scale, dropout_p, seed)))
    return out, lse


class _DocumentAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan, scale, dropout_p, seed):
        q, k, v = _operand(q), _operand(k), _operand(v)
        out, lse = _forward(q, k, v, plan, scale, dropout_p, seed, True)
        ctx.save_for_backward(q, k, v, out, lse, seed)
        ctx.plan, ctx.scale, ctx.dropout_p = plan, scale, dropout_p
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        q, k, v, out, lse, seed = ctx.saved_tensors
        g = _operand(g if g.dtype == q.dtype else g.to(q.dtype))
        dq, dk, dv = q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(k.shape)
        if q.shape[0]:
            a = _args(q, k, v, out, lse, ctx.plan, ctx.scale, ctx.dropout_p, seed)
            delta = torch.empty_like(lse)
            a.grad, (a.g_st, a.g_sh, _) = g.data_ptr(), g.stride()
            a.dq, a.dk, a.dv, a.delta = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr()
            L.launch(L.load_library().ldot_packed_attn_bwd, q.device, ctypes.byref(a))
        return dq, dk, dv, None, None, None, None


def document_attention(q: T, k: T, v: T, plan: DocumentPlan, scale: Optional[float] = None, dropout_p: float = 0.0,
                       seed: Optional[T] = None) -> T:
    """softmax(scale * q k^T) v within every document -> [tokens, heads, dim].

    q [tokens, heads, dim], k and v [tokens, kv_heads, dim], one of float32, bfloat16, float16 on the plan's GPU; dim a multiple of 8, at
    most 128; kv_heads divides heads (query head h reads key head h // (heads // kv_heads)); views, as of one projection that leaves
    query, key and value side by side, are read where they lie.  ``scale``: 1 / sqrt(dim) unless given, positive.  ``dropout_p``: every
    probability is dropped with this probability (held as 1/65536ths) and the others are divided by 1 - p; ``seed``: int64 tensor of one
    element on the GPU, which with head, token and key decides the bits — the same seed gives the same bits, a training loop hands over
    another one for each layer and step.  Rows that no document holds come out as zeros, in the gradients too."""
    for n, t in (('q', q), ('k', k), ('v', v)):
        if not isinstance(t, T) or t.dim() != 3:
            raise ValueError(f'{n} is a tensor [tokens, heads, dim]')
        if not t.is_cuda:
            raise L.LdotError(-2, 'document_attention needs CUDA(HIP) tensors: there is no CPU fallback')
    dtype, device = q.dtype, q.device
    if k.dtype != dtype or v.dtype != dtype or k.device != device or v.device != device:
        raise ValueError('q, k and v have one type and one device')
    if dtype not in _CODES:
        raise ValueError(f'document_attention takes float32, bfloat16 or float16, not {dtype}')
    if not isinstance(plan, DocumentPlan):
        raise ValueError('plan is a DocumentPlan')
    if plan.device != device:
        raise ValueError(f'the plan is on {plan.device}, the tensors are on {device}')
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    if k.shape != v.shape or tokens != k.shape[0] or dim != k.shape[2]:
        raise ValueError(f'shapes do not fit: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}')
    if tokens != plan.total:
        raise ValueError(f'the plan is for {plan.total} tokens, the tensors hold {tokens}')
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f'{heads} heads are no multiple of {kv_heads} key heads')
    if dim < 8 or dim > 128 or dim % 8:
        raise ValueError(f'head size {dim}: a multiple of 8 up to 128 is needed')
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError('scale has to be positive and finite')
    dropout_p = float(dropout_p)
    if not 0.0 <= dropout_p < 1.0 or int(65536 * dropout_p + 0.5) >= 65536:
        raise ValueError('dropout_p has to be in [0, 1)')
    if dropout_p > 0:
        if not isinstance(seed, T) or seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError('dropout needs a seed: an int64 tensor of one element on the same GPU')
    else:
        seed = None
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _DocumentAttention.apply(q, k, v, plan, scale, dropout_p, seed)
    L.values_only('document_attention', q, k, v)
    return _forward(_operand(q), _operand(k), _operand(v), plan, scale, dropout_p, seed, False)[0]

"""What the packed attention, the 8-bit layers and the gradient clipping refuse: through Python, and at the C entry points (every check
there comes before the first GPU call, so wrong arguments are refused without a GPU too)."""
import ctypes

import pytest
import torch

from lightningdot_amd import LdotError, _lib as L, fp8, grad_clip
from lightningdot_amd.packed import DocumentPlan, document_attention


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64)
    with pytest.raises(LdotError):
        DocumentPlan.from_lengths([4], 'cpu')
    with pytest.raises(LdotError):
        document_attention(x, x, x, None)
    with pytest.raises(LdotError):
        fp8.quantize_rows(torch.zeros(4, 64))
    with pytest.raises(LdotError):
        fp8.add_layer_norm(torch.zeros(4, 64), None, torch.ones(64), torch.zeros(64))
    with pytest.raises(LdotError):
        grad_clip.clip_gradients([torch.zeros(4)], 1.0)


def test_plan_arguments():
    with pytest.raises(ValueError):
        DocumentPlan(torch.zeros(3), 4)
    with pytest.raises(ValueError):
        DocumentPlan(torch.zeros((2, 2), dtype=torch.int32), 4)
    with pytest.raises(ValueError):
        DocumentPlan(torch.zeros(0, dtype=torch.int32), 4)
    with pytest.raises(ValueError):
        DocumentPlan(torch.zeros(2, dtype=torch.int32), 1 << 31)
    with pytest.raises(ValueError):
        DocumentPlan.from_lengths([3, -1], 'cpu')
    with pytest.raises(ValueError):
        DocumentPlan.from_lengths([3, 4], 'cpu', total=6)
    with pytest.raises(ValueError):
        DocumentPlan.from_lengths([1 << 30, 1 << 30], 'cpu')


def test_clip_arguments():
    t = torch.zeros(4)
    for kw in (dict(norm_type=1.0), dict(norm_type=0.0)):
        with pytest.raises(ValueError):
            grad_clip.clip_gradients([t], 1.0, **kw)
    for bad in (-1.0, float('nan')):
        with pytest.raises(ValueError):
            grad_clip.clip_gradients([t], bad)
    with pytest.raises(ValueError):
        grad_clip.clip_gradients([1.0], 1.0)
    assert float(grad_clip.clip_grad_norm_([torch.nn.Parameter(t)], 1.0)) == 0.0          # no gradient at all


def _attn(**kw):
    a = L.PackedAttn()
    base = dict(q=4096, k=4096, v=4096, out=4096, grad=4096, dq=4096, dk=4096, dv=4096, lse=4096, delta=4096, plan=4096, q_st=128, q_sh=64, k_st=128,
                k_sh=64, v_st=128, v_sh=64, g_st=128, g_sh=64, ndocs=1, total=8, dropout=0.0, scale=0.125, dtype=L.BF16, heads=2, kv_heads=2, dim=64)
    for n, v in {**base, **kw}.items():
        setattr(a, n, v)
    return ctypes.byref(a)


@pytest.mark.parametrize('kw', [dict(q=None), dict(q=4098), dict(k_st=4), dict(v_sh=3), dict(out=None), dict(plan=None), dict(dim=0), dict(dim=60),
                                dict(dim=136), dict(heads=3), dict(kv_heads=0), dict(heads=0), dict(dtype=7), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=float('nan')), dict(scale=float('inf')), dict(dropout=-0.1), dict(dropout=1.0), dict(dropout=0.999999),
                                dict(dropout=0.1), dict(total=-1), dict(total=1 << 31), dict(ndocs=-1), dict(ndocs=(1 << 30) - 1, heads=64, kv_heads=64)])
def test_attention_entry_refuses(kw):
    lib = L.load_library()
    assert lib.ldot_packed_attn_fwd(_attn(**kw), None) == -1 and lib.ldot_last_error()
    assert lib.ldot_packed_attn_bwd(_attn(**kw), None) == -1


@pytest.mark.parametrize('kw', [dict(grad=None), dict(grad=4100), dict(lse=None), dict(delta=None), dict(dq=None), dict(dk=4104), dict(dv=None), dict(g_st=2)])
def test_attention_backward_entry_refuses(kw):
    assert L.load_library().ldot_packed_attn_bwd(_attn(**kw), None) == -1


def test_nothing_to_do_needs_no_gpu():
    lib = L.load_library()
    assert lib.ldot_packed_attn_fwd(_attn(total=0), None) == 0
    assert lib.ldot_packed_attn_fwd(None, None) == -1
    assert lib.ldot_linear_e4m3(4096, 4096, 64, 4096, 4096, None, 0, 0, 8, 64, 4096, L.BF16, None) == 0
    assert lib.ldot_quantize_e4m3(4096, L.F32, 0, 64, 64, 1, 4096, 4096, None) == 0


def test_plan_entry_refuses():
    lib = L.load_library()
    assert lib.ldot_packed_plan_ints(3, 100) > 0
    assert lib.ldot_packed_plan_ints(-1, 100) == lib.ldot_packed_plan_ints(1, -1) == lib.ldot_packed_plan_ints(1, 1 << 31) == -1
    assert lib.ldot_packed_plan(None, 0, 1, 8, 4096, None) == -1
    assert lib.ldot_packed_plan(4096, 0, 1, 8, 4100, None) == -1
    assert lib.ldot_packed_plan(4096, 0, 1, 1 << 31, 4096, None) == -1


@pytest.mark.parametrize('change', [dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(out=None), dict(k=24), dict(k=0), dict(ldx=48), dict(ldx=72),
                                    dict(n=0), dict(m=-1), dict(x=4104), dict(w=4104), dict(dtype=9), dict(k=(1 << 20) + 16), dict(n=(1 << 24) + 1)])
def test_linear_entry_refuses(change):
    a = dict(x=4096, xs=4096, ldx=64, w=4096, ws=4096, bias=None, gelu=0, m=4, n=8, k=64, out=4096, dtype=L.BF16)
    a.update(change)
    assert L.load_library().ldot_linear_e4m3(*a.values(), None) == -1


@pytest.mark.parametrize('change', [dict(x=None), dict(codes=None), dict(scales=None), dict(k=0), dict(k=16385), dict(ld=63), dict(rows=2), dict(dtype=5), dict(m=-1)])
def test_quantize_entry_refuses(change):
    a = dict(x=4096, dtype=L.F32, m=4, k=64, ld=64, rows=1, codes=4096, scales=4096)
    a.update(change)
    if 'k' in change:
        a['ld'] = 20000
    assert L.load_library().ldot_quantize_e4m3(*a.values(), None) == -1


@pytest.mark.parametrize('change', [dict(x=None), dict(weight=None), dict(bias=None), dict(codes=None), dict(scales=None), dict(k=0), dict(k=16385), dict(ldx=60),
                                    dict(ldr=60), dict(eps=-1.0), dict(eps=float('nan')), dict(dtype=3), dict(m=-2)])
def test_norm_entry_refuses(change):
    a = dict(x=4096, ldx=20000, residual=4096, ldr=20000, dtype=L.BF16, m=4, k=64, weight=4096, bias=4096, eps=1e-12, y=4096, codes=4096, scales=4096)
    a.update(change)
    assert L.load_library().ldot_add_layer_norm_e4m3(*a.values(), None) == -1


def _clip(src, dst, numel, dtype, max_norm=1.0):
    n = len(src)
    vp, i64, i32 = ctypes.c_void_p * n, ctypes.c_int64 * n, ctypes.c_int * n
    return L.load_library().ldot_clip_grad(vp(*src), vp(*dst) if dst is not None else None, i64(*numel), i32(*dtype), n, max_norm, 0, 4096, 4096, None)


def test_clip_entry_refuses():
    f = L.F32
    assert _clip([4096], [4096], [8], [9]) == -1                                   # type
    assert _clip([4098], [4098], [8], [f]) == -1                                   # alignment
    assert _clip([None], [4096], [8], [f]) == -1
    assert _clip([4096], [None], [8], [f]) == -1
    assert _clip([4096], [4096], [-1], [f]) == -1
    assert _clip([4096], [4096], [8], [f], -1.0) == -1
    assert _clip([4096], [4096], [8], [f], float('nan')) == -1
    assert _clip([4096, 4096], [4096, 4096], [8, 8], [f, f]) == -1                 # the same tensor twice
    assert _clip([4096, 4112], [4096, 4112], [8, 8], [f, f]) == -1                 # overlapping
    assert _clip([4096], [4112], [8], [f]) == -1                                   # out overlaps its source, shifted
    assert _clip([4096, 8192], [8192, 4096], [8, 8], [f, f]) == -1                 # out is another one's source
    assert L.load_library().ldot_clip_grad_partials(None, 3) == -1

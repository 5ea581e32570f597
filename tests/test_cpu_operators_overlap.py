"""What the 8-bit kernels write must not overlap what they read: refused at the C entry points, before the first GPU call."""
import pytest

from lightningdot_amd import _lib as L

MB = 1 << 20


def norm(**kw):
    a = dict(x=MB, ldx=64, residual=2 * MB, ldr=64, dtype=L.BF16, m=4, k=64, weight=3 * MB, bias=4 * MB, eps=1e-12, y=5 * MB, codes=6 * MB, scales=7 * MB)
    a.update(kw)
    lib = L.load_library()
    return lib.ldot_add_layer_norm_e4m3(*a.values(), None), lib.ldot_last_error()


@pytest.mark.parametrize('kw', [dict(y=MB + 128), dict(y=MB - 128), dict(y=MB, ldx=72), dict(y=2 * MB, ldr=72), dict(y=2 * MB + 16), dict(codes=MB), dict(codes=2 * MB + 500),
                                dict(scales=MB), dict(scales=3 * MB + 252), dict(y=4 * MB), dict(codes=5 * MB + 500), dict(scales=6 * MB + 240), dict(y=7 * MB - 500)])
def test_norm(kw):
    code, text = norm(**kw)
    assert code == -1 and b'overlap' in text


@pytest.mark.parametrize('rows,codes,scales', [(1, MB + 1000, 7 * MB), (128, MB, 7 * MB), (1, 6 * MB, MB + 1020), (1, 6 * MB, 6 * MB + 248), (128, 6 * MB, 6 * MB)])
def test_quantize(rows, codes, scales):
    lib = L.load_library()
    assert lib.ldot_quantize_e4m3(MB, L.F32, 4, 64, 64, rows, codes, scales, None) == -1 and b'overlap' in lib.ldot_last_error()


@pytest.mark.parametrize('scale', [3e38, 2.4e38])
def test_attention_scale_that_is_infinite_in_base_2(scale):
    """(kept beside the other refusals: nothing but NaN would come out)"""
    from test_cpu_operators_refuse import _attn
    lib = L.load_library()
    assert lib.ldot_packed_attn_fwd(_attn(scale=scale, total=0), None) == -1 and b'scale' in lib.ldot_last_error()
    assert lib.ldot_packed_attn_fwd(_attn(scale=2e38, total=0), None) == 0

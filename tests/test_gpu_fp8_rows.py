"""Rows of the residual norm in 8 bits (lightningdot_amd.fp8.add_layer_norm): statistics, values, scales and codes come from one set of
64-bit numbers, row by row.  Tolerances: a 64-bit sum of k terms is off by k 2^-53 of its largest term; y, scale and code are each rounded
once from there (y of a 16-bit type by way of 32 bits: 2^-24 more)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
EPS = float(torch.tensor(1e-12))          # (the kernel takes eps in 32 bits)


def code(v):
    """nearest e4m3 value of a 64-bit one, ties to even"""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def definition(x, r, w, b):
    """y, scales, y / scale and how far a 64-bit computation may be off y, all in 64 bits"""
    z = x.double() + (r.double() if r is not None else 0)
    m, k = z.shape
    mean = z.mean(1, keepdim=True)
    dev = z - mean
    sd = (dev.square().mean(1, keepdim=True) + EPS).sqrt()
    y = dev / sd * w.double() + b.double()
    off = 2 * k * 2.0 ** -53 * z.abs().amax(1, keepdim=True) * (1 / sd + dev.abs() / sd ** 2) * w.double().abs() + k * 2.0 ** -53 * (y.abs() + b.double().abs())
    pad = torch.nn.functional.pad(y, (0, -k % 128)).view(m, -1, 128).abs().amax(2)
    scale = torch.where(pad > 0, pad / 448, torch.ones_like(pad))
    return y, scale, y / scale.repeat_interleave(128, 1)[:, :k], off


def check(x, r, w, b, got, sure=slice(None)):
    """every value, scale and code of the rows `sure` against the definition"""
    y, scale, v, off = definition(x, r, w, b)
    u = U[x.dtype] + (0 if x.dtype == torch.float32 else 2.0 ** -24)
    assert ((got[0].double() - y).abs() <= off + u * (y.abs() + off) + TINY[x.dtype]).all()
    k = y.shape[1]
    far = torch.nn.functional.pad(off, (0, -k % 128)).view(len(y), -1, 128).amax(2)
    assert ((got[2].double() - scale).abs() <= (2.0 ** -24 + 2.0 ** -40) * scale + far / 448).all()
    wide = scale.repeat_interleave(128, 1)[:, :k]
    e = (off + far.repeat_interleave(128, 1)[:, :k]) / wide + 448 * 2.0 ** -50
    c = got[1].float().double()
    assert ((c >= code(v - e)) & (c <= code(v + e)))[sure].all()


def rows_of_all_kinds(k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x, r = torch.randn(61, k, generator=g), torch.randn(61, k, generator=g)
    for i, (mean, sd) in enumerate(((1.3, 0.0), (0.1, 0.0), (100.1, 1e-3), (8.0, 1.0), (50.0, 1.0), (3e4, 7.0), (1e-3, 1e-6), (0.7, 1e-5))):
        x[7 * i], r[7 * i] = mean + sd * x[7 * i], 0.0
    return x.to(dtype).cuda(), r.to(dtype).cuda()


WIDTHS = [64, 100, 101, 128, 200, 256, 513, 768, 1000, 1022, 2048, 4096]


@pytest.mark.parametrize('k', WIDTHS)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_a_row_does_not_depend_on_its_neighbours(k, dtype):
    """ordinary rows, constant ones, ones of a large mean and a small spread: the same results alone, in the batch and behind other rows"""
    from lightningdot_amd import fp8
    x, r = rows_of_all_kinds(k, dtype, k)
    w, b = (torch.randn(k, generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2))
    whole = fp8.add_layer_norm(x, r, w, b)
    order = torch.randperm(len(x), generator=torch.Generator().manual_seed(3)).cuda()
    mixed = fp8.add_layer_norm(x[order], r[order], w, b)
    for a, c in zip(whole, mixed):
        assert torch.equal(a[order].view(torch.uint8), c.view(torch.uint8))
    for i in range(len(x)):
        for a, c in zip(whole, fp8.add_layer_norm(x[i:i + 1], r[i:i + 1], w, b)):
            assert torch.equal(a[i:i + 1].view(torch.uint8), c.view(torch.uint8)), i
    check(x, r, w, b, whole)


@pytest.mark.parametrize('k', [64, 100, 768, 1022, 1536])
@pytest.mark.parametrize('value', [1.3, 0.1, 3.0, 1e-3, 12345.678])
def test_constant_rows_are_the_bias(k, value):
    from lightningdot_amd import fp8
    x = torch.full((9, k), value).cuda()
    w, b = (torch.randn(k, generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2))
    y, codes, scale = fp8.add_layer_norm(x, None, w, b)
    want = fp8.quantize_rows(b[None].repeat(9, 1))
    assert torch.equal(y, b[None].expand(9, k)) and torch.equal(scale, want[1])
    y, codes, scale = fp8.add_layer_norm(x, x, w, torch.zeros_like(b))
    assert not y.any() and not codes.float().any() and (scale == 1).all()


@pytest.mark.parametrize('k', [100, 513, 768, 2048])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('mean,bias', [(0.0, 0.0), (0.0, -1.0), (8.0, 0.0), (50.0, 0.3)])
def test_all_codes_are_those_of_the_exact_values(k, dtype, mean, bias):
    """small values, where codes have a fixed step, values that cancel against the mean or the bias: none is left out"""
    from lightningdot_amd import fp8
    m = 3_000_000 // k
    g = torch.Generator(device='cuda').manual_seed(k)
    x, r = (torch.randn(m, k, generator=g, device='cuda') + mean).to(dtype), torch.randn(m, k, generator=g, device='cuda').to(dtype)
    w = 1 + 0.1 * torch.randn(k, generator=g, device='cuda')
    b = bias + 0.1 * torch.randn(k, generator=g, device='cuda')
    check(x, r, w, b, fp8.add_layer_norm(x, r, w, b))


def test_weights_that_are_infinite_or_tiny():
    from lightningdot_amd import fp8
    k = 256
    x = torch.randn(5, k, generator=torch.Generator().manual_seed(0)).cuda()
    w, b = torch.ones(k).cuda(), torch.zeros(k).cuda()
    b[3] = float('inf')                       # an infinite value: an infinite scale, the block's others are 0, as in quantize_rows
    y, codes, scale = fp8.add_layer_norm(x, None, w, b)
    assert torch.isinf(scale[:, 0]).all() and torch.isfinite(scale[:, 1]).all()
    c = codes.float()
    assert torch.isnan(c[:, 3]).all() and not c[:, :3].any() and not c[:, 4:128].any() and c[:, 128:].any(1).all()
    for size in (1e-36, 1e-39, 1e-43):        # scales that are no normal numbers: the codes fit the scale that is stored
        y, codes, scale = fp8.add_layer_norm(x, None, w * size, torch.zeros(k).cuda())
        step = torch.maximum(codes.float().abs(), torch.tensor(2.0 ** -6).cuda()).double() * 2.0 ** -4
        wide = scale.double().repeat_interleave(128, 1)
        top = codes.float().abs() == 448      # (a scale that was rounded down: its largest values are cut off)
        assert (((codes.float().double() * wide - y.double()).abs() <= 1.01 * step * wide + 2.0 ** -149) | top).all() and (codes.float().abs() <= 448).all()


@pytest.mark.parametrize('k', [64, 126, 513, 768, 1000, 4096, 16384])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('where', ['x', 'residual'])
def test_y_in_the_place_of_an_operand(k, dtype, where):
    """the C entry with y = x or y = residual: the results of separate tensors"""
    from lightningdot_amd import _lib as L, fp8
    m, g = 301, torch.Generator().manual_seed(k)
    x, r = (torch.randn(m, k, generator=g).to(dtype).cuda() for _ in range(2))
    w, b = torch.randn(k, generator=g).cuda(), torch.randn(k, generator=g).cuda()
    want = fp8.add_layer_norm(x, r, w, b)
    y = x if where == 'x' else r
    codes, scales = torch.empty_like(want[1]), torch.empty_like(want[2])
    L.launch(L.load_library().ldot_add_layer_norm_e4m3, x.device, x.data_ptr(), k, r.data_ptr(), k, fp8._CODES[dtype], m, k, w.data_ptr(), b.data_ptr(), 1e-12,
             y.data_ptr(), codes.data_ptr(), scales.data_ptr())
    for a, c in zip(want, (y, codes, scales)):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))

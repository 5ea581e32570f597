"""The 8-bit layers (lightningdot_amd.fp8) against their definitions in 64 bits.  Tolerances come from arithmetic: w = 2^-24 for an fp32
operation, u = eps / 2 of the output's type for its one rounding, half a step of e4m3 (2^-4 of the value, 2^-10 below 2^-6) for a code."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
W = 2.0 ** -24


def half_step(v):
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)


def blocks_of(x, rows):
    m, k = x.shape
    pad = torch.zeros(-(-m // rows) * rows, -(-k // 128) * 128, dtype=torch.float64)
    pad[:m, :k] = x
    return pad.view(-(-m // rows), rows, -(-k // 128), 128)


def wide(scale, rows, m, k):
    return scale.cpu().double().repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


@pytest.mark.parametrize('rows', [1, 128])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('m,k', [(1, 1), (3, 127), (130, 128), (5, 129), (257, 768), (64, 2056), (2, 5001), (3, 16384)])
def test_quantize(m, k, dtype, rows):
    from lightningdot_amd import fp8
    g = torch.Generator().manual_seed(m * k)
    x = torch.randn(m, k, generator=g) * torch.exp(3 * torch.randn(m, 1, generator=g))
    x[0, :] = 0
    x = x.to(dtype)
    codes, scale = (fp8.quantize_rows if rows == 1 else fp8.quantize_weight)(x.cuda())
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape
    amax = blocks_of(x.double(), rows).abs().amax(dim=(1, 3))
    want = torch.where(amax > 0, (amax.float() / 448.0), torch.ones(())).float()
    assert torch.equal(scale.cpu(), want)                                   # (the largest magnitude is exact, the division IEEE's)
    v = x.double() / wide(scale, rows, m, k)
    # the value that is rounded is off by two fp32 operations (the scale's reciprocal, the product)
    assert ((codes.cpu().float().double() - v).abs() <= half_step(v) * (1 + 1e-9) + 4 * W * v.abs()).all()


def test_quantize_small_values_infinities_and_nan():
    from lightningdot_amd import fp8
    x = torch.zeros(5, 256)
    x[0, :128] = torch.linspace(-1e-40, 1e-40, 128)          # subnormal: the scale is subnormal too
    x[1, 3] = math.inf
    x[2, 200] = math.nan
    x[2, 201] = 448.0
    x[3, 0] = 3e38
    x[4, 5] = -2.0 ** -126
    codes, scale = fp8.quantize_rows(x.cuda())
    back = codes.float().cpu() * scale.cpu().repeat_interleave(128, 1)
    assert (back[0].double() - x[0].double()).abs().max() <= 1e-40 / 16 + 2.0 ** -149
    assert torch.isinf(scale[1, 0]) and scale[1, 1] == 1 and torch.isnan(back[1, 3])
    assert torch.isnan(codes.float()[2, 200]) and float(codes.float()[2, 201]) == 448.0 and scale[2, 1] == 1
    assert abs(float(back[3, 0]) / 3e38 - 1) < 4 * W
    assert abs(float(back[4, 5]) * 2.0 ** 126 + 1) < 2.0 ** -4


def test_quantize_strided_rows():
    from lightningdot_amd import fp8
    g = torch.Generator().manual_seed(0)
    for x in (torch.randn(40, 400, generator=g).cuda()[:, 8:392], torch.randn(40, 400, generator=g).cuda()[:, 3:300], torch.randn(300, 40, generator=g).cuda().t(),
              torch.randn(1, 300, generator=g).cuda().expand(7, 300)):
        a, b = fp8.quantize_rows(x), fp8.quantize_rows(x.contiguous())
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


LINEAR = [(1, 16, 1), (12, 768, 768), (16, 1040, 130), (17, 128, 64), (33, 400, 77), (64, 2048, 256), (65, 256, 128), (100, 144, 1000), (129, 768, 200),
          (300, 1536, 768), (1000, 16, 33), (2000, 784, 1537), (5000, 768, 2304), (8200, 272, 5001)]


@pytest.mark.parametrize('m,k,n', LINEAR)
@pytest.mark.parametrize('dtype,gelu,with_bias', [(torch.bfloat16, False, True), (torch.float32, True, True), (torch.float16, True, False), (torch.bfloat16, True, True),
                                                  (torch.float32, False, False)])
def test_linear(m, k, n, dtype, gelu, with_bias):
    from lightningdot_amd import fp8
    g = torch.Generator(device='cuda').manual_seed(m + k + n)
    x = torch.randn(m, k, generator=g, device='cuda') * (1 + 20 * (torch.rand(k, generator=g, device='cuda') < 0.02).float())
    x8, xs = fp8.quantize_rows(x)
    w8, ws = fp8.quantize_weight(torch.randn(n, k, generator=g, device='cuda') * 0.03)
    bias = torch.randn(n, generator=g, device='cuda') * 0.2 if with_bias else None
    got = fp8.linear(x8, xs, w8, ws, bias, gelu=gelu, out_dtype=dtype)
    assert got.dtype == dtype and got.shape == (m, n)
    kb = -(-k // 128)
    xd = x8.float().double() * xs.double().repeat_interleave(128, 1)[:, :k]
    wd = w8.float().double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if with_bias:
        y, size = y + bias.double(), size + bias.double().abs()
    # 128 products summed in the matrix unit, the two scales, kb blocks added, the bias
    err = 2 * (128 + kb + 4) * W * size
    if dtype != torch.float32:
        # the 8-bit matrix unit adds 8 neighbouring products in fixed point: next to the largest, which it holds exactly (8 bits), each of
        # the other 7 loses less than 2^-13 of it.  The largest product is at most the largest |x| times the largest |w| of the 8
        top = lambda t: torch.nn.functional.pad(t.abs(), (0, -k % 8)).view(t.shape[0], -1, 8).amax(-1)
        err = err + 7 * 2.0 ** -13 * top(xd) @ top(wd).t()
    if gelu:
        # the activation's slope is at most 1.13; its erf is off by 1.5e-7 for 16-bit results, by 2^-22 for fp32 ones
        err = 1.13 * err + y.abs() * (2.0 ** -22 if dtype == torch.float32 else 1.5e-7 + 2.0 ** -21)
        y = 0.5 * y * torch.erfc(-y * math.sqrt(0.5))
    off = (got.double() - y).abs()
    tol = err + U[dtype] * (y.abs() + err) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert (off <= tol).all(), float((off / tol).max())


def test_linear_strided_and_unaligned_codes():
    from lightningdot_amd import fp8
    g = torch.Generator(device='cuda').manual_seed(3)
    big, _ = fp8.quantize_rows(torch.randn(70, 512, generator=g, device='cuda'))
    w8, ws = fp8.quantize_weight(torch.randn(96, 256, generator=g, device='cuda'))
    xs = torch.rand(70, 2, generator=g, device='cuda')
    for x8 in (big[:, 64:320], big[:, 5:261], big[3:60, :256], big[:1, 16:272]):
        s = xs[:x8.shape[0]]
        a = fp8.linear(x8, s, w8, ws, out_dtype=torch.float32)
        b = fp8.linear(x8.clone(memory_format=torch.contiguous_format), s, w8, ws, out_dtype=torch.float32)
        assert torch.equal(a, b)


def test_linear_nan_stays_in_its_row_and_column():
    from lightningdot_amd import fp8
    for m in (20, 200):
        g = torch.Generator(device='cuda').manual_seed(m)
        x = torch.randn(m, 400, generator=g, device='cuda')
        w = torch.randn(150, 400, generator=g, device='cuda')
        x[7, 399] = math.nan
        w[33, 0] = math.nan
        y = fp8.linear(*fp8.quantize_rows(x), *fp8.quantize_weight(w))
        want = torch.zeros_like(y, dtype=torch.bool)
        want[7], want[:, 33] = True, True
        assert torch.equal(torch.isnan(y), want)


NORM = [(1, 1), (12, 768), (5, 7), (33, 129), (257, 768), (70, 1000), (9, 2048), (300, 4096), (3, 4099), (17, 8192), (2, 16384), (4100, 64)]


@pytest.mark.parametrize('m,k', NORM)
@pytest.mark.parametrize('dtype,with_residual', [(torch.bfloat16, True), (torch.float32, True), (torch.float16, False)])
def test_add_layer_norm(m, k, dtype, with_residual):
    from lightningdot_amd import fp8
    g = torch.Generator().manual_seed(m + k)
    x = torch.randn(m, k, generator=g).to(dtype).cuda()
    r = (torch.randn(m, k, generator=g) + 0.5).to(dtype).cuda() if with_residual else None
    w, b = (1 + 0.1 * torch.randn(k, generator=g)).cuda(), (0.1 * torch.randn(k, generator=g)).cuda()
    y, codes, scale = fp8.add_layer_norm(x, r, w, b, 1e-5)
    assert y.dtype == dtype and codes.shape == y.shape == (m, k) and scale.shape == (m, -(-k // 128))
    z = (x.double() + (r.double() if r is not None else 0)).cpu()
    w, b = w.cpu().double(), b.cpu().double()
    mean = z.mean(1, keepdim=True)
    dev = z - mean
    sd = (dev.square().mean(1, keepdim=True) + 1e-5).sqrt()
    want = dev / sd * w + b
    # a sum of k terms over 64 lanes or more: k / 64 + 12 additions deep
    ls = (k / 64 + 12) * W
    e_dev = ls * z.abs().mean(1, keepdim=True) + 2 * W * z.abs()
    e_sd = (ls + 6 * W) + (e_dev * dev.abs()).mean(1, keepdim=True) / sd ** 2
    tol = w.abs() * (e_dev / sd + (dev / sd).abs() * (e_sd + 4 * W)) + 2 * W * (want.abs() + b.abs())
    assert ((y.cpu().double() - want).abs() <= tol + U[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
    amax = blocks_of(want, 1).abs().amax(dim=(1, 3))
    t = blocks_of(tol, 1).amax(dim=(1, 3))
    assert ((scale.cpu().double() - torch.where(amax > 0, amax / 448, torch.ones(()).double())).abs() <= t / 448 + W * amax / 448)[amax > t].all()
    s = wide(scale, 1, m, k)
    v = codes.float().cpu().double()
    # half a step of the code, of a value that is off by tol
    assert ((v * s - want).abs() <= half_step((want.abs() + tol) / s) * s * (1 + 1e-6) + tol + 4 * W * want.abs()).all()


def test_norm_strided_and_unaligned():
    from lightningdot_amd import fp8
    g = torch.Generator().manual_seed(0)
    big = torch.randn(30, 900, generator=g).to(torch.bfloat16).cuda()
    w, b = torch.randn(769, generator=g).cuda()[1:], torch.randn(768, generator=g).cuda()
    ref = fp8.add_layer_norm(big[:, 8:776].contiguous(), big[:, 16:784].contiguous(), w.clone(), b)
    for x, r in ((big[:, 8:776], big[:, 16:784]), (torch.cat([big[:, :1], big], 1)[:, 9:777], big[:, 16:784])):
        got = fp8.add_layer_norm(x, r, w, b)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1].view(torch.uint8), ref[1].view(torch.uint8)) and torch.equal(got[2], ref[2])


def test_norm_constant_rows_and_nonfinite_rows():
    from lightningdot_amd import fp8
    x = torch.randn(5, 300).cuda()
    x[1], x[2, 7], x[3, 8] = 3.0, math.nan, math.inf
    w, b = torch.ones(300).cuda(), torch.zeros(300).cuda()
    y, codes, scale = fp8.add_layer_norm(x, None, w, b, 1e-12)
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all() and torch.isfinite(y[[0, 1, 4]]).all()
    assert not y[1].any() and not codes[1].float().any() and (scale[1] == 1).all()


def test_layers_in_a_row_captured_and_replayed():
    """norm, product, activation, quantisation, product: a feed-forward block of the towers, eager and in a graph"""
    from lightningdot_amd import fp8
    g = torch.Generator(device='cuda').manual_seed(1)
    h, m = 256, 77
    w1, w2 = (fp8.quantize_weight(torch.randn(a, b, generator=g, device='cuda') * 0.05) for a, b in ((4 * h, h), (h, 4 * h)))
    b1, b2, lw, lb = (torch.randn(n, generator=g, device='cuda') * 0.1 for n in (4 * h, h, h, h))
    x, r = (torch.randn(m, h, generator=g, device='cuda').to(torch.bfloat16) for _ in range(2))

    def block():
        y, y8, ys = fp8.add_layer_norm(x, r, lw, lb)
        mid = fp8.linear(y8, ys, *w1, b1, gelu=True)
        return fp8.add_layer_norm(fp8.linear(*fp8.quantize_rows(mid), *w2, b2), y, lw, lb)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = block()
    for i in range(3):
        x.copy_(torch.randn(m, h, generator=g, device='cuda'))
        graph.replay()
        got = [t.clone() for t in static]
        want = block()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    # close to the layers in 32 bits: three quantisations, each off by 2^-4 of its values, uniformly distributed: 2^-4 / sqrt(3) at most
    z = torch.nn.functional.layer_norm(x.float() + r.float(), (h,), lw, lb, 1e-12)
    deq = lambda w: w[0].float() * w[1].repeat_interleave(128, 0)[:w[0].shape[0]].repeat_interleave(128, 1)[:, :w[0].shape[1]]
    mid = torch.nn.functional.gelu(z @ deq(w1).t() + b1)
    full = torch.nn.functional.layer_norm(mid @ deq(w2).t() + b2 + z, (h,), lw, lb, 1e-12)
    assert float((want[0].float() - full).norm() / full.norm()) < 3 * 2.0 ** -4 / math.sqrt(3)


def test_gradients_and_wrong_arguments_are_refused():
    from lightningdot_amd import fp8
    x = torch.randn(4, 64, device='cuda')
    x8, xs = fp8.quantize_rows(x)
    w8, ws = fp8.quantize_weight(torch.randn(32, 64, device='cuda'))
    with pytest.raises(ValueError):
        fp8.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError):
        fp8.linear(x8, xs, w8, ws, torch.zeros(32, device='cuda', requires_grad=True))
    with torch.no_grad():
        fp8.linear(x8, xs, w8, ws, torch.zeros(32, device='cuda', requires_grad=True))
    for bad in (lambda: fp8.linear(x, xs, w8, ws), lambda: fp8.linear(x8, xs[:2], w8, ws), lambda: fp8.linear(x8, xs, w8[:, :48], ws),
                lambda: fp8.linear(x8[:, :40], xs, w8[:, :40], ws), lambda: fp8.linear(x8, xs, w8, ws, torch.zeros(31, device='cuda')),
                lambda: fp8.linear(x8, xs, w8, ws, out_dtype=torch.float64), lambda: fp8.quantize_rows(torch.zeros(2, 16385, device='cuda')),
                lambda: fp8.quantize_rows(x.double()), lambda: fp8.quantize_rows(torch.zeros(3, device='cuda')),
                lambda: fp8.add_layer_norm(x, x[:2], xs[0], xs[0]), lambda: fp8.add_layer_norm(x, None, torch.ones(63, device='cuda'), torch.ones(64, device='cuda'))):
        with pytest.raises(ValueError):
            bad()
    assert fp8.linear(x8[:0], xs[:0], w8, ws).shape == (0, 32) and fp8.quantize_rows(x[:0])[0].shape == (0, 64)


def test_more_rows_than_one_dimension_of_a_launch_holds():
    from lightningdot_amd import fp8
    m = (1 << 27) + 1003
    x = torch.randn(1000, 8, device='cuda', dtype=torch.float16).repeat(m // 1000 + 1, 1)[:m]
    codes, scales = fp8.quantize_rows(x)
    for a, b in ((0, 1000), ((1 << 27) - 500, (1 << 27) + 500), (m - 1000, m)):
        c, s = fp8.quantize_rows(x[a:b])
        assert torch.equal(codes[a:b].view(torch.uint8), c.view(torch.uint8)) and torch.equal(scales[a:b], s)


# more tiles than workgroups, so that a workgroup takes several: one block of k and less, a tail, more scales than are held at once, ragged
# edges, rows of results that begin anywhere
@pytest.mark.parametrize('m,k,n,dtype,gelu', [(9001, 48, 1301, torch.bfloat16, False), (20000, 112, 2304, torch.float16, False), (20000, 128, 2304, torch.bfloat16, True),
                                              (9001, 128, 1301, torch.float32, True), (17000, 272, 2056, torch.bfloat16, False), (8192, 4240, 4104, torch.bfloat16, False),
                                              (6000, 4352, 2047, torch.float16, True), (6001, 8208, 1544, torch.float32, False)])
def test_linear_takes_one_tile_after_another(m, k, n, dtype, gelu):
    from lightningdot_amd import fp8
    test_linear(m, k, n, dtype, gelu, True)
    # the rows' scales differ from block to block by powers of ten: a scale taken from another block or row shows
    g = torch.Generator(device='cuda').manual_seed(k)
    x8, _ = fp8.quantize_rows(torch.randn(m, k, generator=g, device='cuda'))
    xs = torch.pow(10.0, torch.randint(-3, 2, (m, -(-k // 128)), generator=g, device='cuda').float())
    w8, ws = fp8.quantize_weight(torch.randn(n, k, generator=g, device='cuda'))
    rows = torch.randint(0, m, (50,), generator=g, device='cuda')
    got = fp8.linear(x8, xs, w8, ws, out_dtype=torch.float32)[rows].double()
    xd = x8[rows].float().double() * xs[rows].double().repeat_interleave(128, 1)[:, :k]
    wd = w8.float().double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    assert ((got - xd @ wd.t()).abs() <= (2 * (128 + k / 128 + 4) * W + 2 ** -24) * (xd.abs() @ wd.abs().t())).all()


@pytest.mark.parametrize('k', [2, 6, 126, 262, 1022, 1500, 4094, 10010])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_norm_by_pairs_and_by_elements(k, dtype):
    """rows of an even width that begin on a pair's bytes, and that do not: the same results"""
    from lightningdot_amd import fp8
    g = torch.Generator().manual_seed(k)
    m = 23
    x, r = (torch.randn(m, k, generator=g).to(dtype).cuda() for _ in range(2))
    w, b = torch.randn(k, generator=g).cuda(), torch.randn(k, generator=g).cuda()
    odd = lambda t: torch.nn.functional.pad(t, (1, 2))[:, 1:k + 1]           # (rows of k + 3 elements, from the second one on)
    want = fp8.add_layer_norm(x, r, w, b)
    for got in (fp8.add_layer_norm(odd(x), r, w, b), fp8.add_layer_norm(odd(x), odd(r), w, b), fp8.add_layer_norm(x, odd(r), w, b)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1].view(torch.uint8), want[1].view(torch.uint8)) and torch.equal(got[2], want[2])
    c, s = fp8.quantize_rows(x)
    d, t = fp8.quantize_rows(odd(x))
    assert torch.equal(c.view(torch.uint8), d.view(torch.uint8)) and torch.equal(s, t)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_norm_codes_are_those_of_the_exact_values(dtype):
    """Values of 1/4 and more (smaller ones lose more than 4 of their last bits to the mean) of rows without a bias: the code of the value in
    64 bits, whatever border it lies next to."""
    from lightningdot_amd import fp8
    m, k = 6000, 768
    g = torch.Generator(device='cuda').manual_seed(9)
    x, r = (torch.randn(m, k, generator=g, device='cuda').to(dtype) for _ in range(2))
    codes = fp8.add_layer_norm(x, r, torch.ones(k, device='cuda'), torch.zeros(k, device='cuda'))[1].float().double()
    z = x.double() + r.double()
    dev = z - z.mean(1, keepdim=True)
    y = dev / (dev.square().mean(1, keepdim=True) + 1e-12).sqrt()
    v = y / (y.view(m, -1, 128).abs().amax(2) / 448).repeat_interleave(128, 1)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    want = torch.round(v / step) * step
    assert (codes == want)[y.abs() >= 0.25].all()

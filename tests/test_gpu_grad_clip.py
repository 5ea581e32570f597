"""Global gradient norm and clipping (lightningdot_amd.grad_clip) against the definition in 64 bits.  The norm is summed in 64 bits and
rounded to fp32 (2^-24), a result is off by the coefficient's rounding, the product's and the type's: 2 * 2^-24 + u of its value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def definition(grads, max_norm, inf=False):
    g = [t.detach().double().cpu() for t in grads]
    norm = max([float(t.abs().max()) for t in g if t.numel()] + [0.0]) if inf else math.sqrt(sum(float(t.square().sum()) for t in g))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def check(before, after, norm, max_norm, inf=False):
    want, coef = definition(before, max_norm, inf)
    assert abs(float(norm) - want) <= 2.0 ** -23 * want + 2.0 ** -149
    for a, b in zip(before, after):
        y = a.double() * coef
        tiny = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}[a.dtype]
        assert ((b.double() - y).abs() <= (3 * 2.0 ** -24 + U[a.dtype]) * y.abs() + tiny).all()


def tensors(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(sizes)]


SIZES = [[1], [3, 5, 0, 17], [16384, 16385, 16383], [100003, 7], [(64, 64), (64,), (257, 3), (1, 1)] * 60, [40000000, 1]]


@pytest.mark.parametrize('sizes', SIZES, ids=lambda s: f'{len(s)} tensors, first {s[0]}')
@pytest.mark.parametrize('dtypes', [[F32], [BF16], [F16], [F32, BF16, F16]], ids=str)
@pytest.mark.parametrize('norm_type', [2.0, math.inf])
def test_in_place_and_into_another_list(sizes, dtypes, norm_type):
    from lightningdot_amd.grad_clip import clip_gradients, global_grad_norm
    g = tensors(sizes, dtypes)
    inf = math.isinf(norm_type)
    keep = [t.clone() for t in g]
    out = [torch.full_like(t, 9) for t in g]
    norm = clip_gradients(g, 0.7, norm_type, out=out)
    assert all(torch.equal(a, b) for a, b in zip(g, keep))
    check(keep, out, norm, 0.7, inf)
    assert torch.equal(global_grad_norm(g, norm_type), norm)
    assert torch.equal(clip_gradients(g, 0.7, norm_type), norm)
    assert all(torch.equal(a, b) for a, b in zip(g, out))


def test_nothing_changes_below_the_limit():
    from lightningdot_amd.grad_clip import clip_gradients
    g = tensors([1000, 33], [F32, BF16])
    keep = [t.clone() for t in g]
    out = [torch.empty_like(t) for t in g]
    clip_gradients(g, 1e6, out=out)
    clip_gradients(g, 1e6)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(keep, g, out))
    clip_gradients(g, 0.0)
    assert not any(t.any() for t in g)


def test_places_that_are_not_aligned():
    """slices of one buffer that begin at any element, sources and destinations apart"""
    from lightningdot_amd.grad_clip import clip_gradients
    for dtype in (F32, BF16, F16):
        src, dst = torch.randn(200000).to(dtype).cuda(), torch.zeros(200000, dtype=dtype, device='cuda')
        at = [(1, 5), (9, 17000), (17013, 40001), (60000, 1), (60003, 70000)]
        g, o = [src[a:a + n] for a, n in at], [dst[a + 2 * i:a + 2 * i + n] for i, (a, n) in enumerate(at)]
        norm = clip_gradients(g, 1.0, out=o)
        check(g, o, norm, 1.0)
        touched = torch.zeros(200000, dtype=torch.bool)
        for i, (a, n) in enumerate(at):
            touched[a + 2 * i:a + 2 * i + n] = True
        assert not dst.cpu()[~touched].any()


def test_gradients_that_are_not_contiguous():
    from lightningdot_amd.grad_clip import clip_gradients
    base = torch.randn(50, 60).cuda()
    g = [base[:, 10:30], base.t()[:5, 7:], torch.randn(8, 9).cuda().t()]
    keep = [t.clone() for t in g]
    before = base.clone()
    norm = clip_gradients(g[:1] + g[2:], 0.5)
    check(keep[:1] + keep[2:], g[:1] + g[2:], norm, 0.5)
    assert torch.equal(base[:, :10], before[:, :10]) and torch.equal(base[:, 30:], before[:, 30:])


def test_sizes_that_fp32_sums_lose():
    from lightningdot_amd.grad_clip import clip_gradients
    g = [torch.full((1 << 20,), 1e30, device='cuda'), torch.full((100,), 1e-30, device='cuda')]
    keep = [t.clone() for t in g]
    norm = clip_gradients(g, 1.0)
    check(keep, g, norm, 1.0)
    h = [torch.full((5,), 1e-30, device='cuda')]
    assert abs(float(clip_gradients(h, 1.0)) / (1e-30 * math.sqrt(5)) - 1) < 1e-6


@pytest.mark.parametrize('norm_type', [2.0, math.inf])
def test_nan_and_infinity_as_in_torch(norm_type):
    from lightningdot_amd.grad_clip import clip_grad_norm_
    for bad in (math.nan, math.inf, -math.inf):
        ours = [torch.nn.Parameter(torch.zeros(n, device='cuda')) for n in (5, 40000, 3)]
        theirs = [torch.nn.Parameter(torch.zeros(n, device='cuda')) for n in (5, 40000, 3)]
        for p, q in zip(ours, theirs):
            p.grad = torch.randn(p.shape, device='cuda')
            if p.numel() == 40000:
                p.grad[20001] = bad
            q.grad = p.grad.clone()
        with pytest.raises(RuntimeError):
            clip_grad_norm_(ours, 1.0, norm_type, error_if_nonfinite=True)
        assert all(torch.equal(p.grad.nan_to_num(7), q.grad.nan_to_num(7)) for p, q in zip(ours, theirs))
        a = clip_grad_norm_(ours, 1.0, norm_type)
        b = torch.nn.utils.clip_grad_norm_(theirs, 1.0, norm_type)
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        for p, q in zip(ours, theirs):
            assert torch.equal(torch.isnan(p.grad), torch.isnan(q.grad)) and torch.equal(p.grad.nan_to_num(0), q.grad.nan_to_num(0))


def test_parameters_without_gradients_and_one_tensor():
    from lightningdot_amd.grad_clip import clip_grad_norm_
    p = [torch.nn.Parameter(torch.randn(10, device='cuda')) for _ in range(3)]
    p[0].grad, p[2].grad = torch.ones(10, device='cuda'), torch.ones(10, device='cuda') * 2
    assert abs(float(clip_grad_norm_(iter(p), 1.0)) - math.sqrt(50)) < 1e-5 and p[1].grad is None
    assert abs(float(torch.cat([p[0].grad, p[2].grad]).norm()) - 1) < 1e-5
    assert abs(float(clip_grad_norm_(p[0], 10.0)) - math.sqrt(10 / 50)) < 1e-5


def test_wrong_lists_are_refused():
    from lightningdot_amd import LdotError
    from lightningdot_amd.grad_clip import clip_gradients
    a, b = torch.randn(100, device='cuda'), torch.randn(100, device='cuda')
    for g, out in (([a, a], None), ([a, a[50:]], None), ([a[:50], b], [a[25:75], b]), ([a, b], [b, a])):
        with pytest.raises(LdotError):
            clip_gradients(g, 1.0, out=out)
    for g, out in (([a], [b[:50]]), ([a], []), ([a], [b.double()]), ([a.double()], None), ([a, b.cpu()], None), ([a.to_sparse()], None)):
        with pytest.raises(ValueError):
            clip_gradients(g, 1.0, out=out)


def test_runs_are_equal_and_replays_follow_the_gradients():
    from lightningdot_amd.grad_clip import clip_gradients
    g = tensors([100000, 33, 5000] * 50, [F32, BF16])
    out = [torch.empty_like(t) for t in g]
    a, first = clip_gradients(g, 0.3, out=out), [t.clone() for t in out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = clip_gradients(g, 0.3, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(first, out))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients(g, 0.3, out=out)
    for i in range(3):
        for t in g:
            t.mul_(1.5)
        graph.replay()
        got, n = [t.clone() for t in out], norm.clone()
        want = [torch.empty_like(t) for t in g]
        m = clip_gradients(g, 0.3, out=want)
        torch.cuda.synchronize()
        assert torch.equal(n, m) and all(torch.equal(x, y) for x, y in zip(got, want))


def test_written_tensors_count_as_changed():
    from lightningdot_amd.grad_clip import clip_gradients, global_grad_norm
    a, b = tensors([1000, 70], [F32])
    other = [torch.zeros_like(a), torch.zeros_like(b)]
    empty = [torch.empty(0, device='cuda') for _ in range(2)]
    versions = [t._version for t in (a, b, *other)]
    global_grad_norm([a, b, a])
    clip_gradients([a, b, *empty], 1.0, out=[*other, *empty])
    clip_gradients([a, *empty], 1.0, out=[a, *empty])
    assert [t._version for t in (a, b, *other)] == [versions[0] + 1, versions[1], versions[2] + 1, versions[3] + 1]
    w = torch.ones(5, device='cuda', requires_grad=True)
    saved = torch.full((5,), 3.0, device='cuda')
    z = (w * saved).sum()
    clip_gradients([saved], 1.0)
    with pytest.raises(RuntimeError):                   # (the product's gradient needs what was there before)
        z.backward()

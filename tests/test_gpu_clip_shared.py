"""Gradients that share memory: clip_gradients_ of the training loop leaves them to torch's function, clip_gradients refuses them unchanged."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, device='cuda'))
        p.grad = g
        out.append(p)
    return out


LAYOUTS = {
    'the same tensor': lambda f: [f[:9], f[:9]],
    'one behind the other, overlapping': lambda f: [f[:300], f[200:700], f[700:]],
    'one inside the other': lambda f: [f, f[100:110]],
    'columns that share one': lambda f: [f[:900].view(30, 30)[:, :20], f[:900].view(30, 30)[:, 19:]],
    'a transposed view': lambda f: [f[:900].view(30, 30).t(), f[450:460]],
    'apart': lambda f: [f[:300], f[300:301], f[301:]],
    'columns apart': lambda f: [f[:900].view(30, 30)[:, :20], f[:900].view(30, 30)[:, 20:]],
}


@pytest.mark.parametrize('name', LAYOUTS)
def test_training_loop_takes_them_as_torch_does(name):
    """fp32 norms of 1000 terms: 2^-24 a term over a tree of some ten additions, the coefficient's and the product's rounding.  What two
    gradients share is scaled by torch once or twice, as its two writers happen to meet."""
    from lightningdot_amd.train import clip_gradients_
    before = torch.randn(1000, generator=torch.Generator().manual_seed(0)).cuda()
    f, g, shared = before.clone(), before.clone(), torch.zeros_like(before)
    for v in LAYOUTS[name](shared):
        v.add_(1)
    shared = shared > 1
    a = clip_gradients_(params(LAYOUTS[name](f)), 0.5)
    b = torch.nn.utils.clip_grad_norm_(params(LAYOUTS[name](g)), 0.5)
    coef = min(1.0, 0.5 / (float(b) + 1e-6))
    assert abs(float(a) / float(b) - 1) < 16 * 2.0 ** -24 and shared.any() == ('apart' not in name)
    tol = 20 * 2.0 ** -24 * before.abs()
    assert ((f - g).abs() <= tol)[~shared].all()
    assert (((f - before * coef).abs() <= tol) | ((f - before * coef ** 2).abs() <= tol))[shared].all()


REFUSED = {
    'a view twice': lambda f: ([f[:900].view(30, 30).t()] * 2, None),
    'columns that share one': lambda f: ([f[:900].view(30, 30)[:, :20], f[:900].view(30, 30)[:, 19:]], None),
    'a transposed view over a dense one': lambda f: ([f[:900].view(30, 30).t(), f[450:460]], None),
    'one element in many places': lambda f: ([f[:10], f[20:21].expand(50)], None),
    'windows': lambda f: ([f[:10], f[20:40].unfold(0, 5, 2)], None),
    'out over another source': lambda f: ([f[:900].view(30, 30)[:, ::2], f[900:950]], [f[:900].view(30, 30)[:, 1::2], f[870:920]]),
    'out over its own source, turned': lambda f: ([f[:900].view(30, 30)[:, :29]], [f[1:901].view(30, 30)[:, :29]]),
    'out twice': lambda f: ([f[:900].view(30, 30)[:, 0], f[:900].view(30, 30)[:, 1]], [f[:900].view(30, 30)[:, 2]] * 2),
}


@pytest.mark.parametrize('name', REFUSED)
def test_strided_tensors_that_share_memory_are_refused_unchanged(name):
    from lightningdot_amd import LdotError
    from lightningdot_amd.grad_clip import clip_gradients
    f = torch.randn(1000, generator=torch.Generator().manual_seed(0)).cuda()
    before = f.clone()
    g, out = REFUSED[name](f)
    with pytest.raises(LdotError):
        clip_gradients(g, 0.5, out=out)
    assert torch.equal(f, before)


def test_strided_tensors_that_lie_between_each_other():
    from lightningdot_amd.grad_clip import clip_gradients
    before = torch.randn(1000, generator=torch.Generator().manual_seed(0)).cuda()
    for cut in (lambda f: [f[:900].view(30, 30)[:, :20], f[:900].view(30, 30)[:, 20:], f[900:]], lambda f: [f[::2], f[1::2]],
                lambda f: [f[:990].view(3, 30, 11).permute(2, 0, 1)[::2], f[:990].view(3, 30, 11).permute(2, 0, 1)[1::2], f[990:]]):
        f, g = before.clone(), before.clone()
        a, b = clip_gradients(cut(f), 0.5), clip_gradients([g], 0.5)
        # (the sums of squares in 64 bits, in another order; a result's two roundings)
        assert abs(float(a) / float(b) - 1) <= 2.0 ** -23 and ((f - g).abs() <= 4 * 2.0 ** -24 * g.abs()).all()
        f = before.clone()
        out = [torch.zeros_like(f)]
        clip_gradients(cut(f), 0.5, out=cut(out[0]))
        assert torch.equal(f, before) and ((out[0] - g).abs() <= 4 * 2.0 ** -24 * g.abs()).all()
        c = cut(f)
        clip_gradients(c, 0.5, out=cut(f))             # (other views of the same places: each its own source)
        assert ((f - g).abs() <= 4 * 2.0 ** -24 * g.abs()).all()

"""Layouts of q, k, v and of the output's gradient that the kernels do not take where they lie: one token or one head with strides that mean
nothing, rows that begin anywhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def odd(t, token, head, first):
    """the same values with strides larger by so many elements than a dense tensor's, from element `first` of a buffer on"""
    n, h, d = t.shape
    buf = torch.full((n * (h * (d + head) + token) + 64,), float('nan'), dtype=t.dtype, device=t.device)
    return buf.as_strided((n, h, d), (h * (d + head) + token, d + head, 1), first).copy_(t)


@pytest.mark.parametrize('tokens', [1, 2, 70])
@pytest.mark.parametrize('heads,kv_heads', [(1, 1), (12, 12), (4, 1)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('token,head,first', [(1, 0, 0), (0, 1, 0), (3, 5, 16), (3, 5, 1), (8, 0, 1)])
def test_odd_strides_are_copied(tokens, heads, kv_heads, dtype, token, head, first):
    from lightningdot_amd.packed import DocumentPlan, document_attention, _operand
    dim = 64
    g = torch.Generator().manual_seed(tokens)
    q, k, v, go = (torch.randn(tokens, h, dim, generator=g).to(dtype).cuda() for h in (heads, kv_heads, kv_heads, heads))
    plan = DocumentPlan.from_lengths([tokens], 'cuda')
    for t in (q, k, v, go):
        o = _operand(odd(t, token, head, first))
        assert o.data_ptr() % 16 == 0 and all(s * o.element_size() % 16 == 0 for s in o.stride()[:2]) and o.stride(2) == 1
    res = []
    for f in (lambda t: t, lambda t: odd(t, token, head, first)):
        x = [f(t).requires_grad_() for t in (q, k, v)]
        out = document_attention(*x, plan)
        with torch.no_grad():
            assert torch.equal(document_attention(*x, plan), out)
        res.append((out, *torch.autograd.grad(out, x, f(go))))
    assert all(torch.equal(a, b) for a, b in zip(*res))

"""Forward-mode tangents and traces on the GPU: refused, with and without gradients, and ordinary calls beside them are not."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


def test_attention():
    from lightningdot_amd.packed import DocumentPlan, document_attention
    plan = DocumentPlan.from_lengths([5, 70], 'cuda')
    x = torch.randn(75, 2, 32, device='cuda')
    want = document_attention(x, x, x, plan)
    for i in range(3):
        with fw.dual_level():
            args = [x, x, x]
            args[i] = fw.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError):
                document_attention(*args, plan)
            args[(i + 1) % 3] = x.clone().requires_grad_()
            with pytest.raises(NotImplementedError):
                document_attention(*args, plan)
            assert torch.equal(document_attention(x, x, x, plan), want)
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda t: document_attention(t, x, x, plan), (x,), (x,))
    with pytest.raises(RuntimeError, match='traced'):
        torch.jit.trace(lambda t: document_attention(t, t, t, plan), x)
    assert torch.equal(document_attention(x, x, x, plan), want)


def test_layers_and_clipping():
    from lightningdot_amd import fp8, grad_clip
    x, w, b = torch.randn(9, 64, device='cuda'), torch.randn(64, device='cuda'), torch.zeros(64, device='cuda')
    w8, ws = fp8.quantize_weight(torch.randn(32, 64, device='cuda'))
    x8, xs = fp8.quantize_rows(x)
    with fw.dual_level():
        d, e = fw.make_dual(x, x), fw.make_dual(w, w)
        for call in (lambda: fp8.quantize_rows(d), lambda: fp8.quantize_weight(d), lambda: fp8.add_layer_norm(d, x, w, b), lambda: fp8.add_layer_norm(x, x, e, b),
                     lambda: fp8.linear(x8, fw.make_dual(xs, xs), w8, ws), lambda: grad_clip.clip_gradients([d], 1.0), lambda: grad_clip.clip_gradients([x], 1.0, out=[d]),
                     lambda: grad_clip.global_grad_norm([d])):
            with pytest.raises(NotImplementedError):
                call()
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(fp8.quantize_rows(x), (x8, xs)))
    with pytest.raises(RuntimeError, match='traced'):
        torch.jit.trace(lambda t: fp8.add_layer_norm(t, None, w, b)[0], x)
    p = torch.randn(32, 64, device='cuda', requires_grad=True)
    assert torch.equal(fp8.quantize_weight(p)[1], fp8.quantize_weight(p.detach())[1])      # (weights that train are quantised as they are)

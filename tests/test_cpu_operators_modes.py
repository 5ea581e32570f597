"""Forward-mode tangents and traces: the operators that autograd does not see refuse them instead of dropping them."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from lightningdot_amd import LdotError, fp8, grad_clip

X, V, C = torch.zeros(4, 64), torch.ones(64), torch.zeros(4, 64).to(torch.float8_e4m3fn)
CALLS = {
    'quantize_rows': (lambda t: fp8.quantize_rows(t), X),
    'quantize_weight': (lambda t: fp8.quantize_weight(t), X),
    'linear, a scale': (lambda t: fp8.linear(C, t, C, torch.ones(1, 1)), torch.ones(4, 1)),
    'linear, the bias': (lambda t: fp8.linear(C, torch.ones(4, 1), C, torch.ones(1, 1), t), torch.ones(4)),
    'add_layer_norm': (lambda t: fp8.add_layer_norm(t, None, V, V), X),
    'add_layer_norm, the residual': (lambda t: fp8.add_layer_norm(X, t, V, V), X),
    'add_layer_norm, the weight': (lambda t: fp8.add_layer_norm(X, None, t, V), V),
    'clip_gradients': (lambda t: grad_clip.clip_gradients([X, t], 1.0), X),
    'clip_gradients, out': (lambda t: grad_clip.clip_gradients([X], 1.0, out=[t]), X),
    'global_grad_norm': (lambda t: grad_clip.global_grad_norm([t]), X),
}


@pytest.mark.parametrize('name', CALLS)
def test_tangents(name):
    call, t = CALLS[name]
    if name != 'clip_gradients, out':        # (the first list is looked at first)
        with fw.dual_level(), pytest.raises(NotImplementedError):
            call(fw.make_dual(t, torch.ones_like(t)))
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda x: (call(x), x)[1], (t,), (torch.ones_like(t),))
    with fw.dual_level(), pytest.raises(LdotError):          # (no tangent: CPU tensors are refused as ever)
        call(t)


@pytest.mark.parametrize('name', [n for n in CALLS if n != 'clip_gradients, out'])
def test_traces(name):
    call, t = CALLS[name]
    with pytest.raises(RuntimeError, match='traced'):
        torch.jit.trace(lambda x: (call(x), x)[1], t)

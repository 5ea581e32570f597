"""Training on packed towers: each tensor's gradient against 64 bits, and what a seed decides."""
import pytest
import torch

from test_gpu_packed_towers import _args, _batch, _towers

pytestmark = pytest.mark.gpu


def _gradients(be, batch, move=lambda t: t):
    """of a fixed random combination of all pooled outputs"""
    at = {n: {k: move(v) if isinstance(v, torch.Tensor) else v for k, v in batch[n].items()} for n in ('txts', 'imgs')}
    txt, img, _ = be(dict(batch, **at))
    g = torch.Generator().manual_seed(5)
    total = sum((o * torch.randn(o.shape, generator=g).to(o)).sum() for o in (txt, img))
    total.backward()
    return {n: p.grad.cpu().double() for n, p in be.named_parameters() if p.grad is not None}


@pytest.mark.parametrize('packed', [False, True])
def test_every_gradient_against_64_bits(packed):
    """The towers in 64 bits on the CPU, padded, without dropout.  An element is a sum over at most 24 x 31 tokens of terms that went through two
    layers, some 2^4 operations each over sums of 2^6 terms whose errors add up like a random walk (2^3): 2^-24 * 2^5 * 2^3 = 2^-16 a term, and terms
    of random sign leave a sum of 1 / sqrt(744) > 2^-5 of their size: 2^-11 of the tensor's largest element.  A key's bias moves all scores of a row by
    as much: its gradient is 0, and what rounding leaves is measured against the gradient of the key's weights, whose terms it shares."""
    batch = _batch()
    be = _towers(packed_towers=packed)
    got = _gradients(be, batch)
    want = _gradients(_towers().double().cpu(), batch, lambda t: t.cpu().double() if t.is_floating_point() else t.cpu())
    assert got.keys() == want.keys() and len(got) > 60
    off = {}
    for n, w in want.items():
        size = want[n[:-4] + 'weight'] if n.endswith('self.key.bias') else w
        off[n] = float((got[n] - w).abs().max() / size.abs().max())
    worst = max(off, key=off.get)
    assert off[worst] <= 2.0 ** -11, (worst, off[worst])


def _first_step(seed, autocast):
    from lightningdot_amd.loss import train_step_loss
    be, batch = _towers(dropout=0.1, packed_towers=True).train(), _batch()
    torch.manual_seed(seed)
    with torch.autocast('cuda', dtype=torch.bfloat16, enabled=autocast):
        txt, img, _ = be(batch)
    loss = train_step_loss(_args(), txt, img, None, batch)[0]
    loss.backward()
    return be, loss.detach(), {n: p.grad for n, p in be.named_parameters() if p.grad is not None}


@pytest.mark.parametrize('autocast', [False, True])
def test_a_seed_decides_the_first_step(autocast):
    """the same seed: the same loss to the bit and the same gradients (torch adds up the embeddings' by atomics, in any order: 2^-24 a term of up to
    24 x 31 * 2^1, of the largest); another seed: another loss"""
    _, a, ga = _first_step(7, autocast)
    _, b, gb = _first_step(7, autocast)
    _, c, _ = _first_step(8, autocast)
    assert torch.equal(a, b) and not torch.equal(a, c)
    for n in ga:
        if 'embeddings' in n:
            assert float((ga[n] - gb[n]).abs().max()) <= 2.0 ** -13 * float(ga[n].abs().max()), n
        else:
            assert torch.equal(ga[n], gb[n]), n


def test_gradients_with_dropout_are_those_of_the_loss():
    """Central differences of the loss along its gradient, every forward pass with the same seed and so with the same dropped probabilities: a
    backward pass that drops others gives another slope.  The differences of step h and 2 h differ by three times what the one of h is off (h^2);
    a loss is off by 2^-24 of itself for some 2^8 roundings, over h."""
    from lightningdot_amd.loss import train_step_loss
    be, first, grads = _first_step(7, False)
    batch, names = _batch(), dict(be.named_parameters())
    norm = float(sum(g.double().square().sum() for g in grads.values()).sqrt())

    def loss(step):
        with torch.no_grad():
            for n, g in grads.items():
                names[n].add_(g, alpha=step / norm)
        torch.manual_seed(7)
        txt, img, _ = be(batch)
        out = float(train_step_loss(_args(), txt, img, None, batch)[0].detach())
        with torch.no_grad():
            for n, g in grads.items():
                names[n].sub_(g, alpha=step / norm)
        return out
    h = 0.02 * float(first) / norm                  # (moves the loss by 2 % each way)
    slope, wide = ((loss(s) - loss(-s)) / (2 * s) for s in (h, 2 * h))
    noise = 2.0 ** -16 * float(first) / h
    assert abs(slope - norm) <= abs(wide - slope) + noise, (slope, wide, norm, noise)
    assert abs(wide - slope) + noise < 0.02 * norm

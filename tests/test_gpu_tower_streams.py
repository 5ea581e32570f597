"""Towers in 8 bits on several streams: the kept weights are used by streams that did not make them."""
import pytest
import torch

from test_gpu_packed_towers import _batch, _towers

pytestmark = pytest.mark.gpu


def _tower():
    sb = _batch()['txts']
    tower = _towers(fp8_towers=True).eval().txt_model
    return tower, lambda: tower(sb['input_ids'], sb['attention_mask'], sb['position_ids'])[0]


@torch.no_grad()
def test_weights_made_on_one_stream_are_waited_for_on_another():
    tower, run = _tower()
    want = run()
    tower.use_fp8()                           # (drops them)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(50_000_000)         # tens of milliseconds: what is made behind it is not there yet when b asks
        tower.bert._layers_fp8()
    with torch.cuda.stream(b):
        got = run()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@torch.no_grad()
def test_weights_outlive_their_use_on_another_stream():
    from lightningdot_amd import fp8
    tower, run = _tower()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x8, xs = fp8.quantize_rows(torch.randn(300, 64, device='cuda'))
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        want = [fp8.linear(x8, xs, *layer.dense[0]) for layer in tower.bert._layers_fp8()]
        sizes = [t.numel() for layer in tower.bert._layers_fp8() for d in layer.dense for t in d[:1]]
    torch.cuda.synchronize()
    with torch.cuda.stream(b):
        torch.cuda._sleep(50_000_000)
        layers = tower.bert._layers_fp8()
        got = [fp8.linear(x8, xs, *layer.dense[0]) for layer in layers]
    del layers
    tower.train()                             # drops the weights while b still has to read them
    with torch.cuda.stream(a):                # (takes their memory if nothing keeps it)
        junk = [torch.full((n,), 77, dtype=torch.uint8, device='cuda') for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    del junk


def test_a_tower_made_and_changed_under_inference_mode():
    from lightningdot_amd.towers import TowerConfig, TowerEncoder
    cfg = TowerConfig(vocab_size=50, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, intermediate_size=128, max_position_embeddings=16)
    ids, mask, at = torch.randint(0, 50, (3, 9)).cuda(), torch.ones(3, 9, dtype=torch.long).cuda(), torch.arange(9)[None].cuda()
    with torch.inference_mode():
        tower = TowerEncoder(cfg, with_image=False).cuda().eval().use_fp8()
        a, b = tower(ids, mask, at)[0], tower(ids, mask, at)[0]
        tower.bert.encoder.layer[0].output.dense.weight.mul_(1.5)
        c = tower(ids, mask, at)[0]
        tower.use_fp8()
        d = tower(ids, mask, at)[0]
    assert torch.equal(a, b) and not torch.equal(a, c) and torch.equal(c, d)


def test_use_fp8_and_back(monkeypatch):
    """8-bit towers run packed, in training too; switched off, a tower runs as before, bit for bit"""
    from lightningdot_amd.towers import Backbone
    calls, packed = [], Backbone._forward_packed
    monkeypatch.setattr(Backbone, '_forward_packed', lambda self, *a: calls.append(1) or packed(self, *a))
    sb = _batch()['txts']
    tower = _towers().eval().txt_model
    run = lambda: tower(sb['input_ids'], sb['attention_mask'], sb['position_ids'])[0]
    with torch.no_grad():
        before = run()
        assert not calls
        tower.use_fp8()
        run()
        assert len(calls) == 1
    tower.train()
    run()
    assert len(calls) == 2
    tower.eval().use_fp8(False)
    with torch.no_grad():
        assert torch.equal(run(), before) and len(calls) == 2

"""The towers' kept 8-bit weights: which stream waits for them, how long their memory lives, what copies hold (streams and layers are stand-ins here)."""
import copy
import types

import pytest
import torch

from lightningdot_amd import towers


class Stream:
    def __init__(self, number):
        self.cuda_stream, self.waits = number, []

    def record_event(self):
        return 'made on %d' % self.cuda_stream

    def wait_event(self, event):
        self.waits.append(event)


class Layer:
    made = 0

    def __init__(self, layer):
        Layer.made += 1
        self.streams = []

    def record_stream(self, stream):
        self.streams.append(stream.cuda_stream)


@pytest.fixture
def bert(monkeypatch):
    monkeypatch.setattr(towers, '_LayerFp8', Layer)
    monkeypatch.setattr(Layer, 'made', 0)
    cfg = towers.TowerConfig(vocab_size=50, hidden_size=32, num_hidden_layers=2, num_attention_heads=2, intermediate_size=64, max_position_embeddings=16)
    return towers.TowerEncoder(cfg, with_image=False).eval().use_fp8().bert


def on(monkeypatch, stream):
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: stream)


def test_other_streams_wait_once_and_keep_the_memory(bert, monkeypatch):
    a, b = Stream(1), Stream(2)
    on(monkeypatch, a)
    layers = bert._layers_fp8()
    assert bert._layers_fp8() is layers and Layer.made == 2 and not a.waits
    on(monkeypatch, b)
    assert bert._layers_fp8() is layers and bert._layers_fp8() is layers
    assert b.waits == ['made on 1'] and all(l.streams == [2] for l in layers)
    on(monkeypatch, a)
    assert bert._layers_fp8() is layers and not a.waits
    with torch.no_grad():
        bert.encoder.layer[0].output.dense.weight.mul_(2)
    on(monkeypatch, b)
    assert bert._layers_fp8() is not layers and Layer.made == 4 and len(b.waits) == 1


def test_copies_make_their_own(bert, monkeypatch):
    on(monkeypatch, Stream(1))
    bert._layers_fp8()
    other = copy.deepcopy(bert)
    assert other.fp8 and other._fp8_weights is None and bert._fp8_weights is not None
    other._layers_fp8()
    assert Layer.made == 4


def test_every_kept_tensor_is_recorded():
    seen = []

    class T(torch.Tensor):
        def record_stream(self, stream):
            seen.append(id(self))
    tensors = [torch.zeros(2).as_subclass(T) for _ in range(16)]
    layer = towers._LayerFp8.__new__(towers._LayerFp8)
    layer.dense = [tuple(tensors[3 * i:3 * i + 3]) for i in range(4)]
    layer.norm = [(tensors[12], tensors[13], 1e-12), (tensors[14], tensors[15], 1e-12)]
    layer.record_stream(types.SimpleNamespace())
    assert sorted(seen) == sorted(map(id, tensors))


def test_broadcast_parameters_count_as_changed(bert, monkeypatch):
    """on a rank that receives rank 0's parameters in eval mode, weights made from the old ones are not used again"""
    from lightningdot_amd import train

    class Dist:
        def broadcast(self, flat, src):
            flat.fill_(0.5)
    monkeypatch.setattr(train, '_dist', lambda: Dist())
    on(monkeypatch, Stream(1))
    layers = bert._layers_fp8()
    train.broadcast_parameters(bert)
    assert all((p == 0.5).all() for p in bert.parameters())
    assert bert._layers_fp8() is not layers and Layer.made == 4


def test_parameters_made_under_inference_mode(monkeypatch):
    """torch counts no changes of them: nothing is kept"""
    monkeypatch.setattr(towers, '_LayerFp8', Layer)
    monkeypatch.setattr(Layer, 'made', 0)
    on(monkeypatch, Stream(1))
    cfg = towers.TowerConfig(vocab_size=50, hidden_size=32, num_hidden_layers=2, num_attention_heads=2, intermediate_size=64, max_position_embeddings=16)
    with torch.inference_mode():
        bert = towers.TowerEncoder(cfg, with_image=False).eval().use_fp8().bert
        a, b = bert._layers_fp8(), bert._layers_fp8()
    assert a is not b and Layer.made == 4


def test_use_fp8_leaves_use_packed_as_it_was():
    cfg = towers.TowerConfig(vocab_size=50, hidden_size=32, num_hidden_layers=1, num_attention_heads=2, intermediate_size=64, max_position_embeddings=16)
    tower = towers.TowerEncoder(cfg, with_image=False)
    for packed in (False, True, False):
        tower.use_packed(packed)
        tower.use_fp8()
        assert tower.bert.fp8
        tower.use_fp8(False)
        assert tower.bert.packed is packed and not tower.bert.fp8
    tower.use_fp8().use_packed().use_fp8(False)
    assert tower.bert.packed

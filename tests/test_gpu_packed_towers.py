"""The towers on packed batches, in 8 bits, and a training step with clipping: the operators together, as eval_itm / train_itm run them."""
import json
import math
import os
import types

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _golden(golden_dir):
    from lightningdot_amd.towers import TowerConfig, TowerEncoder
    g = np.load(os.path.join(golden_dir, 'g5_tower_small.npz'))
    cfg = TowerConfig(**{('vocab_size' if k == 'vocab_size_or_config_json_file' else k): v for k, v in json.loads(str(g['cfg'])).items()})
    enc = TowerEncoder(cfg, project_dim=int(g['project_dim']), with_image=True)
    enc.load_state_dict({k[4:]: torch.from_numpy(g[k]) for k in g.files if k.startswith('sd__')}, strict=True)
    return g, enc.cuda().eval()


def test_packed_tower_matches_the_reference_outputs(golden_dir):
    """the bounds that the padded tower is held to on the same golden outputs (fp32 against the reference's fp32)"""
    g, enc = _golden(golden_dir)
    enc.use_packed()
    t = lambda k: torch.from_numpy(g[k]).cuda()
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            seq, pooled, _ = enc(t('img_input_ids'), t('img_attn'), t('img_position_ids'), t('img_feat'), t('img_pos_feat'), None, t('gather_index'))
            tseq, tpooled, _ = enc(t('txt_input_ids'), t('txt_attn'), t('txt_position_ids'))
        for got, want, mask in ((seq, 'img_seq', 'img_attn'), (tseq, 'txt_seq', 'txt_attn')):
            real = g[mask].astype(bool)
            np.testing.assert_allclose(got.detach().cpu().numpy()[real], g[want][real], rtol=1e-4, atol=5e-5)
            assert not got.detach().cpu().numpy()[~real].any()
        np.testing.assert_allclose(pooled.detach().cpu().numpy(), g['img_pooled'], rtol=1e-4, atol=5e-5)
        np.testing.assert_allclose(tpooled.detach().cpu().numpy(), g['txt_pooled'], rtol=1e-4, atol=5e-5)


def _towers(dropout=0.0, **kw):
    from lightningdot_amd.towers import BiEncoder, TowerConfig
    cfg = TowerConfig(vocab_size=30000, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, intermediate_size=128,
                      max_position_embeddings=64, hidden_dropout_prob=dropout, attention_probs_dropout_prob=dropout)
    args = types.SimpleNamespace(img_model_type='uniter-base', txt_model_type='bert-base', **kw)
    torch.manual_seed(0)
    return BiEncoder(args, project_dim=48, txt_config=cfg, img_config=cfg).cuda()


def _batch(seed=4, n=24):
    """items of different lengths: captions of 3 to 20 tokens, images of 2 to 30 regions"""
    g = torch.Generator().manual_seed(seed)
    lt, lb = torch.randint(3, 21, (n,), generator=g), torch.randint(2, 31, (n,), generator=g)
    at = lambda l, m: (torch.arange(m)[None] < l[:, None]).long().cuda()
    txt = dict(input_ids=torch.randint(1000, 20000, (n, 20), generator=g).cuda(), position_ids=torch.arange(20)[None].cuda(), attention_mask=at(lt, 20),
               img_feat=None, img_pos_feat=None, img_masks=None, gather_index=None)
    img = dict(input_ids=torch.full((n, 1), 101).cuda(), position_ids=torch.zeros(1, 1, dtype=torch.long).cuda(), attention_mask=at(lb + 1, 31),
               img_feat=torch.randn(n, 30, 2048, generator=g).cuda(), img_pos_feat=torch.rand(n, 30, 7, generator=g).cuda(), img_masks=None,
               gather_index=torch.arange(31)[None].repeat(n, 1).cuda())
    return dict(txts=txt, imgs=img, caps=dict(input_ids=None), sample_size=n, pos_ctx_indices=list(range(n)), neg_ctx_indices=[],
                txt_index=list(range(n)), img_fname=[f'i{j}' for j in range(n)])


def _args(**kw):
    return types.SimpleNamespace(caption_score_weight=0.0, num_hard_negatives=0, max_grad_norm=0.5, gradient_accumulation_steps=1, **kw)


def test_packed_gradients_match_the_padded_ones():
    """fp32, no dropout: both forms compute the same function; their gradients differ by the order of fp32 sums.  Several gradients cancel to
    nothing by definition (a key's bias moves every score of a row, a vector added to all embeddings moves every score of a query), so what
    rounding leaves is measured against the terms of the sums and not against the sums: the terms of a bias's gradient are the token gradients
    that the weights' gradients are made of, and none exceeds the largest weight gradient.  2^-24 a term, at most 24 x 31 tokens in a
    sum, two layers and two products in each: 2^-24 * 2^10 = 2^-14 of it."""
    from lightningdot_amd.loss import train_step_loss
    batch, grads = _batch(), []
    for packed in (False, True):
        be = _towers(packed_towers=packed)
        assert be.txt_model.bert.packed is packed and be.img_model.bert.packed is packed
        txt, img, _ = be(batch)
        train_step_loss(_args(), txt, img, None, batch)[0].backward()
        grads.append({n: p.grad for n, p in be.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys()
    for tower in ('txt_model', 'img_model'):
        names = [n for n in grads[0] if n.startswith(tower)]
        top = max(float(grads[0][n].abs().max()) for n in names)
        for n in names:
            assert float((grads[0][n] - grads[1][n]).abs().max()) <= 2.0 ** -14 * top, n


def test_training_steps_packed_with_dropout_and_clipping():
    """runs, and every parameter that has a gradient in the padded form has a finite one; same seeds give the same step"""
    from lightningdot_amd.train import get_optimizer, train_step
    batch, states = _batch(), []
    for _ in range(2):
        be = _towers(dropout=0.1, packed_towers=True)
        opt = get_optimizer(be, learning_rate=1e-3)
        torch.manual_seed(7)
        losses = [train_step(be, batch, _args(), opt, autocast_bf16=True)[0] for _ in range(3)]
        assert np.isfinite(losses).all()
        states.append([p.detach().clone() for p in be.parameters()])
    assert all(torch.isfinite(a).all() and (a - b).abs().max() <= 1e-2 for a, b in zip(*states))


def test_clipping_of_a_step_is_torchs():
    """one backward pass, clipped by both: coefficients equal to the rounding of an fp32 norm (torch sums squares in fp32: 2^-24 a term over
    trees of some twenty additions) and of one product"""
    from lightningdot_amd.loss import train_step_loss
    from lightningdot_amd.train import clip_gradients_
    be, batch = _towers(packed_towers=True), _batch()
    txt, img, _ = be(batch)
    (train_step_loss(_args(), txt, img, None, batch)[0] * 100).backward()
    with_grad = [p for p in be.parameters() if p.grad is not None]
    keep = [p.grad.clone() for p in with_grad]
    ours = clip_gradients_(be.parameters(), 0.5)
    mine = [p.grad for p in with_grad]
    for p, g in zip(with_grad, keep):
        p.grad = g
    theirs = torch.nn.utils.clip_grad_norm_(with_grad, 0.5)
    assert float(theirs) > 0.5 and abs(float(ours) / float(theirs) - 1) < 32 * 2.0 ** -24
    for a, p in zip(mine, with_grad):
        assert float((a - p.grad).abs().max()) <= 40 * 2.0 ** -24 * float(p.grad.abs().max())


def test_clipping_keeps_torchs_function_for_other_gradients():
    from lightningdot_amd.train import clip_gradients_
    for dev, dtype in (('cpu', torch.float32), ('cuda', torch.float64)):
        p = torch.nn.Parameter(torch.zeros(10, dtype=dtype, device=dev))
        p.grad = torch.ones_like(p)
        assert abs(float(clip_gradients_([p], 1.0)) - math.sqrt(10)) < 1e-6 and abs(float(p.grad.norm()) - 1) < 1e-5


def test_fp8_towers_encode_close_to_the_padded_ones():
    """A layer rounds to 8 bits at eight places (four inputs, four weights), each off by 2^-4 of a value at most and by 2^-4 / sqrt(3) as a
    root mean square of a uniform error; independent errors of two layers and the 16-bit roundings between them add up to less than twice
    sqrt(16) of that, the norms keep the scale."""
    batch, be = _batch(n=60), _towers(fp8_towers=True).eval()
    with torch.no_grad():
        for tower, sb in ((be.txt_model, batch['txts']), (be.img_model, batch['imgs'])):
            run = lambda: tower(sb['input_ids'], sb['attention_mask'], sb['position_ids'], sb['img_feat'], sb['img_pos_feat'], None, sb['gather_index'])
            seq, pooled, _ = run()
            again = run()
            assert torch.equal(seq, again[0]) and torch.equal(pooled, again[1])
            tower.use_fp8(False)
            tower.use_packed(False)
            full, fpooled, _ = run()
            real = sb['attention_mask'].bool()
            off = float((seq[real] - full[real]).norm() / full[real].norm())
            assert 0 < off < 2 * math.sqrt(16) * 2.0 ** -4 / math.sqrt(3), off
            assert seq.dtype == full.dtype and pooled.shape == fpooled.shape and not seq[~real].any()


def test_fp8_weights_follow_the_parameters():
    be, batch = _towers(fp8_towers=True).eval(), _batch()
    sb = batch['txts']
    run = lambda: be.txt_model(sb['input_ids'], sb['attention_mask'], sb['position_ids'])[0]
    with torch.no_grad():
        a = run()
        be.txt_model.bert.encoder.layer[0].output.dense.weight.mul_(1.5)
        b = run()
        assert not torch.equal(a, b)
        state = {k: v.clone() for k, v in be.state_dict().items()}
        be.load_state_dict(state)
        assert torch.equal(run(), b)
    be.train()
    assert be(batch)[0].requires_grad           # (training runs unquantised)
    be.eval()
    assert be(batch)[0].requires_grad


def test_widths_that_the_operators_do_not_take_are_refused():
    from lightningdot_amd.towers import TowerConfig, TowerEncoder
    small = dict(vocab_size=50, num_hidden_layers=1, max_position_embeddings=16)
    with pytest.raises(ValueError):
        TowerEncoder(TowerConfig(hidden_size=36, num_attention_heads=3, intermediate_size=64, **small), with_image=False).use_packed()
    with pytest.raises(ValueError):
        TowerEncoder(TowerConfig(hidden_size=64, num_attention_heads=4, intermediate_size=72, **small), with_image=False).use_fp8()
    TowerEncoder(TowerConfig(hidden_size=64, num_attention_heads=4, intermediate_size=64, **small), with_image=False).use_fp8()


@pytest.mark.parametrize('extra', [{'packed_towers': True}, {'fp8_towers': True}])
def test_evaluation_entry_point_with_the_operators(tmp_path, extra):
    """eval_itm's EVAL_MODEL on synthetic batches, the option in the JSON config as a user sets it"""
    from lightningdot_amd.eval_itm import EVAL_MODEL
    small = dict(vocab_size=28996, hidden_size=64, num_hidden_layers=2, num_attention_heads=4, intermediate_size=128, max_position_embeddings=128,
                 type_vocab_size=2, hidden_dropout_prob=0.1, attention_probs_dropout_prob=0.1, initializer_range=0.02, hidden_act='gelu')
    (tmp_path / 'small.json').write_text(json.dumps(small))
    cfg = dict(txt_model_config=str(tmp_path / 'small.json'), img_model_config=str(tmp_path / 'small.json'), itm_global_file=None, seed=1, output_dir=str(tmp_path),
               max_txt_len=20, conf_th=0.2, max_bb=20, min_bb=5, num_bb=12, project_dim=32, val_txt_db='synthetic', val_img_db='synthetic', test_txt_db=None,
               test_img_db=None, project_name='t', n_workers=0, fp16=True, **extra)
    path = tmp_path / 'cfg.json'
    path.write_text(json.dumps(cfg))
    res = EVAL_MODEL(str(path), '', synthetic_images=40)
    assert res and all(np.isfinite(r['loss']) for r in res.values())


def test_fp8_weights_are_made_anew():
    """after training, after to(), after use_fp8(): each time the weights have been written where no version counts it"""
    be, batch = _towers(fp8_towers=True).eval(), _batch()
    sb, tower = batch['txts'], be.txt_model
    def run():
        with torch.no_grad():
            return tower(sb['input_ids'], sb['attention_mask'], sb['position_ids'])[0]
    outs = [run()]
    for again in (lambda: be.train().eval(), lambda: be.to(torch.float32), lambda: tower.use_fp8()):
        tower.bert.encoder.layer[0].output.dense.weight.data.mul_(1.5)
        again()
        outs.append(run())
        assert not torch.equal(outs[-1], outs[-2]) and torch.equal(run(), outs[-1])


def test_clipping_of_a_gradient_that_two_parameters_share():
    """torch's own function takes it, as before"""
    from lightningdot_amd.train import clip_gradients_
    def params():
        p = [torch.nn.Parameter(torch.ones(9, device='cuda')) for _ in range(2)]
        p[0].grad = p[1].grad = torch.full((9,), 2.0, device='cuda')
        return p
    a, b = params(), params()
    assert torch.equal(clip_gradients_(a, 0.5), torch.nn.utils.clip_grad_norm_(b, 0.5)) and torch.equal(a[0].grad, b[0].grad)

"""Attention masks that the packed towers meet: one for all items, holes, items without any token, shapes that do not fit."""
import pytest
import torch

from test_gpu_packed_towers import _batch, _towers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def towers():
    return _towers().eval().txt_model, _towers(packed_towers=True).eval().txt_model


def run(tower, mask):
    sb = _batch()['txts']
    with torch.no_grad():
        return tower(sb['input_ids'], mask, sb['position_ids'])


@pytest.mark.parametrize('name,mask', [('one row', torch.arange(20)[None] < 13), ('one row of ones', torch.ones(1, 20)),
                                       ('holes', torch.rand(24, 20, generator=torch.Generator().manual_seed(0)) < 0.6), ('ones', torch.ones(24, 20, dtype=torch.int32))])
def test_real_tokens_come_out_as_in_the_padded_form(towers, name, mask):
    """fp32: the bounds that the towers are held to on the reference's outputs"""
    mask = mask.cuda()
    if len(mask) > 1:
        mask[:, 0] = 1
    a, b = run(towers[0], mask), run(towers[1], mask)
    real = (mask != 0).expand(24, 20)
    torch.testing.assert_close(b[0][real], a[0][real], rtol=1e-4, atol=5e-5)
    torch.testing.assert_close(b[1], a[1], rtol=1e-4, atol=5e-5)
    assert not b[0][~real].any()


def test_items_without_tokens_are_zeros_and_change_no_other(towers):
    mask = _batch()['txts']['attention_mask'].clone()
    want = run(towers[1], mask)[0]
    empty = torch.zeros(24, dtype=torch.bool, device='cuda')
    empty[[0, 5, 6, 23]] = True
    mask[empty] = 0
    got = run(towers[1], mask)[0]
    assert not got[empty].any()
    # (not bit for bit: the library's products of fewer rows may take another kernel, which adds the same terms in another order)
    torch.testing.assert_close(got[~empty], want[~empty], rtol=1e-4, atol=5e-5)
    assert not run(towers[1], torch.zeros_like(mask))[0].any()


@pytest.mark.parametrize('shape', [(24, 19), (24, 21), (23, 20), (2, 20)])
def test_shapes_that_do_not_fit_are_refused_by_both(towers, shape):
    for tower in towers:
        with pytest.raises(RuntimeError):
            run(tower, torch.ones(shape, dtype=torch.long).cuda())

"""Packed attention at the largest batch that is taken: 2^31 - 1 tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('total', [2 ** 31 - 1, 2 ** 31 - 130])
def test_rows_behind_the_last_document_of_the_largest_batch(total):
    """one document of 70 tokens and two billion rows that no document holds: zeros, whatever their memory held before"""
    from lightningdot_amd.packed import DocumentPlan, document_attention
    g = torch.Generator().manual_seed(0)
    n, dim = 70, 8
    plan = DocumentPlan(torch.tensor([0, n], dtype=torch.int64, device='cuda'), total)
    rows = total - n
    torch.cuda.synchronize()
    count = plan.data[-6 * (1 + 3) - 8:-6 * (1 + 3)].tolist()         # how many entries each list holds
    assert count[:5] == [-(-rows // 64), -(-rows // 128), -(-rows // 64) + 2, -(-rows // 128) + 1, 1]
    q = torch.randn(1, 1, dim, generator=g).to(torch.bfloat16).cuda().expand(total, 1, dim)           # (every token the same: no memory)
    junk = torch.ones(total, 1, dim, dtype=torch.bfloat16, device='cuda')
    del junk                                                                                          # (the result takes its place)
    out = document_attention(q, q, q, plan)
    # equal keys: a row's result is the value itself, its probabilities' sum and one rounding apart
    assert ((out[:n].float() - q[:n].float()).abs() <= 2.0 ** -7 * q[:n].float().abs()).all()
    assert not any(bool(part.any()) for part in out[n:].view(-1).split(1 << 30))

"""Rows of the table without a token, in every form of the gradient."""
import pytest
import torch

from tests.test_embed_gpu import DEV, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.5, -0.5])
@pytest.mark.parametrize("N,V,D", [(100, 6, 33), (600, 6, 70), (600, 3, 7), (4000, 8, 300), (900, 60, 5), (6000, 700, 24)])
def test_added_to_rows_without_a_token_keep_their_bits(N, V, D, scale):
    """accumulate leaves a row that no token reads as it is: negative zeros, infinities and NaN payloads too."""
    ops = _ops()
    ids = torch.randint(0, V - 1, (N,), generator=torch.Generator().manual_seed(1), dtype=torch.int64)
    ids[ids == V // 2] = -1   # rows V // 2 and V - 1: none
    x = torch.randn(N, D, generator=torch.Generator().manual_seed(2)).to(DEV)
    table = torch.full((V, D), -0.0)
    table[:, 1::3] = float("inf")
    bits = table.view(torch.int32)
    bits[:, 2::3] = 0x7fc01234
    got = table.to(DEV)
    ops.embed_grad(x, ids.to(DEV), V, scale=scale, dtable=got, accumulate=True)
    none = torch.bincount(ids[ids >= 0], minlength=V) == 0
    assert none[V // 2] and none[V - 1]
    assert torch.equal(got.cpu().view(torch.int32)[none], bits[none])
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids[ids >= 0], x.cpu().double()[ids >= 0])[~none] * scale
    fresh = ops.embed_grad(x, ids.to(DEV), V, scale=scale)
    assert torch.equal(got[~none.to(DEV)][:, 0::3], fresh[~none.to(DEV)][:, 0::3])
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids[ids >= 0], x.cpu().double().abs()[ids >= 0])[~none] * 0.5
    assert ((fresh.cpu().double()[~none] - want).abs() <= mag * (N + 2) * 2.0 ** -24).all() and (fresh[none.to(DEV)] == 0).all()

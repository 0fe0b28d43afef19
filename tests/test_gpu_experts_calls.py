"""GPU: calls of blocks.Router, Fp4Matmul and ExpertsFfn at the borders of what they take, against oracle/experts.py."""
import pytest
import torch

from cache_util import assert_within
from oracle import experts as oe
from trinity_amd import blocks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (1, 1, 1), (70, 16, 4), (33, 128, 8), (40, 256, 8)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_what_a_group_counts_means_nothing_where_there_is_one(dev, T, E, k, scores):
    g = torch.Generator().manual_seed(T + E)
    z, b = 1.5 * torch.randn(T, E, generator=g), 0.3 * torch.randn(E, generator=g)
    ids, weights = blocks.Router(k, scores=scores, group_top=2, scale=2.5).route(z.to(dev), b.to(dev))
    want, w = oe.route(z, b, top_k=k, sigmoid=scores == "sigmoid", scale=2.5)
    assert torch.equal(ids.cpu().long(), want)
    assert_within(weights, w, 2.0 ** -24 * w.abs() * 1.01, "weights")

"""A document's result and the accuracy of its gradient do not depend on what else the batch holds."""
import pytest
import torch

from chronicals_b200.ops import _ext
from test_attention_window_gpu import _inputs, _run, _truth

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _roundings(g, g64):
    return ((g.double() - g64).norm() / (g64.to(BF).double() - g64).norm()).item()


@pytest.mark.parametrize("hq,hk,d", [(2, 1, 64), (2, 1, 128)])
@pytest.mark.parametrize("lens", [[4] * 30 + [5000], [3000] + [7] * 20 + [1500]])
def test_short_documents_beside_a_long_one(hq, hk, d, lens):
    """The limit is that of batches of short documents alone: the gradient's own rounding, and that of P or dS before the products, as
    large and independent of it, are the square root of two roundings together."""
    window, sinks = 2000, 1
    qkv, do, cu = _inputs(hq, hk, d, lens, 0)
    g64 = _truth(qkv, do, hq, hk, d, lens, window, sinks)[1]
    g = _run(qkv, do, cu, hq, hk, d, window, sinks)[1]
    bounds = cu.tolist()
    rows = torch.cat([torch.arange(a, b, device=DEV) for a, b in zip(bounds, bounds[1:]) if b - a < 100])
    assert _roundings(g[rows], g64[rows]) <= 1.5


@pytest.mark.parametrize("hq,hk,d", [(2, 1, 64), (16, 4, 64), (2, 1, 128)])
@pytest.mark.parametrize("lens", [[2500], [5, 1300, 40, 700], [9] * 40])
@pytest.mark.parametrize("window,sinks", [(1100, 3), (20, 0)])
def test_empty_documents_behind_the_last_one(hq, hk, d, lens, window, sinks):
    """Lists of boundaries that are filled up to a fixed length."""
    qkv, do, cu = _inputs(hq, hk, d, lens, 11)
    o, g = _run(qkv, do, cu, hq, hk, d, window, sinks)
    more = torch.cat((cu, cu[-1:].expand(64)))
    p, h = _run(qkv, do, more, hq, hk, d, window, sinks)
    _ext.check_status()
    assert torch.equal(o, p)
    # additions into dQ, dK and dV in any order: last bits of 32, then a rounding that may fall the other way
    assert (h.double() - g.double()).norm() <= 2.0 ** -8 * g.double().norm()

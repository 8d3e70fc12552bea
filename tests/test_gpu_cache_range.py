"""GPU: the paged K/V cache where values and numbers are far from ordinary ones: rows of very different sizes, zeros, NaN
alone in a tile, large values of V, batches whose numbers contradict each other.  The tolerances of test_gpu_cache.py hold
unless a test says otherwise."""
import math

import pytest
import torch

from test_gpu_cache import D, U, Case, h  # noqa: F401  (h: the package's fixture)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- factors of a tile
@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length", [(2, 20), (16, 40), (100, 100), (100, 129), (300, 1000)])
def test_zero_queries_and_keys(h, n, length, quantised):
    """All logits are 0: every row is the mean of the values that it sees, however small the powers of two in front of them."""
    c = Case(h, [n], [length], 2, 2, 16, quantised, seed=n)
    c.q = torch.zeros_like(c.q)
    c.k[0] = torch.zeros_like(c.k[0])
    c.fill()
    for causal in (True, False):
        out, lse = c.check(causal)
        assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n", [2, 100])
@pytest.mark.parametrize("scale", [1e-12, 1e-30, 1e-38])
def test_scales_next_to_nothing(h, n, scale, quantised):
    c = Case(h, [n], [n + 37], 2, 2, 16, quantised, seed=n)
    c.q[0] = 0
    c.fill().check(True, softmax_scale=scale)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("n,length,heads", [(10, 129, 4), (100, 129, 2), (130, 257, 2), (40, 130, 2), (300, 385, 4)])
def test_hidden_nan_keys_alone_in_a_tile(h, n, length, heads, quantised):
    """The keys of the last tile are NaN and only the last tokens may see them."""
    c = Case(h, [n], [length], heads, 2, 16, quantised, seed=n)
    first = (length - 1) // 128 * 128
    c.k[0][first:, :, 0] = math.nan
    c.fill()
    out, lse = h.cache_attn(c.q.cuda(), c.cache, c.batch, return_lse=True)
    sees = torch.arange(length - n, length, device="cuda") >= first  # rows for which everything is NaN
    assert torch.isnan(out[sees].float()).all() and torch.isnan(lse[:, sees]).all()
    c.k[0][first:, :, 0] = 0  # hidden from the others: any number will do
    ro, rl, tol, ltol = c.reference(True)
    c.compare(out[~sees], lse[:, ~sees], ro[~sees], rl[:, ~sees], tol[~sees], ltol[:, ~sees])

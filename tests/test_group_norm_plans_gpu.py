"""Group norm where its plans (a warp, a block, a cluster an image, passes over
global memory) have to agree."""

import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu

#: images, spatial, channels, groups: a warp, a block, a cluster that stages
#: its rows, one that reads them again, passes over global memory
PLANS = [(9, 16, 32, 4), (9, 80, 32, 4), (160, 400, 90, 6), (40, 7056, 128, 4), (3, 5879, 64, 2)]


def _context():
    from ttrl_b200.device import context
    return context("cuda:0")


@gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("n,s,c,g", PLANS)
def test_a_bad_value_in_any_row_makes_its_group_nan(n, s, c, g, bad):
    """As the definition gives it: the variance of values among which one is
    infinite is NaN, and so is what it scales; no other group sees it."""
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(n * s, c, device="cuda", generator=gen)
    y, clean = torch.empty_like(x), torch.empty_like(x)
    stats, ref = (torch.empty(n, g, 2, device="cuda") for _ in range(2))
    shape = dict(groups=g, spatial=s, act="none")
    _context().group_norm_fwd(x, None, None, clean, ref, **shape)
    hurt = torch.zeros(n, g, dtype=torch.bool, device="cuda")
    for image, row, col in ((0, 0, 1), (1, s // 2 + 1, c - 1), (n - 1, s - 1, c // 2)):
        x[image * s + row, col] = bad
        hurt[image, col // (c // g)] = True
    _context().group_norm_fwd(x, None, None, y, stats, **shape)
    assert bool(torch.isnan(stats[hurt][:, 1]).all())
    assert torch.equal(stats[~hurt], ref[~hurt])
    wide = hurt[:, None, :, None].expand(n, s, g, c // g).reshape(n * s, c)
    assert bool(torch.isnan(y[wide]).all())
    assert torch.equal(y[~wide], clean[~wide])

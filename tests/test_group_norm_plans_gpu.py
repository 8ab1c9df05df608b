"""Group norm where its plans (a warp, a block, a cluster an image, passes over
global memory) have to agree."""

import ctypes
import subprocess
import sys

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


@gpu
@pytest.mark.parametrize("n,s,c,g,off", [
    (9, 16, 32, 4, 0), (9, 80, 32, 4, 0), (9, 80, 32, 4, 1), (160, 400, 90, 6, 0),
    (3, 5879, 64, 2, 0),
    (300, 441, 128, 8, 0),  # forward by clusters, backward over global memory
    (300, 441, 128, 8, 1),  # and by single floats
])
def test_a_relu_gate_is_the_forwards(n, s, c, g, off):
    """Where z is the rounding of a product, the backward opens the gates that
    the forward opened: dbias counts them (dy is one), and dx is the formula's
    for them."""
    gen = torch.Generator("cuda").manual_seed(2)
    image = torch.randint(-3, 4, (s, c), device="cuda", generator=gen) * 0.37 + 0.11
    x = image.repeat(n, 1)
    w = 1.0 + 0.3 * torch.randn(c, device="cuda", generator=gen)
    y, stats = torch.empty_like(x), torch.empty(n, g, 2, device="cuda")
    shape = dict(groups=g, spatial=s)
    _context().group_norm_fwd(x, w, None, y, stats, act="none", **shape)
    mean, rstd = (stats[0, :, i].repeat_interleave(c // g) for i in (0, 1))
    hat = (image - mean) * rstd
    b = -(hat * w)[0]  # z of a seventh of the elements is a rounding
    _context().group_norm_fwd(x, w, b, y, stats, act="relu", **shape)
    gate = y > 0
    near = (image == image[0]).repeat(n, 1)
    assert 0 < int(gate[near].sum()) < int(near.sum())
    dy = torch.ones(n * s * c + off, device="cuda")[off:].reshape(n * s, c)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    _context().group_norm_bwd(dy, x, w, b, stats, dx, dw, db, act="relu", **shape)
    assert torch.equal(db, gate.sum(0).float())
    d = (gate * w).double().reshape(n, s, g, c // g)
    hat = hat.double().reshape(1, s, g, c // g)
    r = rstd.double().reshape(1, 1, g, c // g)
    want = r * (d - d.mean((1, 3), keepdim=True) - hat * (d * hat).mean((1, 3), keepdim=True))
    # A wrong gate is off by rstd * w, some 1; roundings by some 2^-20 of it.
    assert float((dx.double() - want.reshape(n * s, c)).abs().max()) < 1e-4


_PROBE = """
import hashlib, sys
sys.path.insert(0, "tt-rl_b200")
import torch
from ttrl_b200.device import context
ctx = context("cuda:0")

def backward(n, s, c, g):
    gen = torch.Generator("cuda").manual_seed(3)
    x, dy = (torch.randn(n * s, c, device="cuda", generator=gen) for _ in range(2))
    y, stats = torch.empty_like(x), torch.empty(n, g, 2, device="cuda")
    ctx.group_norm_fwd(x, None, None, y, stats, groups=g, spatial=s)
    dw, db = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    ctx.group_norm_bwd(dy, x, None, None, stats, y, dw, db, groups=g, spatial=s)
    return hashlib.sha1(b"".join(t.cpu().numpy().tobytes() for t in (y, dw, db))).hexdigest()

shapes = {"narrow": (1200, 441, 96, 3), "wide": (800, 32, 2048, 8)}
print({name: backward(*shapes[name]) for name in sys.argv[1:]}["narrow"])
"""


@gpu
def test_results_do_not_depend_on_the_shapes_before():
    """Clusters of 256 and of 512 threads: how many are resident, and so which
    images a column's sums are added up by, is each kind's own."""
    def first(*names):
        run = subprocess.run([sys.executable, "-c", _PROBE, *names], capture_output=True,
                             text=True, timeout=300)
        assert run.returncode == 0, run.stderr
        return run.stdout.strip().splitlines()[-1]

    assert first("narrow") == first("wide", "narrow")


def test_more_channels_than_a_grid_holds_are_refused():
    """By the extents alone: no pointer is looked at."""
    from ttrl_b200._lib import lib
    p, null = ctypes.c_void_p(64), None
    for channels in (65535 * 256 + 1, 1 << 30):
        assert lib().ttrl_group_norm_workspace_bytes(1, 1, channels, 1, 0) == 0
        assert lib().ttrl_group_norm_fwd(p, null, null, p, null, 1, 1, channels, 1, 1e-5, 0, null,
                                         0, null) != 0
        assert b"channels" in lib().ttrl_last_error()
        assert lib().ttrl_group_norm_bwd(p, p, null, null, p, p, null, null, 1, 1, channels, 1, 0,
                                         0, 0, null, 0, null) != 0
        assert b"channels" in lib().ttrl_last_error()
    assert lib().ttrl_group_norm_workspace_bytes(1, 1, 65535 * 256, 1, 0) > 0

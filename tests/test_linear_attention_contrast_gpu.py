"""Linear attention over operands whose sizes differ within a sequence: between
tokens, across a start, between columns, and sums that runs of zeros leave to
older tokens. Each token (or column) is judged by its own float64 norm.

q and dout lean on their token's k and v, so that no result is a small
difference of large terms and its norm is that of its terms, up to a factor of
about two. Tolerance: 2e-6 as in test_linear_attention_gpu.py (four roundings
to 22 bits and the cut of at most 24 tensor core steps at 2^-24 each, 2e-6)."""

import pytest

torch = pytest.importorskip("torch")

from tests.test_linear_attention_gpu import plain  # noqa: E402

gpu = pytest.mark.gpu
TOL = 2e-6

#: steps, lanes, heads, key, value: a few tokens, one chunk, several on either
#: kernel, segments
SHAPES = [(6, 3, 2, 64, 64), (9, 2, 2, 128, 33), (50, 3, 2, 64, 64), (150, 2, 2, 32, 32), (200, 2, 2, 64, 64), (200, 2, 3, 100, 90),
          (1500, 1, 2, 64, 64)]


def draw(t, b, h, kd, vd, seed=0):
    g = torch.Generator().manual_seed(seed + t + kd)
    q, k, v, dout = (torch.randn(t, b, h, n, generator=g) for n in (kd, kd, vd, vd))
    return dict(q=k + 0.5 * q, k=k, v=v, dout=v + 0.5 * dout,
                state=torch.randn(b, h, kd, vd, generator=g),
                dstate=torch.randn(b, h, kd, vd, generator=g),
                starts=torch.zeros(t, b),
                decay=torch.tensor([1.0 - 2.0 ** -(5 + i) for i in range(h)]))


def run(d):
    """{name: (kernel's, float64's)}, tokens as [steps, lanes, heads, width]."""
    from ttrl_b200.device import context
    ctx = context("cuda:0")
    t, b, h, kd = d["k"].shape
    vd = d["v"].shape[-1]
    c = {n: x.cuda().contiguous() for n, x in d.items()}
    qkv = torch.cat([c[n].reshape(t, b, -1) for n in "qkv"], -1)
    dout = c["dout"].reshape(t, b, -1)
    shape = dict(heads=h, key_dim=kd, value_dim=vd, scale=0.3)
    out, new = torch.empty_like(dout), torch.empty_like(c["state"])
    dqkv, first = torch.empty_like(qkv), torch.empty_like(new)
    ctx.linear_attention_fwd(qkv, c["state"], c["starts"], c["decay"], out, new, **shape)
    ctx.linear_attention_bwd(dout, c["dstate"], qkv, c["state"], c["starts"], c["decay"], dqkv,
                             first, **shape)
    want = plain(qkv, c["state"], c["starts"], c["decay"], h, kd, vd, 0.3, dout, c["dstate"])
    cut = [h * kd, h * kd, h * vd]
    pairs = {"out": (out, want[0]), "new": (new, want[1]), "first": (first, want[3])}
    for n, x, y in zip(("dq", "dk", "dv"), dqkv.split(cut, -1), want[2].split(cut, -1)):
        pairs[n] = (x, y)
    for n in ("out", "dq", "dk", "dv"):
        pairs[n] = tuple(x.double().reshape(t, b, h, -1) for x in pairs[n])
    return pairs


def near(pair, dims, tol=TOL):
    got, want = (x.double() for x in pair)
    off = (got - want).pow(2).sum(dims).sqrt()
    size = want.pow(2).sum(dims).sqrt()
    assert torch.isfinite(got).all()
    assert bool((off <= tol * size).all()), float((off / size.clamp_min(1e-300)).max())


@gpu
@pytest.mark.parametrize("factor", [1e3, 1e5, 1e6, 1e8, 1e10, 1e12, 1e14])
@pytest.mark.parametrize("which", ["k", "v", "q", "dout"])
@pytest.mark.parametrize("t,b,h,kd,vd", SHAPES)
def test_a_dropped_episode_leaves_the_next_its_bits(t, b, h, kd, vd, which, factor):
    d = draw(t, b, h, kd, vd)
    at = t // 2 + 1
    d["starts"][at] = 1.0
    d[which][:at] *= factor
    for name, pair in run(d).items():
        near(pair, -1 if name in ("out", "dq", "dk", "dv") else (-1, -2))


@gpu
@pytest.mark.parametrize("factor", [1e3, 1e5, 1e8, 1e12])
@pytest.mark.parametrize("t,b,h,kd,vd", SHAPES)
def test_tokens_before_a_large_one_keep_their_bits(t, b, h, kd, vd, factor):
    d = draw(t, b, h, kd, vd)
    at = t // 2 + 1
    d["k"][at] *= factor
    pairs = run(d)
    near([x[:at] for x in pairs["out"]], -1)
    near([x[:at] for x in pairs["dq"]], -1)
    near(pairs["dv"], -1)
    d = draw(t, b, h, kd, vd, seed=1)
    d["dout"][at] *= factor  # a large gradient, for the tokens behind it
    pairs = run(d)
    near([x[at + 1:] for x in pairs["dk"]], -1)
    near([x[at + 1:] for x in pairs["dv"]], -1)
    near(pairs["dq"], -1)


@gpu
@pytest.mark.parametrize("factor", [1e6, 1e10, 1e14, 1e-6, 1e-10, 1e-14])
@pytest.mark.parametrize("places", ["one", "every fourth"])
@pytest.mark.parametrize("t,b,h,kd,vd", SHAPES)
def test_columns_keep_their_bits(t, b, h, kd, vd, places, factor):
    """A column of v of another size, for the others and for itself, and one
    of k with its inverse in q."""
    cols = slice(2, 3) if places == "one" else slice(1, None, 4)
    d = draw(t, b, h, kd, vd)
    d["v"][..., cols] *= factor
    d["dout"][..., cols] /= factor
    d["state"] *= 0
    d["dstate"] *= 0
    pairs = run(d)
    near(pairs["out"], 0)
    near(pairs["new"], -2)
    near(pairs["dv"], 0)
    d = draw(t, b, h, kd, vd, seed=2)
    d["k"][..., cols] *= factor
    d["q"][..., cols] /= factor
    d["state"] *= 0
    d["dstate"] *= 0
    pairs = run(d)
    near(pairs["out"], -1)
    near(pairs["new"], -1)
    near(pairs["dq"], 0)
    near(pairs["dk"], 0)


@gpu
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("t,b,h,kd,vd", SHAPES)
def test_runs_of_zeros_leave_old_tokens_their_bits(t, b, h, kd, vd, which):
    """A padded run under a strong decay: what is left is 2^-40 of the tokens
    before it, to all its bits."""
    d = draw(t, b, h, kd, vd)
    d["decay"][:] = 0.5
    d[which][t - 40:] = 0.0
    d["state"] *= 0
    pairs = run(d)
    near(pairs["out"], -1)
    near(pairs["new"], (-1, -2))


@gpu
def test_ordinary_sequences_beside_uneven_ones():
    """A lane's operands decide for that lane only: the others' results are bit
    for bit what they are alone."""
    from ttrl_b200.device import context
    ctx = context("cuda:0")
    d = draw(200, 3, 2, 64, 64)
    shape = dict(heads=2, key_dim=64, value_dim=64, scale=0.3)

    def forward(x):
        c = {n: y.cuda().contiguous() for n, y in x.items()}
        qkv = torch.cat([c[n].reshape(200, 3, -1) for n in "qkv"], -1)
        out, new = torch.empty(200, 3, 128, device="cuda"), torch.empty_like(c["state"])
        ctx.linear_attention_fwd(qkv, c["state"], c["starts"], c["decay"], out, new, **shape)
        return out, new

    alone = forward(d)
    d["k"][:90, 1] *= 1e9
    beside = forward(d)
    for lane in (0, 2):
        assert torch.equal(alone[0][:, lane], beside[0][:, lane])
        assert torch.equal(alone[1][lane], beside[1][lane])


@gpu
@pytest.mark.parametrize("sizes", [dict(dout=1e-20, dstate=1e-20), dict(k=1e-24), dict(v=1e-30),
                                   dict(k=1e-17, v=1e-17), dict(q=1e-15, k=1e-17)])
@pytest.mark.parametrize("t,b,h,kd,vd", SHAPES)
def test_tiny_operands_keep_their_bits(t, b, h, kd, vd, sizes):
    """Whole operands, down to what fp32 itself holds (a state of 1e-34)."""
    d = draw(t, b, h, kd, vd)
    d["state"] *= 0
    d["dstate"] *= 0 if "dout" not in sizes else 1
    for name, size in sizes.items():
        d[name] *= size
    pairs = run(d)
    near(pairs["out"], -1)
    near(pairs["new"], (-1, -2))
    near(pairs["first"], (-1, -2))
    for name in ("dq", "dk", "dv"):
        near(pairs[name], -1)

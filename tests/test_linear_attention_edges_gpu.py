"""Linear attention: results over its flags and decays, rows wider than 32-bit
offsets, and states that stay infinite over long sequences."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("name", ["starts", "decay"])
def test_results_over_flags_and_decays_are_refused(name):
    from ttrl_b200._lib import TtrlError
    from ttrl_b200.device import context
    ctx = context("cuda:0")
    t, b, h, kd, vd = 8, 4, 2, 16, 16
    shape = dict(heads=h, key_dim=kd, value_dim=vd, scale=0.25)
    qkv = torch.randn(t, b, h * (2 * kd + vd), device="cuda")
    dout, out = (torch.randn(t, b, h * vd, device="cuda") for _ in range(2))
    state, new = (torch.randn(b, h, kd, vd, device="cuda") for _ in range(2))
    dqkv = torch.empty_like(qkv)

    def inside(x, count):
        return x.view(-1)[8:8 + count].view(count)

    for result in ("out", "new", "dqkv", "dstate", "step out", "step state"):
        starts = torch.zeros(t, b, device="cuda")
        decay = torch.full((h,), 0.9, device="cuda")
        over = {"out": out, "new": new, "dqkv": dqkv, "dstate": new, "step out": out[0],
                "step state": new}[result]
        if name == "starts":
            starts = inside(over, b if "step" in result else t * b)
        else:
            decay = inside(over, h)
        with pytest.raises(TtrlError, match=name):
            if "step" in result:
                ctx.linear_attention_step(qkv[0], state, starts.view(-1)[:b], decay, out[0], new,
                                          **shape)
            elif result in ("out", "new"):
                ctx.linear_attention_fwd(qkv, state, starts, decay, out, new, **shape)
            else:
                ctx.linear_attention_bwd(dout, None, qkv, state, starts, decay, dqkv, new,
                                         **shape)


def test_rows_beyond_32_bit_offsets_are_refused():
    """Offsets within a row are 32 bits: a row of 2^31 floats or more is refused
    by its extents alone (no pointer is looked at)."""
    from ttrl_b200._lib import lib
    p, null = ctypes.c_void_p(64), None
    for heads, kd, vd in ((1 << 24, 128, 1), (1 << 23, 64, 128), (1 << 24, 1, 126)):
        assert heads * (2 * kd + vd) >= 1 << 31
        assert lib().ttrl_linear_attention_workspace_bytes(2, 1, heads, kd, vd) == 0
        calls = (
            lambda: lib().ttrl_linear_attention_fwd(p, null, null, p, p, null, 2, 1, heads, kd,
                                                    vd, 1.0, null, 0, null),
            lambda: lib().ttrl_linear_attention_bwd(p, null, p, null, null, p, p, null, 2, 1,
                                                    heads, kd, vd, 1.0, null, 0, null),
            lambda: lib().ttrl_linear_attention_step(p, p, null, p, p, p, 1, heads, kd, vd, 1.0,
                                                     null))
        for call in calls:
            assert call() != 0
            assert b"row" in lib().ttrl_last_error()


@gpu
@pytest.mark.parametrize("decay", [0.9, 0.5, 0.0])
@pytest.mark.parametrize("t", [700, 9000])
def test_an_infinite_state_stays_infinite(t, decay):
    """decay * inf is inf for every decay but zero, however long the sequence
    (its power over a part of it may be zero in float)."""
    from ttrl_b200.device import context
    ctx = context("cuda:0")
    kd = vd = 64
    g = torch.Generator("cuda").manual_seed(4)
    qkv = torch.randn(t, 1, 2 * kd + vd, device="cuda", generator=g)
    state = torch.randn(1, 1, kd, vd, device="cuda", generator=g)
    state[0, 0, 3, 5], state[0, 0, 7, 9] = float("inf"), float("-inf")
    d = torch.tensor([decay], device="cuda")
    out, new = torch.empty(t, 1, vd, device="cuda"), torch.empty_like(state)
    shape = dict(heads=1, key_dim=kd, value_dim=vd, scale=0.1)
    ctx.linear_attention_fwd(qkv, state, None, d, out, new, **shape)
    want = torch.zeros_like(state)
    want[0, 0, 3, 5], want[0, 0, 7, 9] = (float("inf") * decay, float("-inf") * decay)
    bad = ~torch.isfinite(want)
    assert torch.equal(torch.isfinite(new), ~bad)
    torch.testing.assert_close(new[bad], want[bad], rtol=0, atol=0, equal_nan=True)
    columns = torch.ones(vd, dtype=torch.bool, device="cuda")
    columns[[5, 9]] = False
    assert torch.isfinite(out[:, 0, columns]).all()
    q = qkv[:, 0, [3, 7]]
    first = torch.stack([q[:, 0] * want[0, 0, 3, 5], q[:, 1] * want[0, 0, 7, 9]], 1)
    torch.testing.assert_close(out[:, 0, [5, 9]], first, rtol=0, atol=0, equal_nan=True)

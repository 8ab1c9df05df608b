"""Linear attention: results over its flags and decays, rows wider than 32-bit
offsets, and states that stay infinite over long sequences."""

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

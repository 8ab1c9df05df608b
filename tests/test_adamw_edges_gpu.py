"""AdamW at the edges: 8-bit codes of blocks whose scale is near either end of
float's range, rates that float cannot hold, parameters changed in place, and
clipping over more tensors than one launch of the norm takes."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_adamw_gpu import HYPER, leaves, pack_plain  # noqa: E402

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("scale", [3e38, 1e38, 2.0 ** 126, 2.0 ** 125, 1e-30, 1e-38, 1e-40, 3e-45])
def test_codes_of_very_large_and_small_blocks(scale):
    """Bit for bit those of IEEE arithmetic: 1 / scale runs out of float's range
    at both ends."""
    from ttrl_b200.engine.optim import AdamW
    ps = leaves([1024], 5)
    opt = AdamW(ps, state_bits=8, min_8bit_size=1, **HYPER)
    rng = np.random.default_rng(6)
    share = rng.uniform(-1, 1, 1024).astype(np.float32)
    share[::256] = 1.0
    m = (share * np.float32(scale)).astype(np.float32)
    v = np.abs(m)
    assert np.isfinite(m).all()
    opt.load_moments([torch.from_numpy(m).cuda()], [torch.from_numpy(v).cuda()], t=1)
    for codes, scales, x, signed in ((opt._m8, opt._m_scale, m, True),
                                     (opt._v8, opt._v_scale, v, False)):
        want, size = pack_plain(x, signed)
        assert np.array_equal(codes.cpu().numpy().astype(np.int32)[:1024], want)
        assert np.array_equal(scales.cpu().numpy(), size)


@gpu
def test_an_eps_below_floats_range_is_refused():
    """The kernel divides in float: an eps that is zero there would make NaN of
    every parameter whose gradients have been zero."""
    from ttrl_b200.engine.optim import AdamW
    ps = leaves([300], 7)
    for eps in (1e-50, 1e-40, 2.0 ** -127):
        with pytest.raises(ValueError, match="eps"):
            AdamW(ps, lr=1e-3, eps=eps)
    opt = AdamW(ps, lr=1e-3, eps=2.0 ** -126, weight_decay=0.0)
    before = ps[0].data.clone()
    ps[0].grad = torch.zeros_like(before)
    opt.step()
    assert torch.equal(ps[0].data, before)
    state = opt.state_dict()
    state["eps"] = 1e-50
    with pytest.raises(ValueError, match="eps"):
        opt.load_state_dict(state)


@gpu
@pytest.mark.parametrize("change", ["transposed", "moved over another", "dtype"])
def test_a_parameter_changed_in_place_is_refused(change):
    """The same tensor object, with other strides, memory or type: refused
    before anything is written."""
    from ttrl_b200.engine.optim import AdamW
    ps = leaves([(64, 64), (64, 64), 100], 8)
    opt = AdamW(ps, **HYPER)
    opt.step()
    if change == "transposed":
        ps[0].data.t_()
    elif change == "moved over another":
        ps[0].data.set_(ps[1].data)
    else:
        ps[0].data.data = torch.zeros(64, 64, device="cuda", dtype=torch.int32)
    before = [p.data.clone() for p in ps]
    with pytest.raises(ValueError, match="AdamW"):
        opt.step()
    assert all(torch.equal(p.data, b) for p, b in zip(ps, before))
    assert opt.steps == [1, 1, 1]


@gpu
@pytest.mark.parametrize("count", [64, 65, 130, 400])
def test_clipping_over_many_tensors(count):
    """The norm of any number of gradients, and a clipped step of AdamW. The sum
    of squares is in 64 bits; the factor and out[0] are rounded to float once
    (2^-24), as is each scaled gradient."""
    from ttrl_b200.algos.grads import clip_grad_norm_device, grad_sq_device
    from ttrl_b200.engine.optim import AdamW
    sizes = [1 + 37 * (i % 91) for i in range(count)]
    sizes[-1] = 100_003
    ps, twins = leaves(sizes, 9), leaves(sizes, 9)
    exact = sum(float((p.grad.double() ** 2).sum()) for p in ps)
    assert abs(float(grad_sq_device(ps)) / exact - 1) <= 2.0 ** -23
    opt, ref = AdamW(ps, **HYPER), AdamW(twins, **HYPER)
    out = clip_grad_norm_device(ps, 0.5, opt)
    factor = 0.5 / (exact ** 0.5 + 1e-6)
    assert abs(float(out[0]) / exact - 1) <= 2.0 ** -23
    assert abs(float(out[1]) / factor - 1) <= 2.0 ** -23
    opt.step()
    for p in twins:
        p.grad = p.grad * out[1]
    ref.step()
    for p, q in zip(ps, twins):
        assert torch.equal(p.data, q.data)
    again = clip_grad_norm_device(ps, 0.5)
    assert torch.equal(out, again)


@gpu
def test_clipping_passes_over_empty_tensors_and_replays():
    from ttrl_b200.algos.grads import clip_grad_norm_device
    ps = leaves([5] * 70 + [0], 10)
    want = clip_grad_norm_device(ps[:-1], 0.1).clone()
    assert torch.equal(clip_grad_norm_device(ps, 0.1), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = clip_grad_norm_device(ps, 0.1)
    ps[3].grad.mul_(1.0)
    graph.replay()
    assert torch.equal(got, want)

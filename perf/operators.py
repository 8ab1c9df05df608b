"""The measured cases of three operators: the linear-attention memory, group
norm with an activation, and AdamW over many tensors.

`run` computes a case in its plain form, elementary torch operations in 32
bits, or, with `own` set, by the calls a user of ttrl_b200 makes.
"""

import math
import os
import sys

import torch

own = False

_CHUNK = 64  # tokens a chunk of the plain linear attention
_BLOCK = 256  # elements that share a scale in 8-bit optimizer states

#: The recurrent actor-critic's parameters: Nature-CNN trunk, 512-wide
#: encoder, 256-wide GRU, policy and value heads.
_RECURRENT_NET = ("8192,32,32768,64,36864,64,1605632,512,393216,196608,768,768,"
                  "1536,6,256,1")


def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-rl_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _context():
    _package()
    from ttrl_b200.device import context
    return context("cuda:0")


def listed():
    return [
        # One acting step of a small set of environments: latency.
        {"name": "attention step, 16 lanes", "op": "step", "batch": 16, "heads": 4, "key": 64,
         "value": 64, "starts": True},
        # One acting step of a large vectorised simulator: the state's bytes.
        {"name": "attention step, 4096 lanes", "op": "step", "batch": 4096, "heads": 4,
         "key": 64, "value": 64, "starts": True},
        # The recurrent PPO minibatch (16 sequences of 32 steps), with resets.
        {"name": "attention train, 32x16", "op": "attention", "train": True, "steps": 32,
         "batch": 16, "heads": 4, "key": 64, "value": 64, "starts": True},
        # Few long contexts, odd length: the time axis has to be split.
        {"name": "attention forward, 8191x2", "op": "attention", "train": False, "steps": 8191,
         "batch": 2, "heads": 8, "key": 64, "value": 64, "starts": False},
        # Many episodes of a long rollout, unequal key and value widths.
        {"name": "attention train, 1024x64", "op": "attention", "train": True, "steps": 1024,
         "batch": 64, "heads": 8, "key": 64, "value": 128, "starts": True},
        # The third conv layer of an acting batch: latency.
        {"name": "norm forward, 32x7x7x64", "op": "norm", "train": False, "images": 32,
         "spatial": 49, "channels": 64, "groups": 8, "act": "relu"},
        # The first conv layer of a PPO minibatch.
        {"name": "norm train, 256x20x20x32", "op": "norm", "train": True, "images": 256,
         "spatial": 400, "channels": 32, "groups": 4, "act": "silu"},
        # The head norm behind the memory: one row a token.
        {"name": "norm train, 32768x512", "op": "norm", "train": True, "images": 32768,
         "spatial": 1, "channels": 512, "groups": 8, "act": "silu"},
        # A wide residual stage of a large batch, with groups of odd width.
        {"name": "norm train, 512x42x42x90", "op": "norm", "train": True, "images": 512,
         "spatial": 1764, "channels": 90, "groups": 6, "act": "silu"},
        # The recurrent actor-critic's update.
        {"name": "adamw, recurrent net", "op": "adamw", "sizes": _RECURRENT_NET, "tensors": 16,
         "params": 2277287, "bits": 32},
        # A deep net: hundreds of tensors, most of them short.
        {"name": "adamw, 320 tensors", "op": "adamw", "sizes": "", "tensors": 320,
         "params": 24000000, "bits": 32},
        # The largest: states in 8 bits, read back as a checkpoint reads them.
        {"name": "adamw, 8 bits, 96 tensors", "op": "adamw", "sizes": "", "tensors": 96,
         "params": 100000000, "bits": 8},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "attention", "attention", "norm", "norm", "adamw"])
    if op == "step":
        heads, key, value = rng.choice([1, 2, 4, 8]), rng.randint(8, 128), rng.randint(8, 128)
        most = max(1, 67108864 // (heads * key * value))
        return {"op": op, "batch": _log_int(rng, 1, min(4096, most)), "heads": heads, "key": key,
                "value": value, "starts": rng.random() < 0.5}
    if op == "attention":
        heads = rng.choice([1, 2, 3, 4, 8])
        key, value = rng.choice([16, 32, 48, 64, 100, 128]), rng.choice([16, 32, 64, 90, 128])
        steps = _log_int(rng, 2, 8191)
        most = max(1, 100663296 // (steps * heads * (key + value)))
        return {"op": op, "train": rng.random() < 0.5, "steps": steps,
                "batch": _log_int(rng, 1, min(256, most)), "heads": heads, "key": key,
                "value": value, "starts": rng.random() < 0.5}
    if op == "norm":
        groups, width = rng.choice([1, 2, 4, 8]), rng.randint(2, 64)
        spatial = rng.choice([1, _log_int(rng, 4, 7056)])
        most = max(1, 81285120 // (groups * width * spatial))
        train = rng.random() < 0.5
        # relu's derivative jumps: a rounding next to zero decides a whole
        # gradient, so gradients are measured with the smooth activations.
        return {"op": op, "train": train, "images": _log_int(rng, 1, min(32768, most)),
                "spatial": spatial, "channels": groups * width, "groups": groups,
                "act": rng.choice(["none", "silu"] if train else ["none", "relu", "silu"])}
    tensors = _log_int(rng, 1, 400)
    return {"op": op, "sizes": "", "tensors": tensors,
            "params": max(tensors * 8, _log_int(rng, 5000, 50000000)),
            "bits": rng.choice([8, 32])}


def _sizes(case):
    """Tensor lengths of an AdamW case: given, or a spread of short biases
    and long weights of odd lengths that adds up to `params`."""
    if case["sizes"]:
        return [int(s) for s in case["sizes"].split(",")]
    n, total = case["tensors"], case["params"]
    weights = [1.0 if i % 2 else 50.0 + 13.0 * (i * 7 % 31) for i in range(n)]
    whole = sum(weights)
    sizes = [max(1, int(total * w / whole)) for w in weights]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(shape, device="cuda", generator=g) * scale + shift

    s = dict(case)
    if case["op"] in ("step", "attention"):
        b, h, k, v = case["batch"], case["heads"], case["key"], case["value"]
        t = case.get("steps", 1)
        s["qkv"] = normal(t, b, h * (2 * k + v))
        s["state"] = normal(b, h, k, v)
        s["starts"] = None
        if case["starts"]:
            s["starts"] = (torch.rand((t, b), device="cuda", generator=g) < 0.02).float()
        # One time scale a head: 1 - 2^-5, 2^-6, ...
        s["decay"] = torch.tensor([1.0 - 2.0 ** -(5 + i % 6) for i in range(h)], device="cuda")
        s["scale"] = k ** -0.5
        if case.get("train"):
            s["dout"] = normal(t, b, h * v)
            s["dstate"] = normal(b, h, k, v)
        return s
    if case["op"] == "norm":
        n, p, c = case["images"], case["spatial"], case["channels"]
        s["x"] = normal(n * p, c, scale=1.5, shift=0.3)
        s["weight"] = normal(1, c, scale=0.1, shift=1.0)
        s["bias"] = normal(1, c, scale=0.1)
        if case["train"]:
            s["dy"] = normal(n * p, c)
        return s
    sizes = _sizes(case)
    # One flat buffer, every tensor at a 256-byte boundary, zeros between.
    at = (torch.tensor(sizes, device="cuda") + 63) // 64 * 64
    total = int(at.sum())
    first = torch.cumsum(at, 0) - at
    of = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), at)
    place = torch.arange(total, device="cuda") - first[of]
    there = (place < torch.tensor(sizes, device="cuda")[of]).float()
    s["p"] = normal(total, scale=0.05) * there
    # Every tensor learns at a scale of its own.
    rate = torch.rand(len(sizes), device="cuda", generator=g) * 3 + 0.1
    s["g"] = normal(total, scale=0.01) * rate[of] * there
    s["m"], s["v"] = s["g"] * normal(total, scale=0.3), (s["g"] * normal(total)) ** 2
    s["t"] = 100
    s["hyper"] = dict(lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    if case["bits"] == 8:
        # The block of every element: blocks of 256 start at each tensor.
        blocks = (at + _BLOCK - 1) // _BLOCK
        s["block"] = (torch.cumsum(blocks, 0) - blocks)[of] + place // _BLOCK
        s["blocks"] = int(blocks.sum())
        s["m"], s["v"] = _pack(s["m"], s, True), _pack(s["v"], s, False)
    if own:
        _package()
        from ttrl_b200.engine.autograd import Tensor
        from ttrl_b200.engine.optim import AdamW

        def views(x):
            return [x[f:f + n] for f, n in zip(first.tolist(), sizes)]

        leaves = [Tensor(x, True) for x in views(s["p"])]
        for leaf, x in zip(leaves, views(s["g"])):
            leaf.grad = x
        s["opt"] = AdamW(leaves, state_bits=case["bits"], min_8bit_size=1, **s["hyper"])
        if case["bits"] == 8:
            # The moments are held in 8 bits: read back as a checkpoint reads them.
            s["m"], s["v"] = _unpack(s["m"], s, True), _unpack(s["v"], s, False)
        s["opt"].load_moments(views(s["m"]), views(s["v"]), t=s["t"])
        s["read"] = [views(s["m"]), views(s["v"])]
    return s


# ------------------------------------------------------- 8-bit states

def _pack(x, s, signed):
    """(codes, scales): a block's largest magnitude is its scale. The first
    moment is held as the signed square root of its share of it in 127
    steps, the second (never negative) as the fourth root in 255, a positive
    value at least as 1."""
    size = x.abs()
    scale = torch.zeros(s["blocks"], device="cuda").scatter_reduce(0, s["block"], size, "amax")
    part = size / torch.where(scale > 0, scale, torch.ones_like(scale))[s["block"]]
    if signed:
        return torch.round(torch.sqrt(part) * 127.0) * torch.sign(x), scale
    code = torch.round(torch.sqrt(torch.sqrt(part)) * 255.0)
    return torch.where(x > 0, code.clamp_min(1.0), code), scale


def _unpack(packed, s, signed):
    code, scale = packed
    root = code * (1.0 / (127.0 if signed else 255.0))
    root = root * root.abs()
    return (root if signed else root * root) * scale[s["block"]]


# -------------------------------------------------------- plain forms

def _attend(q, k, v, decay, starts, s0):
    """o_t = q_t S_t of S_t = decay (1 - start_t) S_{t-1} + k_t v_t^T over
    [B, H, T, .] tensors, chunk by chunk; -> (o, S after the last token)."""
    b, h, t, dk = q.shape
    dv = v.shape[-1]
    n = -(-t // _CHUNK)
    pad = n * _CHUNK - t

    def chunks(x):
        return torch.nn.functional.pad(x, (0, 0, 0, pad)).reshape(b, h, n, _CHUNK, -1)

    q, k, v = chunks(q), chunks(k), chunks(v)
    dev = q.device
    log = torch.log2(decay.double())[:, None, None]
    seg = torch.zeros((b, t), device=dev, dtype=torch.long)
    if starts is not None:
        seg = torch.cumsum((starts != 0).long(), 1)
    last = torch.clamp(torch.arange(1, n + 1, device=dev) * _CHUNK, max=t) - 1
    seg_end = torch.cat([torch.zeros_like(seg[:, :1]), seg[:, last]], 1)  # before chunk c
    segc = torch.nn.functional.pad(seg, (0, pad), value=-1).reshape(b, n, _CHUNK)
    i = torch.arange(_CHUNK, device=dev)
    gap = i[:, None] - i[None, :]
    weight = torch.where(gap >= 0, torch.exp2(log * gap.clamp_min(0)), 0.0).float()
    same = (segc[:, :, :, None] == segc[:, :, None, :]).float()
    scores = torch.matmul(q, k.transpose(-1, -2)) * weight[None, :, None] * same[:, None]
    o = torch.matmul(scores, v)
    # Each chunk's own contribution to the state behind it.
    length = torch.clamp(t - torch.arange(n, device=dev) * _CHUNK, max=_CHUNK)
    left = length[:, None] - 1 - i[None, :]
    keep = torch.exp2(log * left.clamp_min(0)).float()[None]
    keep = keep * ((segc == seg_end[:, 1:, None]) & (left >= 0)).float()[:, None]
    local = torch.matmul((k * keep[..., None]).transpose(-1, -2), v)  # B H n K V
    # The state before chunk c (c = n: behind the last): decayed sums of the
    # earlier chunks' contributions and of s0, none across a start.
    begin = torch.clamp(torch.arange(n + 1, device=dev) * _CHUNK, max=t)
    reach = begin[:, None] - begin[None, 1:]
    mix = torch.where(reach >= 0, torch.exp2(log * reach.clamp_min(0)), 0.0).float()[None]
    mix = mix * (seg_end[:, :, None] == seg_end[:, None, 1:]).float()[:, None]
    state = torch.matmul(mix, local.reshape(b, h, n, dk * dv))
    from0 = torch.exp2(log[:, :, 0] * begin).float()[None] * (seg_end == 0).float()[:, None]
    state = (state + from0[..., None] * s0.reshape(b, h, 1, -1)).reshape(b, h, n + 1, dk, dv)
    enter = torch.exp2(log * (i[None, :] + 1)).float()[None]
    enter = enter * (segc == seg_end[:, :-1, None]).float()[:, None]
    o = o + enter[..., None] * torch.matmul(q, state[:, :, :-1])
    return o.reshape(b, h, n * _CHUNK, dv)[:, :, :t], state[:, :, -1]


def _heads(s):
    h, k, v = s["heads"], s["key"], s["value"]
    x = s["qkv"].permute(1, 0, 2)
    b, t, _ = x.shape
    parts = x.split([h * k, h * k, h * v], -1)
    return [p.reshape(b, t, h, -1).transpose(1, 2) for p in parts]


def _rows(x):
    """[B, H, T, D] -> time-major rows [T, B, H * D]."""
    b, h, t, d = x.shape
    return x.permute(2, 0, 1, 3).reshape(t, b, h * d)


def _plain_step(s):
    h, k, v = s["heads"], s["key"], s["value"]
    q, k, v = (x.reshape(s["batch"], h, -1) for x in s["qkv"][0].split([h * k, h * k, h * v], -1))
    keep = s["decay"][None, :]
    if s["starts"] is not None:
        keep = keep * (s["starts"][0] == 0).float()[:, None]
    state = s["state"] * keep[..., None, None] + k[..., :, None] * v[..., None, :]
    out = ((q * s["scale"])[..., :, None] * state).sum(2)
    return {"out": out.reshape(1, s["batch"], -1), "state": state}


def _plain_attention(s):
    q, k, v = _heads(s)
    starts = None if s["starts"] is None else s["starts"].t()
    decay, scale = s["decay"], s["scale"]
    o, state = _attend(q * scale, k, v, decay, starts, s["state"])
    out = {"out": _rows(o), "state": state}
    if not s.get("train"):
        return out
    b, h, t, _ = q.shape
    do = s["dout"].permute(1, 0, 2).reshape(b, t, h, -1).transpose(1, 2)
    dq, _ = _attend(do, v, k, decay, starts, s["state"].transpose(-1, -2))
    # Backwards in time the gradient of the state is the same recurrence.
    after = None
    if starts is not None:
        after = torch.cat([torch.zeros_like(starts[:, :1]), starts.flip(1)[:, :-1]], 1)
    end = s["dstate"] / decay[:, None, None]
    kr, vr, qr, dor = (x.flip(2) for x in (k, v, q * scale, do))
    dv, first = _attend(kr, qr, dor, decay, after, end)
    dk, _ = _attend(vr, dor, qr, decay, after, end.transpose(-1, -2))
    ds = first * decay[:, None, None]
    if starts is not None:
        ds = ds * (starts[:, 0] == 0).float()[:, None, None, None]
    out["dqkv"] = torch.cat([_rows(dq * scale), _rows(dk.flip(2)), _rows(dv.flip(2))], -1)
    out["dstate"] = ds
    return out


def _plain_norm(s):
    n, p, c, groups = s["images"], s["spatial"], s["channels"], s["groups"]
    x = s["x"].reshape(n, p, groups, c // groups)
    w, b = s["weight"].reshape(groups, -1), s["bias"].reshape(groups, -1)
    centred = x - x.mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-5)
    hat = centred * rstd
    z = hat * w + b
    gate = torch.sigmoid(z) if s["act"] == "silu" else None
    y = {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: z * gate}[s["act"]]()
    out = {"y": y.reshape(n * p, c)}
    if not s["train"]:
        return out
    dz = s["dy"].reshape(z.shape)
    if s["act"] == "silu":
        dz = dz * (gate * (1.0 + z * (1.0 - gate)))
    elif s["act"] == "relu":
        dz = dz * (z > 0)
    # Sums over all images and places: long, so in 64 bits.
    out["dweight"] = (dz * hat).sum((0, 1), dtype=torch.float64).float().reshape(1, c)
    out["dbias"] = dz.sum((0, 1), dtype=torch.float64).float().reshape(1, c)
    d = dz * w
    d = rstd * (d - d.mean((1, 3), keepdim=True) - hat * (d * hat).mean((1, 3), keepdim=True))
    out["dx"] = d.reshape(n * p, c)
    return out


def _plain_adamw(s):
    lr, (b1, b2) = s["hyper"]["lr"], s["hyper"]["betas"]
    eps, wd = s["hyper"]["eps"], s["hyper"]["weight_decay"]
    s["t"] += 1
    g = s["g"]
    packed = s["bits"] == 8
    m = _unpack(s["m"], s, True) if packed else s["m"]
    v = _unpack(s["v"], s, False) if packed else s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = torch.sqrt(v) * (1.0 / math.sqrt(1 - b2 ** s["t"])) + eps
    s["p"] = s["p"] * (1 - lr * wd) - (m / root) * (lr / (1 - b1 ** s["t"]))
    s["m"], s["v"] = m, v
    if packed:
        s["m"], s["v"] = _pack(m, s, True), _pack(v, s, False)
        m, v = _unpack(s["m"], s, True), _unpack(s["v"], s, False)
    return {"p": s["p"], "m": m, "v": v}


# ------------------------------------------------- the framework's calls

def _own_attention(s):
    ctx = _context()
    t, b, _ = s["qkv"].shape
    h, k, v = s["heads"], s["key"], s["value"]
    out = torch.empty((t, b, h * v), device="cuda")
    state = torch.empty_like(s["state"])
    shape = dict(heads=h, key_dim=k, value_dim=v, scale=s["scale"])
    if s["op"] == "step":
        ctx.linear_attention_step(s["qkv"][0], s["state"], s["starts"], s["decay"], out[0], state,
                                  **shape)
        return {"out": out, "state": state}
    ctx.linear_attention_fwd(s["qkv"], s["state"], s["starts"], s["decay"], out, state, **shape)
    if not s["train"]:
        return {"out": out, "state": state}
    dqkv, dstate = torch.empty_like(s["qkv"]), torch.empty_like(state)
    ctx.linear_attention_bwd(s["dout"], s["dstate"], s["qkv"], s["state"], s["starts"],
                             s["decay"], dqkv, dstate, **shape)
    return {"out": out, "state": state, "dqkv": dqkv, "dstate": dstate}


def _own_norm(s):
    ctx = _context()
    x, w, b = s["x"], s["weight"], s["bias"]
    y = torch.empty_like(x)
    stats = torch.empty((s["images"], s["groups"], 2), device="cuda") if s["train"] else None
    shape = dict(groups=s["groups"], spatial=s["spatial"], act=s["act"])
    ctx.group_norm_fwd(x, w, b, y, stats, eps=1e-5, **shape)
    if not s["train"]:
        return {"y": y}
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    ctx.group_norm_bwd(s["dy"], x, w, b, stats, dx, dw, db, **shape)
    return {"y": y, "dweight": dw, "dbias": db, "dx": dx}


def _own_adamw(s):
    opt = s["opt"]
    opt.step()
    if s["bits"] == 8:
        opt.read_moments(*s["read"])
        m, v = s["m"], s["v"]
    else:
        m, v = opt.moment_arenas
    return {"p": s["p"], "m": m, "v": v}


def run(state):
    if own:
        return {"step": _own_attention, "attention": _own_attention, "norm": _own_norm,
                "adamw": _own_adamw}[state["op"]](state)
    return {"step": _plain_step, "attention": _plain_attention, "norm": _plain_norm,
            "adamw": _plain_adamw}[state["op"]](state)


# ------------------------------------------------------------ in 64 bits

def _exact_attention(s):
    """Token by token, from the recurrence itself."""
    t, b, _ = s["qkv"].shape
    h, kd, vd = s["heads"], s["key"], s["value"]
    x = s["qkv"].double()
    q = x[:, :, :h * kd].reshape(t, b, h, kd) * s["scale"]
    k = x[:, :, h * kd:2 * h * kd].reshape(t, b, h, kd)
    v = x[:, :, 2 * h * kd:].reshape(t, b, h, vd)
    lam = s["decay"].double()[None, :, None, None]
    go = torch.ones((t, b, 1, 1, 1), device="cuda", dtype=torch.float64)
    if s["starts"] is not None:
        go = (s["starts"] == 0).double()[:, :, None, None, None]
    train = s.get("train", False)
    state, outs, dqs = s["state"].double(), [], []
    do = s["dout"].double().reshape(t, b, h, vd) if train else None
    for i in range(t):
        state = state * (lam * go[i]) + k[i][..., :, None] * v[i][..., None, :]
        outs.append(torch.einsum("bhk,bhkv->bhv", q[i], state))
        if train:
            dqs.append(torch.einsum("bhv,bhkv->bhk", do[i], state) * s["scale"])
    out = {"out": torch.stack(outs).reshape(t, b, h * vd), "state": state}
    if not train:
        return out
    outs.clear()
    dqkv = torch.empty((t, b, x.shape[-1]), device="cuda", dtype=torch.float64)
    dqkv[:, :, :h * kd] = torch.stack(dqs).reshape(t, b, h * kd)
    dqs.clear()
    r = s["dstate"].double()
    for i in reversed(range(t)):
        r = r + q[i][..., :, None] * do[i][..., None, :]
        dqkv[i, :, h * kd:2 * h * kd] = torch.einsum("bhkv,bhv->bhk", r, v[i]).reshape(b, -1)
        dqkv[i, :, 2 * h * kd:] = torch.einsum("bhkv,bhk->bhv", r, k[i]).reshape(b, -1)
        r = r * (lam * go[i])
    out["dqkv"], out["dstate"] = dqkv, r
    return out


def _exact_norm(s):
    n, p, c, g = s["images"], s["spatial"], s["channels"], s["groups"]
    x = s["x"].double().reshape(n, p, c).transpose(1, 2).reshape(n, g, -1)
    count = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / count
    var = (x * x).sum(-1, keepdim=True) / count - mean * mean
    inv = (var + 1e-5) ** -0.5
    hat = ((x - mean) * inv).reshape(n, c, p)
    z = hat * s["weight"].double().reshape(1, c, 1) + s["bias"].double().reshape(1, c, 1)
    act = s["act"]
    y = z.clamp_min(0) if act == "relu" else z / (1 + torch.exp(-z)) if act == "silu" else z
    out = {"y": y.transpose(1, 2).reshape(n * p, c)}
    if not s["train"]:
        return out
    dz = s["dy"].double().reshape(n, p, c).transpose(1, 2)
    if act == "silu":
        e = torch.exp(-z)
        dz = dz * (1 + e + z * e) / (1 + e) ** 2
    elif act == "relu":
        dz = torch.where(z > 0, dz, 0.0)
    out["dweight"] = torch.einsum("ncp,ncp->c", dz, hat).reshape(1, c)
    out["dbias"] = torch.einsum("ncp->c", dz).reshape(1, c)
    d = (dz * s["weight"].double().reshape(1, c, 1)).reshape(n, g, -1)
    hat = hat.reshape(n, g, -1)
    along = torch.einsum("ngi,ngi->ng", d, hat)[..., None] / count
    dx = inv * (d - d.sum(-1, keepdim=True) / count - hat * along)
    out["dx"] = dx.reshape(n, c, p).transpose(1, 2).reshape(n * p, c)
    return out


def _exact_adamw(s):
    lr, (b1, b2) = s["hyper"]["lr"], s["hyper"]["betas"]
    t, g = s["t"] + 1, s["g"].double()
    if s["bits"] == 8:
        c, r = (x.double() for x in s["m"])
        m = torch.sign(c) * (c / 127) ** 2 * r[s["block"]]
        c, r = (x.double() for x in s["v"])
        v = (c / 255) ** 4 * r[s["block"]]
    else:
        m, v = s["m"].double(), s["v"].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
    step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + s["hyper"]["eps"])
    p = s["p"].double()
    p = p - lr * s["hyper"]["weight_decay"] * p - lr * step
    # A code next to the middle of two has no value but what 32 bits give.
    return {"p": p, "m": None, "v": None} if s["bits"] == 8 else {"p": p, "m": m, "v": v}


def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_attention, "attention": _exact_attention, "norm": _exact_norm,
            "adamw": _exact_adamw}[s["op"]](s)


def work(case):
    op = case["op"]
    if op in ("step", "attention"):
        h, k, v = case["heads"], case["key"], case["value"]
        rows = case.get("steps", 1) * case["batch"]
        state = 4 * case["batch"] * h * k * v
        io = 4 * rows * h * (2 * k + v)
        out = 4 * rows * h * v
        if not case.get("train"):
            # A token updates the state and reads it: a multiply and an add
            # an element each.
            return {"bytes": io + out + 2 * state, "flops": 4 * rows * h * k * v}
        return {"bytes": 2 * io + 2 * out + 4 * state, "flops": 12 * rows * h * k * v}
    if op == "norm":
        n = case["images"] * case["spatial"] * case["channels"]
        if not case["train"]:
            return {"bytes": 8 * n, "flops": 8 * n}
        return {"bytes": 16 * n, "flops": 24 * n}
    n = sum(_sizes(case))
    if case["bits"] == 32:
        return {"bytes": 28 * n, "flops": 14 * n}
    return {"bytes": (12 + 4 + 8) * n + 16 * (n // _BLOCK), "flops": 30 * n}

"""What the training operators of this package are measured on: the optimizer's AdamW step over all the tensors of a model
(32-bit or 8-bit states, with the clipping of the gradients' global norm) and the layer norm of the encoder and of the head,
forward and backward.  `own` selects the package's kernels; without it every operator runs in its plain form, elementary
torch operations in 32 bits (64 for the long sum of the gradient norm), rounded once at the end.

The 8-bit states are block-scaled floats: 32 consecutive elements of a tensor share one power-of-two scale (e8m0, 2^(s-127)),
the first moment is held in e4m3, the second in e5m2, both rounded stochastically.  The random bits are a function of
(seed, step, position), so that both forms round every element the same way.
"""
import numpy as np
import torch

own = False

BLOCK = 32                                   # elements that share a scale
BETAS, EPS, LR, DECAY = (0.9, 0.999), 1e-5, 1e-4, 1e-2


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # the last layer of the head alone (256 -> 56, with bias), as when only the regressor is refined on a new basis: latency
        dict(name="adamw_last_layer", op="adamw", part="last", edge=64, views=2, latent=56, depth=0, bits=32, dtype="fp32", clip=False),
        # the whole network at 64^3: 18 tensors, 0.5 M parameters
        dict(name="adamw_64", op="adamw", part="all", edge=64, views=2, latent=56, depth=0, bits=32, dtype="fp32", clip=True),
        # 256^3, two views: 13.5 M parameters, nearly all in the first layer of the head
        dict(name="adamw_256_clip", op="adamw", part="all", edge=256, views=2, latent=56, depth=0, bits=32, dtype="fp32", clip=True),
        # the same with block-scaled 8-bit states
        dict(name="adamw8_256_clip", op="adamw", part="all", edge=256, views=2, latent=56, depth=0, bits=8, dtype="fp32", clip=True),
        # 384^3: 44.6 M parameters, the largest network of the configurations
        dict(name="adamw_384", op="adamw", part="all", edge=384, views=2, latent=56, depth=0, bits=32, dtype="fp32", clip=False),
        # a deep encoder with normalised blocks: 178 small tensors of uneven sizes, bf16 parameters, 8-bit states
        dict(name="adamw8_deep_bf16", op="adamw", part="all", edge=96, views=11, latent=57, depth=40, bits=8, dtype="bf16", clip=True),
        # normalised head at batch 8 (800 features): latency
        dict(name="norm_head_train", op="norm", rows=8, cols=800, dtype="fp32", train=True, act=False),
        # the flattened encoder output of 160^3 at the batch of 30
        dict(name="norm_features_train", op="norm", rows=30, cols=4000, dtype="fp32", train=True, act=False),
        # the first encoder block at 256^3, channels last: a row of 16 channels for each voxel
        dict(name="norm_block0_train", op="norm", rows=256 ** 3, cols=16, dtype="fp32", train=True, act=False),
        # the second block's bf16 activations in inference, LeakyReLU in the same pass, two cases of 128^3 voxels
        dict(name="norm_block1_infer_bf16", op="norm", rows=2 * 128 ** 3, cols=32, dtype="bf16", train=False, act=True),
        # one statistic for each sample over the whole third activation (64^3 voxels, 32 channels): few rows, long ones
        dict(name="norm_sample_train", op="norm", rows=2, cols=32 * 64 ** 3, dtype="fp32", train=True, act=False),
        # odd sizes
        dict(name="norm_odd_train_bf16", op="norm", rows=4099, cols=801, dtype="bf16", train=True, act=False),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    if rng.random() < 0.5:
        part = "last" if rng.random() < 0.15 else "all"
        return dict(op="adamw", part=part, edge=spread(32, 384), views=rng.randint(1, 11), latent=rng.randint(5, 64),
                    depth=rng.choice([0, 0, 0, rng.randint(1, 40)]), bits=rng.choice([32, 8]), dtype=rng.choice(["fp32", "fp32", "bf16"]),
                    clip=rng.random() < 0.5)
    dtype = rng.choice(["fp32", "fp32", "bf16"])
    train = rng.random() < 0.65
    cols = rng.choice([16, 32, spread(4, 4_000_000), spread(4, 40_000), spread(4, 2000)])
    rows = spread(1, max(1, min(256 ** 3, 2 ** 27 // cols)))
    return dict(op="norm", rows=rows, cols=cols, dtype=dtype, train=train, act=not train and rng.random() < 0.5)


def shapes(case):
    """The tensors that the optimizer steps: six 3x3x3 conv blocks (strides 1, 2, 2, 2, 2, 2), `depth` further normalised
    blocks, the head flatten -> 800 -> 256 -> latent."""
    latent, edge = case["latent"], case["edge"]
    last = [(latent, 256), (latent,)]
    if case["part"] == "last":
        return last
    chans = [case["views"] + 1, 16, 32, 32, 32, 32, 32]
    conv = [s for a, b in zip(chans, chans[1:]) for s in ((b, a, 3, 3, 3), (b,))]
    more = [(32, 32, 3, 3, 3), (32,), (32,), (32,)] * case["depth"]
    left = -(-edge // 32)
    return conv + more + [(800, 32 * left ** 3), (800,), (256, 800), (256,)] + last


def blocks_of(n):
    return -(-n // BLOCK)


def sizes(case):
    return [int(np.prod(s)) for s in shapes(case)]


# ----------------------------------------------------------------------------- what a user's program holds
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    dtype = TYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # a convolution's output: every channel with its own offset and spread
        x = (randn(rows, cols) * (randn(cols) * 0.3 + 1.2) + randn(cols) * 0.5).to(dtype)
        state = dict(op="norm", x=x, weight=1 + 0.1 * randn(cols), bias=0.1 * randn(cols), eps=1e-5, train=case["train"],
                     slope=0.2 if case["act"] else 1.0)
        if case["train"]:
            state["gy"] = (randn(rows, cols) * 1e-2).to(dtype)
        return state
    dims, ns = shapes(case), sizes(case)
    offs = np.concatenate([[0], np.cumsum([BLOCK * blocks_of(n) for n in ns])]).tolist()
    total = offs[-1]
    # flat buffers whose tensors start on whole blocks; the padding in between stays zero
    where = torch.zeros(total, device="cuda")
    spans = [slice(o, o + n) for o, n in zip(offs, ns)]
    for s in spans:
        where[s] = 1.0
    flat_p = (0.05 * randn(total) * where).to(dtype)
    spread = torch.exp2(2.0 * torch.randn(total // BLOCK, generator=g, device="cuda")).repeat_interleave(BLOCK)
    flat_g = (1e-3 * randn(total) * spread * where).to(dtype)
    m = 3e-4 * randn(total) * spread * where
    v = 1e-6 * (0.2 + randn(total).square()) * spread.square() * where
    state = dict(op="adamw", step=100, seed=20 + seed, max_norm=1.0 if case["clip"] else None, flat_p=flat_p, flat_g=flat_g,
                 params=[flat_p[s].view(d) for s, d in zip(spans, dims)], grads=[flat_g[s].view(d) for s, d in zip(spans, dims)])
    if case["bits"] == 8:
        bspans = [slice(o // BLOCK, o // BLOCK + blocks_of(n)) for o, n in zip(offs, ns)]
        for name, x, top, kind in (("m", m, 7, torch.float8_e4m3fn), ("v", v, 14, torch.float8_e5m2)):
            s = block_scale(x, top)
            q = torch.ldexp(x, (127 - s).repeat_interleave(BLOCK)).to(kind)
            s = s.to(torch.uint8).view(torch.float8_e8m0fnu)
            state |= {"flat_" + name: q, "flat_" + name + "_scale": s, name: [q[k].view(d) for k, d in zip(spans, dims)],
                      name + "_scale": [s[k] for k in bspans]}
    else:
        state |= dict(flat_m=m, flat_v=v, m=[m[k].view(d) for k, d in zip(spans, dims)], v=[v[k].view(d) for k, d in zip(spans, dims)])
    return state


# ----------------------------------------------------------------------------- plain forms
def block_scale(x, top):
    """The exponent byte s of each block's scale 2^(s-127): the block's largest magnitude lands in [2^top, 2^(top+1))."""
    exponent = (x.view(torch.int32) & 0x7FFFFFFF).view(-1, BLOCK).amax(1) >> 23
    return torch.where(exponent == 255, exponent, (exponent - top).clamp(min=1))


MASK = 0xFFFFFFFF


def mix(x):
    """32 bits to 32 bits, two rounds of xor-shift and multiplication (x: int64 tensor of values below 2^32)."""
    x = x ^ (x >> 16)
    x = (x * 0x0A00F875) & MASK
    x = x ^ (x >> 15)
    x = (x * 0x517B5965) & MASK
    return x ^ (x >> 16)


def random_bits(seed, step, n, device):
    def t(v):
        return torch.tensor(v, dtype=torch.int64, device=device)

    key = mix(t(step & MASK))
    key = mix(key ^ t((seed >> 32) & MASK))
    key = mix(key ^ t(seed & MASK))
    return mix(torch.arange(n, device=device) ^ key)


def to_8_bits(x, top, mantissa, bias, r, kind):
    """(codes, scale bytes): x / scale, magnitudes rounded down after `r` (16 random bits) was added below the last place."""
    s = block_scale(x, top)
    y = torch.ldexp(x.abs(), (127 - s).repeat_interleave(BLOCK))
    drop = 23 - mantissa
    normal = ((y.view(torch.int32) + (r << (drop - 16)).int()) >> drop) - ((127 - bias) << mantissa)
    low = (y * 2.0 ** (bias - 1 + mantissa) + r.float() * 2.0 ** -16).int()
    code = torch.where(y >= 2.0 ** (1 - bias), normal, low)
    if kind is torch.float8_e5m2:              # a second moment that is not zero stays above zero
        code = torch.maximum(code, (y > 0).int())
    code = code | (x.view(torch.int32) >> 31 & 0x80)
    return code.to(torch.uint8).view(kind), s.to(torch.uint8).view(torch.float8_e8m0fnu)


def values(q, s):
    return torch.ldexp(q.float(), (s.view(torch.uint8).int() - 127).repeat_interleave(BLOCK))


def plain_adamw(state):
    (b1, b2), t = BETAS, state["step"]
    g, norm = state["flat_g"].float(), None
    if state["max_norm"] is not None:
        norm = g.double().square().sum().sqrt().float()
        g = g * (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    eight = "m_scale" in state
    m = values(state["flat_m"], state["flat_m_scale"]) if eight else state["flat_m"]
    v = values(state["flat_v"], state["flat_v_scale"]) if eight else state["flat_v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    denom = v.sqrt() / (1 - b2 ** t) ** 0.5 + EPS
    p = state["flat_p"].float() * (1 - LR * DECAY) - m / denom * (LR / (1 - b1 ** t))
    state["flat_p"].copy_(p)
    if eight:
        r = random_bits(state["seed"], t, m.numel(), m.device)
        state["flat_m"], state["flat_m_scale"] = to_8_bits(m, 7, 3, 7, r & 0xFFFF, torch.float8_e4m3fn)
        state["flat_v"], state["flat_v_scale"] = to_8_bits(v, 14, 2, 15, r >> 16, torch.float8_e5m2)
    else:
        state["flat_m"], state["flat_v"] = m, v
    return norm


def plain_norm(state):
    x = state["x"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(xc.square().mean(1, keepdim=True) + state["eps"])
    xhat = xc * rstd
    z = xhat * state["weight"] + state["bias"]
    y = torch.where(z >= 0, z, z * state["slope"]).to(state["x"].dtype)
    if not state["train"]:
        return {"y": y}
    g = state["gy"].float()
    gw = (g * xhat).sum(0)
    gb = g.sum(0)
    g = g * state["weight"]
    gx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return {"y": y, "gx": gx.to(y.dtype), "gw": gw, "gb": gb}


# ----------------------------------------------------------------------------- one pass
def run(state):
    if state["op"] == "norm":
        if not own:
            return plain_norm(state)
        from liftreg_amd import ops, ops_bwd
        x, w, b = state["x"], state["weight"], state["bias"]
        if not state["train"]:
            return {"y": ops.layer_norm(x, w, b, eps=state["eps"], negative_slope=state["slope"])}
        y, stats = ops.layer_norm(x, w, b, eps=state["eps"], return_stats=True)
        gx, gw, gb = ops_bwd.layer_norm_bwd(x, w, b, state["gy"], eps=state["eps"], stats=stats)
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    state["step"] += 1
    if own:
        from liftreg_amd import optim
        norm = optim.adamw_step(state["params"], state["grads"], state["m"], state["v"], step=state["step"], lr=LR, betas=BETAS, eps=EPS,
                                weight_decay=DECAY, max_norm=state["max_norm"], exp_avg_scales=state.get("m_scale"),
                                exp_avg_sq_scales=state.get("v_scale"), seed=state["seed"])
    else:
        norm = plain_adamw(state)
    out = {k: state[k] for k in ("flat_p", "flat_m", "flat_v", "flat_m_scale", "flat_v_scale") if k in state}
    return out if norm is None else out | {"norm": norm}


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["cols"], 4 if case["dtype"] == "fp32" else 2
        if case["train"]:                       # x, gy -> y, gx; weight, bias -> their gradients
            return {"bytes": 4 * n * size + 16 * case["cols"], "flops": 22 * n}
        return {"bytes": 2 * n * size + 8 * case["cols"], "flops": 9 * n}
    n, size = sum(sizes(case)), 4 if case["dtype"] == "fp32" else 2
    state = 16 * n if case["bits"] == 32 else 4 * n + 4 * sum(blocks_of(k) for k in sizes(case))
    return {"bytes": 3 * size * n + state, "flops": (16 if case["clip"] else 13) * n + (30 * n if case["bits"] == 8 else 0)}


# ----------------------------------------------------------------------------- the definition in 64 bits
def _exact_norm(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    xhat = (x - mean) / (var + s["eps"]) ** 0.5
    del x
    z = xhat * w + b
    y = torch.maximum(z, s["slope"] * z)        # the slope is at most one
    if not s["train"]:
        return {"y": y}
    g = s["gy"].double()
    gw, gb = torch.einsum("rc,rc->c", g, xhat), g.sum(0)
    h = g * w
    gx = (h - h.mean(-1, keepdim=True) - xhat * (h * xhat).mean(-1, keepdim=True)) / (var + s["eps"]) ** 0.5
    return {"y": y, "gx": gx, "gw": gw, "gb": gb}


def _exact_hash(h):
    for shift, odd in ((16, 0x0A00F875), (15, 0x517B5965)):
        h = (h ^ (h >> np.uint32(shift))) * np.uint32(odd)
    return h ^ (h >> np.uint32(16))


def _exact_code(x, top, step, least, r):
    """x as code and scale: x / scale on a grid of 2^-step of its binade, never finer than `least`, rounded by chance."""
    peak = x.view(-1, BLOCK).abs().amax(1)
    e = torch.where(peak > 0, torch.frexp(peak).exponent - 1 - top, torch.full_like(peak, -126, dtype=torch.int32)).clamp(min=-126)
    y = torch.ldexp(x.abs(), -e.repeat_interleave(BLOCK))
    grid = torch.exp2(torch.frexp(y).exponent.double() - 1 - step).clamp(min=least)
    q = torch.floor(y / grid + r) * grid
    return q, e


def _exact_adamw(s):
    b1, b2 = BETAS
    t = s["step"] + 1
    g, out = s["flat_g"].double(), {}
    if s["max_norm"] is not None:
        out["norm"] = (g * g).sum() ** 0.5
        g = g * min(1.0, s["max_norm"] / (float(out["norm"]) + 1e-6))
    old = [s["flat_m"].double(), s["flat_v"].double()]
    if "m_scale" in s:
        old = [q * s[k].double().repeat_interleave(BLOCK) for q, k in zip(old, ("flat_m_scale", "flat_v_scale"))]
    m = b1 * old[0] + (1 - b1) * g
    v = b2 * old[1] + (1 - b2) * g ** 2
    step = LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + EPS)
    out["flat_p"] = s["flat_p"].double() * (1 - LR * DECAY) - step
    if "m_scale" not in s:
        return out | {"flat_m": m, "flat_v": v}
    with np.errstate(over="ignore"):
        k = np.zeros(1, np.uint32)
        for part in (t, s["seed"] >> 32, s["seed"]):
            k = _exact_hash(k ^ np.uint32(part & 0xFFFFFFFF))
        r = _exact_hash(np.arange(m.numel(), dtype=np.uint32) ^ k)
    r = torch.from_numpy(r.astype(np.int64)).to(m.device)
    qm, em = _exact_code(m, 7, 3, 2.0 ** -9, (r % 65536).double() / 65536)
    qv, ev = _exact_code(v, 14, 2, 2.0 ** -16, (r // 65536).double() / 65536)
    qv = torch.where((v > 0) & (qv == 0), torch.full_like(qv, 2.0 ** -16), qv)
    return out | {"flat_m": torch.copysign(qm, m), "flat_v": qv, "flat_m_scale": torch.exp2(em.double()), "flat_v_scale": torch.exp2(ev.double())}


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_norm(state) if case["op"] == "norm" else _exact_adamw(state)

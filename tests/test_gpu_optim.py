"""liftreg_amd.optim on the GPU: the AdamW step (32-bit and block-scaled 8-bit states) and the gradients' norm against the
definition in 64 bits."""
import copy

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

B1, B2 = 0.9, 0.999
U32 = 2.0 ** -24          # half a step of fp32
UBF = 2.0 ** -8           # half a step of bf16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def hash32(x):
    with np.errstate(over="ignore"):
        for shift, odd in ((16, 0x0A00F875), (15, 0x517B5965)):
            x = (x ^ (x >> np.uint32(shift))) * np.uint32(odd)
    return x ^ (x >> np.uint32(16))


def random16(seed, step, first, n):
    """The two 16-bit numbers of n elements from position `first`."""
    key = np.zeros(1, np.uint32)
    for part in (step, seed >> 32, seed):
        key = hash32(key ^ np.uint32(part & 0xFFFFFFFF))
    r = hash32(((first + np.arange(n)) % 2 ** 32).astype(np.uint32) ^ key)
    return (r & 0xFFFF).astype(np.float64) / 65536, (r >> 16).astype(np.float64) / 65536


def neighbours8(x, top, step, least, got_e):
    """Scale exponent of each block, and for each element the codes below and above |x| / scale on the format's grid.  fp32 has a
    block's peak with at most 14 half steps of error: within that of a power of two (a bf16 gradient of 1.25 2^k times 1 - b1 = 0.1
    is one) the exponent may come out as its neighbour, and the grid is then that of the exponent that came out."""
    n = x.size
    pad = np.zeros(-(-n // 32) * 32)
    pad[:n] = np.abs(x)
    peak = pad.reshape(-1, 32).max(1)
    lo, hi = (np.where(peak > 0, np.frexp(peak * (1 + k * 14 * U32))[1] - 1 - top, -126).clip(min=-126) for k in (-1, 1))
    assert ((got_e == lo) | (got_e == hi)).all()
    e = got_e
    y = (pad / np.exp2(e.repeat(32).astype(np.float64)))[:n]
    grid = np.maximum(np.exp2(np.frexp(y)[1] - 1.0 - step), least)
    low = np.floor(y / grid) * grid
    return y, low, grid


def tensors(dev, sizes, dtype, seed, misaligned=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    lead = 1 if misaligned else 0

    def one(n, scale):
        t = torch.empty(n + lead, device=dev, dtype=torch.float32)
        t.normal_(0, scale, generator=g)
        return t.to(dtype)[lead:]

    p = [one(n, 0.05) for n in sizes]
    gr = [one(n, 1e-3) for n in sizes]
    return p, gr


def states32(dev, sizes, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    m = [torch.randn(n, device=dev, generator=g) * 3e-4 for n in sizes]
    v = [torch.randn(n, device=dev, generator=g).square() * 1e-6 for n in sizes]
    return m, v


def definition(p, g, m, v, step, lr, eps, wd, max_norm=None, norm=None):
    """All float64 numpy; returns p, m, v, update."""
    if max_norm is not None:
        g = g * min(1.0, max_norm / (norm + 1e-6))
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g * g
    upd = lr / (1 - B1 ** step) * m / (np.sqrt(v) / np.sqrt(1 - B2 ** step) + eps)
    return p * (1 - lr * wd) - upd, m, v, upd


SIZES = [[1], [31, 32, 33], [7, 0, 4096, 4097], [5, 27 * 48, 3, 8191, 70001], [13] * 130, [9] * 200]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("misaligned", [False, True])
@pytest.mark.parametrize("clip", [None, 1e-2, 1e3])
def test_step_with_32_bit_states(dev, sizes, dtype, misaligned, clip):
    from liftreg_amd import optim
    p, g = tensors(dev, sizes, dtype, 1, misaligned)
    m, v = states32(dev, sizes, 2)
    before = [[t.double().cpu().numpy() for t in ts] for ts in (p, g, m, v)]
    step, lr, eps, wd = 7, 1e-3, 1e-8, 0.1
    norm = optim.adamw_step(p, g, m, v, step=step, lr=lr, eps=eps, weight_decay=wd, max_norm=clip)
    want_norm = float(np.sqrt(sum((x ** 2).sum() for x in before[1])))
    if clip is None:
        assert norm is None
    else:
        # fp64 sums of exact squares; one rounding to fp32
        assert abs(float(norm) - want_norm) <= 2 * U32 * want_norm
    for i in range(len(sizes)):
        wp, wm, wv, upd = definition(*(b[i] for b in before), step, lr, eps, wd, clip, want_norm)
        gc = before[1][i] if clip is None else before[1][i] * min(1.0, clip / (want_norm + 1e-6))
        # m: rounding of the coefficient (2 of norm and quotient), g c, the constants, two products and the sum: 8 half steps of the terms
        tol_m = 8 * U32 * (np.abs(B1 * before[2][i]) + np.abs((1 - B1) * gc))
        assert (np.abs(m[i].double().cpu().numpy() - wm) <= tol_m + 1e-45).all()
        # v: the same, the coefficient and g c twice: 14
        tol_v = 14 * U32 * wv
        assert (np.abs(v[i].double().cpu().numpy() - wv) <= tol_v + 1e-44).all()
        # update: m's and half of v's error, square root and reciprocal of 1 step (2 half steps) each, 6 more roundings; m may
        # cancel, so its error is counted in the size of its terms; then p's product, sum and final rounding
        size = lr / (1 - B1 ** step) / (np.sqrt(wv) / np.sqrt(1 - B2 ** step) + eps)
        tol = 24 * U32 * np.abs(upd) + size * tol_m + 3 * U32 * np.abs(wp) + 2 * U32 * np.abs(upd)
        if dtype == torch.bfloat16:
            tol = tol + UBF * np.abs(wp)
        assert (np.abs(p[i].double().cpu().numpy() - wp) <= tol + 1e-44).all()
        assert np.array_equal(g[i].double().cpu().numpy(), before[1][i])


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("misaligned", [False, True])
def test_step_with_8_bit_states(dev, sizes, dtype, misaligned):
    from liftreg_amd import optim
    p, g = tensors(dev, sizes, dtype, 3, misaligned)
    lead = 1 if misaligned else 0
    st = [optim.state8(torch.empty(n + lead, device=dev)) for n in sizes]
    m, v = [s[0][lead:] for s in st], [s[2][lead:] for s in st]
    ms = [torch.zeros(-(-n // 32) + lead, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)[lead:] for n in sizes]
    vs = [torch.zeros(-(-n // 32) + lead, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)[lead:] for n in sizes]
    seed = (5 << 32) + 77
    for step in (1, 2, 3):
        old = [[x.double().cpu().numpy() for x in p], [x.double().cpu().numpy() for x in g],
               [optim.values8(a, b).double().cpu().numpy() for a, b in zip(m, ms)],
               [optim.values8(a, b).double().cpu().numpy() for a, b in zip(v, vs)]]
        optim.adamw_step(p, g, m, v, step=step, lr=1e-3, weight_decay=0.1, exp_avg_scales=ms, exp_avg_sq_scales=vs, seed=seed)
        first = 0
        for i, n in enumerate(sizes):
            if not n:
                continue
            wp, wm, wv, upd = definition(*(o[i] for o in old), step, 1e-3, 1e-8, 0.1)
            rm, rv = random16(seed, step, first, n)
            first += -(-n // 32) * 32
            for q, s, want, r, top, man, least in ((m[i], ms[i], wm, rm, 7, 3, 2.0 ** -9), (v[i], vs[i], wv, rv, 14, 2, 2.0 ** -16)):
                y, low, grid = neighbours8(want, top, man, least, s.view(torch.uint8).cpu().numpy().astype(int) - 127)
                got = q.to(torch.float32).double().cpu().numpy()
                up = np.abs(got) - low
                assert ((up == 0) | (up == grid)).all() if top == 7 else ((up == 0) | (up == grid) | (np.abs(got) == least)).all()
                frac = (y - low) / grid
                # away from the border the choice is decided: fp32 forms y with at most 14 half steps, 2^-20 of y, 2^-16 of a grid step
                sure = np.abs(frac + r - 1) > 2.0 ** -15
                pick = np.where(frac + r >= 1, low + grid, low)
                if top == 14:
                    pick = np.where((want > 0) & (pick == 0), least, pick)
                assert np.array_equal(np.abs(got)[sure], pick[sure])
                assert (np.sign(got)[got != 0] == np.sign(want)[got != 0]).all()
                assert (got[want == 0] == 0).all()
            size = 1e-3 / (1 - B1 ** step) / (np.sqrt(wv) / np.sqrt(1 - B2 ** step) + 1e-8)
            tol_m = 8 * U32 * (np.abs(B1 * old[2][i]) + np.abs((1 - B1) * old[1][i]))
            tol = 26 * U32 * np.abs(upd) + size * tol_m + 3 * U32 * np.abs(wp) + (UBF * np.abs(wp) if dtype == torch.bfloat16 else 0)
            assert (np.abs(p[i].double().cpu().numpy() - wp) <= tol + 1e-44).all()


def test_8_bit_states_keep_their_expectation(dev):
    """With a constant gradient v converges to its square although a step is far below half a code step; deviations are those of
    the code's spacing (25 % below the value, variance <= 1/4 step^2), averaged over 64 K elements."""
    from liftreg_amd import optim
    n = 1 << 16
    p, g = torch.zeros(n, device=dev), torch.full((n,), 1e-2, device=dev)
    m, ms, v, vs = optim.state8(p)
    for t in range(1, 401):
        optim.adamw_step([p], [g], [m], [v], step=t, lr=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], seed=9)
    mean_v = float(optim.values8(v, vs).double().mean())
    mean_m = float(optim.values8(m, ms).double().mean())
    assert abs(mean_v / (1e-4 * (1 - B2 ** 400)) - 1) < 0.05
    assert abs(mean_m / (1e-2 * (1 - B1 ** 400)) - 1) < 0.01


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_values_that_are_not_finite(dev, bad):
    from liftreg_amd import optim
    for bits in (32, 8):
        p, g = tensors(dev, [100], torch.float32, 4)
        g[0][40] = bad
        st = optim.state8(p[0])
        m, v = ([torch.zeros(100, device=dev)], [torch.zeros(100, device=dev)]) if bits == 32 else ([st[0]], [st[2]])
        more = {} if bits == 32 else dict(exp_avg_scales=[st[1]], exp_avg_sq_scales=[st[3]])
        optim.adamw_step(p, g, m, v, step=1, **more)
        assert not torch.isfinite(p[0][40]) and torch.isfinite(p[0][:40]).all() and torch.isfinite(p[0][41:]).all()
        if bits == 8:
            value = optim.values8(m[0], st[1])
            assert torch.isnan(value[32:64]).all() and torch.isfinite(value[:32]).all() and torch.isfinite(value[64:]).all()
            assert torch.isnan(optim.values8(v[0], st[3])[32:64]).all()
    # a norm that is not finite reaches every parameter (inf: 0 * inf at the element, 0 elsewhere; NaN: everywhere)
    p, g = tensors(dev, [100], torch.float32, 4)
    g[0][40] = bad
    norm = optim.adamw_step(p, g, [torch.zeros(100, device=dev)], [torch.zeros(100, device=dev)], step=1, max_norm=1.0)
    assert not torch.isfinite(norm) and torch.isnan(p[0][40])


def test_nothing_outside_the_tensors_is_written(dev):
    from liftreg_amd import optim
    for n in (1, 3, 31, 33, 4095, 4099):
        base = [torch.full((n + 64,), 5.0, device=dev) for _ in range(4)]
        p, g, m, v = (t[32:32 + n] for t in base)
        optim.adamw_step([p], [g], [m], [v], step=1)
        for t in base:
            assert (t[:32] == 5).all() and (t[32 + n:] == 5).all()
        bytes8 = [torch.full((k + 64,), 0x35, dtype=torch.uint8, device=dev) for k in (n, n, -(-n // 32), -(-n // 32))]
        kinds = (torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu, torch.float8_e8m0fnu)
        mq, vq, ms, vs = (t.view(k)[32:t.numel() - 32] for t, k in zip(bytes8, kinds))
        optim.adamw_step([p], [g], [mq], [vq], step=1, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
        for t in bytes8:
            assert (t[:32] == 0x35).all() and (t[-32:] == 0x35).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_norm(dev, dtype):
    from liftreg_amd import optim
    for sizes in SIZES + [[3_000_001]]:
        _, g = tensors(dev, sizes, dtype, 6, misaligned=True)
        want = float(torch.sqrt(sum((t.double() ** 2).sum() for t in g)))
        got = optim.grad_norm(g)
        assert got.dtype == torch.float32 and got.dim() == 0
        assert abs(float(got) - want) <= 2 * U32 * want
        assert torch.equal(got, optim.grad_norm(g))
    assert float(optim.grad_norm([torch.empty(0, device=dev)])) == 0.0
    p = torch.empty(0, device=dev)
    assert float(optim.adamw_step([p], [p.clone()], [p.clone()], [p.clone()], step=1, max_norm=1.0)) == 0.0
    # squares that leave fp32's range
    big = [torch.full((1000,), 1e30, device=dev), torch.full((1000,), 1e-30, device=dev)]
    assert abs(float(optim.grad_norm(big)) / (1e30 * 1000 ** 0.5) - 1) < 1e-6


def test_device_side_step_and_learning_rate_in_a_graph(dev):
    """A captured step follows the step count and the learning rate on the device; two graphs and eager calls in between."""
    from liftreg_amd import optim
    sizes = [33, 5000]
    for bits in (32, 8):
        p, g = tensors(dev, sizes, torch.float32, 8)
        q = [t.clone() for t in p]

        def fresh():
            if bits == 32:
                m, v = [torch.zeros(n, device=dev) for n in sizes], [torch.zeros(n, device=dev) for n in sizes]
                return m, v, {}
            st = [optim.state8(t) for t in p]
            return [s[0] for s in st], [s[2] for s in st], dict(exp_avg_scales=[s[1] for s in st], exp_avg_sq_scales=[s[3] for s in st])

        (m, v, more), (m2, v2, more2) = fresh(), fresh()
        t, lr = torch.zeros((), dtype=torch.int64, device=dev), torch.tensor(1e-3, device=dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs = []
        for clip in (1e-2, None):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                t.add_(1)
                norm = optim.adamw_step(p, g, m, v, step=t, lr=lr, max_norm=clip, seed=3, **more)
            graphs.append((graph, clip, norm))
        torch.cuda.synchronize()
        for k in range(1, 7):
            lr.fill_(1e-3 / k)
            graph, clip, norm = graphs[k % 2]
            for x in g:
                x.normal_(0, 1e-3 * k)
            graph.replay()
            want = optim.adamw_step(q, g, m2, v2, step=k, lr=float(lr), max_norm=clip, seed=3, **more2)
            torch.cuda.synchronize()
            if clip is not None:
                assert torch.equal(norm, want)
            assert all(torch.equal(a, b) for a, b in zip(p, q)), (bits, k)
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(m + v, m2 + v2))


def test_streams(dev):
    from liftreg_amd import optim
    p, g = tensors(dev, [100_003], torch.float32, 10)
    m, v = states32(dev, [100_003], 11)
    a = [t.clone() for t in (p[0], m[0], v[0])]
    optim.adamw_step([a[0]], g, [a[1]], [a[2]], step=1, max_norm=1e-3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        optim.adamw_step(p, g, m, v, step=1, max_norm=1e-3)
    s.synchronize()
    assert torch.equal(a[0], p[0]) and torch.equal(a[1], m[0]) and torch.equal(a[2], v[0])


def test_lists_from_generators(dev):
    """What a generator yields lives until the launches: the workspace of the norm does not take its memory."""
    from liftreg_amd import optim
    sizes = [100] * 100
    p, g = tensors(dev, sizes, torch.float32, 14)
    m, v = states32(dev, sizes, 15)
    a = [[t.clone() for t in ts] for ts in (p, m, v)]
    want = optim.adamw_step(a[0], [t * 3 for t in g], a[1], a[2], step=1, max_norm=1e-3)
    got = optim.adamw_step(iter(p), (t * 3 for t in g), iter(m), tuple(v), step=1, max_norm=1e-3)
    assert torch.equal(got, want) and torch.equal(optim.grad_norm(t * 3 for t in g), want)
    assert all(torch.equal(x, y) for x, y in zip(a[0] + a[1] + a[2], p + m + v))


def test_refusals(dev):
    from liftreg_amd import _hip, optim
    p, g = tensors(dev, [64, 10], torch.float32, 12)
    m, v = states32(dev, [64, 10], 13)
    ok = dict(step=1)
    with pytest.raises(ValueError):
        optim.adamw_step([], [], [], [], **ok)
    with pytest.raises(_hip.LiftRegHipError):
        optim.adamw_step([t.cpu() for t in p], g, m, v, **ok)
    with pytest.raises(_hip.LiftRegHipError):
        optim.adamw_step(p, [g[0].cpu(), g[1]], m, v, **ok)
    with pytest.raises(TypeError):
        optim.adamw_step(p, [t.bfloat16() for t in g], m, v, **ok)
    with pytest.raises(TypeError):
        optim.adamw_step([t.double() for t in p], g, m, v, **ok)
    with pytest.raises(TypeError):
        optim.adamw_step([t.bfloat16() for t in p], [t.bfloat16() for t in g], [t.bfloat16() for t in m], v, **ok)
    with pytest.raises(ValueError):
        optim.adamw_step(p, g[:1], m, v, **ok)
    with pytest.raises(ValueError):
        optim.adamw_step(p, g, [m[0], m[0]], v, **ok)
    with pytest.raises(ValueError):
        optim.adamw_step([p[0], p[0]], [g[0], g[0]], [m[0], m[0].clone()], [v[0], v[0].clone()], **ok)
    with pytest.raises(ValueError):
        optim.adamw_step([torch.zeros(8, 8, device=dev).t(), p[1]], g, m, v, **ok)
    flat = torch.zeros(100, device=dev)
    with pytest.raises(ValueError):      # overlapping views
        optim.adamw_step([flat[:64], flat[60:70]], g, m, v, **ok)
    with pytest.raises(ValueError):      # one element for all of them
        optim.adamw_step([torch.zeros(1, device=dev).expand(64), p[1]], g, m, v, **ok)
    for more in (dict(step=0), dict(step=1, lr=-1.0), dict(step=1, betas=(1.0, 0.9)), dict(step=1, eps=-1e-8), dict(step=1, weight_decay=-1.0),
                 dict(step=1, max_norm=0.0), dict(step=1, grad_norm=torch.ones((), device=dev)),
                 dict(step=torch.ones((), device=dev)), dict(step=1, lr=torch.ones((), device=dev, dtype=torch.float64)),
                 dict(step=1, exp_avg_scales=[torch.zeros(2, device=dev)] * 2)):
        with pytest.raises(ValueError):
            optim.adamw_step(p, g, m, v, **more)
    with pytest.raises(TypeError):
        optim.adamw_step(p, g, m, v, step=1, max_norm=1.0, grad_norm=1.0)
    st = [optim.state8(t) for t in p]
    with pytest.raises(ValueError):      # one scale short
        optim.adamw_step(p, g, [s[0] for s in st], [s[2] for s in st], step=1, exp_avg_scales=[s[1][:1] for s in st],
                         exp_avg_sq_scales=[s[3] for s in st])
    with pytest.raises(TypeError):
        optim.adamw_step(p, g, m, v, step=1, exp_avg_scales=[s[1] for s in st], exp_avg_sq_scales=[s[3] for s in st])


# ------------------------------------------------------------------------------------------------ the optimizer class
class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.a = torch.nn.Linear(37, 65)
        self.b = torch.nn.Linear(65, 3)

    def forward(self, x):
        return self.b(torch.tanh(self.a(x)))


def train(net, opt, steps, seed=0, sched=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for _ in range(steps):
        x = torch.randn(16, 37, device="cuda", generator=g)
        opt.zero_grad()
        net(x).square().mean().backward()
        opt.step()
        if sched:
            sched.step()


def test_class_follows_torch(dev):
    """Ten steps with a schedule next to torch.optim.AdamW.  Both round p once a step and the update in a few fp32 operations:
    p differs by at most 2 half steps a step plus 64 of the update, whose sum is at most 10 lr; nothing amplifies it but the
    gradients, which change by as much relative to weights of about 0.1: a factor of 10 is left for that."""
    from liftreg_amd import optim
    torch.manual_seed(1)
    ref = Net().to(dev)
    net = copy.deepcopy(ref)
    kw = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-5, weight_decay=0.05)
    a, b = torch.optim.AdamW(ref.parameters(), **kw), optim.AdamW(net.parameters(), **kw)
    train(ref, a, 10, sched=torch.optim.lr_scheduler.StepLR(a, 3, 0.5))
    train(net, b, 10, sched=torch.optim.lr_scheduler.StepLR(b, 3, 0.5))
    for x, y in zip(ref.parameters(), net.parameters()):
        assert float((x - y).detach().abs().max()) <= 10 * (20 * U32 * float(x.detach().abs().max()) + 64 * U32 * 10 * 1e-3)
        assert y._version > 0
    # torch's checkpoint continues here
    c = optim.AdamW(net.parameters(), **kw)
    c.load_state_dict(a.state_dict())
    assert all(c.state[p]["step"] == 10 and c.state[p]["exp_avg"].dtype == torch.float32 for p in net.parameters())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpoints_continue_bit_for_bit(dev, bits, capturable, dtype, tmp_path):
    from liftreg_amd import optim
    torch.manual_seed(2)
    net = Net().to(dev)
    kw = dict(lr=1e-2, state_bits=bits, max_grad_norm=0.1, seed=4, capturable=capturable)

    def make(net):
        return optim.AdamW([{"params": net.a.parameters()}, {"params": net.b.parameters(), "lr": 1e-3}], **kw)

    def steps(net, opt, n, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for _ in range(n):
            for p in net.parameters():
                p.grad = torch.randn(p.shape, device="cuda", generator=g).to(p.dtype)
            opt.step()

    net = net.to(dtype)
    opt = make(net)
    steps(net, opt, 3, 0)
    assert opt.grad_norm is not None and float(opt.grad_norm) > 1
    torch.save({"net": net.state_dict(), "opt": opt.state_dict()}, tmp_path / "c.pt")
    steps(net, opt, 3, 1)
    other = Net().to(dev).to(dtype)
    again = make(other)
    saved = torch.load(tmp_path / "c.pt", weights_only=True)
    other.load_state_dict(saved["net"])
    again.load_state_dict(saved["opt"])
    if capturable:
        assert len({id(again.state[p]["step"]) for p in other.parameters()}) == 1
    steps(other, again, 3, 1)
    for x, y in zip(net.parameters(), other.parameters()):
        assert torch.equal(x, y)
        for k in opt.state[x]:
            s, t = opt.state[x][k], again.state[y][k]
            assert (s == t) if not isinstance(s, torch.Tensor) else torch.equal(s.reshape(-1).view(torch.uint8), t.reshape(-1).view(torch.uint8))
    wrong = optim.AdamW(other.parameters(), state_bits=40 - bits)
    with pytest.raises(ValueError):
        wrong.load_state_dict(saved["opt"])


def test_class_steps_only_what_has_a_gradient(dev):
    from liftreg_amd import optim
    net = Net().to(dev)
    net.b.requires_grad_(False)
    opt = optim.AdamW(net.parameters(), max_grad_norm=1.0)
    keep = [p.clone() for p in net.b.parameters()]
    train(net, opt, 2)
    assert all(torch.equal(a, b) for a, b in zip(keep, net.b.parameters())) and len(opt.state) == 2
    # a parameter that joins later has its own count
    net.b.requires_grad_(True)
    train(net, opt, 1)
    assert opt.state[net.a.weight]["step"] == 3 and opt.state[net.b.weight]["step"] == 1
    opt.zero_grad()
    before = [p.clone() for p in net.parameters()]
    opt.step()
    assert opt.grad_norm is None and all(torch.equal(a, b) for a, b in zip(before, net.parameters()))


@pytest.mark.parametrize("bits", [32, 8])
def test_device_counts_of_parameters_without_gradients(dev, bits):
    """Parameters that share a count on the device keep their own when only some of them have gradients."""
    from liftreg_amd import _hip, optim
    torch.manual_seed(9)
    net = Net().to(dev)
    twin = copy.deepcopy(net)
    opts = [optim.AdamW(n.parameters(), lr=1e-2, max_grad_norm=0.5, state_bits=bits, capturable=c) for n, c in ((net, True), (twin, False))]
    for k, absent in enumerate(((), ("a.bias",), (), ("a.weight", "a.bias"), ("a.bias",), ())):
        g = torch.Generator(device="cuda").manual_seed(k)
        for (name, p), q in zip(net.named_parameters(), twin.parameters()):
            p.grad = None if name in absent else torch.randn(p.shape, device=dev, generator=g)
            q.grad = p.grad
        for o in opts:
            o.step()
        for (name, p), q in zip(net.named_parameters(), twin.parameters()):
            assert torch.equal(p, q), (k, name)
            assert int(opts[0].state[p]["step"]) == opts[1].state[q]["step"]
    # within a capture a shared count cannot be parted
    net2 = Net().to(dev)
    opt = optim.AdamW(net2.parameters(), capturable=True, state_bits=bits)
    for p in net2.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    net2.b.bias.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(_hip.LiftRegHipError):
            opt.step()
        torch.zeros(1, device=dev)


def test_a_failed_step_is_not_counted(dev):
    from liftreg_amd import optim
    net = Net().to(dev)
    opt = optim.AdamW(net.parameters())
    train(net, opt, 1)
    opt.param_groups[0]["eps"] = -1.0
    with pytest.raises(ValueError):
        train(net, opt, 1)
    assert all(s["step"] == 1 for s in opt.state.values())


def test_captured_class_step(dev):
    from liftreg_amd import optim
    torch.manual_seed(3)
    net = Net().to(dev)
    twin = copy.deepcopy(net)
    for n in (net, twin):
        for p in n.parameters():
            p.grad = torch.zeros_like(p)
    lr = torch.tensor(1e-2, device=dev)
    opt = optim.AdamW(net.parameters(), lr=lr, capturable=True, max_grad_norm=0.5)
    ref = optim.AdamW(twin.parameters(), lr=1e-2, max_grad_norm=0.5)

    def grads(k):
        g = torch.Generator(device="cuda").manual_seed(k)
        for p, q in zip(net.parameters(), twin.parameters()):
            p.grad.normal_(generator=g)
            q.grad.copy_(p.grad)

    grads(0)
    opt.step(), ref.step()                 # states exist before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(1, 5):
        grads(k)
        lr.fill_(1e-2 / k)
        ref.param_groups[0]["lr"] = float(lr)
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(net.parameters(), twin.parameters())), k
    assert int(opt.state[net.a.weight]["step"]) == 5


def test_captures_that_could_not_be_replayed_are_refused(dev):
    from liftreg_amd import _hip, optim
    for kw, warm in ((dict(), True), (dict(capturable=True), False)):
        net = Net().to(dev)
        for p in net.parameters():
            p.grad = torch.ones_like(p)
        opt = optim.AdamW(net.parameters(), **kw)
        if warm:
            opt.step()
        before = [p.clone() for p in net.parameters()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(_hip.LiftRegHipError):
                opt.step()
            torch.zeros(1, device=dev)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(before, net.parameters()))
    with pytest.raises(ValueError):
        optim.AdamW(net.parameters(), lr=torch.tensor(1e-3, device=dev))


def test_gradients_in_flat_buckets(dev):
    """parallel.GradientAllReduce's views (any 4-byte address) as gradients: the bits of separate tensors."""
    from liftreg_amd import optim
    from liftreg_amd.parallel import GradientAllReduce
    torch.manual_seed(6)
    net = Net().to(dev)
    twin = copy.deepcopy(net)
    ddp = GradientAllReduce(net, head_prefix="b.")
    a, b = optim.AdamW(net.parameters(), max_grad_norm=0.1), optim.AdamW(twin.parameters(), max_grad_norm=0.1)
    for k in range(3):
        x = torch.randn(16, 37, device=dev)
        ddp.zero_grad()
        net(x).square().mean().backward()
        ddp.finish()
        b.zero_grad()
        twin(x).square().mean().backward()
        a.step(), b.step()
        assert all(torch.equal(p, q) for p, q in zip(net.parameters(), twin.parameters())), k


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_copied_optimizer_takes_the_same_steps(dev, bits, capturable):
    from liftreg_amd import optim
    torch.manual_seed(4)
    net = Net().to(dev)
    opt = optim.AdamW(net.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=0.1, seed=5, capturable=capturable)
    train(net, opt, 3)
    other, again = copy.deepcopy((net, opt))
    train(net, opt, 2, seed=1)
    train(other, again, 2, seed=1)
    assert torch.equal(opt.grad_norm, again.grad_norm)
    for p, q in zip(net.parameters(), other.parameters()):
        assert torch.equal(p, q) and int(opt.state[p]["step"]) == int(again.state[q]["step"]) == 5
        for k in set(opt.state[p]) - {"step"}:
            assert torch.equal(opt.state[p][k].view(torch.uint8), again.state[q][k].view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("groups", [1, 2])
def test_a_failed_step_with_device_counts_is_not_counted(dev, bits, groups):
    from liftreg_amd import optim
    net = Net().to(dev)
    ps = [{"params": net.a.parameters()}, {"params": net.b.parameters()}] if groups == 2 else net.parameters()
    opt = optim.AdamW(ps, capturable=True, state_bits=bits)
    train(net, opt, 2)
    opt.param_groups[-1]["eps"] = -1.0
    for _ in range(2):
        with pytest.raises(ValueError):
            train(net, opt, 1)
    assert all(int(s["step"]) == 2 for s in opt.state.values())
    opt.param_groups[-1]["eps"] = 1e-8
    train(net, opt, 1)
    assert all(int(s["step"]) == 3 for s in opt.state.values())


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("clip", [None, 0.1])
def test_a_refused_group_leaves_the_others_where_they_are(dev, capturable, clip):
    """A step that is refused for one group or type writes nothing."""
    from liftreg_amd import optim
    net = Net().to(dev)
    net.b.to(torch.bfloat16)
    opt = optim.AdamW([{"params": [net.a.weight, net.b.weight]}, {"params": [net.a.bias, net.b.bias]}], capturable=capturable, max_grad_norm=clip)

    def step(k):
        g = torch.Generator(device="cuda").manual_seed(k)
        for p in net.parameters():
            p.grad = torch.randn(p.shape, device=dev, generator=g).to(p.dtype)
        opt.step()

    step(0)
    before = [(p.detach().clone(), {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state[p].items()}) for p in net.parameters()]
    opt.param_groups[1]["weight_decay"] = -1.0
    with pytest.raises(ValueError):
        step(1)
    for p, (old, state) in zip(net.parameters(), before):
        assert torch.equal(p, old)
        assert all(torch.equal(v, state[k]) if isinstance(v, torch.Tensor) else v == state[k] for k, v in opt.state[p].items())
    opt.param_groups[1]["weight_decay"] = 0.0
    step(1)
    assert all(not torch.equal(p, old) and int(opt.state[p]["step"]) == 2 for p, (old, _) in zip(net.parameters(), before))


def test_types_of_a_group_round_with_different_bits(dev):
    """A group with parameters of two types or two step counts is stepped in several calls, each with random bits of its own."""
    from liftreg_amd import optim
    n = 4096
    start = torch.randn(n, device=dev).bfloat16()
    ps = [torch.nn.Parameter(start.to(t)) for t in (torch.float32, torch.bfloat16)]
    opt = optim.AdamW(ps, state_bits=8, seed=11)
    g = (torch.randn(n, device=dev) * 1e-2).bfloat16()
    for p in ps:
        p.grad = g.to(p.dtype)
    opt.step()
    a, b = (opt.state[p] for p in ps)
    # the same moments, the same scales, rounded apart: of 4096 codes with a remainder hundreds differ
    assert torch.equal(a["exp_avg_scale"].view(torch.uint8), b["exp_avg_scale"].view(torch.uint8))
    for k in ("exp_avg", "exp_avg_sq"):
        assert int((a[k].view(torch.uint8) != b[k].view(torch.uint8)).sum()) > 100
    # the first call's bits are those of the seed as it is given
    m, ms, v, vs = optim.state8(ps[0])
    optim.adamw_step([ps[0].detach().clone()], [ps[0].grad], [m], [v], step=1, exp_avg_scales=[ms], exp_avg_sq_scales=[vs], seed=11)
    assert torch.equal(a["exp_avg"].view(torch.uint8), m.view(torch.uint8)) and torch.equal(a["exp_avg_sq"].view(torch.uint8), v.view(torch.uint8))


@pytest.mark.parametrize("bits", [32, 8])
def test_subnormal_second_moments_without_eps(dev, bits):
    """Gradients of 2^-50 ... 2^-69: v goes through fp32's subnormal numbers and its root does not.  The update of the first step is lr times the
    gradient's sign within what rounding v to fp32 changes; from that v (rounded as fp32 holds it) the kernel is off by the 26 half steps of
    test_step_with_32_bit_states."""
    from liftreg_amd import optim
    e = torch.arange(-50, -70, -1, device=dev, dtype=torch.float64)
    g = (torch.exp2(e)[:, None] * torch.tensor([1.0, -1.25, 1.5, 1.75], device=dev)).reshape(-1).float()
    lr, n = 1e-3, g.numel()
    p = torch.zeros(n, device=dev)
    if bits == 32:
        m, v, more = torch.zeros(n, device=dev), torch.zeros(n, device=dev), {}
        optim.adamw_step([p], [g], [m], [v], step=1, lr=lr, eps=0.0, weight_decay=0.0)
        m, v = m.double(), v.double()
    else:
        mq, ms, vq, vs = optim.state8(p)
        optim.adamw_step([p], [g], [mq], [vq], step=1, lr=lr, eps=0.0, weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
        m, v = (1 - B1) * g.double(), ((1 - B2) * g.double() ** 2).float().double()
    assert bool((v > 0).all()) and float(v.min()) < 2.0 ** -140
    want = -lr / (1 - B1) * m / (v.sqrt() / (1 - B2) ** 0.5)
    assert float(((p.double() - want) / want).abs().max()) <= 26 * U32
    assert torch.equal(torch.sign(p), -torch.sign(g))


# above 2048 x 1024 elements a launch takes chunks of 4096, above 2048 x 4096 a workgroup takes several of them
LARGE = [[3, 1_000_003, 5000, 4097, 970_001, 1, 200_000], [5_000_001, 33, 3_400_003, 12_289, 7]]


@pytest.mark.parametrize("sizes", LARGE, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_large_steps_with_32_bit_states(dev, sizes, dtype, clip):
    assert 2048 * 1024 < sum(sizes) < 2048 * 4096 or sum(sizes) > 2048 * 4096
    test_step_with_32_bit_states(dev, sizes, dtype, True, clip)


def step_with_8_bit_states(dev, sizes, dtype, steps, clip):
    """test_step_with_8_bit_states with clipping, a step at a time (the moments of a step are formed from the codes that the last one left)."""
    from liftreg_amd import optim
    p, g = tensors(dev, sizes, dtype, 17)
    st = [optim.state8(t) for t in p]
    (m, ms, v, vs), seed = map(list, zip(*st)), (3 << 32) + 12345
    host = lambda ts: [t.double().cpu().numpy() for t in ts]
    grads = host(g)
    want_norm = float(np.sqrt(sum((x ** 2).sum() for x in grads)))
    for step in range(1, steps + 1):
        old = [host(p), grads, host([optim.values8(a, b) for a, b in zip(m, ms)]), host([optim.values8(a, b) for a, b in zip(v, vs)])]
        norm = optim.adamw_step(p, g, m, v, step=step, lr=1e-3, weight_decay=0.1, max_norm=clip, exp_avg_scales=ms, exp_avg_sq_scales=vs, seed=seed)
        assert (norm is None) == (clip is None) and (clip is None or abs(float(norm) - want_norm) <= 2 * U32 * want_norm)
        coef = 1.0 if clip is None else min(1.0, clip / (want_norm + 1e-6))
        assert clip is None or coef < 0.5
        first = 0
        for i, n in enumerate(sizes):
            wp, wm, wv, upd = definition(*(o[i] for o in old), step, 1e-3, 1e-8, 0.1, clip, want_norm)
            rm, rv = random16(seed, step, first, n)
            first += -(-n // 32) * 32
            for q, s, want, r, top, man, least in ((m[i], ms[i], wm, rm, 7, 3, 2.0 ** -9), (v[i], vs[i], wv, rv, 14, 2, 2.0 ** -16)):
                y, low, grid = neighbours8(want, top, man, least, s.view(torch.uint8).cpu().numpy().astype(int) - 127)
                got = q.to(torch.float32).double().cpu().numpy()
                frac = (y - low) / grid
                # moments in fp64: what is off is the coefficient, by a few 2^-53 of terms no larger than 2^17 grid steps
                sure = np.abs(frac + r - 1) > 2.0 ** -30
                assert sure.mean() > 0.99 or n < 100
                pick = np.where(frac + r >= 1, low + grid, low)
                if top == 14:
                    pick = np.where((want > 0) & (pick == 0), least, pick)
                assert np.array_equal(np.abs(got)[sure], pick[sure])
                assert (np.sign(got)[got != 0] == np.sign(want)[got != 0]).all()
            size = 1e-3 / (1 - B1 ** step) / (np.sqrt(wv) / np.sqrt(1 - B2 ** step) + 1e-8)
            tol_m = 8 * U32 * (np.abs(B1 * old[2][i]) + np.abs((1 - B1) * coef * grads[i]))
            tol = 26 * U32 * np.abs(upd) + size * tol_m + 3 * U32 * np.abs(wp) + (UBF * np.abs(wp) if dtype == torch.bfloat16 else 0)
            assert (np.abs(p[i].double().cpu().numpy() - wp) <= tol + 1e-44).all()


@pytest.mark.parametrize("sizes", LARGE, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_large_steps_with_8_bit_states(dev, sizes, dtype, clip):
    step_with_8_bit_states(dev, sizes, dtype, 1, clip)


@pytest.mark.parametrize("sizes", [[31, 32, 33], [7, 4096, 4097], [5, 27 * 48, 3, 8191, 70001], [13] * 130], ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clipped_steps_with_8_bit_states(dev, sizes, dtype):
    step_with_8_bit_states(dev, sizes, dtype, 3, 1e-3)

"""Layer norm on the GPU, forward and backward, against the definition in 64 bits and against differences; the blocks and the model
that use it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U32, UBF = 2.0 ** -24, 2.0 ** -8        # half a step, relative to the value


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def definition(x, w, b, eps, slope, gy=None):
    x = x.double()
    C = x.shape[-1]
    one = torch.ones(C, dtype=torch.float64, device=x.device)
    w, b = (one if w is None else w.double()), (0 * one if b is None else b.double())
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    z = xh * w + b
    y = torch.where(z >= 0, z, slope * z)
    out = {"y": y, "z": z, "xh": xh, "mean": mean, "rstd": rstd}
    if gy is not None:
        g = torch.where(z >= 0, gy.double(), slope * gy.double())
        h = g * w
        rows = tuple(range(x.dim() - 1))
        out |= {"g": g, "h": h, "gx": rstd * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True)),
                "gw": (g * xh).sum(rows), "gb": g.sum(rows)}
    return out


def sum_steps(n):
    """Half steps of a sum of n terms in fp32, in the size of the terms' absolute sum: a lane adds up to 64 in a row, joins of 2^k."""
    return 64 + 2 * max(1, n).bit_length()


def limits(x, d, w, eps):
    """Errors of mean (in x's units), rstd (relative) and xhat (absolute) that fp32 can cause, row by row."""
    C = x.shape[-1]
    k = min(C, sum_steps(C))
    ax = x.double().abs().mean(-1, keepdim=True)
    dm = (k + 2) * U32 * ax                                   # sum, times 1/C
    # var: each difference carries dm and a rounding (dm^2 enters the mean square, the linear term sums to nothing but rounding)
    xc = (x.double() - d["mean"]).abs()
    var = (xc ** 2).mean(-1, keepdim=True)
    dvar = (k + 6) * U32 * var + 4 * dm ** 2 + 4 * dm * U32 * ax
    dr = 0.5 * dvar * d["rstd"] ** 2 + 3 * U32
    dxh = (dm + 2 * U32 * (x.double().abs() + d["mean"].abs())) * d["rstd"] + d["xh"].abs() * (dr + 3 * U32)
    return dm, dr, dxh


def near(got, want, tol, what, dtype=torch.float32):
    err = (got.double() - want).abs()
    tol = tol + (UBF if dtype == torch.bfloat16 else U32) * want.abs() + 1e-44
    assert got.dtype == dtype and bool((err <= tol).all()), f"{what}: off by up to {float((err / tol).max())} of the bound"


def data(dev, rows, cols, dtype, seed, offset=0.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(rows, cols, device=dev, generator=g) * 1.3 + offset).to(dtype)
    w = 1 + 0.2 * torch.randn(cols, device=dev, generator=g)
    b = 0.2 * torch.randn(cols, device=dev, generator=g)
    gy = torch.randn(rows, cols, device=dev, generator=g).to(dtype)
    return x, w, b, gy


def check(dev, x, w, b, gy, eps, slope):
    from liftreg_amd import ops, ops_bwd
    dtype = x.dtype
    y, stats = ops.layer_norm(x, w, b, eps=eps, negative_slope=slope, return_stats=True)
    assert torch.equal(y, ops.layer_norm(x, w, b, eps=eps, negative_slope=slope))
    d = definition(x, w, b, eps, slope)
    dm, dr, dxh = limits(x, d, w, eps)
    aw = 1.0 if w is None else w.double().abs()
    dz = dxh * aw + 3 * U32 * (d["xh"].abs() * aw + d["z"].abs())
    near(y, d["y"], dz * max(1.0, abs(slope)), "y", dtype)
    if stats is not None:
        assert stats.shape == (x.numel() // x.shape[-1], 2)
        near(stats[:, 0], d["mean"].reshape(-1), dm.reshape(-1), "mean")
        near(stats[:, 1], d["rstd"].reshape(-1), (dr * d["rstd"]).reshape(-1), "rstd")
    # a gradient whose sign of z is within the error could go either way: none is sent there
    gy = torch.where(d["z"].abs() <= 2 * dz, torch.zeros_like(gy), gy)
    d = definition(x, w, b, eps, slope, gy)
    C, rows = x.shape[-1], x.numel() // x.shape[-1]
    gx, gw, gb = ops_bwd.layer_norm_bwd(x, w, b, gy, eps=eps, negative_slope=slope, stats=stats)
    k, kr = min(C, sum_steps(C)), min(rows, 64 + sum_steps(rows))
    h = d["h"].abs()
    dh = 2 * U32 * h
    m1, m2 = h.mean(-1, keepdim=True), (h * d["xh"].abs()).mean(-1, keepdim=True)
    e1 = (k + 4) * U32 * m1
    e2 = (k + 6) * U32 * m2 + (h * dxh).mean(-1, keepdim=True)
    inner = h + m1 + d["xh"].abs() * m2
    tol = d["rstd"] * (dh + e1 + d["xh"].abs() * e2 + dxh * m2 + 4 * U32 * inner) + dr * d["gx"].abs()
    near(gx, d["gx"], tol, "gx", dtype)
    over = tuple(range(x.dim() - 1))
    if w is not None:
        near(gw, d["gw"], (d["g"].abs() * dxh).sum(over) + (kr + 4) * U32 * (d["g"] * d["xh"]).abs().sum(over), "gw")
    else:
        assert gw is None
    if b is not None:
        near(gb, d["gb"], (kr + 2) * U32 * d["g"].abs().sum(over), "gb")
    else:
        assert gb is None
    if stats is not None:      # statistics recomputed: the forward's bits
        again = ops_bwd.layer_norm_bwd(x, w, b, gy, eps=eps, negative_slope=slope)
        assert torch.equal(again[0], gx)
    more = ops_bwd.layer_norm_bwd(x, w, b, gy, eps=eps, negative_slope=slope, stats=stats)
    assert torch.equal(more[0], gx) and (gw is None or torch.equal(more[1], gw)) and (gb is None or torch.equal(more[2], gb))


COLS = [1, 2, 3, 5, 8, 16, 17, 31, 32, 33, 64, 100, 128, 200, 256, 257, 500, 512, 513, 800, 1024, 1025, 2000, 2048, 2049, 4000, 4097, 8191,
        8192, 8193, 12000, 16384, 16385, 50001]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths(dev, cols, dtype):
    # one column: gx cancels to rounding of the terms, which the bound counts
    for rows in (1, 2, 37):
        check(dev, *data(dev, rows, cols, dtype, cols + rows), 1e-5, 0.2 if rows == 37 else 1.0)


@pytest.mark.parametrize("rows,cols", [(100_003, 16), (70_001, 32), (40_000, 5), (9_000, 257), (5_000, 800), (1_500, 4096), (700, 9000),
                                       (300, 16384), (130, 20_001), (2, 300_001), (70_000, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(dev, rows, cols, dtype):
    check(dev, *data(dev, rows, cols, dtype, rows), 1e-5, 0.2)


def test_more_long_rows_than_a_grid_has(dev):
    """Above 32768 rows longer than registers hold the launches are cut."""
    check(dev, *data(dev, 32770, 16_400, torch.bfloat16, 5), 1e-5, 1.0)


@pytest.mark.parametrize("rows,cols", [(300_000, 3), (200_000, 13), (30_000, 127), (2_500, 803), (9_000, 803), (6_000, 1503), (400, 4003), (2_100, 4003),
                                       (1_100, 8191), (600, 16_001), (60, 270_001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("slope", [1.0, 0.2])
def test_many_rows_that_end_inside_a_vector(dev, rows, cols, dtype, slope):
    check(dev, *data(dev, rows, cols, dtype, rows), 1e-5, slope)


@pytest.mark.parametrize("cols", [16, 33, 800, 4097, 20_000])
def test_without_weight_or_bias(dev, cols):
    x, w, b, gy = data(dev, 50, cols, torch.float32, 1)
    for ww, bb in ((None, None), (w, None), (None, b)):
        check(dev, x, ww, bb, gy, 1e-5, 0.2)


@pytest.mark.parametrize("cols", [16, 800, 4000, 20_000])
def test_offsets_much_larger_than_the_spread(dev, cols):
    """mean / spread = 1000: a variance from sums of squares would lose every digit; two passes lose what the bound says."""
    x, w, b, gy = data(dev, 40, cols, torch.float32, 2, offset=1300.0)
    check(dev, x, w, b, gy, 1e-5, 1.0)


@pytest.mark.parametrize("cols", [16, 800, 4000, 20_000])
def test_very_small_and_very_large_values(dev, cols):
    """Without eps the output does not depend on the input's scale.  At 1e-19 the squares of the differences are subnormal, with down
    to 12 bits: 2^-11 is allowed; at 1e17 nothing overflows."""
    from liftreg_amd import ops
    x, w, b, _ = data(dev, 9, cols, torch.float32, 11)
    want = definition(x, w, b, 0.0, 1.0)["y"]
    for scale in (2.0 ** -63, 2.0 ** 56):
        got = ops.layer_norm(x * scale, w, b, eps=0.0)
        assert float((got.double() - want).abs().max()) <= 2.0 ** -11 * float(want.abs().max())


@pytest.mark.parametrize("cols", [3, 5, 12, 20, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_constant_rows_of_large_values(dev, cols, dtype):
    """mean / sqrt(eps) is beyond fp32, xhat is 0: gx = (h - mean(h)) / sqrt(eps), lanes without columns add nothing.  h = gy: a sum of
    cols terms, its mean, the difference and the product are off by (cols + 4) half steps of the largest term, twice."""
    from liftreg_amd import ops_bwd
    x = torch.full((5, cols), 2.0 ** 119, device=dev).to(dtype)
    gy = data(dev, 5, cols, torch.float32, 12)[3].to(dtype)
    gx, gw, gb = ops_bwd.layer_norm_bwd(x, torch.ones(cols, device=dev), torch.zeros(cols, device=dev), gy, eps=1e-6)
    g = gy.double()
    want = (g - g.mean(1, keepdim=True)) / float(torch.tensor(1e-6)) ** 0.5
    half = torch.finfo(dtype).eps / 2
    assert float((gx.double() - want).abs().max()) <= (2 * (cols + 4) * 2.0 ** -24 + half) * 2 * float(g.abs().max()) * 1e3
    assert (gw == 0).all() and torch.isfinite(gb).all()


@pytest.mark.parametrize("cols", [16_385, 20_000, 20_001, 300_001, 1_000_000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_constant_rows_of_large_values(dev, cols, dtype):
    """Powers of two, whose sums are exact: the mean is the value, xhat is 0 and the output the bias, however large the square of the value.
    gx = (gy - mean(gy)) / sqrt(eps), within the bound of test_constant_rows_of_large_values with the sums' own number of half steps."""
    from liftreg_amd import ops, ops_bwd
    w, b = data(dev, 1, cols, torch.float32, 13)[1:3]
    gy = data(dev, 3, cols, torch.float32, 14)[3].to(dtype)
    eps = float(torch.tensor(1e-6))
    for e in (56, 57, 64, 100, 119):
        x = torch.full((3, cols), 2.0 ** e, device=dev).to(dtype)
        y, stats = ops.layer_norm(x, w, b, eps=eps, return_stats=True)
        assert torch.equal(y, b.to(dtype).expand(3, cols)), e
        assert bool((stats[:, 0] == 2.0 ** e).all()) and float((stats[:, 1].double() * eps ** 0.5 - 1).abs().max()) <= 4 * U32
        g = gy.double()
        want = (g - g.mean(1, keepdim=True)) / eps ** 0.5
        for s in (stats, None):
            gx, gw, gb = ops_bwd.layer_norm_bwd(x, torch.ones_like(w), b, gy, eps=eps, stats=s)
            half = torch.finfo(dtype).eps / 2
            assert float((gx.double() - want).abs().max()) <= (2 * (sum_steps(cols) + 4) * U32 + half) * 2 * float(g.abs().max()) * 1e3, e
            assert bool((gw == 0).all()) and float((gb.double() - g.sum(0)).abs().max()) <= 4 * U32 * float(g.abs().sum(0).max())


@pytest.mark.parametrize("cols", [16_385, 20_000, 300_001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows_of_large_mean(dev, cols, dtype):
    """Mean 2^63, spread 2^55: the square of the mean leaves fp32, those of the differences do not."""
    x, w, b, gy = data(dev, 5, cols, torch.float32, 15, offset=300.0)
    check(dev, (x * 2.0 ** 55).to(dtype), w, b, gy.to(dtype), 1e-5, 1.0)


@pytest.mark.parametrize("cols", [16_385, 20_001, 300_001])
def test_very_small_and_very_large_values_of_long_rows(dev, cols):
    test_very_small_and_very_large_values(dev, cols)


@pytest.mark.parametrize("cols", [1, 3, 7, 13, 33, 100, 513, 801, 1500, 4097, 5000, 10_001, 16_384, 16_385, 20_000, 20_001, 300_001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_constant_rows_of_any_value(dev, cols, dtype):
    """The mean of a constant row is its value, also where the sum of `cols` of them is not a number of 24 bits or beyond fp32: the output is
    the bias and the weight's gradient zero, exactly.  Without eps such a row is 0 / 0."""
    from liftreg_amd import ops, ops_bwd
    w, b, gy = data(dev, 6, cols, dtype, 16)[1:]
    v = torch.tensor([1000.1, 12345.6, 0.1, -77.7, 3.3e-20, 1.1 * 2.0 ** 120], device=dev).to(dtype)
    x = v[:, None].expand(6, cols).contiguous()
    y, stats = ops.layer_norm(x, w, b, return_stats=True)
    assert torch.equal(y, b.to(dtype).expand(6, cols))
    assert stats is None or torch.equal(stats[:, 0], v.float())
    for s in (stats, None):
        gx, gw, gb = ops_bwd.layer_norm_bwd(x, w, b, gy, stats=s)
        assert bool((gw == 0).all()) and bool(torch.isfinite(gx).all()) and bool(torch.isfinite(gb).all())
    assert bool(torch.isnan(ops.layer_norm(x, w, b, eps=0.0)).all())


@pytest.mark.parametrize("cols", [16, 800, 8192])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("slope", [1.0, 0.2])
def test_arrays_that_pass_the_caches_by(dev, cols, dtype, slope):
    """From 256 MiB on x, gy, y and gx are read and written past the caches."""
    rows = (256 << 20) // (cols * torch.finfo(dtype).bits // 8) + 3
    check(dev, *data(dev, rows, cols, dtype, 18), 1e-5, slope)


@pytest.mark.parametrize("cols", [16, 801, 4097, 20_001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_that_start_anywhere(dev, cols, dtype):
    x, w, b, gy = data(dev, 30, cols, dtype, 3)
    off = [torch.cat([torch.zeros(1, device=dev, dtype=t.dtype), t.reshape(-1)])[1:].view(t.shape) for t in (x, w, b, gy)]
    from liftreg_amd import ops, ops_bwd
    assert torch.equal(ops.layer_norm(*off[:3]), ops.layer_norm(x, w, b))
    for a, c in zip(ops_bwd.layer_norm_bwd(*off), ops_bwd.layer_norm_bwd(x, w, b, gy)):
        assert torch.equal(a, c)
    # other strides are laid out first, leading axes are rows
    xt = x.t().contiguous().t()
    assert torch.equal(ops.layer_norm(xt, w, b), ops.layer_norm(x, w, b))
    assert torch.equal(ops.layer_norm(x.view(5, 3, 2, cols), w, b), ops.layer_norm(x, w, b).view(5, 3, 2, cols))


@pytest.mark.parametrize("cols", [16, 800, 4097, 20_000])
def test_rows_that_are_not_finite_or_constant(dev, cols):
    """A row with NaN or an infinity is NaN, its neighbours in the wave are not; a constant row with eps = 0 is 0 / 0."""
    from liftreg_amd import ops, ops_bwd
    x, w, b, gy = data(dev, 41, cols, torch.float32, 4)
    good = ops.layer_norm(x, w, b)
    x2 = x.clone()
    x2[3, cols // 2], x2[17, 0], x2[40, cols - 1] = float("nan"), float("inf"), float("-inf")
    y = ops.layer_norm(x2, w, b)
    bad = torch.zeros(41, dtype=torch.bool, device=dev)
    bad[[3, 17, 40]] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], good[~bad])
    gx, gw, gb = ops_bwd.layer_norm_bwd(x2, w, b, gy)
    assert torch.isnan(gx[bad]).all() and torch.equal(gx[~bad], ops_bwd.layer_norm_bwd(x, w, b, gy)[0][~bad])
    assert torch.isnan(gw).all()
    c = torch.full((41, cols), 2.0, device=dev)
    assert torch.equal(ops.layer_norm(c, None, b), b.expand(41, cols))
    gx = ops_bwd.layer_norm_bwd(c, w, b, gy)[0]
    assert torch.isfinite(gx).all()
    # rows that fill only part of a workgroup, eps = 0: the lanes without a row add nothing
    x3, w3, b3, gy3 = data(dev, 3, cols, torch.float32, 6)
    check(dev, x3, w3, b3, gy3, 0.0, 1.0)


def test_nothing_outside_is_written(dev):
    from liftreg_amd import _hip
    lib = _hip.lib()
    st = torch.cuda.current_stream().cuda_stream
    for rows, cols, dtype in ((3, 5, torch.float32), (7, 33, torch.bfloat16), (2, 801, torch.float32), (2, 4099, torch.bfloat16),
                              (2, 20_001, torch.float32), (9, 16, torch.bfloat16)):
        x, w, b, gy = data(dev, rows, cols, dtype, 7)
        n = rows * cols
        y, gx = (torch.full((n + 64,), 3.0, device=dev, dtype=dtype) for _ in range(2))
        gw, gb = (torch.full((cols + 64,), 3.0, device=dev) for _ in range(2))
        es = x.element_size()
        need = max(lib.lr_layer_norm_workspace(rows, cols, 0), lib.lr_layer_norm_workspace(rows, cols, 1))
        ws = torch.full((need + 256,), 7, dtype=torch.uint8, device=dev)
        bf = dtype == torch.bfloat16
        _hip.check(lib.lr_layer_norm(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr() + 32 * es, None, ws.data_ptr(), rows, cols, bf,
                                     1e-5, 0.2, st), "fwd")
        _hip.check(lib.lr_layer_norm_bwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), gy.data_ptr(), None, gx.data_ptr() + 32 * es,
                                         gw.data_ptr() + 128, gb.data_ptr() + 128, ws.data_ptr(), rows, cols, bf, 1e-5, 0.2, st), "bwd")
        torch.cuda.synchronize()
        for t, k in ((y, n), (gx, n), (gw, cols), (gb, cols)):
            assert (t[:32] == 3).all() and (t[32 + k:] == 3).all() and not (t[32:32 + k] == 3).all()
        assert (ws[need:] == 7).all()


def test_no_rows(dev):
    from liftreg_amd import ops, ops_bwd
    for cols in (16, 20_000):
        x = torch.empty(0, cols, device=dev)
        w = torch.ones(cols, device=dev)
        y, stats = ops.layer_norm(x, w, w, return_stats=True)
        assert y.shape == (0, cols)
        gx, gw, gb = ops_bwd.layer_norm_bwd(x, w, w, x, stats=stats)
        assert gx.shape == (0, cols) and not gw.any() and not gb.any()


def test_refusals(dev):
    from liftreg_amd import _hip, ops, ops_bwd
    x, w, b, gy = data(dev, 4, 8, torch.float32, 8)
    with pytest.raises(_hip.LiftRegHipError):
        ops.layer_norm(x.cpu())
    with pytest.raises(_hip.LiftRegHipError):
        ops.layer_norm(x, w.cpu())
    for t in (x.double(), x.half(), x.int()):
        with pytest.raises(TypeError):
            ops.layer_norm(t)
    with pytest.raises(TypeError):
        ops.layer_norm(x, w.bfloat16())
    with pytest.raises(TypeError):
        ops_bwd.layer_norm_bwd(x, w, b, gy.bfloat16())
    for call in (lambda: ops.layer_norm(x, w[:4]), lambda: ops.layer_norm(x, w, b[:, None]), lambda: ops.layer_norm(x, w, b, eps=-1e-5),
                 lambda: ops.layer_norm(x, w, b, eps=float("nan")), lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x[0, 0]),
                 lambda: ops_bwd.layer_norm_bwd(x, w, b, gy[:2]), lambda: ops_bwd.layer_norm_bwd(x, w, b, gy, stats=torch.zeros(3, 2, device=dev))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("cols", [16, 800, 4096, 20_000])
def test_gradient_against_differences(dev, cols):
    """(L(x + t u) - L(x - t u)) / 2t of L = sum gy y in 64 bits, along random u in x, w and b."""
    from liftreg_amd import ops_bwd
    x, w, b, gy = data(dev, 6, cols, torch.float32, 9)
    gy[(definition(x, w, b, 1e-5, 0.2)["z"].abs() < 1e-4)] = 0        # no sample on the kink
    gx, gw, gb = ops_bwd.layer_norm_bwd(x, w, b, gy, negative_slope=0.2)
    t = 1e-6
    for k, grad in enumerate((gx, gw, gb)):
        u = torch.randn(grad.shape, device=dev, dtype=torch.float64)
        args = [x.double(), w.double(), b.double()]

        def loss(s):
            a = list(args)
            a[k] = a[k] + s * u
            return float((definition(*a, 1e-5, 0.2)["y"] * gy.double()).sum())

        want = (loss(t) - loss(-t)) / (2 * t)
        # truncation ~ t^2, cancellation ~ 1e-16 |L| / t ~ 1e-8, the kernel's gradient ~ 1e-6 of its size
        assert abs(float((grad.double() * u).sum()) - want) <= 1e-5 * float((grad.double() * u).abs().sum()) + 1e-6


def test_module_matches_torch(dev):
    from liftreg_amd.layers.layers import LayerNorm
    torch.manual_seed(0)
    for shape, lead in ((24, (5, 7)), ((3, 5, 16), (4,)), ((6, 3000), (3,))):
        ref = torch.nn.LayerNorm(shape).to(dev)
        with torch.no_grad():
            ref.weight.normal_(1, 0.2), ref.bias.normal_(0, 0.2)
        net = LayerNorm(shape).to(dev)
        net.load_state_dict(ref.state_dict())
        x = torch.randn(lead + ref.normalized_shape, device=dev)
        a, c = x.clone().requires_grad_(), x.clone().requires_grad_()
        g = torch.randn_like(x)
        ya, yc = ref.double()(a.double()).float(), net(c)
        ya.backward(g), yc.backward(g)
        # C <= 18000 terms in the sums; everything of order one: 200 half steps are far below what a mistake changes
        assert float((ya - yc).detach().abs().max()) < 200 * U32 * 5 and float((a.grad - c.grad).abs().max()) < 200 * U32 * 5
        for p, q in zip(ref.parameters(), net.parameters()):
            assert p.shape == q.shape and float((p.grad - q.grad).abs().max()) < 200 * U32 * 40
    assert LayerNorm((4, 6)).to(dev)(torch.empty(0, 4, 6, device=dev)).shape == (0, 4, 6)
    plain = LayerNorm(24, elementwise_affine=False).to(dev)
    assert not list(plain.parameters())
    x = torch.randn(3, 24, device=dev, requires_grad=True)
    plain(x).sum().backward()
    assert x.grad is not None
    assert [n for n, _ in LayerNorm(24, bias=False).named_parameters()] == ["weight"]
    with pytest.raises(ValueError):
        plain(torch.randn(3, 25, device=dev))
    # frozen parts and an expanded gradient
    net = LayerNorm(24).to(dev)
    net.bias.requires_grad_(False)
    net(torch.randn(9, 24, device=dev)).sum().backward()
    assert net.weight.grad is not None and net.bias.grad is None


def test_graph_replays(dev):
    from liftreg_amd import ops, ops_bwd
    for rows, cols in ((1000, 16), (8, 800), (3, 30_000)):
        x, w, b, gy = data(dev, rows, cols, torch.float32, 10)
        ops_bwd.layer_norm_bwd(x, w, b, gy)
        graphs = []
        for slope in (0.2, 1.0):         # two graphs: their workspaces are their own
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y, stats = ops.layer_norm(x, w, b, negative_slope=slope, return_stats=True)
                out = (y,) + ops_bwd.layer_norm_bwd(x, w, b, gy, negative_slope=slope, stats=stats)
            graphs.append((graph, slope, out))
        for k in range(6):
            x.normal_(), gy.normal_()
            graph, slope, out = graphs[k % 2]
            graphs[(k + 1) % 2][0].replay()
            graph.replay()
            y, stats = ops.layer_norm(x, w, b, negative_slope=slope, return_stats=True)
            want = (y,) + ops_bwd.layer_norm_bwd(x, w, b, gy, negative_slope=slope, stats=stats)
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(out, want)), (rows, cols, k)


# ------------------------------------------------------------------------------------------------ blocks and the model
def reference_model(net, inp):
    """The model with norm="layer" from torch operations in float64 (forward of coefs only, by autograd differentiable)."""
    import torch.nn.functional as F
    from liftreg_amd import ops
    sd = {k: v.detach().double().requires_grad_(v.dtype == torch.float32 and "gaussian" not in k) for k, v in net.state_dict().items()}
    B, _, D, W, H = inp["source"].shape
    vol = ops.backproject(inp["target_proj"], inp["target_poses"][0], (D, W, H))
    x = torch.cat([inp["source"], vol], 1).double()
    for i in range(6):
        x = F.conv3d(x, sd[f"encoders.{i}.conv.weight"], sd[f"encoders.{i}.conv.bias"], stride=net.strides[i], padding=1)
        x = F.layer_norm(x.permute(0, 2, 3, 4, 1), (x.shape[1],), sd[f"encoders.{i}.norm.weight"], sd[f"encoders.{i}.norm.bias"], 1e-5)
        x = F.leaky_relu(x.permute(0, 4, 1, 2, 3), 0.2)
    x = x.flatten(1)
    for i in (1, 2):
        x = F.linear(x, sd[f"encoders.6.{i}.fc.weight"], sd[f"encoders.6.{i}.fc.bias"])
        x = F.leaky_relu(F.layer_norm(x, x.shape[1:], sd[f"encoders.6.{i}.norm.weight"], sd[f"encoders.6.{i}.norm.bias"], 1e-5), 0.2)
    return F.linear(x, sd["encoders.6.3.fc.weight"], sd["encoders.6.3.fc.bias"]), sd


def make_model(dev, size=(32, 32, 32), **opt):
    from liftreg_amd.models.LiftRegDeformSubspaceBackproj import model
    torch.manual_seed(5)
    net = model(list(size), {"drr_feature_num": 2, "latent_dim": 6, "pca_path": "synthetic:7", **opt}).to(dev)
    with torch.no_grad():
        for n, p in net.named_parameters():
            if ".norm." in n:
                p.add_(0.1 * torch.randn_like(p))
    return net


def batch(dev, B=2, size=(32, 32, 32)):
    import numpy as np
    from liftreg_amd.utils.sdct_projection_utils import scan_poses
    g = torch.Generator(device=dev).manual_seed(3)
    rnd = lambda *s: torch.rand(*s, generator=g, device=dev) * 2 - 1
    poses = scan_poses(30, 2, size[1]).astype(np.float32)
    return {"source": rnd(B, 1, *size), "target": rnd(B, 1, *size), "target_proj": rnd(B, 2, 32, 32),
            "target_poses": torch.from_numpy(np.broadcast_to(poses, (B, 2, 3)).copy())}


@pytest.mark.parametrize("size", [(32, 32, 32), (32, 40, 36)])
def test_model_with_norm(dev, size):
    """Coefficients and every parameter's gradient against float64 autograd of the same graph.  The fp32 convolutions of six blocks
    and the norms that follow them (each divides by a spread of the size of what it norms) carry 1e-6 to 1e-5 relative to scale;
    a LeakyReLU mask that flips within that changes single terms of sums over thousands of voxels."""
    net, inp = make_model(dev, size, norm="layer"), batch(dev, 2, size)
    net.train()
    coefs = net.encode(inp["source"], inp["target_proj"], inp["target_poses"])
    want, sd = reference_model(net, inp)
    assert float((coefs.double() - want).detach().abs().max()) <= 1e-4 * float(want.detach().abs().max())
    g = torch.randn_like(coefs)
    coefs.backward(g)
    want.backward(g.double())
    for k, p in net.named_parameters():
        w = sd[k].grad
        # a conv bias in front of ... a norm over channels still has a gradient; compare in the 2-norm
        err = float((p.grad.double() - w).norm() / w.norm().clamp_min(1e-12))
        assert err <= 2e-3, (k, err)
    net.eval()
    with torch.no_grad():
        assert torch.equal(net.encode(inp["source"], inp["target_proj"], inp["target_poses"]), coefs)


def test_model_norm_is_off_by_default_and_refuses_what_is_not_built(dev):
    from liftreg_amd import ops
    from liftreg_amd.layers.layers import convBlock
    from liftreg_amd.parallel import LocalComm, SlabShardedRegistration
    net = make_model(dev)
    assert not any(".norm." in k for k in net.state_dict())
    for bad in (dict(norm="batch"), dict(norm="layer", conv_dtype="bf16"), dict(norm="layer", fuse_backproject=True)):
        with pytest.raises(ValueError):
            make_model(dev, **bad)
    with pytest.raises(ValueError):
        convBlock(3, 16, layernorm=True, out_layout=ops.LAYOUT_NDHWC_HPS)
    with pytest.raises(ValueError):
        SlabShardedRegistration(make_model(dev, norm="layer"), LocalComm(1))


def test_inference_mode_and_shared_weights(dev):
    from liftreg_amd import ops
    from liftreg_amd.layers.layers import LayerNorm
    torch.manual_seed(1)
    net = LayerNorm(40, negative_slope=0.2).to(dev)
    x = torch.randn(7, 40, device=dev)
    want = net(x).detach()
    with torch.inference_mode():
        assert torch.equal(net(x), want) and torch.equal(ops.layer_norm(x.clone(), net.weight, net.bias, negative_slope=0.2), want)
    # one weight used twice, a broadcast input, an expanded gradient: autograd adds them up
    row = torch.randn(40, device=dev, requires_grad=True)
    (net(row.expand(5, 40)).sum() + net(x).sum()).backward()
    g = [p.grad.clone() for p in net.parameters()]
    gr = row.grad.clone()
    net.zero_grad(), row.grad.zero_()
    net(row.expand(5, 40).contiguous()).backward(torch.ones(5, 40, device=dev))
    net(x).backward(torch.ones(7, 40, device=dev))
    assert all(torch.equal(a, p.grad) for a, p in zip(g, net.parameters())) and torch.equal(gr, row.grad)


def test_graphed_registration_of_the_normalised_model(dev):
    from liftreg_amd.pipeline import GraphedRegistrar
    net, inp = make_model(dev, norm="layer").eval(), batch(dev)
    reg = GraphedRegistrar(net, inp)
    for k in range(3):
        inp["source"].uniform_(-1, 1), inp["target_proj"].uniform_(-1, 1)
        out, _ = reg(inp)
        with torch.no_grad():
            want = net(inp)
        torch.cuda.synchronize()
        assert torch.equal(out["pca_coefs"], want["pca_coefs"]) and torch.equal(out["warped"], want["warped"]), k


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_of_the_normalised_model(dev, bits):
    """Norm layers, gradients, clipping and the update together: three steps of the whole model; the same three steps a second time
    give the same bits; every parameter moves; a later inference sees the new weights."""
    from liftreg_amd.losses.SubspaceLoss import loss as SubspaceLoss
    from liftreg_amd.optim import AdamW
    inp = batch(dev)
    crit = SubspaceLoss({"initial_reg_factor": 0.01, "min_reg_factor": 0.01, "reg_factor_decay_from": 2})

    def go():
        net = make_model(dev, norm="layer").train()
        start = {k: p.detach().clone() for k, p in net.named_parameters()}
        net.eval()
        with torch.no_grad():
            before = net(inp)["pca_coefs"].clone()     # packs the weights
        net.train()
        opt = AdamW(net.parameters(), lr=1e-3, eps=1e-5, state_bits=bits, max_grad_norm=1.0, seed=1)
        for ep in range(3):
            opt.zero_grad()
            out = net(inp)
            out["epoch"] = ep
            crit(out)["total_loss"].backward()
            grads = [p.grad.double() for p in net.parameters() if p.grad is not None]
            opt.step()
            want = float(sum((g ** 2).sum() for g in grads).sqrt())
            assert abs(float(opt.grad_norm) - want) <= 1e-6 * want
        net.eval()
        with torch.no_grad():
            after = net(inp)["pca_coefs"].clone()
            net.invalidate_packed()
            assert torch.equal(after, net(inp)["pca_coefs"]) and not torch.equal(after, before)
        return start, {k: p.detach().clone() for k, p in net.named_parameters()}

    start, end = go()
    assert all(not torch.equal(start[k], end[k]) and torch.isfinite(end[k]).all() for k in end)
    _, again = go()
    assert all(torch.equal(end[k], again[k]) for k in end)

"""CPU: argument checks of the layer norm and of the AdamW step that answer without a GPU (Python and C entry points), and the
optimizer's state bookkeeping."""
import ctypes as C

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def hip():
    from liftreg_amd import _hip
    _hip.lib()
    return _hip


def test_c_entries_refuse(hip):
    lib = hip.lib()
    f = C.addressof(C.c_float(0))
    n = np.array([5, 0], dtype=np.int64)
    bad = np.array([5, -1], dtype=np.int64)
    ptr = np.array([f, 0], dtype=np.uint64)
    null = np.zeros(2, dtype=np.uint64)
    at = lambda a: a.ctypes.data
    assert lib.lr_grad_norm_partials(None, 2) == -2 and lib.lr_grad_norm_partials(at(n), 0) == -1
    assert lib.lr_grad_norm_partials(at(bad), 2) == -1 and lib.lr_grad_norm_partials(at(n), 2) == 1
    assert lib.lr_grad_norm(None, at(n), 2, 0, f, f, None) == -2 and lib.lr_grad_norm(at(null), at(n), 2, 0, f, f, None) == -2
    assert lib.lr_grad_norm(at(ptr), at(bad), 2, 0, f, f, None) == -1

    def step(p=ptr, g=ptr, m=ptr, v=ptr, ms=None, vs=None, numel=n, count=2, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, t=1, clip=0.0,
             norm_in=None, partial=None):
        adr = lambda a: None if a is None else at(a)
        return lib.lr_adamw_step(adr(p), adr(g), adr(m), adr(v), adr(ms), adr(vs), adr(numel), count, 0, lr, b1, b2, eps, wd, t, None, None,
                                 clip, norm_in, partial, None, 0, None)

    for k in ("p", "g", "m", "v", "numel"):
        assert step(**{k: None}) == -2
    for k in ("p", "g", "m", "v"):
        assert step(**{k: null}) == -2
    assert step(ms=ptr) == -2 and step(vs=ptr) == -2 and step(ms=null, vs=ptr) == -2
    for more in (dict(count=0), dict(numel=bad), dict(b1=1.0), dict(b1=-0.1), dict(b2=1.0), dict(b2=float("nan")), dict(eps=-1.0), dict(t=0),
                 dict(norm_in=f), dict(partial=f), dict(norm_in=f, partial=f, clip=1.0)):
        assert step(**more) == -1, more

    assert lib.lr_layer_norm_workspace(-1, 4, 0) == -1 and lib.lr_layer_norm_workspace(4, 0, 1) == -1
    assert lib.lr_layer_norm_workspace(4, 4, 0) == 0 and lib.lr_layer_norm_workspace(0, 4, 1) == 0
    long = lib.lr_layer_norm_resident_cols() + 1
    assert lib.lr_layer_norm_workspace(4, long, 0) > 0
    assert lib.lr_layer_norm(f, None, None, f, None, None, 1, 0, 0, 1e-5, 1.0, None) == -1
    assert lib.lr_layer_norm(f, None, None, f, None, None, -1, 4, 0, 1e-5, 1.0, None) == -1
    assert lib.lr_layer_norm(f, None, None, f, None, None, 1, 4, 0, -1e-5, 1.0, None) == -1
    assert lib.lr_layer_norm(None, None, None, f, None, None, 1, 4, 0, 1e-5, 1.0, None) == -2
    assert lib.lr_layer_norm(f, None, None, f, None, None, 1, long, 0, 1e-5, 1.0, None) == -2
    assert lib.lr_layer_norm(None, None, None, None, None, None, 0, 4, 0, 1e-5, 1.0, None) == 0
    assert lib.lr_layer_norm_bwd(f, None, None, None, None, f, None, None, f, 1, 4, 0, 1e-5, 1.0, None) == -2
    assert lib.lr_layer_norm_workspace(4, 800, 1) == 0 and lib.lr_layer_norm_workspace(4000, 800, 1) > 0
    assert lib.lr_layer_norm_bwd(f, None, None, f, None, f, None, None, None, 4000, 800, 0, 1e-5, 1.0, None) == -2
    assert lib.lr_layer_norm_bwd(f, None, None, f, None, None, None, None, f, 1, 4, 0, 1e-5, 1.0, None) == 0


def test_python_refuses_cpu_tensors(hip):
    from liftreg_amd import ops, ops_bwd, optim
    x = torch.zeros(3, 4)
    for call in (lambda: ops.layer_norm(x), lambda: ops_bwd.layer_norm_bwd(x, None, None, x), lambda: optim.grad_norm([x]),
                 lambda: optim.adamw_step([x], [x], [x], [x], step=1)):
        with pytest.raises(hip.LiftRegHipError):
            call()
    for call in (lambda: ops.layer_norm([1.0]), lambda: ops.layer_norm(x.int()), lambda: optim.grad_norm([1.0])):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: optim.grad_norm([]), lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x, eps=-1.0)):
        with pytest.raises(ValueError):
            call()


def test_optimizer_arguments():
    from liftreg_amd.optim import AdamW
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(state_bits=4),
                dict(max_grad_norm=0.0)):
        with pytest.raises(ValueError):
            AdamW(p, **bad)
    opt = AdamW(p, lr=0.5)
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))], "lr": -1.0})
    opt.step()                              # no gradient: nothing to do, nothing launched
    assert opt.grad_norm is None and not opt.state


def test_load_state_dict_checks_the_states():
    from liftreg_amd.optim import AdamW, state8
    p = [torch.nn.Parameter(torch.ones(40))]
    ref = torch.optim.AdamW(p, lr=0.1)
    p[0].grad = torch.full((40,), 0.5)
    ref.step()
    opt = AdamW(p)
    opt.load_state_dict(ref.state_dict())
    s = opt.state[p[0]]
    assert s["step"] == 1 and torch.equal(s["exp_avg"], ref.state[p[0]]["exp_avg"]) and opt.param_groups[0]["lr"] == 0.1
    with pytest.raises(ValueError):
        AdamW(p, state_bits=8).load_state_dict(ref.state_dict())
    with pytest.raises(ValueError):
        AdamW(p).load_state_dict(torch.optim.AdamW(p, amsgrad=True).state_dict())
    coupled = torch.optim.Adam(p, weight_decay=0.1)
    with pytest.raises(ValueError):
        AdamW(p).load_state_dict(coupled.state_dict())
    AdamW(p).load_state_dict(torch.optim.Adam(p).state_dict())
    other = [torch.nn.Parameter(torch.ones(41))]
    fresh = AdamW(other, lr=0.25)
    with pytest.raises(ValueError):
        fresh.load_state_dict(ref.state_dict())
    assert fresh.param_groups[0]["lr"] == 0.25 and not fresh.state
    eight = AdamW(p, state_bits=8)
    m, ms, v, vs = state8(p[0])
    eight.state[p[0]] = {"step": 3, "exp_avg": m, "exp_avg_scale": ms, "exp_avg_sq": v, "exp_avg_sq_scale": vs}
    again = AdamW(p, state_bits=8)
    again.load_state_dict(eight.state_dict())
    s = again.state[p[0]]
    assert s["step"] == 3 and s["exp_avg"].dtype == torch.float8_e4m3fn and s["exp_avg_sq"].dtype == torch.float8_e5m2
    assert s["exp_avg_scale"].dtype == torch.float8_e8m0fnu and s["exp_avg"].data_ptr() != m.data_ptr()


def test_values8():
    from liftreg_amd.optim import values8
    q = torch.arange(40, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.tensor([127, 130], dtype=torch.uint8).view(torch.float8_e8m0fnu)
    got = values8(q, s)
    assert torch.equal(got[:32], q[:32].float()) and torch.equal(got[32:], 8 * q[32:].float())
    assert torch.isnan(values8(q, torch.tensor([255, 127], dtype=torch.uint8).view(torch.float8_e8m0fnu))[:32]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_and_pickles_of_the_optimizer(bits):
    import copy
    import pickle

    from liftreg_amd.optim import AdamW, state8
    p = torch.nn.Parameter(torch.ones(40))
    opt = AdamW([p], lr=0.5, state_bits=bits, max_grad_norm=2.0, seed=(7 << 32) + 3, capturable=True)
    count = torch.tensor(4)
    q = torch.nn.Parameter(torch.ones(9))
    opt.add_param_group({"params": [q], "lr": 0.25})
    for t in (p, q):
        m, ms, v, vs = state8(t)
        opt.state[t] = {"step": count, "exp_avg": m, "exp_avg_sq": v, "exp_avg_scale": ms, "exp_avg_sq_scale": vs} if bits == 8 else \
            {"step": count, "exp_avg": torch.zeros(t.shape), "exp_avg_sq": torch.ones(t.shape)}
    opt.grad_norm = torch.tensor(1.5)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        for k in ("state_bits", "max_grad_norm", "seed", "capturable", "grad_norm"):
            assert getattr(other, k) == getattr(opt, k), k
        assert [g["lr"] for g in other.param_groups] == [0.5, 0.25]
        a, b = (other.state[g["params"][0]] for g in other.param_groups)
        assert a["step"] is b["step"] and int(a["step"]) == 4 and a["step"] is not count
        assert a["exp_avg_sq"].dtype == (torch.float8_e5m2 if bits == 8 else torch.float32)
        other.step()                        # no gradient: nothing to do, nothing launched
        assert other.grad_norm is None and opt.grad_norm is not None


def test_an_eps_that_fp32_holds_with_fewer_bits_is_refused(hip):
    """eps is added in fp32: 0, or a normal number."""
    from liftreg_amd import optim
    f = C.addressof(C.c_float(0))
    n, ptr = np.array([5], dtype=np.int64), np.array([f], dtype=np.uint64)
    at = lambda a: a.ctypes.data
    x = torch.zeros(3)
    for eps in (1e-40, 5e-324, 2.0 ** -127):
        assert hip.lib().lr_adamw_step(at(ptr), at(ptr), at(ptr), at(ptr), None, None, at(n), 1, 0, 1e-3, 0.9, 0.999, eps, 0.0, 1, None, None, 0.0,
                                       None, None, None, 0, None) == -1
        with pytest.raises(ValueError):
            optim.adamw_step([x], [x], [x], [x], step=1, eps=eps)
        with pytest.raises(ValueError):
            optim.AdamW([torch.nn.Parameter(x)], eps=eps)
    optim.AdamW([torch.nn.Parameter(x)], eps=2.0 ** -126), optim.AdamW([torch.nn.Parameter(x)], eps=0.0)


def test_the_host_module_belongs_to_the_torch_that_is_loaded(hip, monkeypatch):
    """_host.so is compiled against torch's C++ headers: under another torch it is refused, not called."""
    assert hip.host().torch_version == torch.__version__
    monkeypatch.setattr(hip, "_host", None)
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    with pytest.raises(hip.LiftRegHipError, match="0.0.0"):
        hip.host()
    monkeypatch.undo()
    assert hip.host().torch_version == torch.__version__


def test_load_state_dict_refuses_states_before_it_changes_anything():
    from liftreg_amd.optim import AdamW, state8
    p = [torch.nn.Parameter(torch.ones(40))]

    def checkpoint(**more):
        opt = AdamW(p, lr=0.5, state_bits=8)
        m, ms, v, vs = state8(p[0])
        opt.state[p[0]] = {"step": 3, "exp_avg": m, "exp_avg_scale": ms, "exp_avg_sq": v, "exp_avg_sq_scale": vs} | more
        return opt.state_dict()

    without = checkpoint()
    del without["state"][0]["step"]
    scales = torch.zeros(3, dtype=torch.uint8)
    for bad in (without, checkpoint(exp_avg_scale=scales.view(torch.float8_e8m0fnu)), checkpoint(exp_avg_sq_scale=scales[:2])):
        opt = AdamW(p, lr=0.25, state_bits=8)
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]["lr"] == 0.25 and not opt.state


def test_a_layer_norm_eps_that_fp32_rounds_to_zero_is_refused(hip):
    """It would divide a constant row's 0 by 0."""
    from liftreg_amd import ops, ops_bwd
    x = torch.zeros(3, 4)
    for eps in (1e-46, 1e-300):
        with pytest.raises(ValueError):
            ops.layer_norm(x, eps=eps)
        with pytest.raises(ValueError):
            ops_bwd.layer_norm_bwd(x, None, None, x, eps=eps)
    for eps in (0.0, 1e-44):
        with pytest.raises(hip.LiftRegHipError):         # next in line: a tensor on the CPU
            ops.layer_norm(x, eps=eps)

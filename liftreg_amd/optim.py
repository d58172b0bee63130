"""The update of the parameters on the HIP kernels (liftreg_amd/csrc/optim.hip): the AdamW step over all the tensors of a model,
64 of them a launch, its states in 32 bits or in block-scaled 8 bits, and the global norm of the gradients that it clips by.

The reference trains with `torch.optim.Adam(eps=1e-5)` (src/liftreg/networks/RegistrationNet.py:245), which `AdamW` with
`weight_decay=0` is.  GPU tensors only; launches go to torch's current stream of the tensors' device.
"""
from collections import Counter, defaultdict

import torch

from . import _hip, ops

BLOCK = 32                              # consecutive elements that share a scale in the 8-bit states
_TYPES8 = {"exp_avg": torch.float8_e4m3fn, "exp_avg_scale": torch.float8_e8m0fnu, "exp_avg_sq": torch.float8_e5m2,
           "exp_avg_sq_scale": torch.float8_e8m0fnu}
_T = torch.Tensor


def grad_norm(grads):
    """The 2-norm of all `grads` together (0-dim float32 tensor): fp64 sums in a fixed order, two launches, no synchronisation.
    grads: contiguous float32 or bfloat16 GPU tensors of one type and device, any shapes."""
    if ops._timer is None:
        return _hip.host().grad_norm(grads)
    grads = list(grads)
    with ops._timed("grad_norm", bytes=sum(g.numel() * g.element_size() for g in grads)):
        return _hip.host().grad_norm(grads)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None,
               grad_norm=None, exp_avg_scales=None, exp_avg_sq_scales=None, seed=0):
    """One AdamW step over lists of tensors, in place:

        g = grad c,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    params, grads: contiguous float32 or bfloat16 tensors (one type; bfloat16 parameters are rounded to nearest — where lr times
    the update is below 2^-9 of a parameter it no longer moves: keep those in float32).  What is written may not overlap itself
    (checked) or the gradients.
    exp_avgs, exp_avg_sqs: float32, of the parameters' sizes; or, with exp_avg_scales and exp_avg_sq_scales, block-scaled 8-bit
    states: float8_e4m3fn / float8_e5m2 codes of the parameters' sizes and one float8_e8m0fnu scale for each 32 consecutive
    elements (`state8` makes them, `values8` reads them).  They are rounded stochastically: the random bits are a function of
    (seed, step, position of the element in the call's tensors), so equal calls give equal bits.  A block with an element that is
    not finite becomes NaN as a whole.
    eps: 0 or at least 2^-126 (it is added in fp32).  With 0 a v below 2^-149, which fp32 holds as 0, divides by 0.
    step: 1 for the first step; lr: both numbers, or one-element device tensors (int64, float32) that a captured graph reads
    at each replay (a number is captured as it is).
    max_norm: the gradients are scaled by min(1, max_norm / (norm + 1e-6)) on the way in (they are not written); norm is
    `grad_norm` (0-dim float32 tensor) or, if that is None, the 2-norm of all of `grads`, computed here.  A norm that is not finite
    reaches the parameters.  The lists may be any iterables.  Returns the norm (0-dim float32 tensor), None without max_norm."""
    b1, b2 = betas
    if ops._timer is not None:
        params = list(params)
    args = (params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, step, lr, b1, b2, eps, weight_decay, max_norm, grad_norm, seed)
    if ops._timer is None:
        return _hip.host().adamw_step(*args)
    with ops._timed("adamw_step", bytes=sum(p.numel() * (3 * p.element_size() + (16 if exp_avg_scales is None else 4)) for p in params)):
        return _hip.host().adamw_step(*args)


def _steps(calls):
    """Several adamw_step calls (tuples of the host function's arguments), all of them checked before the first one writes."""
    if ops._timer is None:
        return _hip.host().adamw_steps(*calls)
    size = sum(p.numel() * (3 * p.element_size() + (16 if c[4] is None else 4)) for c in calls for p in c[0])
    with ops._timed("adamw_step", bytes=size):
        return _hip.host().adamw_steps(*calls)


def state8(p):
    """(codes e4m3, scales, codes e5m2, scales): the 8-bit states of parameter `p`, at zero."""
    def zeros(shape, dtype):
        return torch.zeros(shape, dtype=torch.uint8, device=p.device).view(dtype)

    blocks = (-(-p.numel() // BLOCK),)
    return (zeros(p.shape, torch.float8_e4m3fn), zeros(blocks, torch.float8_e8m0fnu), zeros(p.shape, torch.float8_e5m2),
            zeros(blocks, torch.float8_e8m0fnu))


def values8(codes, scales):
    """The float32 values that 8-bit states stand for: code * scale of its block of 32 consecutive elements."""
    s = scales.to(torch.float32).repeat_interleave(BLOCK)[:codes.numel()]
    return codes.to(torch.float32) * s.view(codes.shape)


class AdamW(torch.optim.Optimizer):
    """AdamW on the kernel above, in torch.optim's manner: parameter groups, closures, LR schedulers, state_dict (32-bit states
    have the keys of torch.optim.Adam / AdamW, whose checkpoints load), copies and pickles.  `weight_decay=0` is Adam, the reference's optimizer.

        opt = AdamW(net.parameters(), lr=1e-4, eps=1e-5, weight_decay=0.0, max_grad_norm=1.0)

    state_bits: 32, or 8 for block-scaled 8-bit states (2.06 bytes an element instead of 8).
    max_grad_norm: clip the 2-norm of all gradients, inside the step; `opt.grad_norm` is the last step's norm (0-dim tensor).
    seed: of the stochastic rounding of 8-bit states.
    capturable: the step count lives on the device (int64 tensor), so that `step()` can be captured in a graph; the groups'
    "lr" may then be a one-element float32 device tensor, which a replay reads.  A replay does not run Python: call the model's
    `invalidate_packed()` before inference with parameters that replays have changed.  A graph keeps the state tensors and counts of its
    capture: load checkpoints before it, and step the same parameters between replays (others would part from a shared count).
    These four are the constructor's: copies and pickles keep them, state_dict (groups and states) does not hold them.
    Parameters: contiguous float32 or bfloat16 GPU tensors; gradients of the parameter's type, dense."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_grad_norm=None, seed=0,
                 capturable=False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"max_grad_norm must be positive, got {max_grad_norm}")
        self.state_bits, self.max_grad_norm, self.seed, self.capturable = state_bits, max_grad_norm, int(seed), bool(capturable)
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        # of copies and pickles; the base class keeps its own attributes only, and pickle refuses the 8-bit types
        state = super().__getstate__() | {k: getattr(self, k) for k in ("state_bits", "max_grad_norm", "seed", "capturable", "grad_norm")}
        if self.state_bits == 8:
            state["state"] = {p: {k: v.view(torch.uint8) if k in _TYPES8 else v for k, v in s.items()} for p, s in self.state.items()}
        return state

    def __setstate__(self, state):
        super().__setstate__(state)
        if self.state_bits == 8:
            self.state = defaultdict(dict, {p: {k: v.view(_TYPES8[k]) if k in _TYPES8 and v.dtype == torch.uint8 else v for k, v in s.items()}
                                            for p, s in self.state.items()})

    def add_param_group(self, group):
        b1, b2 = group.get("betas", self.defaults["betas"])
        lr = group.get("lr", self.defaults["lr"])
        eps = group.get("eps", self.defaults["eps"])
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0) or not lr >= 0.0 or not (eps == 0.0 or eps >= 2.0 ** -126) or \
                group.get("weight_decay", self.defaults["weight_decay"]) < 0.0:
            raise ValueError("betas must be in [0, 1), eps 0 or at least 2^-126, lr and weight_decay not negative")
        if isinstance(lr, _T) and lr.is_cuda and not self.capturable:
            raise ValueError("a learning rate on the device needs capturable=True")
        super().add_param_group(group)

    def _new_state(self, p, steps):
        if self.state_bits == 8:
            m, ms, v, vs = state8(p)
            s = {"exp_avg": m, "exp_avg_scale": ms, "exp_avg_sq": v, "exp_avg_sq_scale": vs}
        else:
            s = {"exp_avg": torch.zeros(p.shape, dtype=torch.float32, device=p.device),
                 "exp_avg_sq": torch.zeros(p.shape, dtype=torch.float32, device=p.device)}
        if self.capturable:          # parameters that start together share their count
            if p.device not in steps:
                steps[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
            return {"step": steps[p.device], **s}
        return {"step": 0, **s}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.grad_norm = None
        calls, fresh, skipped = [], {}, False
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            skipped |= len(ps) < len(group["params"])
            if not ps:
                continue
            if ps[0].is_cuda and torch.cuda.is_current_stream_capturing():
                if not self.capturable:
                    raise _hip.LiftRegHipError("a captured step needs capturable=True: the step count would be captured as a number")
                if not all(self.state[p] for p in ps):
                    raise _hip.LiftRegHipError("run one step before the capture: the states would start from zero at every replay")
            gs, ss = [p.grad for p in ps], [self.state[p] for p in ps]
            for p, s in zip(ps, ss):
                if not s:
                    s.update(self._new_state(p, fresh))
            calls += self._calls(gi, ps, [g if g.is_contiguous() else g.contiguous() for g in gs], ss)
        if self.capturable and skipped:
            self._part_counts(calls)
        norm = None
        if self.max_grad_norm is not None and len(calls) > 1:
            kinds = {}
            for _, ps, gs, _ in calls:
                kinds.setdefault((ps[0].dtype, ps[0].device), []).extend(gs)
            if len({device for _, device in kinds}) > 1:
                raise ValueError("max_grad_norm: all parameters must be on one device")
            norms = [grad_norm(gs) for gs in kinds.values()]
            norm = norms[0] if len(norms) == 1 else grad_norm([torch.stack(norms)])
        if not calls:
            return loss
        eight, steps, nth = self.state_bits == 8, [], Counter()
        for gi, ps, gs, ss in calls:
            group, t, lr = self.param_groups[gi], ss[0]["step"], self.param_groups[gi]["lr"]
            b1, b2 = group["betas"]
            steps.append((ps, gs, [s["exp_avg"] for s in ss], [s["exp_avg_sq"] for s in ss], [s["exp_avg_scale"] for s in ss] if eight else None,
                          [s["exp_avg_sq_scale"] for s in ss] if eight else None, t if isinstance(t, _T) else t + 1,
                          float(lr) if isinstance(lr, _T) and not lr.is_cuda else lr, b1, b2, group["eps"], group["weight_decay"],
                          self.max_grad_norm, norm, self.seed + (gi << 32) + (nth[gi] << 48)))      # groups and a group's calls draw different bits
            nth[gi] += 1
        # counts on the device go ahead of the launches that read them (one that several calls share once), and back if one is refused
        ahead = list({id(s[6]): s[6] for s in steps if isinstance(s[6], _T)}.values())
        for t in ahead:
            t.add_(1)
        try:
            self.grad_norm = _steps(steps)
        except BaseException:
            for t in ahead:
                t.sub_(1)
            raise
        for (*_, ss), s in zip(calls, steps):
            if not isinstance(s[6], _T):
                for state in ss:
                    state["step"] = s[6]
        return loss

    def _part_counts(self, calls):
        """Parameters that step now leave the device counts that they share with parameters that do not."""
        now = {id(s) for *_, ss in calls for s in ss}
        left = {id(s["step"]) for s in self.state.values() if s and id(s) not in now}
        own = {}
        for *_, ss in calls:
            t = ss[0]["step"]
            if id(t) in left:
                if torch.cuda.is_current_stream_capturing():
                    raise _hip.LiftRegHipError("run one step with the same parameters' gradients before the capture: their step count is shared "
                                               "with parameters that have none")
                own.setdefault(id(t), t.clone())
                for s in ss:
                    s["step"] = own[id(t)]

    @staticmethod
    def _calls(gi, ps, gs, ss):
        """[(group index, params, grads, states)]: one for the parameters of a group that have one type, device and step count."""
        t = ss[0]["step"]
        if all(s["step"] is t or (not isinstance(t, _T) and s["step"] == t) for s in ss) and len({p.dtype for p in ps}) == 1 and \
                len({p.device for p in ps}) == 1:
            return [(gi, ps, gs, ss)]
        calls = {}
        for p, g, s in zip(ps, gs, ss):
            t = s["step"]
            c = calls.setdefault((p.dtype, p.device, id(t) if isinstance(t, _T) else t), (gi, [], [], []))
            c[1].append(p), c[2].append(g), c[3].append(s)
        return list(calls.values())

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("amsgrad and maximize are not built")
            if group.get("weight_decay") and group.get("decoupled_weight_decay") is False:
                raise ValueError("the checkpoint's weight_decay is an L2 term of the gradient (torch.optim.Adam), which is not built")
        want = set(_TYPES8) if self.state_bits == 8 else {"exp_avg", "exp_avg_sq"}
        for s in state_dict["state"].values():
            if set(s) != want | {"step"}:
                raise ValueError(f"the checkpoint's states {sorted(s)} are not those of state_bits={self.state_bits}")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        ours = [p for g in self.param_groups for p in g["params"]]
        held = [(p, state_dict["state"][i]) for i, p in zip(ids, ours) if i in state_dict["state"]]
        for p, src in held:
            for k in sorted(want):
                dtype = _TYPES8[k] if self.state_bits == 8 else torch.float32
                shape = (-(-p.numel() // BLOCK),) if k.endswith("_scale") else tuple(p.shape)
                if tuple(src[k].shape) != shape or src[k].dtype != dtype:
                    raise ValueError(f"the checkpoint's {k} is {src[k].dtype} {tuple(src[k].shape)}, needed: {dtype} {shape}")
        super().load_state_dict(state_dict)
        # the base class casts every state to its parameter's type: take the checkpoint's own values again
        shared = {}
        for p, src in held:
            t = int(src["step"])
            if self.capturable:
                if (p.device, t) not in shared:
                    shared[p.device, t] = torch.tensor(t, dtype=torch.int64, device=p.device)
                t = shared[p.device, t]
            self.state[p] = {"step": t, **{k: src[k].detach().to(device=p.device, copy=True).contiguous() for k in sorted(want)}}
        for group in self.param_groups:
            for k, v in self.defaults.items():
                group.setdefault(k, v)

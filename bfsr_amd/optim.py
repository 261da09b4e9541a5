"""The end of a training step on the HIP kernels, for the modules that `linf/train.py` trains: gradient clipping by the global norm and Adam (the optimizer
of LINF-LP/train.py:46-62).  Both take any list of dense float32 / float16 / bfloat16 parameters on one GPU in a few launches (ops.tensor_list, ops.adam),
and neither waits for the device; but the first step with a set of parameters that have gradients makes its table, and waits for the current stream once.

`Adam` is a `torch.optim.Optimizer`: parameter groups, learning-rate schedulers and checkpoints work as with `torch.optim.Adam` / `AdamW`, whose
state dicts it reads and whose state it writes (`step`, `exp_avg`, `exp_avg_sq`; moments are float32 whatever the parameter's type)."""
import torch

from .ops import HipOps, _order

_shared = {}
PLANS = 4                  # sets of parameters with gradients that a group remembers (64 bytes of table a parameter each)


def _ops_of(t, ops=None):
    """The ops object for the device of `t`: the given one, or one that calls without it share."""
    if t.device.type != "cuda":
        raise ValueError("bfsr_amd.optim: need parameters on a GPU, got one on %s" % t.device)
    if ops is None:
        ops = _shared.get(t.device)
        if ops is None:
            ops = _shared[t.device] = HipOps(t.device)
    return ops


def clip_grad_norm(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, ops=None):
    """Scales the gradients of `parameters` (those that have one) in place so that their global norm (2 or inf) is at most `max_norm`; returns the norm before,
    a 0-d float32 tensor on the device.  error_if_nonfinite: waits for the norm and raises if it is infinite or NaN (the gradients are then scaled already:
    zero or NaN).  May be captured into a graph."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    ops = ops or _ops_of(grads[0])
    norm = ops.clip_grads(grads, max_norm, norm_type)
    if error_if_nonfinite and not torch.isfinite(norm):
        raise RuntimeError("bfsr_amd.optim.clip_grad_norm: the norm of the gradients is %r" % float(norm))
    return norm


class Adam(torch.optim.Optimizer):
    """Adam, with L2 regularisation (`weight_decay`) or, with `decoupled_weight_decay`, AdamW's decay.

    max_grad_norm     clip the gradients of all groups by their global norm, within the update: p.grad is left as it is
    skip_nonfinite    a step whose gradients' norm is infinite or NaN changes nothing, step counts included
    `grad_norm` holds the last step's norm (0-d, on the device) where one of the two is asked for.
    A group's lr may be a tensor of one float32 on the device; a step captured into a graph then follows it.  Capture after one ordinary step with the
    same parameters' gradients, and again after load_state_dict: state and rate are new tensors then, and a graph goes on with the old ones, which it holds."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled_weight_decay=False, max_grad_norm=None, skip_nonfinite=False,
                 ops=None):
        self._check(lr, betas, eps, weight_decay)
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError("Adam: max_grad_norm %r is out of range" % (max_grad_norm,))
        self.max_grad_norm, self.skip_nonfinite, self.grad_norm = max_grad_norm, skip_nonfinite, None
        self._ops, self._plans = ops, {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled_weight_decay=decoupled_weight_decay))

    @staticmethod
    def _check(lr, betas, eps, weight_decay):
        if isinstance(lr, torch.Tensor):                 # its value now, where it can be waited for
            ok = lr.numel() == 1 and (lr.is_cuda and torch.cuda.is_current_stream_capturing() or float(lr) >= 0.0)
        else:
            ok = lr >= 0.0
        if not ok or not eps >= 0.0 or not weight_decay >= 0.0 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("Adam: lr %r, eps %r, weight_decay %r or betas %r out of range" % (lr, eps, weight_decay, betas))

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            self._check(**{k: param_group.get(k, self.defaults[k]) for k in ("lr", "betas", "eps", "weight_decay")})
        super().add_param_group(param_group)

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans = {}
        for name, value in (("_ops", None), ("max_grad_norm", None), ("skip_nonfinite", False), ("grad_norm", None)):
            self.__dict__.setdefault(name, value)
        for group in self.param_groups:
            group.setdefault("decoupled_weight_decay", False)

    def __getstate__(self):
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm, skip_nonfinite=self.skip_nonfinite)

    def load_state_dict(self, state_dict):
        loading = {}

        def last(_, d):
            """What the program's own hooks have made of the dict."""
            if any(g.get("amsgrad") or g.get("maximize") for g in d["param_groups"]):
                raise ValueError("Adam: amsgrad and maximize are not supported")
            # AdamW did not always write the key: such a group goes on with the decay that it has here
            groups = [dict(g) for g in d["param_groups"]]
            for group, here in zip(groups, self.param_groups):
                group.setdefault("decoupled_weight_decay", here["decoupled_weight_decay"])
            loading.update(d, param_groups=groups)
            return loading

        hook = self.register_load_state_dict_pre_hook(last)
        try:
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
        state_dict = loading
        # torch casts loaded moments to the parameter's type and leaves `step` where it was: take both from the dict as they are
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, [p for g in self.param_groups for p in g["params"]]):
            loaded = state_dict["state"].get(i)
            if loaded:
                self.state[p] = {"step": torch.as_tensor(loaded["step"], dtype=torch.float32).detach().clone().reshape(()).to(p.device)}
                for name in ("exp_avg", "exp_avg_sq"):
                    self.state[p][name] = self._moment(p).copy_(loaded[name].detach())

    @staticmethod
    def _moment(p):
        return torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format, requires_grad=False)

    def _state_of(self, params):
        state = [self.state[p] for p in params]
        if all(state):
            return state
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("Adam: take an ordinary step before the capture begins (it makes the state)")
        new = [p for p, s in zip(params, state) if not s]
        for p, step in zip(new, torch.zeros(len(new), dtype=torch.float32, device=new[0].device).unbind()):
            self.state[p] = {"step": step, "exp_avg": self._moment(p), "exp_avg_sq": self._moment(p)}
        return [self.state[p] for p in params]

    @staticmethod
    def _where(params, state):
        """What tells the memory of a step: its addresses, and the parameters' orders of axes (set anew, one may be a transposed view of what it was)."""
        where = [t.stride() for t in params]
        where += [t.data_ptr() for t in params]
        for name in ("exp_avg", "exp_avg_sq", "step"):
            where += [s[name].data_ptr() for s in state]
        return where

    def _fitting(self, at, ops, where, grads):
        """A plan of the group that names this memory and takes these gradients, and where they are."""
        for held in self._plans.get(at, ()):
            if held[0] is ops and held[1] == where:
                found = held[2].fit(grads)
                if found is not None:
                    return held[2], found
        return None, None

    @staticmethod
    def _refuse_sparse(grads):
        if any(g.is_sparse for g in grads):
            raise RuntimeError("Adam: sparse gradients are not supported")

    def _plan(self, at, params, grads):
        """The group's plan of these parameters, if one still names the memory that they and their state have, or a new one; the gradients in its order of axes, and where they are."""
        if at not in self._plans:
            self._refuse_sparse(grads)
        ops = self._ops or _ops_of(params[0])
        state = self._state_of(params)
        where = self._where(params, state)
        plan, found = self._fitting(at, ops, where, grads)
        if found is None:
            self._refuse_sparse(grads)               # which no plan fits
            grads = [g if _order(g) == _order(p) and not g.is_neg() else torch.empty_like(p, dtype=g.dtype).copy_(g) for p, g in zip(params, grads)]
            plan, found = self._fitting(at, ops, where, grads)
        if found is None:
            bring = all(g.dtype == p.dtype for p, g in zip(params, grads))
            plan = ops.adam(params, None if bring else grads, *[[s[k] for s in state] for k in ("exp_avg", "exp_avg_sq", "step")])
            plan.grads = None                        # every step brings its own: these are not held, since zero_grad may want to free them
            found = plan.fit(grads)
            if found is None:                        # without addresses the plan would go by its own column, which may be the parameters
                raise ValueError("Adam: gradients that do not go with their parameters")
            # older plans of other memory go: they hold what parameters and state were before
            kept = [h for h in self._plans.get(at, ()) if all(self.state.get(p) for p in h[3]) and h[1] == self._where(h[3], [self.state[p] for p in h[3]])]
            self._plans[at] = [(ops, where, plan, params)] + kept[:PLANS - 1]
        return plan, grads, found

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for at, group in enumerate(self.param_groups):
            params = group["params"]
            grads = [p.grad for p in params]
            if any(g is None for g in grads):
                params = [p for p, g in zip(params, grads) if g is not None]
                grads = [g for g in grads if g is not None]
            if params:
                work.append((group, *self._plan(at, params, grads)))
        self.grad_norm = None
        wants = self.max_grad_norm is not None or self.skip_nonfinite
        norm = None
        if wants and len(work) > 1:
            ops = work[0][1].ops
            norm = ops.grad_norm([g for w in work for g in w[2]])
        for group, plan, _, found in work:
            lr = group["lr"]
            if isinstance(lr, torch.Tensor) and lr.device.type == "cpu":
                lr = float(lr)
            got = plan._run(found, lr, group["betas"], group["eps"], group["weight_decay"], group["decoupled_weight_decay"], self.max_grad_norm, 2.0, norm,
                            self.skip_nonfinite)
            self.grad_norm = got if norm is None else norm
        return loss

"""AdamW whose step is one launch for all tensors of a parameter group, on top of the C ABI.

Counterpart of the optimizer of the reference's repro_torch (Adam / AdamW over repro_nn_cuda/repro_nn.cuh:12-21), with
the moments held in FP32 or in 8 bits.  Every value goes through the same fixed sequence of IEEE single operations
(include/rgb200_train.h, rgb200_adamw_step), so the parameters' bits depend on the gradients and the hyper-parameters alone.
CUDA float32 parameters only; there is no CPU path.
"""
import ctypes as C
import operator
import sys

import numpy as np
import torch

from . import _lib
from .repro_gemm import ReproGemmError, _on, _raw_stream, cudaSuccess

_torch_optimizer = sys.modules[torch.optim.Optimizer.__module__]        # torch.optim hides the module's own name

STATE_BLOCK = 256           # values of a tensor that share one scale (8-bit states)

# What torch's AdamW keeps in a group beside the hyper-parameters: variants of the step, with the value that means the plain one, and switches between
# equivalent ways to compute it.
_VARIANTS = dict(amsgrad=False, maximize=False, differentiable=False, decoupled_weight_decay=True)
_SWITCHES = ("foreach", "fused", "capturable")

_nbytes = operator.attrgetter("nbytes")

# one row of the C ABI's rgb200_adamw_tensor
_ROW = np.dtype([(n, np.uint64) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")] +
                [("count", np.int64)])


def _counter(n):
    """A number of steps done, as a tensor that several states can share."""
    return torch.tensor(int(n), dtype=torch.int64, device="cpu")


def _same(a, b):
    """Whether two lists hold the same objects (parameters have an == of their own)."""
    return len(a) == len(b) and all(map(operator.is_, a, b))


def _blocks(n):
    return -(-n // STATE_BLOCK)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay: ``step()`` is one kernel launch per parameter group (per 448 tensors).

    ``state_bits``: 32, or 8 for codes with one scale per 256 values (2.03 instead of 8 bytes of state a parameter).
    ``capturable``: steps are counted on the device, so that ``step()`` can be captured into a CUDA graph and replayed; all
    parameters must then have gradients, and the captured learning rate and other hyper-parameters stay as they were.
    Without it a step under capture is refused, and so is the first step of a group's parameters: it makes their states.  Parameters must not overlap in memory.  The tensors in ``state`` are updated in
    place; to put others in their place use ``adopt`` or ``load_state_dict``.

    ``state_dict()`` holds the moments' values in float32 whatever ``state_bits`` is, and ``load_state_dict`` takes such a
    dict into either width (values pass through the codes again, which returns the same codes)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, capturable=False):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self.state_bits, self.capturable = state_bits, capturable
        self._tables, self._held = {}, []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            _check_hyper(group)
            seen = set()
            for p in group["params"]:
                if id(p) in seen:
                    raise ValueError("a parameter appears twice in the group")
                seen.add(id(p))
                _check_param(p, "parameter")
            if len({p.device for p in group["params"]}) > 1:
                raise ValueError("the parameters of one group must be on one device")
        except Exception:
            self.param_groups.pop()
            raise

    def __getstate__(self):
        for index, t in self._tables.items():
            self._steps(t)
        return {**super().__getstate__(), "state_bits": self.state_bits, "capturable": self.capturable}

    def __setstate__(self, state):
        self._tables, self._held = {}, []            # addresses of the original's tensors do not travel
        super().__setstate__(state)

    # -- states --------------------------------------------------------------------------------------------------
    def _state(self, p):
        s = self.state[p]
        if not s:
            n, dev = p.numel(), p.device
            s["step"] = 0
            if self.state_bits == 32:
                s["exp_avg"], s["exp_avg_sq"] = torch.zeros_like(p), torch.zeros_like(p)
            else:
                s["exp_avg"] = torch.zeros(n, dtype=torch.int8, device=dev)
                s["exp_avg_sq"] = torch.zeros(n, dtype=torch.uint8, device=dev)
                s["exp_avg_scale"] = torch.zeros(_blocks(n), device=dev)
                s["exp_avg_sq_scale"] = torch.zeros(_blocks(n), device=dev)
        return s

    def _names(self):
        return ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if self.state_bits == 8 else ())

    def adopt(self, states, step):
        """Continues from state tensors the caller already holds, without copying them: for each parameter (in group
        order) ``(exp_avg, exp_avg_sq)`` in float32, or with 8-bit states ``(exp_avg int8, exp_avg_sq uint8, exp_avg_scale,
        exp_avg_sq_scale)``.  ``step``: the number of steps done.  The tensors are updated in place from then on.  A step
        captured into a CUDA graph before goes on using the states it was captured with, which stay allocated: capture it again."""
        params = [p for g in self.param_groups for p in g["params"]]
        names = self._names()
        if len(states) != len(params):
            raise ValueError("%d states for %d parameters" % (len(states), len(params)))
        if int(step) < 0:
            raise ValueError("step must not be negative")
        types = (torch.float32,) * 2 if self.state_bits == 32 else (torch.int8, torch.uint8, torch.float32, torch.float32)
        for p, st in zip(params, states):
            if len(st) != len(names):
                raise ValueError("each state is %s" % ", ".join(names))
            for t, name, dtype in zip(st, names, types):
                n = _blocks(p.numel()) if name.endswith("scale") else p.numel()
                if t.dtype != dtype or t.device != p.device or t.numel() != n or not t.is_contiguous():
                    raise ValueError("%s must be a contiguous %s tensor of %d values on %s" % (name, dtype, n, p.device))
        for p, st in zip(params, states):
            self.state[p] = dict(step=int(step), **dict(zip(names, st)))
        old, self._tables = list(self._tables.values()), {}
        self._hold(old)
        for index, group in enumerate(self.param_groups):
            if group["params"]:
                with _on(group["params"][0].device):
                    self._table(index)

    def _table(self, index):
        """The C ABI's rows for one group; parameter and gradient addresses are filled in at each call.  A table belongs to the parameters it was
        made for: a group that has others by now (exchanged, reordered, more, or another group in its place) gets one of its own."""
        group = self.param_groups[index]
        t = self._tables.get(index)
        if t is None or not _same(t["params"], group["params"]):
            if torch.cuda.is_current_stream_capturing():      # states and counters made here would be set to zero by every replay
                raise RuntimeError("AdamW needs a step of these parameters, adopt() or load_state_dict() before it is captured")
            self._settle()
            t = self._tables.get(index)
        if t is None:
            states = [self._state(p) for p in group["params"]]
            rows = np.zeros(len(states), _ROW)
            for name in self._names():
                rows[name] = [s[name].data_ptr() for s in states]
            counts = [s["exp_avg"].numel() for s in states]
            rows["count"] = counts
            steps = {int(s["step"]) for s in states}
            device_step = shared = None
            if len(steps) == 1:                      # one counter for all parameters, until a missing gradient parts them
                shared = _counter(steps.pop())
                for s in states:
                    s["step"] = shared
                if self.capturable:
                    device_step = shared.to(group["params"][0].device)
            elif self.capturable and states:
                raise ValueError("capturable: all parameters of a group must have done the same number of steps")
            else:
                for s in states:
                    s["step"] = _counter(s["step"])
            # `kept`: the rows hold addresses, so the tensors behind them must live as long
            t = self._tables[index] = dict(params=list(group["params"]), rows=rows, counts=counts, bytes=[4 * n for n in counts], states=states, step=shared,
                                           kept=[s[n] for s in states for n in self._names()], device_step=device_step,
                                           captured=False)
        return t

    def _settle(self):
        """Reads every counter back from the device, and keeps the tables of the groups that there are, each at its group's index."""
        old = list(self._tables.values())
        for t in old:
            self._steps(t)
        self._tables = {}
        for index, group in enumerate(self.param_groups):
            for t in old:
                if _same(t["params"], group["params"]):
                    self._tables[index] = t
        self._hold(old)

    def _hold(self, tables):
        """Keeps the memory of tables that go out of use, where a CUDA graph was captured with them: a replay still reads and writes it."""
        used = [id(t) for t in self._tables.values()]
        self._held += [t["kept"] + [t["device_step"]] for t in tables if t["captured"] and id(t) not in used]

    def _steps(self, t):
        if t["device_step"] is not None:
            t["step"].fill_(t["device_step"].item())

    # -- the step ------------------------------------------------------------------------------------------------
    def step(self, closure=None):
        # torch wraps step() of every optimizer in a profiler range and its hooks, which takes longer than the step of a small
        # model; here the wrapped form runs only when a hook is registered (or the profiler is on)
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or torch.autograd.profiler._is_profiler_enabled or
                getattr(_torch_optimizer, "_global_optimizer_pre_hooks", None) or
                getattr(_torch_optimizer, "_global_optimizer_post_hooks", None)):
            return _hooked_step(self, closure)
        return self._step(closure)

    step.hooked = True                  # tells torch.optim.Optimizer not to wrap it again

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for index, group in enumerate(self.param_groups):
            if group["params"]:
                with _on(group["params"][0].device):
                    self._step_group(index, group)
        return loss

    def _step_group(self, index, group):
        capturing = torch.cuda.is_current_stream_capturing()
        if capturing and not self.capturable:
            raise RuntimeError("AdamW.step under CUDA graph capture needs capturable=True")
        t = self._table(index)
        if capturing:
            t["captured"] = True
        if t["step"] is None or not self._ready(t, group["params"]):
            return self._step_checked(group, t)
        torch.autograd.graph.increment_version(group["params"])
        if t["device_step"] is not None:
            self._launch(group, t["rows"], 0, t["device_step"].data_ptr())
        else:
            self._launch(group, t["rows"], int(t["step"]) + 1, None)
            t["step"].add_(1)                        # a refused launch is not a step

    @staticmethod
    def _ready(t, params):
        """Enters the addresses of the usual case, every parameter and gradient a contiguous float32 tensor of its size on the group's device;
        False for anything else.  A few passes over the list in C: a step over many small tensors costs what the host spends on each."""
        T, nbytes, dev = torch.Tensor, _nbytes, {t["kept"][0].get_device()}
        try:
            grads = [p.grad for p in params]
            # of the floating types only float32 has four bytes
            if not (list(map(nbytes, params)) == t["bytes"] == list(map(nbytes, grads)) and set(map(T.get_device, params)) == dev == set(map(T.get_device, grads)) and
                    all(map(T.is_contiguous, params)) and all(map(T.is_contiguous, grads))):
                return False
            addresses = list(map(T.data_ptr, params)), list(map(T.data_ptr, grads))
        except (AttributeError, TypeError, RuntimeError):        # a gradient that is None or not dense
            return False
        t["rows"]["param"], t["rows"]["grad"] = addresses
        return True

    def _step_checked(self, group, t):
        """Missing gradients, gradients to be laid out, parameters that have done different numbers of steps; and the errors."""
        params, states, rows, counts = group["params"], t["states"], t["rows"], t["counts"]
        grads = [p.grad for p in params]
        live = [i for i, g in enumerate(grads) if g is not None]
        if len(live) != len(params):
            if self.capturable:
                raise RuntimeError("capturable: every parameter of the group needs a gradient")
            if not live:
                return
            params, states, grads = ([x[i] for i in live] for x in (params, states, grads))
            rows, counts = np.ascontiguousarray(rows[live]), [counts[i] for i in live]
        T, dev = torch.Tensor, {t["kept"][0].get_device()}
        if {g.dtype for g in grads} != {torch.float32} or {g.layout for g in grads} != {torch.strided} or set(map(T.get_device, grads)) != dev:
            raise TypeError("gradients must be dense float32 tensors on the parameter's device")
        if not all(map(T.is_contiguous, grads)):
            grads = [g.detach().contiguous() for g in grads]          # alive until the launch below is enqueued
        if {p.dtype for p in params} != {torch.float32} or set(map(T.get_device, params)) != dev or not all(map(T.is_contiguous, params)):
            raise ValueError("parameters must stay contiguous float32 tensors on the device they were on")
        if list(map(T.numel, params)) != counts or list(map(T.numel, grads)) != counts:
            raise ValueError("parameters and gradients must keep the size the states were made for")
        rows["param"], rows["grad"] = list(map(T.data_ptr, params)), list(map(T.data_ptr, grads))
        # the kernel writes through addresses: tell autograd, so that a graph that saved the old values refuses them
        torch.autograd.graph.increment_version(params)
        if t["device_step"] is not None:
            self._launch(group, rows, 0, t["device_step"].data_ptr())
            return
        if t["step"] is not None and len(live) == len(group["params"]):
            self._launch(group, rows, int(t["step"]) + 1, None)
            t["step"].add_(1)
            return
        if t["step"] is not None:                    # from here on each parameter counts for itself
            t["step"] = None
            for s in t["states"]:
                s["step"] = s["step"].clone()
        steps = [int(s["step"]) + 1 for s in states]
        for n in sorted(set(steps)):
            these = [i for i, k in enumerate(steps) if k == n]
            self._launch(group, np.ascontiguousarray(rows[these]), n, None)
            for i in these:
                states[i]["step"].add_(1)

    def _launch(self, group, rows, n, device_step):
        b1, b2 = group["betas"]
        h = _lib.AdamwHyper(float(group["lr"]), float(b1), float(b2), float(group["eps"]), float(group["weight_decay"]), n,
                            device_step, self.state_bits)
        rc = _lib.lib().rgb200_adamw_step(rows.ctypes.data, len(rows), C.byref(h), _raw_stream(group["params"][0].device))
        if rc != cudaSuccess:
            raise ReproGemmError(rc, "adamw_step")

    # -- values of the moments -----------------------------------------------------------------------------------
    @torch.no_grad()
    def read_states(self, exp_avgs, exp_avg_sqs):
        """Writes the moments' values into the given contiguous float32 tensors, one for each parameter in group order."""
        self._values("rgb200_adamw_states_read", exp_avgs, exp_avg_sqs)

    @torch.no_grad()
    def write_states(self, exp_avgs, exp_avg_sqs):
        """The reverse of read_states: the moments become the given values (their nearest codes with 8-bit states)."""
        self._values("rgb200_adamw_states_write", exp_avgs, exp_avg_sqs)

    def _values(self, call, ms, vs):
        count = sum(len(g["params"]) for g in self.param_groups)
        if len(ms) != count or len(vs) != count:
            raise ValueError("one tensor is needed for each of the %d parameters" % count)
        at = 0
        for index, group in enumerate(self.param_groups):
            params = group["params"]
            if not params:
                continue
            t = self._table(index)
            gm, gv, dev = ms[at:at + len(params)], vs[at:at + len(params)], params[0].device
            at += len(params)
            both, T = [*gm, *gv], torch.Tensor
            if {x.dtype for x in both} != {torch.float32} or set(map(T.get_device, both)) != {dev.index} or list(map(T.numel, both)) != t["counts"] * 2 or \
                    not all(map(T.is_contiguous, both)):
                raise ValueError("the moments' values are contiguous float32 tensors of the parameters' sizes on their device")
            with _on(dev):
                if self.state_bits == 32:
                    for s, m, v in zip(t["states"], gm, gv):
                        pairs = ((m, s["exp_avg"]), (v, s["exp_avg_sq"]))
                        for x, own in pairs:
                            (x.view(-1).copy_(own.view(-1)) if call.endswith("read") else own.view(-1).copy_(x.view(-1)))
                    continue
                rows = t["rows"].copy()
                rows["param"], rows["grad"] = list(map(T.data_ptr, gm)), list(map(T.data_ptr, gv))
                rc = getattr(_lib.lib(), call)(rows.ctypes.data, len(rows), _raw_stream(dev))
                if rc != cudaSuccess:
                    raise ReproGemmError(rc, call[7:])

    def state_dict(self):
        for hook in list(self._optimizer_state_dict_pre_hooks.values()):
            hook(self)
        made = self._state_dict()
        for hook in list(self._optimizer_state_dict_post_hooks.values()):
            changed = hook(self, made)
            made = made if changed is None else changed
        return made

    def _state_dict(self):
        params = [p for g in self.param_groups for p in g["params"]]
        ms, vs = ([torch.zeros(p.shape, dtype=torch.float32, device=p.device) for p in params] for _ in range(2))
        self.read_states(ms, vs)
        for index in range(len(self.param_groups)):
            if self.param_groups[index]["params"]:
                self._steps(self._tables[index])
        at, groups = 0, []
        for g in self.param_groups:
            n = len(g["params"])
            groups.append({**{k: v for k, v in g.items() if k != "params"}, "params": list(range(at, at + n))})
            at += n
        state = {i: dict(step=int(self.state[p]["step"]), exp_avg=ms[i], exp_avg_sq=vs[i]) for i, p in enumerate(params)}
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, state_dict):
        """Takes what state_dict returns, or the state_dict of torch.optim.AdamW with the same groups.  A dictionary that cannot be taken as it is
        (other groups or sizes, hyper-parameters out of range, variants of the step that this class has not) is refused before anything changes."""
        state_dict = dict(state_dict)                # hooks may change the dictionary, not the caller's
        for hook in list(self._optimizer_load_state_dict_pre_hooks.values()):
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        self._load_state_dict(state_dict)
        for hook in list(self._optimizer_load_state_dict_post_hooks.values()):
            hook(self)

    def _load_state_dict(self, state_dict):
        groups, params = state_dict["param_groups"], [p for g in self.param_groups for p in g["params"]]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the loaded state has other parameter groups")
        new = []
        for mine, theirs in zip(self.param_groups, groups):
            other = [name for name, plain in _VARIANTS.items() if bool(theirs.get(name, plain)) != plain]
            if other:
                raise ValueError("the loaded state was made with %s, which this AdamW has not" % ", ".join("%s=%s" % (n, theirs[n]) for n in other))
            new.append({k: v for k, v in theirs.items() if k != "params" and k not in _VARIANTS and k not in _SWITCHES})
            _check_hyper({**mine, **new[-1]})
        state = state_dict["state"]
        ids = [i for g in groups for i in g["params"]]
        for p, i in zip(params, ids):
            if i in state:
                missing = [k for k in ("step", "exp_avg", "exp_avg_sq") if k not in state[i]]
                if missing:
                    raise ValueError("the loaded state lacks %s" % ", ".join(missing))
                if any(state[i][k].numel() != p.numel() for k in ("exp_avg", "exp_avg_sq")):
                    raise ValueError("the loaded state has other sizes")
                if int(state[i]["step"]) < 0:
                    raise ValueError("step must not be negative")
        if self.capturable and any(len({int(state[i]["step"]) if i in state else 0 for i in g["params"]}) > 1 for g in groups):
            raise ValueError("capturable: all parameters of a group must have done the same number of steps")
        ms, vs = ([state[i][name].to(device=p.device, dtype=torch.float32).contiguous() if i in state else torch.zeros(p.shape, device=p.device)
                   for p, i in zip(params, ids)] for name in ("exp_avg", "exp_avg_sq"))
        for mine, theirs in zip(self.param_groups, new):
            mine.update(theirs)
        for p, i in zip(params, ids):
            self._state(p)["step"] = int(state[i]["step"]) if i in state else 0
        self.write_states(ms, vs)                    # into the tensors there are: a captured step stays valid
        for t in self._tables.values():
            steps = {int(s["step"]) for s in t["states"]}
            if len(steps) == 1:                      # one counter again, and the captured step's
                t["step"] = _counter(steps.pop())
                for s in t["states"]:
                    s["step"] = t["step"]
                if t["device_step"] is not None:
                    t["device_step"].fill_(int(t["step"]))
            else:
                t["step"] = None
                for s in t["states"]:
                    s["step"] = _counter(s["step"])


def _check_hyper(group):
    for name in ("lr", "eps", "weight_decay"):
        if not float(group[name]) >= 0.0:
            raise ValueError("%s must not be negative" % name)
    if len(group["betas"]) != 2 or not all(0.0 <= float(b) < 1.0 for b in group["betas"]):
        raise ValueError("betas must be two numbers in [0, 1)")


_hooked_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)


def _check_param(p, name):
    if p.dtype != torch.float32:
        raise TypeError("%s must be float32" % name)
    if not p.is_cuda:
        raise RuntimeError("%s is not a CUDA tensor: this library has no CPU path" % name)
    if not p.is_contiguous():
        raise ValueError("%s must be contiguous" % name)

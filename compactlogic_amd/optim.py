"""The optimizer half of a CompactLogic training step on the HIP kernels.

The reference trains with (experiments/experiment_script.py:280-293, :362)::

    loss.backward()
    torch.nn.utils.clip_grad_norm_(model.parameters(), max_norm=grad_clip_norm)   # 10.0
    optimizer.step()                                                              # torch.optim.Adam

`FusedAdam` does both in two launches over all parameters (cl_adam_clip_step): the global
gradient norm, the clipped gradients written back into ``p.grad`` as clip_grad_norm_ leaves
them, and the Adam update of every parameter.  The step count is a device tensor, so a step
captured in a HIP graph replays with correct bias corrections.  Sums have a fixed order: the
update is bitwise reproducible.

`FusedAdamW` is the same with decoupled weight decay over tensors of any type, and with moments in 8
bits (cl_adamw_step); the reference has no counterpart of it.

Differences from torch.optim.Adam: every parameter of the optimizer shares one step count,
which advances on every call (torch advances a parameter's count only when it has a
gradient); amsgrad and maximize are not supported, weight decay by `FusedAdamW` alone.  State dicts interchange
with torch.optim.Adam's: ``state_dict()`` gives each parameter its step as a float32 host
scalar, as Adam keeps it, and after ``load_state_dict`` the shared count resumes from the
loaded steps (which must agree), so the bias corrections continue where they stopped.
"""
from __future__ import annotations

import ctypes
import warnings

import torch

from . import _capi, _native
from . import difflogic_hip as _dl
from . import timing


class _OneCount(torch.optim.Optimizer):
    """An optimizer whose parameters share one step count, a device tensor."""

    _step_t = None

    def _loaded_step(self) -> float:
        """The step count held in the state (after load_state_dict, one of torch's Adam
        optimizers or of these): equal for every parameter that has one, else an error; 0 when
        no parameter has one yet."""
        steps = set()
        for p, _ in self._params():
            st = self.state.get(p, {})
            if "step" in st:
                v = st["step"]
                steps.add(float(v.item() if torch.is_tensor(v) else v))
        if len(steps) > 1:
            raise RuntimeError(f"{type(self).__name__} shares one step count, but the loaded state holds "
                               f"several: {sorted(steps)}")
        return steps.pop() if steps else 0.0

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the shared count is taken from the loaded per-parameter steps at the next step()
        self._step_t = None

    def state_dict(self):
        """torch.optim.Adam's layout: per-parameter step as a float32 host scalar."""
        sd = super().state_dict()
        state, counts = {}, {}
        for k, st in sd["state"].items():
            st = dict(st)
            t = st.get("step")
            if torch.is_tensor(t):
                if id(t) not in counts:      # the parameters share one
                    counts[id(t)] = float(t.item())
                st["step"] = torch.tensor(counts[id(t)], dtype=torch.float32)
            state[k] = st
        sd["state"] = state
        return sd

    def _params(self):
        out = []
        for group in self.param_groups:
            for p in group["params"]:
                out.append((p, group))
        return out


class FusedAdam(_OneCount):
    """clip_grad_norm_(params, max_norm) followed by Adam(lr, betas, eps), fused.

    ``max_norm=None`` (or <= 0) skips the clipping.  All parameters must be HIP tensors of one
    dtype (float32 or float64) on one device."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 max_norm: float | None = 10.0):
        if lr < 0 or eps < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError(f"invalid Adam hyper-parameters lr={lr} betas={betas} eps={eps}")
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps)
        super().__init__(params, defaults)
        self.max_norm = max_norm
        self._step_t = None     # shared device step count
        self._workspace = None

    def load_state_dict(self, state_dict):
        if any("exponents" in st for st in state_dict["state"].values()):
            raise RuntimeError("FusedAdam holds no moments in 8 bits; load them into a FusedAdamW with "
                               "state_bits=32, and its state dict here")
        super().load_state_dict(state_dict)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        items = [(p, g) for p, g in self._params() if p.grad is not None]
        if not items:
            return loss
        p0 = items[0][0]
        dev, dtype = p0.device, p0.dtype
        code = _dl.dtype_code(p0)
        for p, _ in items:
            _dl._check(p, "parameter")
            if p.device != dev or p.dtype != dtype:
                raise RuntimeError("FusedAdam needs all parameters on one device in one dtype")
            if p.grad.dtype != dtype or not p.grad.is_contiguous():
                raise RuntimeError("FusedAdam needs contiguous gradients of the parameter dtype")
            if p.grad.is_sparse:
                raise RuntimeError("FusedAdam does not support sparse gradients")
        groups = {id(g): g for _, g in items}
        hp = {(g["lr"], g["betas"], g["eps"]) for g in groups.values()}
        if len(hp) != 1:
            raise RuntimeError("FusedAdam applies one set of hyper-parameters per call; "
                               "use one optimizer per parameter group setting")
        lr, (beta1, beta2), eps = next(iter(hp))
        if self._step_t is None or self._step_t.device != dev or self._step_t.dtype != dtype:
            start = self._loaded_step() if self._step_t is None else float(self._step_t)
            self._step_t = torch.full((), start, dtype=dtype, device=dev)
        for p, _ in items:
            st = self.state[p]
            if "exp_avg" not in st:
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            for key in ("exp_avg", "exp_avg_sq"):   # loaded moments: the kernel's layout
                t = st[key]
                if t.shape != p.shape:
                    raise RuntimeError(f"FusedAdam state {key} has shape {tuple(t.shape)}, "
                                       f"the parameter {tuple(p.shape)}")
                if not t.is_contiguous() or t.device != dev or t.dtype != dtype:
                    st[key] = t.to(device=dev, dtype=dtype).contiguous()
            st["step"] = self._step_t
        max_t = ctypes.c_int64()
        _capi.call("cl_adam_clip_max_tensors", ctypes.byref(max_t))
        if len(items) > max_t.value:
            raise RuntimeError(f"FusedAdam updates at most {max_t.value} parameter tensors "
                               f"per optimizer, got {len(items)}")
        max_norm = float(self.max_norm) if self.max_norm is not None else 0.0
        ps = [p for p, _ in items]
        n = len(ps)
        arr = ctypes.c_void_p * n
        numels = (ctypes.c_int64 * n)(*[p.numel() for p in ps])
        nparts = ctypes.c_int64()
        _capi.call("cl_adam_clip_workspace", n, numels, ctypes.byref(nparts))
        if self._workspace is None or self._workspace.numel() < max(nparts.value, 1) \
                or self._workspace.device != dev or self._workspace.dtype != dtype:
            self._workspace = torch.empty(max(nparts.value, 1), dtype=dtype, device=dev)
        ptrs = [arr(*[t.data_ptr() for t in ts]) for ts in
                (ps, [p.grad for p in ps], [self.state[p]["exp_avg"] for p in ps],
                 [self.state[p]["exp_avg_sq"] for p in ps])]
        with torch.cuda.device(dev):
            timing.timed(f"cl_adam_clip_step[{sum(numels)}]", lambda: _capi.call(
                "cl_adam_clip_step", code, n, *ptrs, numels, self._step_t.data_ptr(),
                float(lr), float(beta1), float(beta2), float(eps), max_norm,
                self._workspace.data_ptr(), self._workspace.numel(), _dl.stream_of(p0)))
        return loss


class FusedAdamW(_OneCount):
    """clip_grad_norm_(params, max_norm) followed by AdamW(lr, betas, eps, weight_decay) over any
    number of tensors of any of float32, float64, float16 and bfloat16, fused (cl_adamw_step).

    Arithmetic is float32 (float64 for float64 parameters), a parameter of 16 bits is rounded once.
    state_bits=32 holds the moments in that wide type.  state_bits=8 holds them in a byte each, with
    two more for 256 elements (float64 parameters have none): ``exp_avg`` float8_e4m3fn,
    ``exp_avg_sq`` uint8 codes and the blocks' ``exponents``; `moments` gives their values.  The
    update itself takes the new moments before they are rounded to 8 bits.

    rounding="random" rounds them up or down so that they are right on average, by a hash of the step
    count, the parameter's place among those that have a gradient, and the element: a run gives the same
    bits again.  rounding="nearest" is for betas up to 0.9 alone, and warns above: a step that changes a
    moment by less than half of its codes' distance (1/32 to 1/16 of it) does not change it at all.  With a
    beta of 0.9 a moment then stays within 2.25 times of where it belongs.  With
    beta2 = 0.999 exp_avg_sq then stays where the first steps took it: 0.02 of what it should be after 3000
    steps of constant gradients, or a hundred times too much once gradients shrink tenfold.

    lr, betas, eps, weight_decay, state_bits and rounding may differ between parameter groups (at most 32);
    ``max_norm`` is one for all, on the norm over all of them (float64 sums in a fixed order: steps
    are bitwise reproducible); None or <= 0 skips the clipping.  The gradients are left as they are:
    unlike clip_grad_norm_ and FusedAdam, ``p.grad`` is not scaled.  An infinite norm scales finite
    gradients to 0, a norm of NaN scales nothing; what is not finite stays in its own elements.
    Hyper-parameters are read at every call; a step captured in a graph keeps those of its capture, and
    the first step of a parameter, which makes its moments, cannot be captured.

    State dicts interchange with torch.optim.AdamW's (of float32 moments for parameters of any type)
    and between 32 and 8 bits, and FusedAdam's are taken, with the weight_decay that the groups have.
    Tensors that are of the type and on the device already are taken as
    they are, without a copy."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, max_norm: float | None = 10.0, state_bits: int = 32,
                 rounding: str = "nearest"):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, rounding=rounding))
        self.max_norm = max_norm

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:         # (pickled before there was a choice)
            group.setdefault("rounding", "nearest")
        self.defaults.setdefault("rounding", "nearest")

    def add_param_group(self, param_group):
        params = param_group["params"]
        if not isinstance(params, torch.Tensor):
            params = param_group["params"] = list(params)
            if len({id(p) for p in params}) != len(params):
                raise ValueError("a parameter group holds a parameter twice")
        g = {**self.defaults, **param_group}
        b1, b2 = g["betas"]
        if not (g["lr"] >= 0 and g["eps"] >= 0 and g["weight_decay"] >= 0 and 0 <= b1 < 1
                and 0 <= b2 < 1):
            raise ValueError(f"invalid AdamW hyper-parameters lr={g['lr']} betas={g['betas']} "
                             f"eps={g['eps']} weight_decay={g['weight_decay']}")
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {g['state_bits']}")
        if g["rounding"] not in ("nearest", "random"):
            raise ValueError(f"rounding must be 'nearest' or 'random', got {g['rounding']!r}")
        super().add_param_group(param_group)
        if g["state_bits"] == 8 and g["rounding"] == "nearest" and max(b1, b2) > 0.9:
            warnings.warn("FusedAdamW: 8-bit moments rounded to the nearest stay where they are under "
                          f"betas above 0.9, got {tuple(g['betas'])}: pass rounding=\"random\"",
                          stacklevel=4)

    def load_state_dict(self, state_dict):
        if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
            raise RuntimeError("FusedAdamW has no amsgrad and no maximize")
        if any(k not in g for g in state_dict["param_groups"] for k in ("lr", "betas", "eps")):
            raise RuntimeError("the state dict's groups have no lr, betas and eps: it is not one of Adam's")
        before = [dict(g) for g in self.param_groups]
        super().load_state_dict(state_dict)
        for group, old in zip(self.param_groups, before):
            group["state_bits"] = old["state_bits"]     # how moments are held stays as it was
            group["rounding"] = old["rounding"]
            for key, value in old.items():              # (FusedAdam has no weight_decay)
                group.setdefault(key, value)
        # torch has cast the moments to the parameters' types: take them as they were given
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        with torch.no_grad():
            for i, (p, group) in zip(ids, self._params()):
                given = state_dict["state"].get(i)
                if given is not None and "exp_avg" in given:
                    self._hold(p, group, {k: given[k] for k in
                                          ("exp_avg", "exp_avg_sq", "exponents") if k in given})

    def _hold(self, p, group, given):
        """The parameter's moments in the form of its group, from given ones in either."""
        small = group["state_bits"] == 8
        st = self.state[p]
        for name in ("exp_avg", "exp_avg_sq"):
            if given[name].shape != p.shape:
                raise RuntimeError(f"FusedAdamW state {name} has shape "
                                   f"{tuple(given[name].shape)}, the parameter {tuple(p.shape)}")
        given = {k: t.to(p.device).contiguous() for k, t in given.items()}
        if small and p.dtype == torch.float64:
            raise RuntimeError("FusedAdamW holds no moments of float64 parameters in 8 bits")
        if ("exponents" in given) == small:
            wide = torch.float64 if p.dtype == torch.float64 else torch.float32
            if small:
                st.update(given)
            else:
                st.pop("exponents", None)
                st.update({k: t.to(wide) for k, t in given.items()})
        elif small:
            _dl._check(p, "parameter")
            self._empty_small(p, st)
            _native.load().adamw_hold(p, st, given["exp_avg"].float(), given["exp_avg_sq"].float())
        else:
            held = _native.load().adamw_held([p], [given])
            st.pop("exponents", None)
            st["exp_avg"], st["exp_avg_sq"] = (t[0].float() for t in held)

    @staticmethod
    def _empty_small(p, st):
        st["exp_avg"] = torch.zeros(p.shape, dtype=torch.uint8,
                                    device=p.device).view(torch.float8_e4m3fn)
        st["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
        st["exponents"] = torch.ones(2 * (-(-p.numel() // 256)), dtype=torch.uint8, device=p.device)

    @staticmethod
    def _refuse_in_capture():
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW makes its state in the first step, which a graph would make "
                               "again at every replay: step once before the capture")

    def _prepare_states(self):
        """Moments for the parameters that have a gradient and none yet, checked for the others."""
        self._refuse_in_capture()
        for p, group in self._params():
            if p.grad is None:
                continue
            _dl._check(p, "parameter")
            _dl.storage_dtype_code(p)
            st = self.state[p]
            if "exp_avg" in st:
                self._hold(p, group, {k: st[k] for k in ("exp_avg", "exp_avg_sq", "exponents")
                                      if k in st})
            elif group["state_bits"] == 8:
                if p.dtype == torch.float64:
                    raise RuntimeError("FusedAdamW holds no moments of float64 parameters in 8 bits")
                self._empty_small(p, st)
            else:
                wide = torch.float64 if p.dtype == torch.float64 else torch.float32
                for name in ("exp_avg", "exp_avg_sq"):
                    st[name] = torch.zeros(p.shape, dtype=wide, device=p.device)
            st["step"] = self._step_t

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        native = _native.load()
        max_norm = float(self.max_norm) if self.max_norm is not None else 0.0
        if self._step_t is None:
            first = next((p for p, _ in self._params() if p.grad is not None), None)
            if first is None:
                return loss
            _dl._check(first, "parameter")
            self._refuse_in_capture()
            self._step_t = torch.full((), self._loaded_step(), dtype=torch.float64,
                                      device=first.device)
            for st in self.state.values():
                st["step"] = self._step_t
        if not native.adamw_step(self.param_groups, self.state, self._step_t, max_norm):
            with torch.no_grad():
                self._prepare_states()
            if not native.adamw_step(self.param_groups, self.state, self._step_t, max_norm):
                raise RuntimeError("FusedAdamW's state does not fit its parameters")
        return loss

    @torch.no_grad()
    def moments(self, params=None):
        """(first, second): lists of the exponential averages of the gradient and of its square of
        `params` (default: every parameter that has them), in float32 (float64) where they are held
        in 32 bits, and in bfloat16, which holds all of their values from 2^-130 on, where in 8."""
        held = [(p, self.state[p]) for p, _ in self._params() if "exp_avg" in self.state.get(p, {})] \
            if params is None else [(p, self.state.get(p, {})) for p in params]
        first, second, small = [], [], []
        for p, st in held:
            if "exp_avg" not in st:
                raise RuntimeError("a parameter has no moments before its first step")
            small.append("exponents" in st)
            first.append(st["exp_avg"])
            second.append(st["exp_avg_sq"])
        if all(small):
            return _native.load().adamw_held([p for p, _ in held], [st for _, st in held]) \
                if small else (first, second)
        if any(small):
            at = [i for i, s in enumerate(small) if s]
            values = _native.load().adamw_held([held[i][0] for i in at], [held[i][1] for i in at])
            for i, m, v in zip(at, *values):
                first[i], second[i] = m, v
        return first, second

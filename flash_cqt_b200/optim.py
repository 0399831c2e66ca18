"""``AdamW``: the optimizer's step of a training loop around the transform.

The update of every tensor -- and, with ``max_norm``, the global gradient norm
that scales the gradients -- runs in the library's kernels (``csrc/optim.cu``):
one launch for up to 360 tensors, moments in 32 or in 8 bits, nothing read
back to the host.  Counts of steps live on the device, so a captured graph that
holds a step advances them with every replay.

    opt = AdamW([x], lr=1e-2, max_norm=1.0)
    loss = t.mse_loss(*t.fwd(x), target)
    loss.backward()
    opt.step()
"""
import ctypes
import sys

import torch

from . import _native
from .engine import _raw_stream_of

BLOCK = 256   # elements that share a scale in the 8-bit moments
_TYPES = {torch.float32: _native.CQT_F32, torch.bfloat16: _native.CQT_BF16,
          torch.float16: _native.CQT_F16, torch.complex64: _native.CQT_F32}


def _fills(shape, strides):
    """whether elements at these strides fill one stretch of memory"""
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(strides, shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _dense(t):
    """whether the elements fill one stretch of memory, in any order of dims"""
    return t.is_contiguous() or _fills(t.shape, t.stride())


def _same_order(a, b):
    """whether element i of a's memory is element i of b's (both dense)"""
    return all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n != 1)


def _order(p):
    """the memory order of a dense tensor: its sizes over its strides"""
    return torch.tensor([*p.shape, *p.stride()], dtype=torch.int64).view(2, p.dim())


def _ordered_like(order, p):
    shape, strides = order.tolist()
    return shape == list(p.shape) and (strides == list(p.stride()) or all(
        a == b for a, b, n in zip(strides, p.stride(), shape) if n != 1))


def _values8(codes, scales):
    """8-bit moments as float32"""
    return codes.float() * scales.float().repeat_interleave(BLOCK)[:codes.numel()]


def _codes8(x, dtype):
    """(codes, scales) of flat float32 values, rounded to nearest"""
    b = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    top = torch.where(b.isfinite(), b.abs(), 0.0).amax(1)
    # the least 2^k with top <= 1.75 * 2^8 (e4m3) or 1.75 * 2^15 (e5m2) of it
    k = ((top.view(torch.int32) + 0x1fffff >> 23) - (8 if dtype == torch.float8_e4m3fn else 15)
         ).clamp_min(1)
    y = b * (254 - k << 23).view(torch.float32)[:, None]
    if dtype == torch.float8_e5m2:   # a denominator must not vanish
        y = torch.where(b > 0, y.clamp_min(2.0 ** -14), y)
    return (y.view(-1)[:x.numel()].to(dtype),
            k.to(torch.uint8).view(torch.float8_e8m0fnu))


def _relaid(x, order, p):
    """flat values of the elements of ``p`` in another memory order, in p's own"""
    def as_p(x, shape, strides):
        if p.is_complex():   # (re, im) of an element lie together
            shape, strides = [*shape, 2], [*(2 * s for s in strides), 1]
        return x.as_strided(shape, strides)
    out = torch.empty_like(x)
    as_p(out, p.shape, p.stride()).copy_(as_p(x, *order.tolist()))
    return out


def _written(tensors):
    """autograd refuses a backward pass through what it saved of these before"""
    torch.autograd.graph.increment_version(
        [t for t in tensors if torch.is_tensor(t) and not t.is_inference()])


def _reals(t):
    return t.numel() * (2 if t.is_complex() else 1)


def _watched(opt):
    """whether anyone listens to an optimizer's steps: hooks or a profiler"""
    o = sys.modules[torch.optim.Optimizer.__module__]
    return (getattr(torch.autograd.profiler, "_is_profiler_enabled", True)
            or getattr(opt, "_optimizer_step_pre_hooks", True)
            or getattr(opt, "_optimizer_step_post_hooks", True)
            or getattr(o, "_global_optimizer_pre_hooks", True)
            or getattr(o, "_global_optimizer_post_hooks", True))


class AdamW(torch.optim.Optimizer):
    """AdamW over all parameters at once.

    With t the number of steps that a parameter has taken (one with no gradient
    is left out of a step), per real element::

        g' = g * min(1, max_norm / (norm + 1e-6))      norm over all parameters
        m  = b1 m + (1 - b1) g'
        v  = b2 v + (1 - b2) g'^2
        p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    in 32 bits.  Real and imaginary parts of a complex64 parameter are elements
    of their own.  float32, bfloat16, float16 and complex64 parameters on one
    CUDA device, dense in memory (in any order of dimensions).  A gradient in
    another order than its parameter is copied first.

    ``lr`` may be a 0-dim float32 tensor on the device (read by the kernel, so a
    captured step follows it); any other number is fixed when a graph is
    captured.

    ``state_bits=8`` holds the moments in 8 bits: ``exp_avg`` as float8_e4m3fn
    and ``exp_avg_sq`` as float8_e5m2 values in the parameter's memory order
    (``order``: its sizes and strides, int64 [2, dim] on the host; a state without
    it is of a contiguous parameter), 256 of which share a power-of-two scale
    (``exp_avg_scale``, ``exp_avg_sq_scale``, float8_e8m0fnu).  A step refuses a
    parameter whose order has changed; a state that was saved in another order is
    laid out anew when it is loaded, which rounds only what is small beside its
    new neighbours.  They are rounded stochastically by a
    hash of (``seed``, t, the parameter's number, element): the same run gives
    the same bits.  A first moment below 2^-6 of its block's scale is held as 0: an
    element whose gradients stay under about 5e-5 of the largest in its block hardly
    moves (3e-5 of it: 6 % of the update that 32-bit moments give; 1e-4: all of it).  ``master=True`` keeps a 32-bit copy of a 16-bit parameter,
    which is then its rounding; without it a 16-bit parameter loses updates
    below half a step of its type.  Both may differ between parameter groups.

    ``max_norm`` scales the gradients as they are read (they stay as they are
    in memory); ``grad_norm`` is the norm before scaling, a 0-dim float32
    device tensor that every step overwrites, or None without ``max_norm``.
    Gradients that are not finite go through as the formulas say.

    Steps of one optimizer must be ordered on one stream at a time.  State is
    made at a parameter's first step; before a step is captured it has to be
    there (``init_state()``, or a step).  ``load_state_dict`` (which also takes the
    state of ``torch.optim.AdamW``, for 32-bit moments: there is no conversion
    between the widths) writes into the state, and into a rate on the
    device, that are there, so a captured step goes on from what was loaded (a
    parameter that the dictionary has no state for goes back to zeros).
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *,
                 state_bits=32, master=False, max_norm=None, seed=0):
        if max_norm is not None and not float(max_norm) > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        self.max_norm = None if max_norm is None else float(max_norm)
        self.seed = int(seed) & 0xffffffff
        self._reset()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, master=master))

    def _reset(self):
        self._dev = self._ws = self._plan = self.grad_norm = None
        self._retired = []
        self._need = None, 0   # a number of tensors and the workspace for it

    def __getstate__(self):
        return dict(super().__getstate__(), max_norm=self.max_norm, seed=self.seed)

    def __setstate__(self, state):
        super().__setstate__(state)
        if "_retired" not in self.__dict__:   # a new object (load_state_dict comes here too)
            self._reset()
        for g in self.param_groups:
            self._dev = g["params"][0].device if g["params"] else self._dev
        self._total = sum(len(g["params"]) for g in self.param_groups)

    # ------------------------------------------------------------------ checks
    @staticmethod
    def _check_options(g):
        lr, (b1, b2) = g["lr"], g["betas"]
        if torch.is_tensor(lr):
            if lr.numel() != 1:
                raise ValueError(f"a tensor lr must hold one number, got {tuple(lr.shape)}")
            if lr.device.type == "cuda" and lr.dtype != torch.float32:
                raise TypeError(f"a device lr must be float32, got {lr.dtype}")
        if (not torch.is_tensor(lr) or lr.device.type == "cpu") and not float(lr) >= 0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError(f"betas must lie in [0, 1), got {(b1, b2)}")
        if not g["eps"] >= 0 or not g["weight_decay"] >= 0:
            raise ValueError("eps and weight_decay must not be negative")
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {g['state_bits']}")

    def _check_param(self, p):
        if p.dtype not in _TYPES:
            raise TypeError("parameters must be float32, bfloat16, float16 or complex64, "
                            f"got {p.dtype}")
        if p.is_conj() or p.is_neg() or not _dense(p):
            raise ValueError("parameters must be dense in memory (no gaps, no elements "
                             "that share a place, no lazy conjugate)")
        if p.device.type != "cuda":
            raise RuntimeError(f"the optimizer step runs on CUDA devices only, got {p.device} "
                               "(there is no CPU fallback)")
        if self._dev is not None and p.device != self._dev:
            raise ValueError(f"parameters must be on one device: {p.device}, {self._dev}")

    def add_param_group(self, group):
        group = dict(group)
        params = group["params"]
        if isinstance(params, (set, frozenset)):
            raise TypeError("parameters must be in an order of their own: a set has none")
        params = [params] if torch.is_tensor(params) else list(params)
        group["params"] = params
        self._check_options({**self.defaults, **group})
        tensors = [p[1] if isinstance(p, tuple) else p for p in params]
        spans = [s for g in self.param_groups for p in g["params"] for s in self._span(p)]
        for p in tensors:
            if not torch.is_tensor(p):
                raise TypeError(f"parameters must be tensors, got {type(p).__name__}")
            self._check_param(p)
            self._dev = p.device
            spans += self._span(p)
        spans.sort()
        for (_, end), (start, _) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError("two parameters share memory, or one is given twice")
        super().add_param_group(group)
        self._total = sum(len(g["params"]) for g in self.param_groups)

    @staticmethod
    def _span(p):
        a = p.data_ptr()
        return [(a, a + p.numel() * p.element_size())] if p.numel() else []

    # ------------------------------------------------------------------- state
    def _new_state(self, p, g):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the optimizer's state must be there before a step is captured: "
                               "call init_state(), or take a step, first")
        zeros = lambda n, dt: torch.zeros(n, dtype=torch.uint8, device=p.device).view(dt)  # noqa: E731
        s = dict(step=torch.zeros((), dtype=torch.int64, device=p.device))
        if g["state_bits"] == 8:
            n = _reals(p)
            s["exp_avg"] = zeros(n, torch.float8_e4m3fn)
            s["exp_avg_sq"] = zeros(n, torch.float8_e5m2)
            for k in ("exp_avg_scale", "exp_avg_sq_scale"):
                s[k] = zeros(-(-n // BLOCK), torch.float8_e8m0fnu)
                s[k].view(torch.uint8).fill_(1)
            s["order"] = _order(p)
        else:
            dt = torch.complex64 if p.is_complex() else torch.float32
            s["exp_avg"] = torch.zeros_like(p, dtype=dt, requires_grad=False)
            s["exp_avg_sq"] = torch.zeros_like(p, dtype=dt, requires_grad=False)
        if g["master"] and p.dtype in (torch.bfloat16, torch.float16):
            s["master"] = p.detach().float()
        return s

    @staticmethod
    def _check_state(s, p, g):
        """a parameter's state as the kernels take it, or ValueError"""
        eight = g["state_bits"] == 8
        n = _reals(p)
        want = {"exp_avg": torch.float8_e4m3fn, "exp_avg_sq": torch.float8_e5m2,
                "exp_avg_scale": torch.float8_e8m0fnu,
                "exp_avg_sq_scale": torch.float8_e8m0fnu} if eight else \
               dict.fromkeys(("exp_avg", "exp_avg_sq"),
                             torch.complex64 if p.is_complex() else torch.float32)
        if g["master"] and p.dtype in (torch.bfloat16, torch.float16):
            want["master"] = torch.float32
        want["step"] = torch.int64
        for k, dt in want.items():
            t = s.get(k)
            if not torch.is_tensor(t) or t.dtype != dt or t.device != p.device \
                    or t.layout != torch.strided or t.is_conj() or t.is_neg():
                raise ValueError(f"state {k!r} must be a {dt} tensor on {p.device}")
            if k == "step":
                fits = t.numel() == 1
            elif eight and k != "master":
                fits = t.is_contiguous() and t.numel() == (
                    -(-n // BLOCK) if k.endswith("scale") else n)
            else:
                fits = t.shape == p.shape and _dense(t) and _same_order(t, p)
            if not fits:
                raise ValueError(f"state {k!r} does not fit its parameter {tuple(p.shape)}")
        if eight:
            o = s.get("order")
            if o is None:
                if not p.is_contiguous():
                    raise ValueError("state 'order' is missing: 8-bit moments without it are "
                                     "those of a contiguous parameter")
            elif not torch.is_tensor(o) or o.dtype != torch.int64 or o.shape != (2, p.dim()) \
                    or not _ordered_like(o, p):
                raise ValueError("state 'order': the 8-bit moments lie in another memory order "
                                 f"than their parameter {tuple(p.shape)}, {p.stride()}")

    @torch.no_grad()
    def init_state(self):
        """make what a step needs and is not there yet: the state of every
        parameter (zero moments), the workspace"""
        if self._dev is not None:
            self._workspace(self._total)
        for g in self.param_groups:
            for p in g["params"]:
                if not self.state.get(p):
                    self.state[p] = self._new_state(p, g)

    def load_state_dict(self, state_dict):
        """take over the options and the state of ``state_dict``; on a state that
        does not fit, ValueError, and the optimizer is as it was"""
        taken = {}

        def take(_, dictionary):
            # as the user's own hooks left it.  The base class would cast the state
            # to the parameters' types: it only takes the groups
            if any(g.get("amsgrad") or g.get("maximize") for g in dictionary["param_groups"]):
                raise ValueError("amsgrad and maximize do not exist here")
            taken.update(dictionary)
            return dict(dictionary, state={})
        before, was = self.state, self.param_groups   # the base class brings its own
        hooks = [self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(
                     lambda opt: opt._take(taken, before, was), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    @torch.no_grad()
    def _take(self, state_dict, before, was):
        """the state of a dictionary whose groups the base class has taken over"""
        try:
            for g, old in zip(self.param_groups, was):
                for k, v in self.defaults.items():   # what is not said there stays
                    g.setdefault(k, old.get(k, v))
            rates = self._keep_rates(was)
            new = {}
            for old, g in zip(state_dict["param_groups"], self.param_groups):
                for i, p in zip(old["params"], g["params"]):
                    if state_dict["state"].get(i):
                        new[p] = self._loaded(state_dict["state"][i], p, g)
                    elif before.get(p):   # it has taken no step: back to zeros
                        new[p] = self._new_state(p, g)
        except Exception:
            self.state, self.param_groups = before, was
            raise
        for at, rate in rates.items():
            at.fill_(rate)
        for p, s in new.items():
            # into the tensors that are there: a captured step goes on with them
            for k, v in s.items():
                at = before.get(p, {}).get(k)
                if torch.is_tensor(at) and at.dtype == v.dtype and at.shape == v.shape \
                        and at.device == v.device and at.stride() == v.stride():
                    s[k] = at.copy_(v)
        self.state.clear()
        self.state.update(new)

    def _keep_rates(self, was):
        """puts rates that are device tensors back into groups that were loaded (a
        captured step reads them): {tensor: the number that was loaded}"""
        rates = {}
        for g, old in zip(self.param_groups, was):
            at, lr = old["lr"], g["lr"]
            if not torch.is_tensor(at) or at.device != self._dev:
                continue
            if torch.is_tensor(lr) and lr.numel() != 1:
                raise ValueError(f"a tensor lr must hold one number, got {tuple(lr.shape)}")
            if rates.setdefault(at, float(lr)) != float(lr):
                raise ValueError("parameter groups that share one lr tensor cannot take "
                                 f"different rates: {rates[at]}, {float(lr)}")
            g["lr"] = at
        return rates

    def _loaded(self, saved, p, g):
        """a parameter's saved state as new tensors, laid out for the kernels"""
        s = {}
        eight = g["state_bits"] == 8
        for k, v in saved.items():
            if k == "order":
                continue
            if k == "step":
                s[k] = torch.as_tensor(v).detach().to(p.device, torch.int64).reshape(()).clone()
            elif torch.is_tensor(v):
                v = v.detach().to(p.device, copy=True)
                if not eight and v.dtype in (torch.bfloat16, torch.float16):
                    v = v.float()   # moments that were kept in the parameter's type
                if v.shape == p.shape and not _same_order(v, p):
                    v = torch.empty_like(p, dtype=v.dtype, requires_grad=False).copy_(v)
                s[k] = v
        if g["master"] and "master" not in s and p.dtype in (torch.bfloat16, torch.float16):
            s["master"] = p.detach().float()
        order = saved.get("order")
        if eight and order is not None:
            s["order"] = _order(p)
        self._check_state(s, p, g)
        if eight and order is not None:
            order = torch.as_tensor(order).cpu()
            if order.shape != (2, p.dim()) or order[0].tolist() != list(p.shape) \
                    or not _fills(*order.tolist()):
                raise ValueError(f"state 'order' does not fit its parameter {tuple(p.shape)}")
            if not _ordered_like(order, p):
                for k in ("exp_avg", "exp_avg_sq"):
                    s[k], s[k + "_scale"] = _codes8(
                        _relaid(_values8(s[k], s[k + "_scale"]), order, p), s[k].dtype)
        return s

    # -------------------------------------------------------------------- step
    def _grad(self, p):
        g = p.grad
        if g.is_sparse or g.layout != torch.strided:
            raise RuntimeError("sparse gradients are not supported")
        if g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
            raise ValueError(f"a gradient must be {p.dtype} {tuple(p.shape)} on {p.device}, got "
                             f"{g.dtype} {tuple(g.shape)} on {g.device}")
        if g.is_conj() or g.is_neg() or not _dense(g) or not _same_order(g, p):
            g = torch.empty_like(p, requires_grad=False).copy_(g)
        return g

    def _workspace(self, count):
        """grow-only; an outgrown one is kept: a captured graph may address it"""
        if self._need[0] != count:
            self._need = count, _native.lib().cqt_adamw_workspace_bytes(count)
        need = self._need[1]
        if self._ws is None or self._ws.numel() < need or (
                self.max_norm is not None and self.grad_norm is None):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the optimizer's workspace must be there before a step is "
                                   "captured: call init_state(), or take a step, first")
            self._retired.append(self._ws)
            self._ws = torch.zeros(need, dtype=torch.uint8, device=self._dev)
            if self.max_norm is not None and self.grad_norm is None:
                self.grad_norm = torch.zeros((), dtype=torch.float32, device=self._dev)
        return self._ws

    def step(self, closure=None):
        """one step of every parameter that has a gradient; returns what
        ``closure`` (evaluated first, with gradients enabled) returns"""
        if _watched(self):
            return _hooked_step(self, closure)
        return self._step(closure)

    # the base class would wrap step() in its profiler label and hooks at every
    # call (8 us); _watched() takes that way when there is one to serve
    step.hooked = True

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._dev is None:
            return loss
        mod = _native.torch_ops()
        if mod is None:
            self._python_step()
        elif self._plan is None or not self._plan_step():
            # the first step, or states, parameters or groups were replaced
            self._lists(plan=True)
            if self._plan is not None and self._plan.captured:
                self._retired.append(self._plan)   # a graph writes to its tensors
            self._plan = mod.AdamWPlan(
                self._dev.index, *[_native.fn_address(n) for n in (
                    "cqt_grad_norm", "cqt_adamw_step", "cqt_last_error")],
                self.param_groups, self.state)
            if not self._plan_step():
                raise RuntimeError("the optimizer's parameters changed during the step")
        return loss

    def _plan_step(self):
        ws = self._workspace(self._total)
        return self._plan.step(self.param_groups, self.state, self.max_norm, self.seed, ws,
                               self.grad_norm)

    @torch.no_grad()
    def _lists(self, plan=False):
        """the tensors of every group that have gradients, as the library takes
        them (states are made and checked), and (gradient or its copy, parameter,
        state) of each; for a plan, which looks at the rest itself, states only"""
        lists, keep = [], []
        first = 0
        for g in self.param_groups:
            self._check_options(g)
            todo = []
            for k, p in enumerate(g["params"]):
                if p.grad is None or not p.numel():
                    continue
                self._check_param(p)   # its storage may have been exchanged
                s = self.state.get(p)
                if s:
                    self._check_state(s, p, g)
                else:
                    s = self.state[p] = self._new_state(p, g)
                if g["state_bits"] == 8 and "order" not in s:
                    s["order"] = _order(p)
                if plan:
                    continue
                grad = self._grad(p)
                keep.append((grad, p, s))
                at = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
                todo.append(_native.CqtAdamwTensor(
                    p.data_ptr(), grad.data_ptr(), at("master") if g["master"] else None,
                    at("exp_avg"), at("exp_avg_sq"), at("exp_avg_scale"), at("exp_avg_sq_scale"),
                    at("step"), _reals(p), _TYPES[p.dtype], first + k))
            first += len(g["params"])
            lists.append((_native.CqtAdamwTensor * len(todo))(*todo))
        return lists, keep

    def _python_step(self):
        with torch.cuda.device(self._dev):
            lists, keep = self._lists()
            if self.max_norm is not None:
                self._workspace(self._total)
                n = self.grad_norm
                if n.device != self._dev or n.numel() != 1 or n.dtype != torch.float32:
                    raise ValueError(f"grad_norm must hold one float32 number on {self._dev}")
                _written([n])
            _written([t for _, p, s in keep for t in (p, *s.values())])
            if torch.cuda.is_current_stream_capturing():
                # the graph addresses these even when they have been replaced
                self._retired.append((self.grad_norm, [g["lr"] for g in self.param_groups],
                                      [(p, *s.values()) for _, p, s in keep]))
            self._launch(lists)

    def _launch(self, lists):
        L, stream = _native.lib(), _raw_stream_of(self._dev.index)
        ws = self._workspace(self._total)
        if self.max_norm is not None:
            every = lists[0] if len(lists) == 1 else (
                (_native.CqtAdamwTensor * sum(map(len, lists)))(*(t for x in lists for t in x)))
            _native._check(L.cqt_grad_norm(every, len(every), self.grad_norm.data_ptr(),
                                           ws.data_ptr(), ws.numel(), stream), "cqt_grad_norm")
        use_norm = 0 if self.max_norm is None else 2   # 1 after the launch behind the norm
        for g, todo in zip(self.param_groups, lists):
            if not len(todo):
                continue
            lr = g["lr"]
            on_device = torch.is_tensor(lr) and lr.device == self._dev
            args = _native.CqtAdamwArgs(
                0.0 if on_device else float(lr), *map(float, g["betas"]), float(g["eps"]),
                float(g["weight_decay"]), self.max_norm or 0.0,
                lr.data_ptr() if on_device else None, use_norm, self.seed)
            _native._check(L.cqt_adamw_step(todo, len(todo), g["state_bits"], ctypes.byref(args),
                                            ws.data_ptr(), ws.numel(), stream), "cqt_adamw_step")
            use_norm = min(use_norm, 1)


_hooked_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)

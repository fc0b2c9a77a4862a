"""AdamW over the library's batched update kernel.

The reference trains with ``torch.optim.AdamW`` (models/regression.py:298-301).  The update rule here is the same
(decoupled weight decay, bias-corrected moments; no amsgrad, no maximize); what differs is the launch: one library
kernel for all parameter tensors of a group (``cfh_adamw_step_batch``) instead of the framework's multi-tensor
machinery, which for a model of many small tensors is bound by its bookkeeping.  The step count lives on the device,
so a captured step keeps counting from replay to replay; ``lr`` and the other scalars are read on the host when
``step`` is called (a captured step replays the values of its capture: a learning-rate scheduler, as the
reference's trainer uses, needs the step captured again, or run eagerly, whenever it changes ``lr``).  The step
count is one word per parameter GROUP, not per parameter as in torch.optim.AdamW: all parameters of a group take
their first step together (a parameter that gets its first gradient later is bias-corrected with the group's count).

Parameters are float32, bfloat16 or float16 (rounded to their type after every step: in 16 bits, steps below half a unit of a
parameter's last place are lost).  ``state_bits`` (an option of a group): the moments in 32 bits, or in 8, a quarter of the
memory and of the traffic (``cfh_adamw_step_moments`` in the C header defines both formats: 64 consecutive elements of a
parameter share a power of two, rounding is stochastic and a function of the step and of the element alone, so that equal
runs give equal bits).  ``max_grad_norm``: the gradients of all groups are clipped by their common norm, as
``torch.nn.utils.clip_grad_norm_`` does before a step (models/regression.py:137-156 of the reference: backward, clip, step), but
inside the step: the gradients are read once more and not written (``grad_norm``; a captured step has one of its own, written
by every replay).  The first step, which makes the moments, is taken before a capture.  A group of float32 parameters with moments in 32 bits and
no clipping takes ``cfh_adamw_step_batch``, anything else ``cfh_adamw_step_moments``.
"""
import collections
import contextlib
import ctypes

import torch

from . import _lib


_here = contextlib.nullcontext()


def _on(dev):
    """A guard for ``dev``, or nothing where it is the current device already."""
    return _here if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


class AdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_grad_norm=None):
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas {betas} must lie in [0, 1)")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"max_grad_norm {max_grad_norm} must not be negative")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits {state_bits}: 8 or 32")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))
        self._flat = {}
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None      # of the last step with max_grad_norm: the norm before clipping, a float32 scalar on the device

    def __getstate__(self):
        # (the flat buffers are made anew from the moments in ``state``, as after a load; 8-bit floats go as bytes: the framework writes
        # them into a pickle, but does not read them from it)
        whole = super().__getstate__()
        state = collections.defaultdict(dict)
        for p, own in whole["state"].items():
            state[p] = own if not isinstance(own, dict) else {
                name: t.view(torch.uint8) if torch.is_tensor(t) and t.dtype == torch.float8_e4m3fn else t for name, t in own.items()}
        return dict(whole, state=state, max_grad_norm=self.max_grad_norm, grad_norm=self.grad_norm)

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("_flat", {})
        self.__dict__.setdefault("max_grad_norm", None)          # (of a copy written without it)
        self.__dict__.setdefault("grad_norm", None)
        for group in self.param_groups:          # (of a checkpoint written without it)
            group.setdefault("state_bits", 32)
        for own in self.state.values():
            codes = own.get("exp_avg") if isinstance(own, dict) and "exp_avg_scale" in own else None
            if torch.is_tensor(codes) and codes.dtype == torch.uint8:
                own["exp_avg"] = codes.view(torch.float8_e4m3fn)

    def _group_state(self, group):
        """Moments of all parameters of a group in flat buffers and the step word; ``self.state[p]`` holds the
        parameter's views of them under torch.optim.AdamW's names (and, in 8 bits, of the scales), so that ``state_dict()``
        saves them.  What ``self.state`` held before (a loaded checkpoint) moves into the buffers."""
        st = self._flat.setdefault(id(group), {})
        if st and st["bits"] != group["state_bits"]:
            raise RuntimeError(f"state_bits of a group that has moments in {st['bits']} bits changed to {group['state_bits']}")
        if not st:
            ps = [p for p in group["params"] if p.requires_grad]
            if not ps:
                return None
            dev, bits = ps[0].device, group["state_bits"]
            if bits not in (8, 32):
                raise ValueError(f"state_bits {bits}: 8 or 32")
            for p in ps:
                if p.dtype not in _lib.ELEMENT_TYPES or not p.is_cuda or p.device != dev:
                    raise RuntimeError("AdamW of crystalframer_amd needs float32 (or bfloat16, float16) parameters on one HIP device")
            plain = bits == 32 and all(p.dtype == torch.float32 for p in ps)
            if not (plain and self.max_grad_norm is None) and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first step of a group makes its moments (every replay would clear them): take it, or load a "
                                   "state, before the capture")
            offs, total, align = [], 0, _lib.MOMENT_BLOCK
            for p in ps:
                offs.append(total)
                total += (p.numel() + align - 1) // align * align          # every view aligned, every scale of one parameter
            self._check_loaded(ps, bits)
            zeros = lambda n, dtype: torch.zeros(n, dtype=dtype, device=dev)  # noqa: E731
            if bits == 8:
                flat = dict(exp_avg=zeros(total, torch.uint8).view(torch.float8_e4m3fn), exp_avg_sq=zeros(total, torch.uint8),
                            exp_avg_scale=zeros(total // align, torch.uint8), exp_avg_sq_scale=zeros(total // align, torch.uint8))
            else:
                flat = dict(exp_avg=zeros(total, torch.float32), exp_avg_sq=zeros(total, torch.float32))
            step = zeros(1, torch.int64)
            loaded = [self.state.get(p) or {} for p in ps]
            for p, o, old in zip(ps, offs, loaded):
                own = dict(step=step)
                for name, t in flat.items():
                    if name.endswith("scale"):
                        own[name] = t[o // align:(o + p.numel() + align - 1) // align]
                    else:
                        own[name] = t[o:o + p.numel()].view_as(p)
                    if old:
                        own[name].copy_(old[name])
                if old:
                    step.fill_(int(old["step"]))
                self.state[p] = own
            st.update(flat, step=step, bits=bits, scratch=zeros(16, torch.float32), offset={id(p): o for p, o in zip(ps, offs)},
                      numel={id(p): p.numel() for p in ps},
                      legacy=plain)
        return st

    def _check_loaded(self, ps, bits):
        """Loaded moments have the parameter's size and the group's number of bits."""
        names = ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if bits == 8 else ())
        for p in ps:
            old = self.state.get(p)
            if not old:
                continue
            blocks = (p.numel() + _lib.MOMENT_BLOCK - 1) // _lib.MOMENT_BLOCK
            types = (torch.float8_e4m3fn, torch.uint8, torch.uint8, torch.uint8)
            for name, want in zip(names, types):
                t = old.get(name)
                if t is None or t.numel() != (blocks if name.endswith("scale") else p.numel()) or (bits == 8 and t.dtype != want) or \
                        (bits == 32 and not (t.is_floating_point() and t.element_size() > 1)):
                    raise RuntimeError(f"{name} of a loaded state does not fit a parameter of {p.numel()} elements with moments in {bits} bits")

    def load_state_dict(self, state_dict):
        """Loads like torch.optim.AdamW, hooks included, then moves the loaded moments into the flat buffers.  A checkpoint brings the
        options of its groups with it, ``state_bits`` among them."""
        given = {}

        def keep(_, state):
            given.update(state)

        def types_as_given(_):
            # (the base class gives floating-point parameters' states the type of their parameter: the moments keep theirs)
            saved = [i for group in given["param_groups"] for i in group["params"]]
            for i, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
                own = self.state.get(p) or {}
                for name, t in (given["state"].get(i) or {}).items():
                    now = own.get(name)
                    if torch.is_tensor(t) and torch.is_tensor(now) and now.dtype != t.dtype:
                        own[name] = t.to(now.device)
        # between the hooks before the load, whose dict it is, and those after it, which may change the state
        handles = [self.register_load_state_dict_pre_hook(keep), self.register_load_state_dict_post_hook(types_as_given, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()
        self._flat = {}
        for group in self.param_groups:
            self._group_state(group)

    @torch.no_grad()
    def moments(self):
        """(exp_avg, exp_avg_sq) of every group that has taken a step, as flat float32 tensors: in 32 bits the moments
        themselves, in 8 the values that they stand for.  The parameters that require a gradient stand in them one after the other,
        each from a multiple of 64 elements on."""
        out, lib = [], _lib.load()
        for group in self.param_groups:
            st = self._flat.get(id(group))
            if not st:
                continue
            m, v = st["exp_avg"], st["exp_avg_sq"]
            if st["bits"] == 8:
                dev, state = m.device, self._moments_struct(st)
                m, v = (torch.empty(m.numel(), dtype=torch.float32, device=dev) for _ in range(2))
                with _on(dev):
                    rc = lib.cfh_adamw_moments(ctypes.byref(state), m.data_ptr(), v.data_ptr(), _lib.raw_stream(dev))
                _lib.check(rc, "cfh_adamw_moments")
            out.append((m, v))
        return out

    @staticmethod
    def _moments_struct(st):
        s = _lib.CfhMoments()
        s.exp_avg, s.exp_avg_sq = st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
        s.size, s.bits = st["exp_avg"].numel(), st["bits"]
        if s.bits == 8:
            s.exp_avg_scale, s.exp_avg_sq_scale = st["exp_avg_scale"].data_ptr(), st["exp_avg_sq_scale"].data_ptr()
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.load()
        work = []
        for group in self.param_groups:
            st = self._group_state(group)
            if st is not None:
                work.append((group, st, self._plan(group, st)))
        clipped = self.max_grad_norm is not None
        typed = [w for w in work if clipped or not w[1]["legacy"]]
        if typed:
            self._step_moments(lib, typed)
        for group, st, plan in work:
            if clipped or not st["legacy"]:
                continue
            jobs = plan["jobs"]
            m0, v0 = st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr()
            n, keep = plan["native"].fill(ctypes.addressof(jobs), m0, v0), None
            if n < 0:
                n, keep = self._fill(plan, m0, v0)      # a gradient that has to be looked at
            if n == 0:
                continue
            dev = plan["device"]
            b1, b2 = group["betas"]
            if torch.cuda.current_device() != dev.index:
                with torch.cuda.device(dev):
                    rc = self._launch(lib, jobs, n, group, b1, b2, st, dev)
            else:
                rc = self._launch(lib, jobs, n, group, b1, b2, st, dev)
            _lib.check(rc, "cfh_adamw_step_batch")
            del keep      # the gradients stay alive through p.grad (or, made contiguous here, through the stream order)
        return loss

    def _step_moments(self, lib, work):
        """The step of groups of any type, with moments in 32 or 8 bits; the gradients' common norm first if they are clipped."""
        filled = []
        for group, st, plan in work:
            jobs = plan.get("param_jobs")
            if jobs is None:
                if len({id(p) for p in plan["params"]}) != len(plan["params"]):
                    raise RuntimeError("a parameter is in its group twice")
                jobs = plan["param_jobs"] = (_lib.CfhParamJob * max(len(plan["params"]), 1))()
            n, keep = plan["native"].fill_params(ctypes.addressof(jobs)), None
            if n < 0:
                n, keep = self._fill_moments(plan, jobs)      # a gradient that has to be looked at
            if n:
                filled.append((group, st, plan, jobs, n, keep))
        clip = sums = None
        if self.max_grad_norm is not None and filled:
            clip, sums = self._clip(lib, filled)      # (the sums live until the steps are on their way)
        elif self.max_grad_norm is not None:
            self.grad_norm = None
        for group, st, plan, jobs, n, keep in filled:
            dev, (b1, b2) = plan["device"], group["betas"]
            state = self._moments_struct(st)
            with _on(dev):
                rc = lib.cfh_adamw_step_moments(
                    jobs, n, ctypes.byref(state), float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                    float(group["weight_decay"]), None if clip is None else ctypes.byref(clip), st["step"].data_ptr(),
                    st["scratch"].data_ptr(), _lib.raw_stream(dev))
            _lib.check(rc, "cfh_adamw_step_moments")

    def _clip(self, lib, filled):
        """The sums of squares of the gradients of all groups are on their way: what the steps need of them."""
        dev = filled[0][2]["device"]
        if any(plan["device"] != dev for _, _, plan, *_ in filled):
            raise RuntimeError("max_grad_norm needs the parameters of all groups on one device")
        total = sum(n for *_, n, _ in filled)
        jobs = filled[0][3]
        if len(filled) > 1:
            jobs, at = (_lib.CfhParamJob * total)(), 0
            for *_, part, n, _ in filled:
                ctypes.memmove(ctypes.addressof(jobs) + at * ctypes.sizeof(_lib.CfhParamJob), part, n * ctypes.sizeof(_lib.CfhParamJob))
                at += n
        clip = _lib.CfhGradClip()
        clip.count = lib.cfh_grad_square_sums_count(jobs, total)
        if clip.count < 0:
            _lib.check(clip.count, "cfh_grad_square_sums_count")
        # (memory of its own for every step: two captured steps never share it)
        sums = torch.empty(clip.count, dtype=torch.float64, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        clip.sums, clip.norm, clip.max_norm = sums.data_ptr(), norm.data_ptr(), float(self.max_grad_norm)
        with _on(dev):
            rc = lib.cfh_grad_square_sums(jobs, total, clip.sums, clip.count, _lib.raw_stream(dev))
        _lib.check(rc, "cfh_grad_square_sums")
        self.grad_norm = norm
        return clip, sums

    @staticmethod
    def _fill_moments(plan, jobs):
        """The job table of ``cfh_adamw_step_moments`` parameter by parameter: (jobs, gradients made contiguous here)."""
        n, keep = 0, None
        for p, off, count in zip(plan["params"], plan["offs"], plan["counts"]):
            g = p.grad
            if g is None:
                continue
            g = AdamW._gradient(p, g, off, count, plan["device"])
            if g.dtype != p.dtype or p.dtype not in _lib.ELEMENT_TYPES:
                raise RuntimeError("AdamW of crystalframer_amd needs float32 (or bfloat16, float16) parameters and gradients of the same type")
            if not g.is_contiguous():
                g = g.contiguous()
                keep = (keep, g)
            j = jobs[n]
            j.param, j.grad, j.n, j.first, j.dtype = p.data_ptr(), g.data_ptr(), count, off, _lib.ELEMENT_TYPES[p.dtype]
            n += 1
        return n, keep

    @staticmethod
    def _gradient(p, g, off, count, device):
        """``g`` if the kernels can take it with the parameter and its moments."""
        if off is None:
            raise RuntimeError("a parameter that was not in the group, or did not require a gradient, at the first step "
                               "has a gradient now")
        if g.is_sparse:
            raise RuntimeError("sparse gradients are not supported")
        if not p.is_contiguous():
            raise RuntimeError("AdamW of crystalframer_amd needs contiguous parameters")
        if p.numel() != count or g.numel() != count or p.device != device or g.device != device:
            raise RuntimeError("a parameter or its gradient has another size or device than at the first step")
        return g

    @staticmethod
    def _fill(plan, m0, v0):
        """The job table parameter by parameter: (jobs, gradients made contiguous here)."""
        n, keep = 0, None
        for p, off, count in zip(plan["params"], plan["offs"], plan["counts"]):
            g = p.grad
            if g is None:
                continue
            AdamW._gradient(p, g, off, count, plan["device"])
            if p.dtype != torch.float32 or g.dtype != torch.float32:
                raise RuntimeError("AdamW of crystalframer_amd needs float32 parameters and gradients")
            if not g.is_contiguous():
                g = g.contiguous()
                keep = (keep, g)
            a = plan["jobs"][n]
            a.param, a.exp_avg, a.exp_avg_sq, a.n = p.data_ptr(), m0 + 4 * off, v0 + 4 * off, p.numel()
            a.grad = g.data_ptr()
            n += 1
        return n, keep

    def zero_grad(self, set_to_none: bool = True):
        if not set_to_none or not self._flat:
            return super().zero_grad(set_to_none=set_to_none)
        for group in self.param_groups:
            st = self._flat.get(id(group))
            if st:
                self._plan(group, st)["native"].drop()
            else:
                for p in group["params"]:
                    p.grad = None

    @staticmethod
    def _launch(lib, jobs, n, group, b1, b2, st, dev):
        return lib.cfh_adamw_step_batch(jobs, n, float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                        float(group["weight_decay"]), st["step"].data_ptr(), _lib.raw_stream(dev))

    def _plan(self, group, st):
        """Job table of the group's launch, kept from step to step (made again when the group holds other parameters)."""
        plan = st.get("plan")
        if plan is None or not plan["native"].of(group["params"]) or plan["moments"] != st["exp_avg"].data_ptr():
            ps = list(group["params"])
            offs = [st["offset"].get(id(p)) for p in ps]
            counts = [st["numel"].get(id(p), 0) for p in ps]
            plan = st["plan"] = dict(params=ps, offs=offs, counts=counts, moments=st["exp_avg"].data_ptr(),
                                     jobs=(_lib.CfhAdamWJob * max(len(ps), 1))(), device=st["exp_avg"].device,
                                     native=_lib.load_host().Updates(ps, [-1 if o is None else o for o in offs], counts,
                                                                     st["exp_avg"]))
        return plan

"""Drop-in for `torch.optim.AdamW` over the parameters a spn4cir_amd model exposes (train_negplus.py:77-84 builds
`optim.AdamW([{'params': ..., 'lr': ..., 'betas': (0.9, 0.999), 'eps': 1e-7}])`; change that one line to
`spn4cir_amd.optim.AdamW(...)` with the same arguments).

The models' nn.Parameters are slices of ONE flat fp32 buffer per tower and their `.grad`s are slices of one flat gradient
buffer (gradsink.py), so the whole update is a single launch of the fused AdamW kernel (spn_adamw_step_scaled, the kernel
Stage2Trainer uses) instead of torch's ~10 multi-tensor passes (2.9 ms -> 0.6 ms per step for ViT-L/14's text tower).
Same arithmetic as torch.optim.AdamW (decoupled weight decay, bias correction, eps outside the square root).  The step
count that enters the bias correction lives on the DEVICE (one fp32 counter shared by every parameter's state["step"],
advanced by spn_adamw_tick only when found_inf == 0): a step GradScaler skips on overflow does not advance it, exactly as
torch - which does not call optimizer.step() on such a step - leaves its per-parameter counters alone.

torch.amp.GradScaler: the class declares `_step_supports_amp_scaling`, so `scaler.step(optimizer)` hands over
`optimizer.grad_scale` / `optimizer.found_inf` (device tensors) and the kernel unscales the gradients and skips the step on
overflow itself - no `unscale_` pass over the gradients and no host synchronisation.

Parameters that are not part of such a flat run of several (or whose gradients are not the matching slices) are updated together by the
many-tensor form of the same kernel (spn_adamw_multi: one launch, the same bits per tensor), so the class works for any fp32 CUDA
parameter list; their gradients may be bf16 or fp16.  That launch's tables are built once (some 0.5 ms for 330 tensors) and again at a step
that finds a parameter's data replaced.

state_bits=8 keeps both moments in 8 bits (2.02 instead of 8 bytes per parameter; ops.AdamWPlan): all parameters of all groups go through
spn_adamw_multi in one launch, whatever buffers they live in.  The moments are rounded stochastically by a hash of (seed, step, element),
so equal runs give equal bits.  state_dict() holds codes and scale bytes.

In a graph: init_state() or one step() first, then capture step().  A 32-bit first step that is captured all the same records the creation of its
state, so that every replay is a first step (with a warning); an 8-bit one is refused, its tables cannot be uploaded there.  Keep the optimizer as long as
such a graph; load_state_dict() and p.data = ... give the optimizer new memory, which a graph captured before does not know."""
import ctypes as C
import warnings

import torch

from ._lib import check, lib
from .ops import _DTYPE_OF, ADAMW_GROUPS, AdamWPlan, _p, _stream, adamw_multi, ranges_overlap


def _flat_view(t, numel):
    """1-D fp32 tensor over t's storage starting at t's first element."""
    return torch.empty(0, dtype=t.dtype, device=t.device).set_(t.untyped_storage(), t.storage_offset(), (numel,), (1,))


def _counters(params):
    """Parameters whose version counters cover all of theirs: one, if they are views of a tensor, else each."""
    before = [p._version for p in params]
    torch.autograd.graph.increment_version(params[:1])
    return params[:1] if all(p._version > v for p, v in zip(params, before)) else params


class AdamW(torch.optim.Optimizer):
    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, on_step=None, state_bits=32, seed=0):
        if lr < 0 or eps < 0 or weight_decay < 0 or not (0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("invalid AdamW hyper-parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits: 8 or 32, not {state_bits!r}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.seed = state_bits, int(seed)
        self._plans = None                  # [(AdamWPlan, its parameters, the slice of its groups)]: 8-bit moments, or the tensors outside flat runs
        self._on_step = on_step             # e.g. model.parameters_changed (the models also notice the update themselves)
        self._runs = None                   # per group: [dict(params, p_flat, m, v, numel, counters, addresses)]
        self._step_dev = None               # 0-dim fp32 device counter of APPLIED steps (shared by every state["step"])
        self._captured = []                 # what captured steps read and write: kept as long as the optimizer, their graphs hold addresses only

    # -------------------------------------------------------------------------------- layout
    def _make_plans(self, members):
        """members: per group a list of (parameter, m, v) (moments None for 8 bits) -> [(AdamWPlan, its parameters, the slice of its
        groups)], one for each 16 groups.  Parameters that share memory (tied weights held twice) are updated one after the other, each by a plan of its own.
        Nothing of the optimizer changes here: a plan that cannot be built (out of memory) leaves it as it was."""
        plans = []
        for g0 in range(0, len(members), ADAMW_GROUPS):
            part = [(i, t) for i, group in enumerate(members[g0:g0 + ADAMW_GROUPS]) for t in group]
            if not part:
                continue
            tied = ranges_overlap([p.data_ptr() for _, (p, _, _) in part], [p.nbytes for _, (p, _, _) in part])
            for some in ([t] for t in part) if tied else (part,):
                state = None if self.state_bits == 8 else [(m, v) for _, (_, m, v) in some]
                plan = AdamWPlan([p for _, (p, _, _) in some], state_bits=self.state_bits, groups=[i for i, _ in some], state=state)
                plans.append((plan, [p for _, (p, _, _) in some], slice(g0, g0 + ADAMW_GROUPS)))
        return plans

    def _device(self):
        """The device of the first parameter that is trained (of the first one if none is)."""
        every = lambda: (p for g in self.param_groups for p in g["params"])  # noqa: E731
        return next((p for p in every() if p.requires_grad), next(every())).device

    def _build_8bit(self):
        ps = [[p for p in g["params"] if p.requires_grad] for g in self.param_groups]
        dev = self._device()
        for p in (p for g in ps for p in g):
            if p.dtype != torch.float32 or not p.is_cuda or not p.is_contiguous():
                raise TypeError("spn4cir_amd.optim.AdamW: parameters must be contiguous fp32 CUDA tensors")
        step_dev = torch.zeros((), dtype=torch.float32, device=dev)
        plans = self._make_plans([[(p, None, None) for p in g] for g in ps])
        for plan, params, _ in plans:
            for p, off, n in zip(params, plan.offsets, plan.numels):
                end = off + (n + 127) // 128 * 128
                self.state[p].update(step=step_dev, exp_avg=plan.m[off:end], exp_avg_sq=plan.v[off:end],
                                     exp_avg_scale=plan.m_scale[off // 128:end // 128], exp_avg_sq_scale=plan.v_scale[off // 128:end // 128])
        self._plans, self._step_dev = plans, step_dev        # (last: a failed build is tried again by the next step)

    @staticmethod
    def _own_grad(p):
        g = p.grad
        if g is None:
            return None
        g = g if g.dtype in (torch.float32, torch.bfloat16, torch.float16) else g.float()
        return g if g.is_contiguous() else g.contiguous()

    def add_param_group(self, param_group):
        if getattr(self, "_step_dev", None) is not None and self.state_bits == 8:
            raise ValueError("state_bits=8: add all parameters before the first step")
        super().add_param_group(param_group)

    def _moved(self):
        """Whether a parameter's data was replaced since the plans were built."""
        return any(list(map(torch.Tensor.data_ptr, params)) != plan.addresses for plan, params, _ in self._plans)

    def _refresh_plans(self):
        for k, (plan, params, groups) in enumerate(self._plans):
            if list(map(torch.Tensor.data_ptr, params)) != plan.addresses:       # p.data was replaced: the moments stay, the addresses do not
                state = plan.own_moments if self.state_bits == 32 else (plan.m, plan.v, plan.m_scale, plan.v_scale)
                if [p.numel() for p in params] != plan.numels:
                    raise ValueError("a parameter changed its size after the first step")
                plan = AdamWPlan(params, state_bits=self.state_bits, groups=plan.groups, state=state)
                self._plans[k] = (plan, params, groups)

    def _plan_calls(self, grads_of, exact_betas):
        """[(plan, gradients, hyper-parameters)] of one adamw_multi per plan; grads_of(p) -> its gradient or None."""
        calls = []
        for plan, params, groups in self._plans:
            grads = [grads_of(p) for p in params]
            if all(g is None for g in grads):
                continue
            calls.append((plan, grads, [dict(g, betas=g["betas"] if exact_betas else tuple(C.c_float(b).value for b in g["betas"]))
                                        for g in self.param_groups[groups]]))
        return calls

    def _build_runs(self):
        all_runs = []
        dev = self._device()
        step_dev = torch.zeros((), dtype=torch.float32, device=dev)
        for group in self.param_groups:
            ps = [p for p in group["params"] if p.requires_grad]
            for p in ps:
                if p.dtype != torch.float32 or not p.is_cuda or not p.is_contiguous():
                    raise TypeError("spn4cir_amd.optim.AdamW: parameters must be contiguous fp32 CUDA tensors")
            ps.sort(key=lambda p: (p.untyped_storage().data_ptr(), p.storage_offset()))
            runs, cur = [], []
            for p in ps:
                if cur and (p.untyped_storage().data_ptr() == cur[-1].untyped_storage().data_ptr()
                            and p.storage_offset() == cur[-1].storage_offset() + cur[-1].numel()):
                    cur.append(p)
                else:
                    if cur:
                        runs.append(cur)
                    cur = [p]
            if cur:
                runs.append(cur)
            out = []
            for r in runs:
                n = sum(p.numel() for p in r)
                m = torch.zeros(n, dtype=torch.float32, device=r[0].device)
                v = torch.zeros(n, dtype=torch.float32, device=r[0].device)
                out.append(dict(params=r, p_flat=_flat_view(r[0], n), m=m, v=v, numel=n, counters=None,
                                addresses=[p.data_ptr() for p in r]))
            all_runs.append(out)
        for run in (run for runs in all_runs for run in runs):
            off = 0
            for p in run["params"]:                          # torch-compatible per-parameter state (views of the run's state)
                end = off + p.numel()
                self.state[p].update(step=step_dev, exp_avg=run["m"][off:end].view_as(p), exp_avg_sq=run["v"][off:end].view_as(p))
                off = end
        self._runs, self._step_dev = all_runs, step_dev      # (last: a failed build is tried again by the next step)

    def load_state_dict(self, state_dict):
        """torch semantics; the loaded per-parameter moments are copied into the flat state of the runs.  A state that is refused leaves the
        optimizer as it was."""
        kept = ("state", "param_groups", "_runs", "_plans", "_step_dev")
        before = [getattr(self, name) for name in kept]
        try:
            super().load_state_dict(state_dict)
            self._adopt()
        except BaseException:
            for name, value in zip(kept, before):
                setattr(self, name, value)
            raise

    def _adopt(self):
        """What torch has just put into self.state becomes the content of fresh runs or plans."""
        loaded = {p: dict(st) for p, st in self.state.items()}
        if self.state_bits == 8:
            self._load_8bit(loaded)
            return
        if any("exp_avg_scale" in st for st in loaded.values()):
            raise ValueError("this state holds 8-bit moments: build the optimizer with state_bits=8")
        self._plans = None
        self._build_runs()                                   # fresh flat state, self.state[p] re-pointed at its views
        steps = 0.0
        for p, old in loaded.items():
            st = self.state[p]
            if "exp_avg" in old:
                st["exp_avg"].copy_(old["exp_avg"].to(st["exp_avg"].device, torch.float32).view_as(st["exp_avg"]))
                st["exp_avg_sq"].copy_(old["exp_avg_sq"].to(st["exp_avg_sq"].device, torch.float32).view_as(st["exp_avg_sq"]))
            if "step" in old:
                steps = max(steps, float(old["step"]))
        self._step_dev.fill_(steps)

    def _load_8bit(self, loaded):
        """Codes and scale bytes are copied as they are (torch casts a loaded state to the parameter's fp32: bytes survive that)."""
        self._build_8bit()
        steps = 0.0
        for p, old in loaded.items():
            st = self.state[p]
            if "exp_avg" in old:
                if "exp_avg_scale" not in old:
                    raise ValueError("this state holds 32-bit moments: build the optimizer with state_bits=32")
                for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
                    if old[k].numel() != st[k].numel():
                        raise ValueError(f"state {k}: {old[k].numel()} bytes for a parameter that needs {st[k].numel()}")
                    st[k].copy_(old[k])
            if "step" in old:
                steps = max(steps, float(old["step"]))
        self._step_dev.fill_(steps)

    @staticmethod
    def _grads_flat(run):
        """The run's gradients as one flat tensor if they are consecutive slices of one buffer and the parameters are where they were when the run was
        laid out (p.data = ... moves them), else None."""
        params, T = run["params"], torch.Tensor
        grads = [p.grad for p in params]
        g0 = grads[0]
        if any(g is None for g in grads) or list(map(T.data_ptr, params)) != run["addresses"]:
            return None
        if set(map(_DTYPE_OF, grads)) != {torch.float32} or not all(map(T.is_contiguous, grads)) or g0.device != params[0].device:
            return None
        base, first = run["addresses"][0], g0.data_ptr()
        if [x - first for x in map(T.data_ptr, grads)] != [x - base for x in run["addresses"]]:
            return None
        if g0.untyped_storage().nbytes() < 4 * (g0.storage_offset() + run["numel"]):       # neighbours by chance
            return None
        return _flat_view(g0, run["numel"])

    # -------------------------------------------------------------------------------- step
    def _launch(self, p, g, m, v, group, scale, found):
        b1, b2 = group["betas"]
        check(lib().spn_adamw_step_dev(_p(p), _p(g), _p(m), _p(v), p.numel(), float(group["lr"]), float(b1), float(b2),
                                       float(group["eps"]), float(group["weight_decay"]), _p(self._step_dev), _p(scale),
                                       _p(found), _stream()), "adamw_step_dev")

    def init_state(self):
        """Creates the moments (zeros), the step counter and the tables of 8-bit moments, which the first step() does otherwise.  A program that captures
        step() in a graph without a step before it calls this first: what a capture creates is created again by every replay."""
        if self._step_dev is None:
            self._build_8bit() if self.state_bits == 8 else self._build_runs()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # launches go to the current stream of the parameters' device
        di = self._device().index
        if di is not None and di != torch.cuda.current_device():
            with torch.cuda.device(di):
                self._step()
        else:
            self._step()
        if self._on_step is not None:
            self._on_step()
        return loss

    def _step(self):
        capturing = torch.cuda.is_current_stream_capturing()
        if self._step_dev is None:
            if capturing and self.state_bits == 8:
                raise RuntimeError("state_bits=8: call init_state() (or take one step) before step() is captured in a graph")
            if capturing:
                warnings.warn("AdamW: the first step is being captured, so the graph zeroes the moments and the step counter too and every replay is a "
                              "first step; call init_state() (or take one step) before the capture", stacklevel=5)
            self.init_state()
        scale = getattr(self, "grad_scale", None)          # set by torch.amp.GradScaler.step around this call
        found = getattr(self, "found_inf", None)
        for t in (scale, found):
            if t is not None and (t.dtype != torch.float32 or not t.is_cuda or t.numel() != 1):
                raise TypeError("grad_scale / found_inf must be 1-element fp32 CUDA tensors")
        # everything that can fail for want of memory or a wrong layout is done before the step is counted and the first kernel launched
        updated = []                                         # parameters, one at least for each version counter
        if self.state_bits == 8:
            if capturing and self._moved():
                raise RuntimeError("state_bits=8: a parameter's data was replaced; take one step before step() is captured in a graph")
            self._refresh_plans()
            launches, calls = [], self._plan_calls(self._own_grad, True)
        else:
            loose, launches, calls, pending = set(), [], [], []          # launches: (p, g, m, v, group)
            one_by_one = capturing and (self._plans is None or self._moved())          # a plan's upload cannot be captured
            for group, runs in zip(self.param_groups, self._runs):
                for run in runs:
                    if run["numel"] == 0 or all(p.grad is None for p in run["params"]):
                        continue
                    g = self._grads_flat(run) if len(run["params"]) > 1 else None
                    if g is not None:
                        launches.append((run["p_flat"], g, run["m"], run["v"], group))
                        if run["counters"] is None:
                            run["counters"] = _counters(run["params"])
                        updated += run["counters"]
                    else:                                    # a tensor by itself, or gradients elsewhere
                        pending.append((run, group))
            # one tensor alone goes through the single-tensor kernel (64 M elements: 350 us, in the many-tensor launch 369; 1000: 29 and 34 us of host
            # time); several are faster together (4 x 16 M: 363 one by one, 368 together; 12 x 2 M: 190 and 142)
            alone = len(pending) == 1 and len(pending[0][0]["params"]) == 1
            for run, group in pending:
                off = 0
                if sum(map(torch.Tensor.numel, run["params"])) != run["numel"]:
                    raise ValueError("a parameter changed its size after the first step")
                for p in run["params"]:
                    g, n = p.grad, p.numel()
                    if g is not None and g.numel() != n:
                        raise ValueError("a parameter changed its size after its gradient was computed")
                    if p.dtype != torch.float32 or not p.is_cuda or not p.is_contiguous():
                        raise TypeError("spn4cir_amd.optim.AdamW: parameters must be contiguous fp32 CUDA tensors")
                    if g is not None and n:
                        if one_by_one or (alone and g.dtype == torch.float32 and g.is_contiguous()):
                            launches.append((_flat_view(p, n), g.contiguous().float().view(-1), run["m"][off:off + n], run["v"][off:off + n], group))
                            updated.append(p)
                        else:                                # all such in one launch
                            loose.add(p)
                    off += n
            if loose:
                if self._plans is None:
                    self._plans = self._make_plans([[(p, self.state[p]["exp_avg"].view(-1), self.state[p]["exp_avg_sq"].view(-1)) for run in runs
                                                     for p in run["params"]] for runs in self._runs])
                else:
                    self._refresh_plans()
                # (betas as the single-tensor kernel takes them, in fp32: a tensor's update does not depend on which of the two serves it)
                calls = self._plan_calls(lambda p: self._own_grad(p) if p in loose else None, False)
        if capturing:
            self._captured.append((self._step_dev, self._runs, [plan for plan, _, _ in calls]))
        check(lib().spn_adamw_tick(_p(self._step_dev), _p(found), _stream()), "adamw_tick")
        for p, g, m, v, group in launches:
            self._launch(p, g, m, v, group, scale, found)
        for plan, grads, hyper in calls:
            adamw_multi(plan, grads, 0, hyper, seed=self.seed, step_dev=self._step_dev, grad_scale=scale, found_inf=found)
        # the version counter of every parameter that was updated: autograd's check of saved tensors and the models, which re-derive their bf16
        # operands when it has moved, read it (parameters over one buffer need not share a counter)
        for plan, grads, _ in calls:
            updated += [p for p, g in zip(plan.params, grads) if g is not None]
        torch.autograd.graph.increment_version(updated)

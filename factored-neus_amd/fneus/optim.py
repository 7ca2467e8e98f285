"""FlatAdam: torch.optim.Adam with its step() replaced by ONE fneus_adam launch over the whole model.

Same hyper-parameters, same per-parameter state (`step`, `exp_avg`, `exp_avg_sq`) and therefore the same
state_dict()/load_state_dict() format as the reference's optimiser (exp_runner.py:108, checkpoint key "optimizer"), but
* the moments of adjacent parameters live in one arena (the Parameters of a fused MLP are views of one flat buffer, so
  a whole network is a single contiguous segment for the kernel);
* `step` is one device scalar shared by every parameter, `lr` a device scalar: the step is hipGraph-capturable;
* the kernel clears each gradient after using it (zero_grad() becomes a no-op for the owner of this optimiser).
Every parameter that takes part must have a persistent `.grad` buffer when step() is first called (the trainer guarantees
it); a parameter whose `.grad` is None is skipped like torch.optim.Adam skips it (no state, no update): the reference hands
the never-evaluated background NeRF of the wmask configuration to Adam in exactly that way (exp_runner.py:89, 96).
"""
from __future__ import annotations

import ctypes as C
from typing import List

import torch

from . import _lib
from ._lib import lib, check


class FlatAdam(torch.optim.Adam):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, clear_grads: bool = True):
        super().__init__(params, lr=float(lr), betas=betas, eps=eps)
        if len(self.param_groups) != 1:
            raise NotImplementedError("FlatAdam supports a single parameter group (as the reference uses)")
        self.clear_grads = clear_grads
        self._segs = None          # ctypes array of FneusAdamSegment
        self._keys = None          # (param ptr, grad ptr) per parameter at build time
        self._arenas = []
        self._step_dev = None
        self._lr_dev = None
        self._lr_host = None

    # ---- learning rate: a device scalar (graph replays see updates) ----
    def set_lr(self, lr: float):
        self.param_groups[0]["lr"] = float(lr)
        if self._lr_dev is not None:
            self._lr_dev.fill_(float(lr))
            self._lr_host = float(lr)

    def _params(self) -> List[torch.nn.Parameter]:
        """the parameters this step updates: those with a gradient (torch.optim.Adam's rule)"""
        return [p for p in self.param_groups[0]["params"] if p.requires_grad and p.grad is not None]

    def _build(self):
        ps = self._params()
        if not ps:
            raise RuntimeError("FlatAdam.step(): no parameter has a gradient")
        dev = ps[0].device
        for p in ps:
            if p.dtype != torch.float32 or not p.is_contiguous() or not p.grad.is_contiguous():
                raise RuntimeError("FlatAdam needs contiguous fp32 parameters with persistent .grad buffers")
        # the shared step counter: continue from a loaded state if there is one
        steps = [float(self.state[p]["step"]) for p in ps if p in self.state and "step" in self.state[p]]
        # (fneus_adam: float[2] = the step count and the launch's arrival counter; the state's `step` is the 0-d view of [0])
        self._step_buf = torch.zeros(2, dtype=torch.float32, device=dev)
        self._step_buf[0] = max(steps) if steps else 0.0
        self._step_dev = self._step_buf[0]
        self._lr_host = float(self.param_groups[0]["lr"])
        self._lr_dev = torch.full((), self._lr_host, dtype=torch.float32, device=dev)
        # merge parameters whose storage AND gradient storage are adjacent
        runs, cur = [], [ps[0]]
        for prev, p in zip(ps, ps[1:]):
            adj = (p.data_ptr() == prev.data_ptr() + prev.numel() * 4 and
                   p.grad.data_ptr() == prev.grad.data_ptr() + prev.numel() * 4)
            if adj:
                cur.append(p)
            else:
                runs.append(cur)
                cur = [p]
        runs.append(cur)
        self._arenas = []
        segs = (_lib.FneusAdamSegment * len(runs))()
        for i, run in enumerate(runs):
            count = sum(p.numel() for p in run)
            m = torch.zeros(count, dtype=torch.float32, device=dev)
            v = torch.zeros(count, dtype=torch.float32, device=dev)
            off = 0
            for p in run:
                st = self.state[p]
                mv, vv = m[off: off + p.numel()].view_as(p), v[off: off + p.numel()].view_as(p)
                if "exp_avg" in st:                       # loaded (or previously stepped) moments move into the arena
                    mv.copy_(st["exp_avg"])
                    vv.copy_(st["exp_avg_sq"])
                st["exp_avg"], st["exp_avg_sq"], st["step"] = mv, vv, self._step_dev
                off += p.numel()
            self._arenas.append((m, v))
            segs[i].param, segs[i].grad = run[0].data_ptr(), run[0].grad.data_ptr()
            segs[i].exp_avg, segs[i].exp_avg_sq, segs[i].count = m.data_ptr(), v.data_ptr(), count
        self._segs = segs
        self._keys = [(p.data_ptr(), p.grad.data_ptr()) for p in ps]

    def _stale(self):
        if self._segs is None:
            return True
        ps = self._params()
        if len(ps) != len(self._keys):
            return True
        for p, (pp, gp) in zip(ps, self._keys):
            st = self.state.get(p)
            if p.grad is None or p.data_ptr() != pp or p.grad.data_ptr() != gp or st is None or st.get("step") is not self._step_dev:
                return True
        return False

    @torch.no_grad()
    def step(self, closure=None):
        if closure is not None:
            raise NotImplementedError("FlatAdam.step() takes no closure")
        if self._stale():                    # first call, re-attached parameters, or a load_state_dict()
            self._build()
        lr = self.param_groups[0]["lr"]
        if float(lr) != self._lr_host:       # someone assigned param_groups[0]["lr"] directly (reference style)
            self.set_lr(float(lr))
        device = self._lr_dev.device
        if device.index != torch.cuda.current_device():      # the launch goes to the device of the parameters, whichever is current
            with torch.cuda.device(device):
                return self._launch()
        self._launch()

    def _launch(self):
        b1, b2 = self.param_groups[0]["betas"]
        check(lib.fneus_adam(self._segs, len(self._segs), C.c_void_p(self._lr_dev.data_ptr()),
                             C.c_void_p(self._step_dev.data_ptr()), float(b1), float(b2), float(self.param_groups[0]["eps"]),
                             int(self.clear_grads), C.c_void_p(torch.cuda.current_stream().cuda_stream)), "fneus_adam")

    def state_dict(self):
        """torch.optim.Adam's format, with an independent `step` tensor per parameter (inside this optimiser all
        parameters share one device scalar; a consumer such as torch.optim.Adam increments each entry separately)"""
        sd = super().state_dict()
        for st in sd["state"].values():
            if torch.is_tensor(st.get("step")):
                st["step"] = st["step"].detach().clone().cpu()
        return sd

    def load_state_dict(self, state_dict):
        """torch shares tensors of the right dtype / device with the dict it is given; the moments move into this
        optimiser's arenas at the next step(), so take private copies now (the source may keep training)"""
        # torch maps the saved state onto the parameters BY POSITION and checks only the count: a state_dict of another
        # parameter order would put, say, the background NeRF's moments on the SDF network.  Check the shapes first.
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        ps = [p for g in self.param_groups for p in g["params"]]
        if len(ids) != len(ps):
            raise ValueError(f"optimizer state_dict holds {len(ids)} parameters, this optimiser {len(ps)}")
        for i, p in zip(ids, ps):
            st = saved.get(i)
            if st is not None and torch.is_tensor(st.get("exp_avg")) and tuple(st["exp_avg"].shape) != tuple(p.shape):
                raise ValueError(f"optimizer state of parameter {i} has shape {tuple(st['exp_avg'].shape)}, the parameter "
                                 f"{tuple(p.shape)}: the parameter lists differ in order")
        super().load_state_dict(state_dict)
        for st in self.state.values():
            for k in ("step", "exp_avg", "exp_avg_sq"):
                if torch.is_tensor(st.get(k)):
                    st[k] = st[k].clone()
        self._segs = None

    @property
    def n_segments(self):
        return 0 if self._segs is None else len(self._segs)


def _capturing(device) -> bool:
    if device.type != "cuda":
        return False
    if device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


class FlatMuon(torch.optim.Optimizer):
    """Muon for a model's weight matrices, FlatAdam for everything else, one learning rate for both (adjust="match_rms" gives a matrix's
    update Adam's rms).  Every matrix of the model takes part in the same launches of fneus_muon (momentum, Newton-Schulz
    orthogonalisation, step); learning rate and step count are device scalars, gradients are cleared by the kernels: capturable in a
    hipGraph like FlatAdam, behind an eager step that allocates the state (else refused), with its methods (set_lr, state_dict /
    load_state_dict).

    params: parameters; the 2-D ones with no side shorter than `min_side` are Muon's (a layer with a handful of outputs has no spectrum to
    level), the others Adam's (fp32, as FlatAdam's are; weight_decay is Muon's alone).  State: `momentum_buffer` a matrix, torch.optim.Adam's of the others.  A parameter without a gradient is
    skipped."""

    def __init__(self, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="match_rms", coefficients=None, steps=5,
                 eps=1e-7, prec=None, betas=(0.9, 0.999), adam_eps=1e-8, min_side=32):
        from . import ops
        if not 0.0 <= momentum < 1.0 or steps < 1 or eps <= 0.0 or weight_decay < 0.0:
            raise ValueError("FlatMuon: 0 <= momentum < 1, steps >= 1, eps > 0, weight_decay >= 0")
        ops.muon_adjust(adjust, 1, 1)
        super().__init__(params, dict(lr=float(lr), momentum=float(momentum), nesterov=bool(nesterov), weight_decay=float(weight_decay),
                                      adjust=adjust, coefficients=tuple(coefficients or ops.NS_COEFFICIENTS), steps=int(steps), eps=float(eps)))
        if len(self.param_groups) != 1:
            raise NotImplementedError("FlatMuon supports a single parameter group")
        ps = self.param_groups[0]["params"]
        self.prec = prec
        self.matrices = [p for p in ps if p.dim() == 2 and min(p.shape) >= min_side]
        rest = [p for p in ps if not (p.dim() == 2 and min(p.shape) >= min_side)]
        self.adam = FlatAdam(rest, lr=lr, betas=betas, eps=adam_eps) if rest else None
        self._table = self._keys = self._lr_dev = self._lr_host = None

    def set_lr(self, lr: float):
        self.param_groups[0]["lr"] = float(lr)
        if self.adam is not None:
            self.adam.set_lr(lr)
        if self._lr_dev is not None:
            self._lr_dev.fill_(float(lr))
            self._lr_host = float(lr)

    def _live(self):
        return [p for p in self.matrices if p.requires_grad and p.grad is not None]

    def _table_keys(self, ps):
        """all that the table of jobs holds or was checked for: it is built anew where any of it differs"""
        keys = [self.param_groups[0]["adjust"]]
        for p in ps:
            m = self.state[p].get("momentum_buffer")
            keys.append((p.data_ptr(), p.grad.data_ptr(), 0 if m is None else m.data_ptr(), p.dtype, p.shape, p.stride(), p.grad.stride()))
        return keys

    def _build(self, ps):
        from . import ops
        for p in ps:
            st = self.state[p]
            if "momentum_buffer" not in st:
                st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
        self._table = ops.muon_jobs([p.detach() for p in ps], [p.grad for p in ps], [self.state[p]["momentum_buffer"] for p in ps],
                                    self.param_groups[0]["adjust"])
        self._keys = self._table_keys(ps)
        if self._lr_dev is None or self._lr_dev.device != ps[0].device:
            self._lr_host = float(self.param_groups[0]["lr"])
            self._lr_dev = torch.full((), self._lr_host, dtype=torch.float32, device=ps[0].device)

    def _capturable(self, ps):
        """refuses a captured step that would clear its state or write its learning rate: a replay would do so again every time"""
        lr, adam = float(self.param_groups[0]["lr"]), self.adam
        if self._lr_dev is None or self._lr_dev.device != ps[0].device or any("momentum_buffer" not in self.state[p] for p in ps) or \
                (adam is not None and adam._params() and adam._stale()):
            raise RuntimeError("FlatMuon.step(): take an eager step (it allocates the state) before the step is captured")
        if lr != self._lr_host or (adam is not None and adam._params() and lr != adam._lr_host):
            raise RuntimeError("FlatMuon.step(): use set_lr() before the capture, not param_groups: a captured step does not change its learning rate")

    @torch.no_grad()
    def step(self, closure=None):
        if closure is not None:
            raise NotImplementedError("FlatMuon.step() takes no closure")
        from . import ops
        if len(self.param_groups) != 1:
            raise NotImplementedError("FlatMuon supports a single parameter group")
        g = self.param_groups[0]
        ps = self._live()
        if ps and _capturing(ps[0].device):
            self._capturable(ps)
        if self.adam is not None:
            if self.adam.param_groups[0]["lr"] != g["lr"]:       # someone assigned param_groups[0]["lr"] directly
                self.adam.set_lr(g["lr"])
            if self.adam._params():
                self.adam.step()
        if not ps:
            return
        if self._keys != self._table_keys(ps):
            self._build(ps)
        if float(g["lr"]) != self._lr_host:
            self._lr_dev.fill_(float(g["lr"]))
            self._lr_host = float(g["lr"])
        ops.muon_launch(self._table, self._lr_dev, g["momentum"], g["nesterov"], g["weight_decay"], g["coefficients"], g["steps"], g["eps"],
                        self.prec, True)

    def state_dict(self):
        if self.adam is not None:
            for p in self.adam.param_groups[0]["params"]:
                if p in self.adam.state:
                    self.state[p] = dict(self.adam.state[p])
        sd = super().state_dict()
        for st in sd["state"].values():
            if torch.is_tensor(st.get("step")):
                st["step"] = st["step"].detach().clone().cpu()
        return sd

    def load_state_dict(self, state_dict):
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        ps = self.param_groups[0]["params"]
        if len(ids) != len(ps):
            raise ValueError(f"optimizer state_dict holds {len(ids)} parameters, this optimiser {len(ps)}")
        muon = set(map(id, self.matrices))
        for i, p in zip(ids, ps):
            st = state_dict["state"].get(i)
            key = "momentum_buffer" if id(p) in muon else "exp_avg"
            if st is not None and (not torch.is_tensor(st.get(key)) or tuple(st[key].shape) != tuple(p.shape)):
                raise ValueError(f"optimizer state of parameter {i} holds no {key} of shape {tuple(p.shape)}: another optimiser's, or another order")
        super().load_state_dict(state_dict)
        for p in ps:
            st = self.state.get(p)
            if st:
                for k, v in st.items():
                    if torch.is_tensor(v):
                        st[k] = v.clone()              # (torch shares tensors with the dict it is given)
        if self.adam is not None:
            self.adam.state.clear()                    # (a parameter that the loaded state does not hold starts anew)
            for p in self.adam.param_groups[0]["params"]:
                if p in self.state:
                    self.adam.state[p] = dict(self.state[p])
            self.adam._segs = None
        self._table = self._keys = None
        self.set_lr(float(self.param_groups[0]["lr"]))

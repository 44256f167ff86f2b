"""AdamW over many separate parameter tensors on MI355X, for training loops that go through torch autograd (the dense network of
`hubconf.MPMAE`, `main_pretrain.py --fast_path False`): a few kernel launches for the whole parameter list, moments in fp32 or in 8 bits, clip by
the global gradient norm in the same call. The fused pretraining step has its own AdamW over one flat buffer (`Engine.optimizer_step`).

    opt = AdamW(param_groups_weight_decay(model, 0.05), lr=1.5e-4, betas=(0.9, 0.95), state_bits=8, max_norm=1.0)
    loss.backward(); opt.step(); opt.zero_grad()

The update is torch.optim.AdamW's (main_pretrain.py:312-320); `state_dict()` has its layout, so checkpoints go both ways. There is no CPU form.
"""
import ctypes as C

import numpy as np
import torch

from . import _lib

BLOCK = 256          # elements that share a scale of the 8-bit moments; every tensor starts at a multiple of it in the moment buffers
CHUNK = 2048         # elements per workgroup (ADAMW_CHUNK of csrc/optim.cuh)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TABLE = np.dtype([("n", "<i8"), ("off", "<i8"), ("p", "<u8"), ("group", "<i4"), ("dt", "<i4")])      # MpmaeAdamwTensor

def moment_layout(numels):
    """Offsets of the tensors in the flat moment buffers (each starts a block of its own) and the buffers' length."""
    offsets, at = [], 0
    for n in numels:
        offsets.append(at)
        at += -(-n // BLOCK) * BLOCK
    return offsets, at


def quantize_moments(m, v):
    """fp32 moments (flat, whole blocks) -> (int8 codes of m, uint8 codes of v, scales of m, scales of v); decided in 64 bits."""
    m, v = m.reshape(-1, BLOCK).double(), v.reshape(-1, BLOCK).double()
    ms, vs = m.abs().amax(1), v.amax(1)
    bad_m, bad_v = ~torch.isfinite(ms), ~torch.isfinite(vs)
    dm = torch.where(bad_m | (ms == 0), 1.0, ms)[:, None]
    dv = torch.where(bad_v | (vs == 0), 1.0, vs)[:, None]
    km = torch.floor(127.0 * (m.abs() / dm).sqrt() + 0.5).clamp(max=127.0) * torch.sign(m)
    kv = torch.floor(255.0 * (v / dv).sqrt().sqrt() + 0.5).clamp(max=255.0)
    kv = torch.where(v > 0, kv.clamp(min=1.0), kv)
    km = torch.where(bad_m[:, None], 0.0, km).to(torch.int8)
    kv = torch.where(bad_v[:, None], 0.0, kv).to(torch.uint8)
    nan = float("nan")
    return km.reshape(-1), kv.reshape(-1), torch.where(bad_m, nan, ms).float(), torch.where(bad_v, nan, vs).float()


class _Plan:
    """Device tables and state of one parameter list."""

    def __init__(self, params, counts, device, bits, max_norm):
        self.params, self.counts, self.device, self.bits = params, counts, device, bits          # counts: parameters of every group
        self.shapes = [(p.shape, p.stride()) for p in params]          # the moments lie in this element order, also where a parameter is laid out anew later
        numels = [p.numel() for p in params]
        self.offsets, self.size = moment_layout(numels)
        nt = len(params)
        self.table = np.zeros(nt, _TABLE)
        self.table["n"], self.table["off"], self.table["group"] = numels, self.offsets, np.repeat(np.arange(len(counts)), counts)
        self.table["dt"], self.table["p"] = [_DTYPES[p.dtype] for p in params], [p.data_ptr() for p in params]
        per = -(-self.table["n"] // CHUNK)
        self.chunk_first = np.zeros(nt + 1, np.int32)
        self.chunk_first[1:] = np.cumsum(per)
        chunks = np.empty((int(per.sum()), 2), np.int32)
        chunks[:, 0] = np.repeat(np.arange(nt), per)
        chunks[:, 1] = np.arange(len(chunks)) - np.repeat(self.chunk_first[:-1], per)
        self.grads, self.orders = np.zeros(nt, np.uint64), np.zeros(nt, np.uint64)
        new = lambda n, dtype: torch.zeros(n, dtype=dtype, device=device)  # noqa: E731
        self.d_table = torch.from_numpy(self.table.view(np.uint8).copy()).to(device)
        self.d_chunks = torch.from_numpy(chunks).to(device)
        self.steps = new(nt, torch.int32)
        self.hyper = new(nt * _lib.ADAMW_HYPER_BYTES, torch.uint8)
        npart = _lib.ADAMW_NORM_BLOCKS * (nt // 480 + 1)
        self.partials = new(npart if max_norm else 1, torch.float64)
        self.norm_skip = new(2, torch.float32)
        self.norm, self.skip = self.norm_skip[0], self.norm_skip[1]
        if bits == 32:
            self.m, self.v, self.ms, self.vs = new(self.size, torch.float32), new(self.size, torch.float32), None, None
        else:
            self.m, self.v = new(self.size, torch.int8), new(self.size, torch.uint8)
            self.ms, self.vs = new(self.size // BLOCK, torch.float32), new(self.size // BLOCK, torch.float32)
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.args = _lib.AdamwArgs(tensors=at(self.d_table), chunks=at(self.d_chunks), chunk_first=self.chunk_first.ctypes.data, steps=at(self.steps),
                                   hyper=at(self.hyper), partials=at(self.partials), norm_skip=at(self.norm_skip), m=at(self.m), v=at(self.v),
                                   ms=at(self.ms), vs=at(self.vs), max_norm=float(max_norm or 0.0), nt=nt, npartials=npart, bits=bits)
        self.at, self.stale = C.addressof(self.args), False          # stale: parameters have moved and the device table does not know
        self.captured = False                                     # a graph holds the addresses of these buffers
        self.table_at, self.grads_at, self.orders_at = self.table.ctypes.data, self.grads.ctypes.data, self.orders.ctypes.data
        _lib.host_tensors().gather(params, self.table_at, device.index, self.grads_at, self.orders_at, False)      # (holds them to the order that offsets go by)
        torch.cuda.current_stream(device).synchronize()      # the tables and zeroed moments are there for whatever stream steps first

    def values(self):
        """Both moments as flat fp32 buffers: the state itself (32 bits) or what its codes stand for (8 bits)."""
        if self.bits == 32:
            return self.m, self.v
        m, v = torch.empty(self.size, dtype=torch.float32, device=self.device), torch.empty(self.size, dtype=torch.float32, device=self.device)
        a = self.args
        self.launch("adamw_values", lambda stream: _lib.load().mpmae_adamw_values(a.m, a.v, a.ms, a.vs, m.data_ptr(), v.data_ptr(), self.size, stream))
        return m, v

    def launch(self, what, call):
        """call(stream) with this plan's device as the current one."""
        if torch._C._cuda_getDevice() != self.device.index:
            with torch.cuda.device(self.device):
                return self.launch(what, call)
        self.captured |= torch.cuda.is_current_stream_capturing()
        err = call(torch._C._cuda_getCurrentRawStream(self.device.index))
        _lib.check(err, what)

    def views(self, flat):
        """A flat moment buffer as one tensor per parameter."""
        return [flat.as_strided(shape, stride, o) for (shape, stride), o in zip(self.shapes, self.offsets)]

    def store(self, m, v):
        """The inverse: flat fp32 moments into the state."""
        if self.bits == 32:
            self.m.copy_(m)
            self.v.copy_(v)
            return
        step = 1 << 22
        for a in range(0, self.size, step):
            b = min(self.size, a + step)
            km, kv, sm, sv = quantize_moments(m[a:b], v[a:b])
            self.m[a:b], self.v[a:b] = km, kv
            self.ms[a // BLOCK:b // BLOCK], self.vs[a // BLOCK:b // BLOCK] = sm, sv


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW over fp32 / bf16 / fp16 parameters of one GPU (types may be mixed), in a few launches for the whole list.

    state_bits   32: fp32 moments. 8: both moments in one byte per element and one fp32 scale per 256 elements.
    max_norm     not None: the gradients enter the update scaled by min(1, max_norm / (norm + 1e-6)), norm over all of them as in
                 torch.nn.utils.clip_grad_norm_ (the gradients themselves stay as they are); `grad_norm` is that norm, fp32, on the device. A step whose
                 norm is not finite changes nothing (`skipped` is then 1), as the fused pretraining step does.

    Parameters without a gradient are left alone. The update is formed in fp32 and rounded once to the parameter's type. Steps are counted on the
    device: a captured step replays as the next one, with the learning rate it was captured with; run one eager step before the capture. The graph
    holds the addresses of the optimizer's buffers: the optimizer has to outlive it, and takes no further groups after a capture.
    `param_groups` hold lr, betas, eps, weight_decay and may be changed between steps; lr is a number. Their lists of parameters stay those of the first
    step, object for object (a call after another edit than `add_param_group` is refused; `model.load_state_dict(assign=True)` puts new parameters into the
    model, for a new optimizer). The moments are in `flat_moments()` and `state_dict()`; `state` stays empty.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_norm=None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, not {state_bits!r}")
        if max_norm is not None and not 0.0 < max_norm < float("inf"):
            raise ValueError(f"max_norm is a positive number or None, not {max_norm!r}")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        self._check_group(defaults)
        self._state_bits, self._max_norm, self._plan = state_bits, max_norm, None
        super().__init__(params, defaults)

    # (both are built into the state and its launches: set on an optimizer that runs, they would do nothing)
    state_bits = property(lambda self: self._state_bits)
    max_norm = property(lambda self: self._max_norm)

    @staticmethod
    def _check_group(g):
        lr, (b1, b2) = g["lr"], g["betas"]
        if isinstance(lr, torch.Tensor):
            raise ValueError("lr is a number: a tensor would have to be read back on every step")
        if not 0.0 <= lr < float("inf") or not 0.0 <= g["eps"] < float("inf") or not 0.0 <= g["weight_decay"] < float("inf"):
            raise ValueError(f"lr, eps and weight_decay are finite and not negative: {lr}, {g['eps']}, {g['weight_decay']}")
        if not 0.0 <= b1 < 1.0 or not 0.0 <= b2 < 1.0:
            raise ValueError(f"betas lie in [0, 1): {g['betas']}")

    def add_param_group(self, group):
        if self._plan is not None and self.plan.captured:
            raise RuntimeError("a captured step of this optimizer holds its buffers, which a longer parameter list replaces: add groups before the capture")
        super().add_param_group(group)
        try:
            self._check_group(self.param_groups[-1])
            seen = {id(p) for g in self.param_groups[:-1] for p in g["params"]}          # (torch refuses a parameter of another group, and warns of one given twice)
            device = next((p.device for g in self.param_groups for p in g["params"]), None)
            for p in self.param_groups[-1]["params"]:
                if id(p) in seen:
                    raise ValueError("a parameter appears twice")
                seen.add(id(p))
                if p.dtype not in _DTYPES:
                    raise ValueError(f"parameters are fp32, bf16 or fp16, not {p.dtype}")
                if p.layout != torch.strided or not _dense(p):
                    raise ValueError("a parameter's elements have to lie densely in memory, each once")
                if p.device.type != "cuda":
                    raise ValueError(f"this optimizer runs on the GPU only: a parameter is on {p.device}")
                if p.device != device:
                    raise ValueError(f"the parameters of one optimizer are on one device: {device} and {p.device}")
            self._check_apart()
            if self._plan is not None:
                self._rebuild()
        except Exception:
            self.param_groups.pop()
            raise

    def _check_apart(self):
        """Two workgroups update two parameters at once: their memory must not overlap."""
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for g in self.param_groups for p in g["params"] if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("two parameters share memory")

    def _build(self):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("run one eager step before capturing one: the state is made on the first")
        _lib.host_tensors()
        params = [p for g in self.param_groups for p in g["params"]]
        self._check_apart()
        return _Plan(params, [len(g["params"]) for g in self.param_groups], params[0].device, self.state_bits, self.max_norm)

    def _rebuild(self):
        """The state for a longer parameter list, with the moments and step counts of the old one."""
        old, new = self._plan, self._build()
        values = old.values()
        where = {id(p): i for i, p in enumerate(new.params)}
        if any(new.orders[where[id(p)]] != order for p, order in zip(old.params, old.orders)):
            raise ValueError("a parameter has another shape or its elements in another order than when the optimizer first ran")
        into = [torch.zeros(new.size, device=new.device) for _ in range(2)]
        for i, p in enumerate(old.params):
            j = where[id(p)]
            for a, b in zip(into, values):
                a[new.offsets[j]:new.offsets[j] + p.numel()] = b[old.offsets[i]:old.offsets[i] + p.numel()]
            new.steps[j] = old.steps[i]
        new.store(*into)
        torch.cuda.current_stream(new.device).synchronize()      # the old buffers go back to the stream that made them, which may be another one
        self._plan = new

    @property
    def plan(self):
        if self._plan is None:
            self._plan = self._build()
        elif not _lib.host_tensors().same_lists(self.param_groups, self._plan.params, self._plan.counts):
            raise RuntimeError("the groups' parameters are not those of the first step: add_param_group adds some, others take a new optimizer")
        return self._plan

    @property
    def grad_norm(self):
        """Norm of all gradients before the last step's clip (0-d fp32 tensor on the device); needs max_norm."""
        if self.max_norm is None:
            raise RuntimeError("the gradient norm is formed with max_norm only")
        return self.plan.norm

    @property
    def skipped(self):
        """1 if the last step was skipped for a gradient norm that is not finite (0-d fp32 tensor on the device)."""
        return self.plan.skip

    @property
    def offsets(self):
        """First element of every parameter, in the order of the groups, in the buffers of `flat_moments()`."""
        return list(self.plan.offsets)

    def flat_moments(self):
        """(exp_avg, exp_avg_sq) of all parameters as two flat fp32 tensors, parameter i at `offsets[i]` in its own element order, zeros between
        them. With 32 bits the state itself, with 8 bits a copy of the values its codes stand for."""
        return self.plan.values()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        plan = self.plan
        grads, moved, other = _lib.host_tensors().gather(plan.params, plan.table_at, plan.device.index, plan.grads_at, plan.orders_at, True)
        plan.stale |= moved
        if plan.stale:                                 # (`p.data = ...`)
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a parameter has moved in memory: run one eager step before capturing one")
            self._check_apart()
            plan.d_table.copy_(torch.from_numpy(plan.table.view(np.uint8)))
            plan.stale = False
        if not grads:
            plan.captured |= torch.cuda.is_current_stream_capturing()
            plan.norm_skip.zero_()
            return loss
        copies = []                                    # gradients in another element order than their parameter's, alive until the launches are queued
        for i in other or ():
            p = plan.params[i]
            copies.append(torch.empty_like(p, memory_format=torch.preserve_format).copy_(p.grad))
            plan.grads[i] = copies[-1].data_ptr()
        done = _lib.host_tensors().adamw(plan.at, plan.grads_at, self.param_groups, plan.device.index)
        plan.captured |= bool(done & 1)
        if done > 1:
            for g in self.param_groups:                # (what the native call refuses, in words)
                self._check_group(g)
            _lib.check(done >> 1, "adamw_multi")
        return loss

    # ---- checkpoints: torch.optim.AdamW's layout -------------------------------------------------------------------------------------------
    def state_dict(self):
        """torch.optim.AdamW.state_dict() layout: per-parameter step / exp_avg / exp_avg_sq, fp32, all copies (an optimizer that
        loads them keeps the tensors it is given). With 8 bits they are the values of the codes, and loading them gives the same codes again."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        groups, at = [], 0
        for g in self.param_groups:
            groups.append({**{k: v for k, v in g.items() if k != "params"}, "amsgrad": False, "maximize": False, "foreach": None, "capturable": False,
                           "differentiable": False, "fused": None, "decoupled_weight_decay": True, "params": list(range(at, at + len(g["params"])))})
            at += len(g["params"])
        state = {}
        if self._plan is not None:
            plan, steps = self.plan, self._plan.steps.tolist()
            for i, (m, v) in enumerate(zip(*map(plan.views, plan.values()))):
                if steps[i]:
                    state[i] = {"step": torch.tensor(float(steps[i])), "exp_avg": m.clone(), "exp_avg_sq": v.clone()}
        out = {"state": state, "param_groups": groups}
        for hook in self._optimizer_state_dict_post_hooks.values():
            done = hook(self, out)
            out = out if done is None else done
        return out

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """What this class or torch.optim.AdamW wrote for the same parameter groups."""
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            done = hook(self, state_dict)
            state_dict = state_dict if done is None else done
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("loaded state dict has other parameter groups than the optimizer")
        if any(g.get("amsgrad") or g.get("maximize") for g in groups):
            raise ValueError("amsgrad and maximize are not supported")
        for g in groups:
            self._check_group({**self.defaults, **{k: v for k, v in g.items() if k != "params"}})
        plan = self.plan
        ids = [i for g in groups for i in g["params"]]
        entries = [state_dict["state"].get(i) or None for i in ids]          # (an empty entry, as reading `state[p]` leaves one behind, is none)
        for (shape, _), st in zip(plan.shapes, entries):
            for key in ("exp_avg", "exp_avg_sq") if st is not None else ():
                if not isinstance(st.get(key), torch.Tensor) or st[key].shape != shape or st[key].is_complex():
                    raise ValueError(f"loaded {key} is {getattr(st.get(key), 'shape', None)} for a parameter of shape {tuple(shape)}")
        steps = [0 if st is None else float(st.get("step", -1)) for st in entries]
        if not all(0 <= t < 2 ** 31 and t == int(t) for t in steps):
            raise ValueError(f"loaded step counts are whole numbers from 0 on: {steps}")
        for mine, g in zip(self.param_groups, groups):
            mine.update({k: v for k, v in g.items() if k in self.defaults or k not in _TORCH_ONLY})
        into = [plan.m, plan.v] if self.state_bits == 32 else [torch.zeros(plan.size, device=plan.device) for _ in range(2)]
        for flat, key in zip(into, ("exp_avg", "exp_avg_sq")):
            views = plan.views(flat)
            there = [(view, st[key]) for view, st in zip(views, entries) if st is not None]
            absent = [view for view, st in zip(views, entries) if st is None]
            if there:
                torch._foreach_copy_(*map(list, zip(*there)))
            if absent:
                torch._foreach_zero_(absent)
        if self.state_bits == 8:
            plan.store(*into)
        plan.steps.copy_(torch.tensor([int(t) for t in steps], dtype=torch.int32))
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def __getstate__(self):
        raise TypeError("the state lives in device buffers: use state_dict()")


_TORCH_ONLY = {"params", "amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay"}


def _dense(p):
    """Whether the elements fill one stretch of memory, each once, in some order of the dimensions."""
    if p.is_contiguous():
        return True
    at = 1
    for size, stride in sorted(((n, s) for n, s in zip(p.shape, p.stride()) if n != 1), key=lambda x: x[1]):
        if stride != at:
            return False
        at *= size
    return True

"""``AdamW`` and ``AdamW8bit``: AdamW with decoupled weight decay over many
tensors in one launch, and the norm of a set of gradients.

They stand beside ``SMO`` / ``SMO8bit`` for parameters whose moments are kept at
full resolution: ``AdamW`` holds both moments in fp32 whatever the parameters'
type, ``AdamW8bit`` in one byte each (square-root companded codes with a scale
for every block of 64, 128 or 256 elements).  For bf16 and fp16 parameters
``master_weights=True`` keeps the parameters themselves in fp32 too and hands the
model their rounding.  The arithmetic is stated in include/smo_b200.h
(``smo_adamw_tensor``).

As with the other optimizers here the parameters are CUDA tensors (fp32, bf16
or fp16) with gradients of their own type, the work runs on the current stream,
and there is no CPU path.  All tensors of a step are written in one launch or in
launches that overlap: parameters that share memory are refused.
"""

from __future__ import annotations

from itertools import chain

import numpy as np
import torch
from torch.optim.optimizer import Optimizer, _global_optimizer_post_hooks, _global_optimizer_pre_hooks

from . import _host, _lib
from .optimizers import _DTYPE_CODES, _host_ext, _named, _same_dense_layout, protected_param_groups

__all__ = ["AdamW", "AdamW8bit", "clip_grad_norm_", "grad_norm"]

BLOCK_SIZES = (64, 128, 256)

_LEAST_NORM = 2.0 ** -149  # as fp32 numbers smaller bounds are 0, which stands for no bound

_FLOAT_KEYS = ("exp_avg", "exp_avg_sq")
_CODE_KEYS = ("m_q", "m_s", "v_q", "v_s")
_STATE_DTYPES = {"exp_avg": torch.float32, "exp_avg_sq": torch.float32, "master": torch.float32, "m_q": torch.int8,
                 "m_s": torch.float32, "v_q": torch.uint8, "v_s": torch.float32}


def _check_options(name, group, defaults):
    """Refuses options of torch's AdamW and Adam under which the step would be another one, and values that it cannot
    take."""
    for key in ("maximize", "amsgrad"):
        if group.get(key):
            raise ValueError(f"{name} has no {key}")
    if not group.get("decoupled_weight_decay", True) and group.get("weight_decay", defaults["weight_decay"]):
        raise ValueError(f"{name} decays the weights themselves: decoupled_weight_decay=False is another step")
    # the 8-bit step's quotient takes smaller denominators as 0
    if name == "AdamW8bit" and 0.0 < group.get("eps", defaults["eps"]) < 2.0 ** -126:
        raise ValueError(f"Invalid epsilon value: {group.get('eps', defaults['eps'])} is below fp32's normal numbers")


def _check_writable(what, tensors):
    if not torch.is_inference_mode_enabled() and any(t.is_inference() for t in tensors):
        raise RuntimeError(f"{what} writes inference tensors in inference mode only")


def _stream(dev) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


# ---------------------------------------------------------------- gradient norms


def _norm(parameters, max_norm, what):
    lib = _lib.load()
    ext, fn, ws = _host_ext(), _lib.address("smo_grad_norm"), _lib.address("smo_grad_norm_workspace_size")
    parameters = [parameters] if torch.is_tensor(parameters) else list(parameters)
    got = ext.grad_norm(parameters, max_norm, fn, ws)
    if got is None:
        got = _norm_of_copies(parameters, max_norm, what, ext, fn, ws)
        if got is None:
            return torch.zeros((), dtype=torch.float32, device="cpu")
    if got[0]:
        _lib.check(got[0], what)
    return got[1]


def _once(t):
    """Index of one of each of t's repeated elements, or None where they overlap in another way than by strides of 0."""
    extent = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if stride and size > 1:
            if stride < extent:
                return None
            extent += stride * (size - 1)
    return tuple(slice(0, 1) if stride == 0 else slice(None) for stride in t.stride())


@torch.no_grad()
def _norm_of_copies(parameters, max_norm, what, ext, fn, ws):
    """Refusals, no gradients at all (None), parameters given twice (taken once),
    and gradients with gaps or repeated elements: those are taken as copies,
    written back when clipped (a repeated element once)."""
    grads = [p.grad for p in {id(p): p for p in parameters}.values() if p.grad is not None]
    for g in grads:
        if g.is_sparse:
            raise RuntimeError(f"{what} does not support sparse gradients.")
        if g.device.type != "cuda":
            raise RuntimeError(f"{what} (B200 build) takes CUDA tensors only; got a gradient on {g.device}")
        if g.dtype not in _DTYPE_CODES:
            raise TypeError(f"{what} (B200 build) takes fp32, bf16 or fp16 gradients; got {g.dtype}")
        if g.device != grads[0].device:
            raise RuntimeError(f"{what} takes the gradients of one device; got {grads[0].device} and {g.device}")
    if not grads:
        return None
    once = [_once(g) for g in grads] if max_norm > 0 else []
    if max_norm > 0:
        _check_writable(what, grads)
    if None in once:
        raise RuntimeError(f"{what} cannot scale a gradient whose elements overlap")
    holders = []
    for g in grads:
        # only its gradient counts: a parameter of g's shape without that much memory
        holder = torch.nn.Parameter(g.new_empty(()).expand(g.shape))
        holder.grad = g.contiguous()
        holders.append(holder)
    got = ext.grad_norm(holders, max_norm, fn, ws)
    if got is None:
        raise RuntimeError(f"{what}: two parameters share one gradient or, to be scaled, a part of it")
    if max_norm > 0:
        for g, h, index in zip(grads, holders, once):
            if h.grad.data_ptr() != g.data_ptr():
                g[index].copy_(h.grad[index])
    return got


def grad_norm(parameters) -> torch.Tensor:
    """The 2-norm over the gradients of all ``parameters`` (an iterable, or one
    parameter) as one vector: an fp32 tensor of no dimensions on their device.

    Parameters without a gradient are left out.  Each gradient is read once;
    squares and sums are held in double, in an order that depends on the sizes and
    the addresses' alignment alone, so a call repeated gives the same bits.  Nothing
    synchronises.  A parameter given twice counts once.  Without any gradient:
    0, on the CPU."""
    return _norm(parameters, 0.0, "grad_norm")


def clip_grad_norm_(parameters, max_norm: float) -> torch.Tensor:
    """Multiplies the gradients of all ``parameters`` in place by
    ``min(1, max_norm / (norm + 1e-6))`` and returns ``norm``, their 2-norm before
    (see ``grad_norm``).  A norm that is NaN makes every gradient NaN.  Gradients
    that share elements are refused.

    ``AdamW`` and ``AdamW8bit`` clip within the step (``max_grad_norm``), without
    writing the gradients; this is for ``SMO``, ``SMO8bit`` and any other user of
    the gradients."""
    max_norm = float(max_norm)
    if not max_norm >= _LEAST_NORM:
        raise ValueError(f"Invalid max_norm: {max_norm}")
    return _norm(parameters, max_norm, "clip_grad_norm_")


# ---------------------------------------------------------------- optimizers


def _check_apart(name, items):
    """Refuses parameters that share elements, with each other (as far as each is one span of memory) or within."""
    spans = []
    for p, _, _, _ in items:
        if p.is_contiguous():
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        elif _once(p) is None or any(stride == 0 and size > 1 for stride, size in zip(p.stride(), p.shape)):
            raise ValueError(f"{name}: elements of a parameter share memory")
    spans.sort()
    if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
        raise ValueError(f"{name}: two parameters share memory")


class _AdamWBase(Optimizer):
    _name = "AdamW"

    def __init__(self, params, lr, betas, eps, weight_decay, master_weights, max_grad_norm, capturable, extra):
        if torch.is_tensor(lr) and not capturable:
            raise ValueError("lr as a tensor needs capturable=True")
        if not torch.is_tensor(lr) and not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 0: {betas[0]}")
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 1: {betas[1]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if max_grad_norm is not None and not max_grad_norm >= _LEAST_NORM:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, **extra))
        self.master_weights = bool(master_weights)
        self.capturable = bool(capturable)
        self.max_grad_norm = max_grad_norm
        # norm of the gradients that the last step saw, before clipping; kept
        # only with max_grad_norm, and overwritten by the next step
        self.last_grad_norm = None
        # the C++ host path of what it was made of: (state, param groups, capsule,
        # device index, number of tensors)
        self._plan = None
        self._workspace = {}    # device index -> (workspace, norm)
        self._scalars = {}      # device index -> scalars of each tensor (capturable)
        self._kept = []         # outgrown and replaced ones of the two, which captured graphs may hold
        self._captured = False  # a step was captured: graphs hold the states' addresses

    # ---------------------------------------------------------------- state

    # torch's Optimizer pickles (and deep-copies) its groups and state only
    _SETTINGS = ("master_weights", "max_grad_norm", "capturable")

    def __getstate__(self):
        return dict(super().__getstate__(), **{k: getattr(self, k) for k in self._SETTINGS})

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plan = None
        self._kept = getattr(self, "_kept", [])
        self._captured = getattr(self, "_captured", False)
        if not self._captured:
            for held in ("_workspace", "_scalars"):
                self._kept += getattr(self, held, {}).values()
                setattr(self, held, {})
            self.last_grad_norm = None
        for p, held, old in self.__dict__.pop("_incoming", ()):
            self.state[p] = self._in_place(held, old) if self._captured and old else held

    @torch.no_grad()
    def _in_place(self, held, old):
        """A loaded state, in the tensors of the old one (whose addresses captured graphs hold) where it is laid out
        like it."""
        if held.keys() != old.keys() or any(not torch.is_tensor(t) or t.dtype != held[k].dtype or
                                            t.device != held[k].device or t.shape != held[k].shape for k, t in old.items()):
            return held
        for k, t in old.items():
            t.copy_(held[k])
        return old

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            _check_options(self._name, param_group, self.defaults)
        super().add_param_group(param_group)
        # torch only warns of a parameter that a group holds twice; stepped in one
        # launch, the two would write the same memory
        params = self.param_groups[-1]["params"]
        if len(set(map(id, params))) < len(params):
            self.param_groups.pop()
            raise ValueError("a parameter appears more than once in a parameter group")

    def _eight_bit(self, p, group) -> bool:
        return False

    def _init_state(self, p, group):
        state = self.state[p]
        state["step"] = torch.zeros((), dtype=torch.float32, device=p.device) if self.capturable else 0
        if self._eight_bit(p, group):
            block = group["block_size"]
            nb = _host.num_blocks(p.numel(), block)
            for q, s, dtype in (("m_q", "m_s", torch.int8), ("v_q", "v_s", torch.uint8)):
                state[q] = torch.zeros((nb, block), dtype=dtype, device=p.device)
                state[s] = torch.zeros((nb, 1), dtype=torch.float32, device=p.device)
        else:
            for key in _FLOAT_KEYS:
                state[key] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)

    def _ready(self):
        """Checks every parameter with a gradient and gives it its state."""
        found = []
        for group in self.param_groups:
            for p in group["params"]:
                grad = p.grad
                if grad is None:
                    continue
                if grad.is_sparse:
                    raise RuntimeError(f"{self._name} does not support sparse gradients.")
                if p.device.type != "cuda":
                    raise RuntimeError(f"{self._name} (B200 build) steps CUDA tensors only; "
                                       f"got a parameter on {p.device}")
                if p.dtype not in _DTYPE_CODES or grad.dtype != p.dtype:
                    raise TypeError(f"{self._name} (B200 build) steps fp32, bf16 or fp16 parameters with "
                                    f"gradients of the same dtype; got {p.dtype} / {grad.dtype}")
                _check_writable(self._name, (p,))
                state = self.state[p]
                master = self.master_weights and p.dtype != torch.float32 and "master" not in state
                if ("step" not in state or master) and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(f"{self._name}: the first step of a parameter cannot be captured (replays would "
                                       "make its state anew); take one before the capture")
                if "step" not in state:
                    self._init_state(p, group)
                if master:
                    state["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)
                state["step"] = self._step_value(p, state["step"])
                found.append((p, grad, state, group))
        return found

    def _step_value(self, p, step):
        """A step count as this optimizer keeps it."""
        if not self.capturable:
            return step if type(step) is int else int(step)
        if torch.is_tensor(step):
            if step.dtype == torch.float32 and step.device == p.device and step.numel() == 1:
                return step
            return step.to(dtype=torch.float32, device=p.device).reshape(())
        return torch.full((), float(step), dtype=torch.float32, device=p.device)

    def load_state_dict(self, state_dict):
        """Loads what ``state_dict()`` of this class, of the other one here or of
        ``torch.optim.AdamW`` returned: moments are kept in 32 bits, and brought
        into 8 bits or out of them (or to another block size) where this
        optimizer holds them so.  The loaded tensors are copied.  Groups with
        ``maximize``, ``amsgrad`` or a decay that is not decoupled are refused; a
        load that is refused leaves the optimizer as it was."""
        def prepare(opt, sd):
            groups = [{**self.defaults, **g} for g in sd["param_groups"]]
            for group in groups:
                _check_options(self._name, group, self.defaults)
            if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
                return None  # torch refuses it
            own = chain.from_iterable(g["params"] for g in self.param_groups)
            names = [(name, g) for g in groups for name in g["params"]]
            self._incoming = [(p, self._loaded(p, sd["state"][name], group), self.state.get(p))
                              for p, (name, group) in zip(own, names) if sd["state"].get(name)]
            # torch's loader would cast every tensor to the parameter's type
            taken = {name for name, _ in names}
            return dict(sd, state={k: v for k, v in sd["state"].items() if k not in taken})

        rates, states = ([g["lr"] for g in self.param_groups], dict(self.state)) if self._captured else ((), {})
        # registered last: sees the dict as the other hooks leave it
        hook = self.register_load_state_dict_pre_hook(prepare)
        try:
            super().load_state_dict(state_dict)  # its __setstate__() takes what comes in
        finally:
            hook.remove()
            self._incoming = ()
        for group in self.param_groups:
            for key, value in self.defaults.items():
                group.setdefault(key, value)
        # what captured graphs hold stays alive, and a learning rate on the device is theirs still, unless the groups
        # that share it have come apart
        self._kept += [st for p, st in states.items() if self.state.get(p) is not st]
        for lr in {id(lr): lr for lr in rates if torch.is_tensor(lr)}.values():
            groups = [g for g, r in zip(self.param_groups, rates) if r is lr]
            if len({float(g["lr"]) for g in groups}) == 1:
                lr.fill_(float(groups[0]["lr"]))
                for g in groups:
                    g["lr"] = lr
            else:
                self._kept.append(lr)

    def _loaded(self, p, saved, group):
        """A saved state as this optimizer holds it, in tensors of its own."""
        step = saved.get("step", 0)
        state = {"step": self._step_value(p, step.clone() if torch.is_tensor(step) else step)}
        for key, dtype in _STATE_DTYPES.items():
            if torch.is_tensor(saved.get(key)):
                state[key] = saved[key].to(device=p.device, dtype=dtype, copy=True)
        if not self.master_weights or p.dtype == torch.float32:
            state.pop("master", None)
        return self._adopt(p, state, group)

    def _adopt(self, p, state, group):
        """A loaded state as this optimizer holds it."""
        shape = tuple(p.shape)
        for key in _FLOAT_KEYS + ("master",):
            if key in state and tuple(state[key].shape) != shape:
                raise ValueError(f"state['{key}'] has the shape {tuple(state[key].shape)}; the parameter's is {shape}")
        coded = all(k in state for k in _CODE_KEYS)
        if coded:
            q = state["m_q"]
            block = q.shape[1] if q.dim() == 2 else 0
            nb = _host.num_blocks(p.numel(), block) if block in BLOCK_SIZES else -1
            for key in _CODE_KEYS:
                want = (nb, block) if key.endswith("_q") else (nb, 1)
                if tuple(state[key].shape) != want:
                    raise ValueError(f"state['{key}'] has the shape {tuple(state[key].shape)}, which no block size of "
                                     f"{BLOCK_SIZES} gives a parameter of {p.numel()} elements")
                state[key] = state[key].contiguous()
        elif not all(k in state for k in _FLOAT_KEYS):
            raise ValueError("the loaded state has neither exp_avg and exp_avg_sq nor m_q, m_s, v_q and v_s")
        eight = self._eight_bit(p, group)
        if coded and not (eight and group["block_size"] == block):
            state.update(zip(_FLOAT_KEYS, _decode([(p, state)])[0]))
            coded = False
            for key in _CODE_KEYS:
                del state[key]
        if eight and not coded:
            state.update(_encode(p, state, group["block_size"]))
            for key in _FLOAT_KEYS:
                del state[key]
        return state

    # ---------------------------------------------------------------- step

    def step(self, closure=None, grad_scale=None):
        """One step of every parameter that has a gradient.

        ``grad_scale``: an fp32 tensor of one element on the parameters' device;
        the step multiplies every gradient by it (and leaves the gradients as
        they are).  ``max_grad_norm`` bounds the scaled gradients' norm."""
        # torch's wrapper around step() costs 7.6 us, more than a small step's own
        # host work: entered only for what it does, hooks and profiler records
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_optimizer_pre_hooks
                or _global_optimizer_post_hooks or torch.autograd._profiler_enabled()):
            return self._hooked_step(closure, grad_scale)
        return self._step(closure, grad_scale)

    step.hooked = True  # torch's Optimizer wraps a step() without this mark

    def _step(self, closure, grad_scale):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if grad_scale is not None:
            if not torch.is_tensor(grad_scale) or grad_scale.dtype != torch.float32 or grad_scale.numel() != 1:
                raise TypeError("grad_scale must be an fp32 tensor of one element")
        plan = self._plan
        if plan is not None and plan[0] is self.state and plan[1] is self.param_groups:
            rc = self._run_plan(grad_scale)
            if rc >= 0:
                return loss
        with torch.no_grad():
            items = self._ready()
            self._plan = None
            if not items:
                self.last_grad_norm = None
                return loss
            _check_apart(self._name, items)
            made = _host_ext().adamw_plan(self.param_groups, self.state, _lib.address("smo_adamw_step"),
                                          _lib.address("smo_adamw_advance") if self.capturable else 0)
            if made is not None:
                self._plan = (self.state, self.param_groups, *made)
            if made is None or self._run_plan(grad_scale) < 0:
                self._plan = None
                self._slow_step(items, grad_scale)
        return loss

    _hooked_step = Optimizer.profile_hook_step(_step)

    def _scale_address(self, grad_scale, index):
        if grad_scale is None:
            return 0
        if grad_scale.device.type != "cuda" or grad_scale.device.index != index:
            raise RuntimeError(f"grad_scale must be on the parameters' device (cuda:{index}); got {grad_scale.device}")
        return grad_scale.data_ptr()

    def _norm_buffers(self, index, tensors):
        """(max_norm, norm address, workspace address, bytes) of a step over so many tensors of a device."""
        if self.max_grad_norm is None:
            self.last_grad_norm = None
            return 0.0, 0, 0, 0
        if not self.max_grad_norm >= _LEAST_NORM:
            raise ValueError(f"Invalid max_grad_norm: {self.max_grad_norm}")
        need = _lib.load().smo_grad_norm_workspace_size(tensors)
        kept = self._workspace.get(index)
        if kept is None or kept[0].numel() < need:
            if kept is not None:
                self._kept.append(kept)
            dev = torch.device("cuda", index)
            kept = (torch.empty(need, dtype=torch.uint8, device=dev), torch.zeros((), dtype=torch.float32, device=dev))
            self._workspace[index] = kept
        self.last_grad_norm = kept[1]
        return float(self.max_grad_norm), kept[1].data_ptr(), kept[0].data_ptr(), kept[0].numel()

    def _scalar_address(self, index, tensors):
        """Device memory for the scalars of so many tensors (capturable), or 0."""
        if not self.capturable:
            return 0
        kept = self._scalars.get(index)
        if kept is None or kept.shape[0] < tensors:
            if kept is not None:
                self._kept.append(kept)
            kept = torch.empty((tensors, len(_lib.ADAMW_HYPER_DTYPE)), dtype=torch.float32,
                               device=torch.device("cuda", index))
            self._scalars[index] = kept
        return kept.data_ptr()

    def _run_plan(self, grad_scale) -> int:
        _, _, cap, index, tensors = self._plan
        if self.capturable and not self._captured:
            self._captured = torch.cuda.is_current_stream_capturing()
        scale = self._scale_address(grad_scale, index)
        rc = _host_ext().adamw_run(cap, self._scalar_address(index, tensors), scale, *self._norm_buffers(index, tensors))
        if rc > 0:
            self._check(rc)
        return rc

    def _check(self, rc):
        if rc == _lib.SMO_ERR_CAPTURE:
            raise RuntimeError(f"{self._name}.step cannot be captured into a CUDA graph: the step count and the learning "
                               "rate are host values, which every replay would repeat (see capturable=True)")
        _lib.check(rc, "smo_adamw_step")

    def _slow_step(self, items, grad_scale):
        """Several devices, or parameters, gradients or moments that do not share
        one layout: the latter are stepped on contiguous copies, written back in
        stream order."""
        per_dev = {}
        if self.capturable and not self._captured:
            self._captured = torch.cuda.is_current_stream_capturing()
        for item in items:
            per_dev.setdefault(item[0].device, []).append(item)
        if len(per_dev) > 1 and (self.max_grad_norm is not None or grad_scale is not None):
            raise RuntimeError(f"{self._name}: max_grad_norm and grad_scale need all parameters on one device")
        for dev, items in per_dev.items():
            table = np.zeros(len(items), dtype=_lib.ADAMW_DTYPE)
            back, keep = [], []
            for rec, (p, grad, state, group) in zip(table, items):
                self._fill(rec, p, grad, state, group, back, keep)
            with torch.cuda.device(dev):
                scale = self._scale_address(grad_scale, dev.index)
                max_norm, norm, ws, nbytes = self._norm_buffers(dev.index, len(items))
                if self.capturable:
                    self._advance(dev, items, table)
                self._check(_lib.load().smo_adamw_step(table.ctypes.data, len(table), scale, max_norm, norm, ws, nbytes,
                                                       _stream(dev)))
                for dst, src in back:
                    dst.copy_(src)
            # autograd sees that the parameters were written
            torch.autograd.graph.increment_version([p for p, _, _, _ in items])
            if not self.capturable:
                for p, grad, state, group in items:
                    state["step"] += 1

    def _advance(self, dev, items, table):
        """Step counts and scalars of a slow step on the device."""
        schedule = np.zeros(len(items), dtype=_lib.SCHEDULE_DTYPE)
        out = self._scalar_address(dev.index, len(items))
        for i, (rec, (p, grad, state, group)) in enumerate(zip(schedule, items)):
            lr = group["lr"]
            if torch.is_tensor(lr):
                if lr.dtype != torch.float32 or lr.device != dev or lr.numel() != 1:
                    raise TypeError(f"lr must be a number or an fp32 tensor of one element on {dev}")
                rec["lr_dev"] = lr.data_ptr()
            else:
                rec["lr"] = lr
            rec["step"] = state["step"].data_ptr()
            rec["beta1"], rec["beta2"] = group["betas"]
            rec["eps"], rec["weight_decay"] = group["eps"], group["weight_decay"]
            table[i]["hp_dev"] = out + i * _lib.ADAMW_HYPER_DTYPE.itemsize
        self._check(_lib.load().smo_adamw_advance(schedule.ctypes.data, len(schedule), out, _stream(dev)))

    def _fill(self, rec, p, grad, state, group, back, keep):
        coded = all(k in state for k in _CODE_KEYS)
        floats = ("master",) if "master" in state else ()
        floats += () if coded else _FLOAT_KEYS
        for key in floats:
            t = state.get(key)
            _check_state_tensor(p, key, t)
            if t.shape != p.shape:
                raise ValueError(f"state['{key}'] must have the parameter's shape {tuple(p.shape)}")
        held = {k: state[k] for k in floats}
        direct = _same_dense_layout(p, *held.values()) and (not coded or p.is_contiguous())

        def local(t, out):
            # the tensor itself, or a contiguous copy of it that is written back
            if direct or t.is_contiguous():
                return t
            c = t.contiguous()
            keep.append(c)
            if out:
                back.append((t, c))
            return c

        if direct:
            g = grad
            if grad.shape != p.shape or grad.stride() != p.stride():
                g = torch.empty_like(p).copy_(grad)  # empty_like keeps the dense layout of p
        else:
            g = grad.contiguous()
        keep.append(g)
        rec["param"], rec["grad"] = local(p.detach(), True).data_ptr(), g.data_ptr()
        for k, t in held.items():
            rec[k] = local(t, True).data_ptr()
        rec["n"], rec["dtype"] = p.numel(), _DTYPE_CODES[p.dtype]
        if coded:
            _coded_row(rec, p, state)
        else:
            rec["kind"] = _lib.SMO_ADAMW_F32
        if not self.capturable:
            rec["hp"] = _host.adamw_scalars(group["lr"], group["betas"], group["eps"], group["weight_decay"],
                                            state["step"] + 1)


class AdamW(_AdamWBase):
    """AdamW (decoupled weight decay), both moments in fp32.

    ``master_weights``: keep an fp32 copy of each bf16 or fp16 parameter
    (``state[p]["master"]``), step that, and write its rounding to the parameter.
    The copy is made of the parameter at its first step; a parameter that is
    changed from outside afterwards needs its copy changed too.
    ``max_grad_norm``: scale the gradients of each step by
    ``min(1, max_grad_norm / (norm + 1e-6))`` within the step;
    ``last_grad_norm`` is then the norm (a device tensor, overwritten by the next
    step).  As with ``clip_grad_norm_`` a norm that is NaN makes the step NaN.
    ``capturable``: the step can be captured into a CUDA graph and replayed.  The
    step counts are then fp32 device tensors and the scalars are formed on the
    device (one more launch); ``lr`` may be an fp32 device tensor, which replays
    read.  Take a step before the capture: it makes the state.  Graphs hold addresses:
    after a capture ``load_state_dict`` writes to the states' present tensors, and
    the optimizer, its parameters and their gradients have to outlive the graphs.

    ``state[p]``: ``step`` (int), ``exp_avg``, ``exp_avg_sq``, with master weights
    ``master``."""
    _name = "AdamW"

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, master_weights=False,
                 max_grad_norm=None, capturable=False):
        super().__init__(params, lr, betas, eps, weight_decay, master_weights, max_grad_norm, capturable, {})


class AdamW8bit(_AdamWBase):
    """AdamW with moments of one byte an element.

    The first moment m and u, the root of the second, are kept in blocks of
    ``block_size`` (64, 128 or 256) consecutive elements as codes ``c`` that stand
    for ``s * sign(c) * (c / 127)**2`` and ``s * (c / 255)**2``, ``s`` the block's
    largest value: relative steps of 2 / c, so the larger values, which steer the
    update, are held most finely.  The update itself uses the moments before they
    are coded.

    Codes round to the nearest, so a moment that changes by less than half a code
    in a step keeps its code, however many steps follow.  Without a gradient a
    step shrinks codes by ``sqrt(beta1)`` and ``beta2 ** (1 / 4)``, or, in a block
    without any gradient, the scale alone.  So beside an element that keeps the
    block's scale up, m falls to 0.5 % of the block's largest and no further
    (``beta1`` = 0.9), u to 2.3 % with ``beta2`` = 0.95, to 61 % with 0.99, and with
    0.999 not at all; where m stays above 0 the parameter keeps moving.  With
    gradients of a steady size u is right within 8 % (its median within 0.4 %) at
    ``beta2`` of 0.99 and below; at 0.999 its median is 10 % too large after 3,000
    steps, 16 % after 6,000 and 36 % after 12,000 (blocks of 128), and the updates
    are that much too small.  Long runs want a ``beta2`` of 0.99 or less, or
    ``AdamW``.

    Tensors of fewer than ``min_8bit_numel`` elements, and those of groups with
    ``compress=False``, keep fp32 moments as in ``AdamW``; ``protect_output``
    makes such groups by the parameters' names, as for ``SMO8bit``.

    ``state[p]``: ``step``, ``m_q`` (int8) and ``v_q`` (uint8) of shape
    (blocks, block_size), ``m_s`` and ``v_s`` (fp32) of shape (blocks, 1)."""
    _name = "AdamW8bit"
    _SETTINGS = _AdamWBase._SETTINGS + ("min_8bit_numel",)

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, block_size=128,
                 min_8bit_numel=4096, master_weights=False, max_grad_norm=None, protect_output=False,
                 capturable=False):
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"Invalid block_size: {block_size}. Must be one of {BLOCK_SIZES}")
        if not 0 <= min_8bit_numel:
            raise ValueError(f"Invalid min_8bit_numel: {min_8bit_numel}")
        if protect_output:
            params = protected_param_groups(_named(params), protect_output)
        self.min_8bit_numel = int(min_8bit_numel)
        super().__init__(params, lr, betas, eps, weight_decay, master_weights, max_grad_norm, capturable,
                         dict(block_size=block_size))

    def _eight_bit(self, p, group) -> bool:
        return bool(group.get("compress", True)) and p.numel() >= max(1, self.min_8bit_numel)

    def moments(self, params=None, out=None):
        """``[(exp_avg, exp_avg_sq)]`` of ``params`` (default: every parameter
        that has a state) as fp32 tensors of the parameters' shapes: what the
        codes stand for, all tensors in one launch.  A parameter whose moments
        are kept in fp32 gives those.  ``out``: pairs of contiguous fp32 tensors
        to write to."""
        if params is None:
            params = [p for g in self.param_groups for p in g["params"] if self.state.get(p)]
        params = [params] if torch.is_tensor(params) else list(params)
        if out is None:
            return self._moments(params)
        out = list(out)
        plan = self._plan
        plan = plan[2] if plan is not None and plan[0] is self.state else None
        got = _host_ext().adamw_moments(self.state, params, out, _lib.address("smo_adamw_decode"), plan)
        if got < 0:
            return self._moments(params, out)
        if got > 0:
            _lib.check(got, "smo_adamw_decode")
        return out

    @torch.no_grad()
    def _moments(self, params, out=None):
        """Refusals, parameters with fp32 moments among the others, several devices."""
        if out is not None and len(out) != len(params):
            raise ValueError(f"{len(params)} parameters, {len(out)} outputs")
        for p in params:
            if not self.state.get(p):
                raise KeyError("moments of a parameter that has no state yet")
        coded = [i for i, p in enumerate(params) if "m_q" in self.state[p]]
        pairs = [None if "m_q" in self.state[p] else tuple(self.state[p][k] for k in _FLOAT_KEYS) for p in params]
        if out is None:
            for i, pair in zip(coded, _decode([(params[i], self.state[params[i]]) for i in coded])):
                pairs[i] = pair
            return pairs
        for p, pair in zip(params, out):
            _check_writable("moments", pair)
            for t in pair:
                if t.dtype != torch.float32 or t.device != p.device or t.shape != p.shape or not t.is_contiguous():
                    raise TypeError(f"out must be contiguous fp32 tensors of the parameters' shapes on {p.device}")
        _decode([(params[i], self.state[params[i]]) for i in coded], [out[i] for i in coded])
        torch.autograd.graph.increment_version([t for i in coded for t in out[i]])
        for pair, dst in zip(pairs, out):
            if pair is not None:
                for d, s in zip(dst, pair):
                    d.copy_(s)
        return out


def _check_state_tensor(p, key, t):
    if not torch.is_tensor(t) or t.dtype != _STATE_DTYPES[key] or t.device != p.device:
        raise TypeError(f"state['{key}'] must be a {_STATE_DTYPES[key]} tensor on {p.device}")


def _coded_row(rec, p, state):
    for k in _CODE_KEYS:
        _check_state_tensor(p, k, state.get(k))
    block = state["m_q"].shape[-1] if state["m_q"].dim() else 0
    nb = _host.num_blocks(p.numel(), block) if block in BLOCK_SIZES else -1
    for k in _CODE_KEYS:
        t = state[k]
        if t.numel() != (nb * block if k.endswith("_q") else nb) or not t.is_contiguous():
            raise ValueError(f"state['{k}'] must be contiguous, with a block size of {BLOCK_SIZES}")
        rec[k] = t.data_ptr()
    rec["kind"], rec["q_block"], rec["n"] = _lib.SMO_ADAMW_8BIT, block, p.numel()


def _launch_codes(name, rows):
    """smo_adamw_decode / smo_adamw_encode over [(p, state, exp_avg, exp_avg_sq)], one call a device."""
    per_dev = {}
    for row in rows:
        if row[0].device.type != "cuda":
            raise RuntimeError(f"8-bit moments (B200 build) are kept on CUDA devices only; got {row[0].device}")
        per_dev.setdefault(row[0].device, []).append(row)
    for dev, rows in per_dev.items():
        table = np.zeros(len(rows), dtype=_lib.ADAMW_DTYPE)
        for rec, (p, state, m, v) in zip(table, rows):
            _coded_row(rec, p, state)
            rec["exp_avg"], rec["exp_avg_sq"] = m.data_ptr(), v.data_ptr()
        with torch.cuda.device(dev):
            _lib.check(getattr(_lib.load(), name)(table.ctypes.data, len(table), _stream(dev)), name)


def _decode(items, out=None):
    """fp32 moments of [(p, state)] with codes."""
    if out is None:
        out = [tuple(torch.empty(p.shape, dtype=torch.float32, device=p.device) for _ in range(2)) for p, _ in items]
    _launch_codes("smo_adamw_decode", [(p, st, m, v) for (p, st), (m, v) in zip(items, out)])
    return out


def _encode(p, state, block):
    """Codes and scales of a state's exp_avg and exp_avg_sq."""
    nb = _host.num_blocks(p.numel(), block)
    got = {}
    for q, s, dtype in (("m_q", "m_s", torch.int8), ("v_q", "v_s", torch.uint8)):
        got[q] = torch.zeros((nb, block), dtype=dtype, device=p.device)
        got[s] = torch.zeros((nb, 1), dtype=torch.float32, device=p.device)
    m, v = state["exp_avg"].contiguous(), state["exp_avg_sq"].contiguous()
    _launch_codes("smo_adamw_encode", [(p, got, m, v)])
    return got

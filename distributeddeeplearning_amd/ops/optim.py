"""Fused optimizers (K10 SGD+momentum, K11 LARS, AdamW) and gradient clipping.

The reference updates 161 ResNet-50 tensors with framework foreach kernels;
here the whole model updates in ONE multi-tensor HIP kernel launch: a chunk
table (pointers + sizes, built once — gradient pointers are stable views
into the persistent flat buckets) drives a single grid over every parameter.
fp32 master weights + momentum state under bf16/fp16 model parameters; the
1/loss_scale unscale folds into the same pass (K13).

Math matches torch.optim.SGD (weight_decay as L2, dampening=0) so the CPU
path is bit-comparable with the stock optimizer in tier-0 tests; LARS
implements You et al. 2017 (layer-wise trust ratio, excluded for BN params
and biases) as required by the batch-8k config (BASELINE.json:9).
"""
from __future__ import annotations

import itertools

import torch
from torch.optim.optimizer import (_global_optimizer_post_hooks,
                                   _global_optimizer_pre_hooks)

from ._ext import load_kernels_ext

CHUNK = 1 << 16  # elements per kernel block


class FusedSGD(torch.optim.Optimizer):
    """SGD + momentum with fp32 master weights, fused on GPU.

    ``lars=True`` turns on layer-wise adaptive rate scaling for tensors with
    ``ndim > 1`` (conv/linear weights); BN parameters and biases always take
    the plain momentum update (standard LARS exclusion list).
    """

    def __init__(self, params, lr, momentum=0.9, weight_decay=0.0,
                 nesterov=False, lars=False, lars_eta=0.001, lars_eps=1e-9,
                 grad_scale=1.0):
        defaults = dict(lr=lr, momentum=momentum, weight_decay=weight_decay,
                        nesterov=nesterov, lars=lars, lars_eta=lars_eta,
                        lars_eps=lars_eps)
        super().__init__(params, defaults)
        self.grad_scale = grad_scale  # multiply grads by 1/scale during update
        self._tables = {}  # per-param-group cached GPU chunk tables

    # ---- state ------------------------------------------------------------

    def _init_state(self, p):
        st = self.state[p]
        if "master" not in st:
            st["master"] = p.detach().to(torch.float32).clone()
            st["momentum_buffer"] = torch.zeros_like(st["master"])
        return st

    def refresh_master(self):
        """Re-copy params into masters (after load_state_dict of the model
        or broadcast_parameters)."""
        for group in self.param_groups:
            for p in group["params"]:
                st = self._init_state(p)
                st["master"].copy_(p.detach().to(torch.float32))

    # ---- GPU fused path ----------------------------------------------------

    def _build_table(self, group):
        """Chunk table: one row per block = [param_ptr, grad_ptr, master_ptr,
        mom_ptr, numel, use_lars, tensor_idx]."""
        ext = load_kernels_ext()
        rows = []
        norms_len = 0
        tensors = []
        for p in group["params"]:
            if p.grad is None:
                continue
            st = self._init_state(p)
            tensors.append((p, st))
        for ti, (p, st) in enumerate(tensors):
            n = p.numel()
            use_lars = 1 if (group["lars"] and p.dim() > 1) else 0
            esz = p.element_size()
            for off in range(0, n, CHUNK):
                cnt = min(CHUNK, n - off)
                rows.append([
                    p.data_ptr() + off * esz,
                    p.grad.data_ptr() + off * esz,
                    st["master"].data_ptr() + off * 4,
                    st["momentum_buffer"].data_ptr() + off * 4,
                    cnt, use_lars, ti,
                ])
        table = torch.tensor(rows, dtype=torch.int64, device=tensors[0][0].device)
        return table, len(tensors)

    def _sig(self, group):
        return tuple(
            (p.data_ptr(), p.grad.data_ptr() if p.grad is not None else 0)
            for p in group["params"]
        )

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            if params[0].is_cuda:
                self._step_gpu(gi, group)
            else:
                self._step_cpu(group)
        return loss

    def _step_gpu(self, gi, group):
        ext = load_kernels_ext()
        sig = self._sig(group)
        cached = self._tables.get(gi)
        if cached is None or cached[0] != sig:
            table, ntensors = self._build_table(group)
            norms = torch.zeros(2, ntensors, dtype=torch.float32,
                                device=table.device)
            cached = (sig, table, norms)
            self._tables[gi] = cached
        _, table, norms = cached
        dt = group["params"][0].dtype
        if group["lars"]:
            norms.zero_()
            ext.lars_norms(table, norms, _dtype_code(dt),
                           float(group["weight_decay"]),
                           float(1.0 / self.grad_scale))
        ext.fused_sgd(
            table, norms if group["lars"] else None,
            _dtype_code(dt),
            float(group["lr"]), float(group["momentum"]),
            float(group["weight_decay"]), bool(group["nesterov"]),
            float(group["lars_eta"]), float(group["lars_eps"]),
            float(1.0 / self.grad_scale),
        )

    def _step_cpu(self, group):
        inv_scale = 1.0 / self.grad_scale
        for p in group["params"]:
            if p.grad is None:
                continue
            st = self._init_state(p)
            master, buf = st["master"], st["momentum_buffer"]
            g = p.grad.detach().to(torch.float32)
            if inv_scale != 1.0:
                g = g * inv_scale
            if group["weight_decay"]:
                g = g.add(master, alpha=group["weight_decay"])
            if group["lars"] and p.dim() > 1:
                wn = master.norm()
                gn = g.norm()
                ratio = torch.where(
                    (wn > 0) & (gn > 0),
                    group["lars_eta"] * wn / (gn + group["lars_eps"]),
                    torch.ones_like(wn),
                )
                g = g * ratio
            if group["momentum"]:
                buf.mul_(group["momentum"]).add_(g)
                g = g.add(buf, alpha=group["momentum"]) if group["nesterov"] else buf
            master.add_(g, alpha=-group["lr"])
            p.data.copy_(master.to(p.dtype))

    def state_dict(self):
        sd = super().state_dict()
        return sd

    def load_state_dict(self, sd):
        """Exact-dtype state restore.

        torch's default ``Optimizer.load_state_dict`` casts floating state
        tensors to the PARAM dtype — under bf16/fp16 params that would
        truncate the fp32 masters and momentum (and break the fused kernel,
        which reads them as 4-byte words).  Restore manually, moving device
        but never changing dtype."""
        _restore_exact(self, sd)
        self._tables = {}

    def invalidate_table(self):
        self._tables = {}


def _restore_exact(opt, sd):
    groups = opt.param_groups
    saved_groups = sd["param_groups"]
    if len(groups) != len(saved_groups):
        raise ValueError("loaded state dict has a different number of "
                         "parameter groups")
    id_map = {}
    for g, sg in zip(groups, saved_groups):
        if len(g["params"]) != len(sg["params"]):
            raise ValueError("parameter group size mismatch in "
                             "load_state_dict")
        for p, pid in zip(g["params"], sg["params"]):
            id_map[pid] = p
        for k, v in sg.items():
            if k != "params":
                g[k] = v
    opt.state.clear()
    for pid, st in sd["state"].items():
        p = id_map.get(pid, pid)
        dev = p.device if torch.is_tensor(p) else None
        opt.state[p] = {
            k: (v.to(device=dev) if torch.is_tensor(v) and dev is not None
                else v)
            for k, v in st.items()
        }


def _dtype_code(dt: torch.dtype) -> int:
    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt]


# --------------------------------------------------------------------------
# AdamW
# --------------------------------------------------------------------------

MOMENT_BLOCK = 256  # elements that share one scale of an 8-bit moment
_E4M3_MAX = 448.0


def _flat(t: torch.Tensor) -> torch.Tensor:
    """The elements of a dense tensor in the order of its storage."""
    return torch.as_strided(t.detach(), (t.numel(),), (1,),
                            t.storage_offset())


def _is_dense(t: torch.Tensor) -> bool:
    need = 1
    for stride, size in sorted((t.stride(d), t.size(d))
                               for d in range(t.dim()) if t.size(d) > 1):
        if stride != need:
            return False
        need *= size
    return True


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.shape == b.shape and all(
        a.size(d) < 2 or a.stride(d) == b.stride(d) for d in range(a.dim()))


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Of two tensors whose address ranges overlap."""
    if _is_dense(a) and _is_dense(b):
        return True
    if a.element_size() != b.element_size():
        return True  # as far as can be told
    places = []
    for t in (a, b):
        at = torch.tensor(t.data_ptr())
        for size, stride in zip(t.shape, t.stride()):
            at = at[..., None] + torch.arange(size) * (
                stride * t.element_size())
        places.append(at.flatten())
    return bool(torch.isin(*places).any())


def _bytes(t: torch.Tensor) -> int:
    """From a tensor's first element to its last one's end."""
    if t.is_contiguous():
        return t.numel() * t.element_size()
    return t.element_size() * (1 + sum(
        (size - 1) * stride for size, stride in zip(t.shape, t.stride())))


def _shared_pair(tensors):
    """Places of two tensors that share memory, or None."""
    spans = [(t.get_device(), t.data_ptr(), _bytes(t), i)
             for i, t in enumerate(tensors) if t.numel()]
    spans.sort()
    for k, (device, at, size, i) in enumerate(spans):
        for other, start, _, j in itertools.islice(spans, k + 1, None):
            if other != device or start >= at + size:
                break
            if _share_memory(tensors[i], tensors[j]):
                return min(i, j), max(i, j)
    return None


def _mix32(x: torch.Tensor) -> torch.Tensor:
    """The kernel's hash of 32 bits (held in int64)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x5DB3D743) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _blocks(x: torch.Tensor) -> torch.Tensor:
    pad = -x.numel() % MOMENT_BLOCK
    return torch.nn.functional.pad(x, (0, pad)).view(-1, MOMENT_BLOCK)


def quantize_moment(x: torch.Tensor, r16: torch.Tensor, least: bool = False):
    """8-bit codes (uint8 bits of e4m3) and block scales of a flat float32
    tensor.  A magnitude between two codes takes the upper one where the part
    above the lower, in 2^-16 of their distance, plus ``r16`` (int64 in
    [0, 2^16)) reaches 2^16.  Values that are not finite become NaN codes and
    do not enter their block's scale; a block below 2^-100 becomes zeros.
    ``least``: magnitudes above zero take at least the smallest code, 2^-9
    (of sqrt(v), whose zero would leave a step without its denominator)."""
    n = x.numel()
    finite = torch.isfinite(x)
    top = _blocks(torch.where(finite, x.abs(), 0.0)).amax(1)
    tiny = top < 2.0 ** -100
    scale = torch.where(tiny, 0.0, top * (1.0 / _E4M3_MAX))
    inv = torch.where(tiny, 0.0, top.reciprocal() * _E4M3_MAX)
    inv = inv.repeat_interleave(MOMENT_BLOCK)[:n]
    y = torch.where(finite, x.abs() * inv, 0.0).clamp(max=_E4M3_MAX)
    bits = (y.view(torch.int32).long() + (r16 << 4)) & ~0xFFFFF
    normal = bits.int().view(torch.float32)
    small = torch.floor(y * 512.0 + r16.float() * 2.0 ** -16) / 512.0
    q = torch.where(y < 2.0 ** -6, small, normal)
    if least:
        q = torch.where(y > 0, q.clamp(min=2.0 ** -9), q)
    q = torch.where(finite, torch.copysign(q, x), float("nan"))
    return q.to(torch.float8_e4m3fn).view(torch.uint8), scale


def dequantize_moment(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The float32 values of flat 8-bit codes."""
    value = code.view(torch.float8_e4m3fn).float()
    return value * scale.repeat_interleave(MOMENT_BLOCK)[:code.numel()]


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay), one fused pass over all tensors on GPU.

    The mathematics is that of ``torch.optim.AdamW``::

        w <- w - lr * weight_decay * w
        m <- beta1 m + (1 - beta1) g,   v <- beta2 v + (1 - beta2) g^2
        w <- w - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    Parameters in bfloat16 or float16 have a float32 master that is updated
    and then rounded; float32 parameters are their own master.

    ``state_bits=8`` (also an option of a parameter group) holds ``m`` and
    ``sqrt(v)`` as 8-bit e4m3 codes with one float32 scale for 256
    consecutive elements: 2 bytes a parameter for both moments instead of 8.
    Codes are rounded up or down by chance, so that they are right on
    average; the chance is a hash of ``seed``, the step, the tensor and the
    element, so that a run can be repeated bit for bit.  ``sqrt(v)`` below
    1 / 229376 of the largest of its 256 is held as that: such an element's
    steps are shorter than with float32 moments.

    ``max_grad_norm`` clips the global norm of all gradients of the optimizer
    (as ``clip_grad_norm_`` before the step would, without writing the
    gradients); ``grad_norm`` then holds the norm of the last step.
    ``grad_scale`` is the loss scale that the gradients still carry.

    State tensors are updated in place; to replace them, load a state dict.
    Step counts are held on the device, so a step captured into a graph
    counts on at each replay, with the learning rate that it was captured
    with.  Each parameter has to be dense in memory (channels_last is).
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=1e-2, state_bits=32, max_grad_norm=None,
                 grad_scale=1.0, seed=0):
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps,
                        weight_decay=weight_decay, state_bits=state_bits,
                        seed=seed)
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise ValueError(f"max_grad_norm must be positive: {max_grad_norm}")
        self._plans = None
        super().__init__(params, defaults)
        self.max_grad_norm = max_grad_norm  # None (later also 0): no clipping
        self.grad_scale = grad_scale  # multiply grads by 1/scale in the update
        self.grad_norm = None

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
        except (ValueError, TypeError):
            self.param_groups.pop()
            raise
        self._plans = None

    @staticmethod
    def _check_group(group):
        if not group["lr"] >= 0:
            raise ValueError(f"invalid learning rate: {group['lr']}")
        if len(group["betas"]) != 2 or not all(0 <= b < 1
                                               for b in group["betas"]):
            raise ValueError(f"betas lie in [0, 1): {group['betas']}")
        if not group["eps"] >= 0:
            raise ValueError(f"invalid eps: {group['eps']}")
        if not group["weight_decay"] >= 0:
            raise ValueError(f"invalid weight_decay: {group['weight_decay']}")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32: {group['state_bits']}")
        ids = [id(p) for p in group["params"]]
        if len(set(ids)) != len(ids):
            raise ValueError("a parameter appears twice in its group")
        for p in group["params"]:
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise TypeError(f"parameters are float32, bfloat16 or "
                                f"float16, not {p.dtype}")
            if not _is_dense(p):
                raise ValueError("a parameter is not dense in memory: the "
                                 "update runs over its storage")
            if p.is_neg():
                raise ValueError("a parameter is a lazy negation: the update "
                                 "runs over its storage")

    # ---- state ------------------------------------------------------------

    def _init_state(self, p, bits):
        st = self.state[p]
        if "step" in st:
            return st
        st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
        if p.dtype != torch.float32:
            st["master"] = p.detach().to(torch.float32)
        kind = torch.uint8 if bits == 8 else torch.float32
        for name in ("exp_avg", "exp_avg_sq"):
            st[name] = torch.zeros_like(p, dtype=kind, requires_grad=False)
            if bits == 8:
                st[name + "_scale"] = torch.zeros(
                    -(-p.numel() // MOMENT_BLOCK), dtype=torch.float32,
                    device=p.device)
        return st

    def moments(self, p):
        """(exp_avg, exp_avg_sq) of a parameter as float32 tensors; copies
        where they are held in 8 bits."""
        st = self.state[p]
        if "step" not in st:
            raise KeyError("the parameter has no state yet")
        if "exp_avg_scale" not in st:
            return st["exp_avg"], st["exp_avg_sq"]
        out = []
        for name in ("exp_avg", "exp_avg_sq"):
            value = torch.empty_like(p, dtype=torch.float32,
                                     requires_grad=False)
            _flat(value).copy_(dequantize_moment(_flat(st[name]),
                                                 st[name + "_scale"]))
            out.append(value)
        return out[0], out[1].square_()

    def refresh_master(self):
        """Re-copy params into masters (after load_state_dict of the model
        or broadcast_parameters)."""
        for group in self.param_groups:
            for p in group["params"]:
                if "master" in self.state.get(p, {}):
                    self.state[p]["master"].copy_(p.detach())

    def load_state_dict(self, sd):
        """Exact-dtype restore, as FusedSGD's; the state tensors of ``sd``
        are taken over without a copy where they are on the right device.
        The state of a ``torch.optim.AdamW`` is understood too.  A state that
        is refused leaves the optimizer as it was."""
        saved = sd["param_groups"]
        if len(saved) != len(self.param_groups):
            raise ValueError("loaded state dict has a different number of "
                             "parameter groups")
        options, owners = [], {}
        for group, new in zip(self.param_groups, saved):
            for option in ("amsgrad", "maximize"):
                if new.get(option):
                    raise ValueError(f"{option} is not supported")
            if len(group["params"]) != len(new["params"]):
                raise ValueError("parameter group size mismatch in "
                                 "load_state_dict")
            ids = new["params"]
            new = {**group, **new, "params": group["params"]}
            new["betas"] = tuple(new["betas"])
            self._check_group(new)
            options.append(new)
            for p, pid in zip(group["params"], ids):
                owners[pid] = p, new["state_bits"]
        state = {}
        for pid, st in sd["state"].items():
            if pid in owners:
                p, bits = owners[pid]
                state[p] = self._adopted(p, st, bits)
            else:
                state[pid] = dict(st)
        self._part(state)
        for group, new in zip(self.param_groups, options):
            group.update(new)
        self.state.clear()
        self.state.update(state)
        self._plans = None

    @staticmethod
    def _part(state):
        """Copies state tensors that share memory with others or with a
        parameter: each is updated by itself, at the same time."""
        owners = [(st, k) for p, st in state.items() if torch.is_tensor(p)
                  for k, v in st.items() if torch.is_tensor(v)]
        params = [p.detach() for p in state if torch.is_tensor(p)]
        while True:
            pair = _shared_pair(params + [st[k] for st, k in owners])
            if pair is None or pair[1] < len(params):
                return
            st, k = owners[pair[1] - len(params)]
            st[k] = st[k].clone()

    @staticmethod
    def _adopted(p, st, bits):
        """A loaded state entry as the optimizer holds it."""
        st = {k: v.to(device=p.device) if torch.is_tensor(v) else v
              for k, v in st.items()}
        if not st:
            return st
        names = ["exp_avg", "exp_avg_sq"]
        scales = [name + "_scale" for name in names]
        if ("exp_avg_scale" in st) != (bits == 8):
            raise ValueError("the loaded moments and the group's state_bits "
                             "do not agree")
        for name in names + (scales if bits == 8 else []) + ["step"]:
            if name not in st:
                raise ValueError(f"the loaded state has no {name}")
        if bits == 8:
            blocks = -(-p.numel() // MOMENT_BLOCK)
            for name, scale in zip(names, scales):
                if st[name].dtype != torch.uint8:
                    raise ValueError(f"{name} holds uint8 codes, not "
                                     f"{st[name].dtype}")
                if st[scale].shape != (blocks,):
                    raise ValueError(f"{scale} holds {blocks} scales")
                st[scale] = st[scale].to(torch.float32).contiguous()
        elif not all(st[name].is_floating_point() for name in names):
            raise ValueError("moments of 32 bits are floating point")
        if p.dtype == torch.float32:
            st.pop("master", None)
        elif "master" not in st:
            st["master"] = p.detach().to(torch.float32)
        for name in ["master"] + names:
            t = st.get(name)
            if t is None or _same_layout(t, p):
                continue
            if t.shape != p.shape:
                raise ValueError(f"{name} has another shape than its "
                                 "parameter")
            if bits == 8 and name != "master":
                raise ValueError("8-bit moments belong to the memory layout "
                                 "that they were saved in")
            st[name] = torch.empty_like(
                p, dtype=t.dtype, requires_grad=False).copy_(t)
        # torch holds the moments in the parameter's dtype
        for name in ["master"] + (names if bits == 32 else []):
            if name in st:
                st[name] = st[name].to(torch.float32)
        if not torch.is_tensor(st["step"]):
            st["step"] = torch.tensor(float(st["step"]))
        if st["step"].numel() != 1:
            raise ValueError("step holds one number")
        st["step"] = st["step"].to(p.device, torch.float32)
        return st

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans = None

    def __getstate__(self):
        state = super().__getstate__()
        state.update(max_grad_norm=self.max_grad_norm,
                     grad_scale=self.grad_scale, grad_norm=None, _plans=None)
        return state

    def invalidate_table(self):
        """Looks the parameters up anew at the next step, after some were
        replaced in ``param_groups``.  Gradients always are."""
        self._plans = None

    # ---- step -------------------------------------------------------------

    def step(self, closure=None):
        # The base class would wrap this for hooks and profiles, 6 us of the
        # host a step, where the kernels of a small model take as long.
        if (closure is not None or _global_optimizer_pre_hooks
                or _global_optimizer_post_hooks
                or self._optimizer_step_pre_hooks
                or self._optimizer_step_post_hooks
                or torch.autograd._profiler_enabled()):
            return self._hooked_step(closure)
        self._update()

    step.hooked = True

    def _closure_step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._update()
        return loss

    _hooked_step = torch.optim.Optimizer.profile_hook_step(_closure_step)

    def _bound(self):
        bound = self.max_grad_norm or 0.0
        if not bound >= 0:
            raise ValueError(f"max_grad_norm must be positive: {bound}")
        return bound

    def _update(self):
        if self._plans is not None or any(
                p.is_cuda for g in self.param_groups for p in g["params"]):
            self._step_gpu()
        else:
            self._step_cpu()

    def _check_overlap(self):
        """Tensors of one launch are updated at the same time."""
        if _shared_pair([p for g in self.param_groups for p in g["params"]
                         if p.grad is not None or p in self.state]):
            raise ValueError("two parameters with gradients share memory")

    def _build_plans(self):
        ext = load_kernels_ext()
        self._check_overlap()
        plans = []
        index = 0
        for group in self.param_groups:
            parts = {}
            for p in group["params"]:
                if not p.is_cuda:
                    raise ValueError("parameters on the CPU and on a GPU in "
                                     "one optimizer")
                parts.setdefault((p.device, p.dtype), []).append((index, p))
                index += 1
            for members in parts.values():
                states = [self.state.get(p, {}) for _, p in members]
                columns = [[st.get(k) for st in states]
                           for k in ("master", "exp_avg", "exp_avg_sq",
                                     "exp_avg_scale", "exp_avg_sq_scale",
                                     "step")]
                plan = ext.AdamWPlan([p for _, p in members], *columns,
                                     [i for i, _ in members],
                                     group["state_bits"])
                plans.append((plan, group, [p for _, p in members]))
        self._plans = plans

    def _step_gpu(self):
        if self._plans is None:
            self._build_plans()
        missing = []  # parameters with their first gradient
        for plan, group, members in self._plans:
            missing += [(i, members, group["state_bits"])
                        for i in plan.collect()]
        if missing:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("take a step before capturing one: a "
                                   "replay would begin with new states")
            with torch.no_grad():
                for i, members, bits in missing:
                    self._init_state(members[i], bits)
            self._build_plans()
            for plan, _, _ in self._plans:
                plan.collect()
        if any(plan.moved() for plan, _, _ in self._plans):
            self._check_overlap()
            for plan, _, _ in self._plans:
                plan.settle()
        norm = load_kernels_ext().adamw_step(
            [plan for plan, _, _ in self._plans],
            [(g["lr"], *g["betas"], g["eps"], g["weight_decay"],
              int(g["seed"]) & 0xFFFFFFFF) for _, g, _ in self._plans],
            1.0 / self.grad_scale, self._bound())
        if norm is not None:
            self.grad_norm = norm

    @torch.no_grad()
    def _step_cpu(self):
        self._check_overlap()
        mul = 1.0 / self.grad_scale
        if self._bound():
            grads = [p.grad for g in self.param_groups for p in g["params"]
                     if p.grad is not None]
            self.grad_norm, coef = _norm_cpu(grads, mul, self.max_grad_norm)
            mul = mul * float(coef)
        index = -1
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            lr, bits = group["lr"], group["state_bits"]
            for p in group["params"]:
                index += 1
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("sparse gradients are not supported")
                st = self._init_state(p, bits)
                grad = p.grad.detach()
                if not _same_layout(grad, p):
                    grad = torch.empty_like(p).copy_(grad)
                g = _flat(grad).to(torch.float32) * mul
                w = _flat(st.get("master", p))
                m, v = _flat(st["exp_avg"]), _flat(st["exp_avg_sq"])
                st["step"] += 1
                t = float(st["step"])
                if bits == 8:
                    codes = m, v
                    m = dequantize_moment(m, st["exp_avg_scale"])
                    v = dequantize_moment(v, st["exp_avg_sq_scale"])
                    v = v * v
                m_new = beta1 * m + (1.0 - beta1) * g
                v_new = beta2 * v + (1.0 - beta2) * (g * g)
                root = v_new.double().sqrt().float()  # correctly rounded
                denom = root * (1.0 - beta2 ** t) ** -0.5 + group["eps"]
                w.mul_(1.0 - lr * group["weight_decay"])
                w.sub_((lr / (1.0 - beta1 ** t) * m_new) / denom)
                if bits == 8:
                    r = self._random_bits(group["seed"], index, int(t),
                                          m.numel())
                    for name, code, new, bits16 in (
                            ("exp_avg", codes[0], m_new, r & 0xFFFF),
                            ("exp_avg_sq", codes[1], root, r >> 16)):
                        q, scale = quantize_moment(
                            new, bits16, least=name == "exp_avg_sq")
                        code.copy_(q)
                        st[name + "_scale"].copy_(scale)
                else:
                    m.copy_(m_new)
                    v.copy_(v_new)
                if "master" in st:
                    _flat(p).copy_(w)

    @staticmethod
    def _random_bits(seed, index, step, n):
        stream = _mix32(torch.tensor(
            (int(seed) + 0x9E3779B9 * (index + 1)) & 0xFFFFFFFF))
        key = _mix32((stream + step) & 0xFFFFFFFF)
        return _mix32((torch.arange(n) & 0xFFFFFFFF) ^ key)


# --------------------------------------------------------------------------
# Clipping of the global gradient norm
# --------------------------------------------------------------------------

def _norm_cpu(grads, mul, max_norm):
    total = sum((g.detach().double().square().sum() for g in grads),
                torch.zeros((), dtype=torch.float64))
    norm = (total.sqrt() * mul).float()
    return norm, (max_norm / (norm + 1e-6)).clamp(max=1.0)


def clip_grad_norm_(params, max_norm, grad_scale=1.0) -> torch.Tensor:
    """Scale all gradients in place so that their global 2-norm is at most
    ``max_norm``; returns the norm before (0-dim float32, no host sync).

    ``grad_scale`` is the loss scale that the gradients carry: the norm, and
    the bound, are of the gradients divided by it, and they keep carrying it.
    As in ``torch.nn.utils.clip_grad_norm_``, a norm that is not finite is
    not caught: it makes the gradients zero or NaN.

    Under data parallelism call it after ``DistributedOptimizer.synchronize``;
    every rank then computes the same norm.  Gradients are not touched where
    the norm is within bounds.
    """
    params = [params] if torch.is_tensor(params) else list(params)
    if not max_norm > 0:
        raise ValueError(f"max_norm must be positive: {max_norm}")
    if not grad_scale > 0:
        raise ValueError(f"grad_scale must be positive: {grad_scale}")
    first = next((p.grad for p in params if p.grad is not None), None)
    if first is None:
        device = params[0].device if params else None
        return torch.zeros((), dtype=torch.float32, device=device)
    if first.is_cuda:
        return load_kernels_ext().clip_grads(params, 1.0 / grad_scale,
                                             float(max_norm))
    grads = [p.grad for p in params if p.grad is not None]
    if (len({id(g) for g in grads}) != len(grads)
            or _shared_pair([g for g in grads if not g.is_sparse])):
        raise RuntimeError("a gradient appears twice, or two share memory")
    for g in grads:
        if g.device != first.device:
            raise RuntimeError("all gradients are on one device")
        if not g.is_floating_point():
            raise RuntimeError(f"expected gradients of real numbers, got "
                               f"{g.dtype}")
    norm, coef = _norm_cpu(grads, 1.0 / grad_scale, max_norm)
    if not float(coef) == 1.0:
        with torch.no_grad():
            for g in grads:
                wide = torch.promote_types(g.dtype, torch.float32)
                g.copy_(g.to(wide) * coef)
    return norm

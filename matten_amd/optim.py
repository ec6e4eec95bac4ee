"""AdamW over all parameter tensors of a model at once (tfc_adamw_step), with moments in 32 or in 8 bits and the gradients
optionally limited to a largest global norm, in the same launches.

Takes the place of torch.optim.AdamW in the `class_path` of a config (the reference's trainer steps whatever optimizer its yaml
names, eigenn/model/model.py:410-426), and of torch.optim.Adam, which the reference's own configs name, where `weight_decay: 0` is
written out: Adam's default is no decay and its decay is part of the gradient, here it is 0.01 and apart from it.  A
`torch.optim.Optimizer` with param groups, schedulers, closures and `state_dict`.  Everything a step needs lives on the device - the step counts too - so that a step can be part of a captured
graph (matten_amd.graphs.GraphedStep)."""
from __future__ import annotations

import ctypes as C
import math
from operator import is_
from typing import Iterable, Optional

import torch

from . import _lib, ops

__all__ = ["AdamW"]

BLOCK = 256  # elements that share a scale in the 8-bit moments
_STATE = {  # state entry -> dtype, by the width of the moments ("step" besides)
    32: {"exp_avg": torch.float32, "exp_avg_sq": torch.float32},
    8: {"exp_avg": torch.float8_e4m3fn, "exp_avg_scale": torch.float8_e8m0fnu, "exp_avg_sq_root": torch.float8_e4m3fn,
        "exp_avg_sq_root_scale": torch.float8_e8m0fnu},
}


# (unbound: a step asks for these of every tensor, and host time is what a step of a small model costs)
_address, _numel, _device, _packed = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device, torch.Tensor.is_contiguous
_type, _layout = torch.Tensor.dtype.__get__, torch.Tensor.layout.__get__


class _Table:
    """The descriptors of the tensors one call steps: everything but the gradients' addresses is set once."""

    def __init__(self, group, params, states, indexes, bits: int):
        self.group, self.params, self.states = group, params, states
        self.device, self.dtype = params[0].device, params[0].dtype
        self.entries = [t for st in states for t in st.values()]  # (alive as long as their addresses are used)
        self.at = list(map(_address, (*params, *self.entries)))
        self.sizes = [p.numel() for p in params]
        self.rows = (_lib.AdamwTensor * len(params))()
        self.each = list(self.rows)
        names = list(_STATE[bits])
        for row, p, st, i in zip(self.each, params, states, indexes):
            row.p, row.n, row.index, row.step = p.data_ptr(), p.numel(), i, st["step"].data_ptr()
            if bits == 32:
                row.m, row.v = (st[k].data_ptr() for k in names)
            else:
                row.m, row.m_scale, row.v, row.v_scale = (st[k].data_ptr() for k in names)

    def holds(self, state) -> bool:
        """Whether parameters and state still lie where the descriptors say, every parameter with a gradient."""
        entries = []
        for p, st in zip(self.params, self.states):
            if p.grad is None or state.get(p) is not st:
                return False
            entries += st.values()
        try:
            return (list(map(_address, (*self.params, *entries))) == self.at and list(map(_numel, self.params)) == self.sizes
                    and all(map(_packed, self.params)))
        except TypeError:  # (not a tensor: for _check_state to name)
            return False


class AdamW(torch.optim.Optimizer):
    """With g the gradient and t the tensor's step count:

        m = beta1 m + (1 - beta1) g,    v = beta2 v + (1 - beta2) g^2,
        p = (1 - lr weight_decay) p - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    in fp32 for fp32, bf16 and fp16 parameters (a 16-bit parameter is rounded to the nearest once, at the end).

    * `state_bits=32`: state entries `exp_avg`, `exp_avg_sq` (fp32).  `state_bits=8`: `exp_avg` and `exp_avg_sq_root` (the root
      of the second moment) as float8_e4m3fn, flat and padded to whole blocks of 256, each block with a power-of-two scale
      (`*_scale`, float8_e8m0fnu): a quarter of the state.  They are rounded up or down at random so that they are kept on
      average; the random bits follow from `seed`, the step and the element, so runs repeat bit for bit.
    * `max_grad_norm`: all gradients are scaled by min(1, max_grad_norm / (norm + 1e-6)) as they are read (`.grad` itself is
      left alone).  After a step `grad_norm` holds the norm before scaling (a device scalar; None without `max_grad_norm`).
      A norm that is not finite reaches the parameters: check `grad_norm` where that can happen.
    * `lr` is a number or a 0-dim fp32 tensor on the parameters' device, read when the step runs: inside a captured graph a
      number is fixed, a tensor can be written to between replays.

    Parameters and gradients are contiguous and on a ROCm device (gradients that are not contiguous are copied); a sparse gradient
    raises, and so do parameters that share memory (they are stepped at the same time).  `amsgrad` and `maximize` do not exist.  A parameter without a gradient is skipped and its step count stands.  The first step allocates the state and
    therefore must not be inside a graph capture; a captured step drops its gradients (`zero_grad()`, set to None) rather than
    zeroing them, as matten_amd.graphs asks of every captured backward pass."""

    def __init__(self, params: Iterable, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 max_grad_norm: Optional[float] = None, seed: int = 0):
        if state_bits not in _STATE:
            raise ValueError(f"AdamW: state_bits must be 32 or 8, got {state_bits}")
        if max_grad_norm is not None and not 0.0 < float(max_grad_norm) < math.inf:
            raise ValueError(f"AdamW: max_grad_norm must be positive and finite, got {max_grad_norm}")
        self.state_bits = int(state_bits)
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        self.seed = int(seed) & 0xFFFFFFFF
        self.grad_norm: Optional[torch.Tensor] = None
        self._tables = None  # the last step's, and the parameters it left alone
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def add_param_group(self, group):
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            self._check_group(g)
            for p in g["params"]:
                if p.dtype not in ops._dtype_codes:
                    raise TypeError(f"AdamW: parameters must be float32, bfloat16 or float16, got {p.dtype}")
            if len(set(g["params"])) != len(g["params"]):
                raise ValueError("AdamW: a parameter is in its group twice")
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(g):
        lr, (b1, b2) = g["lr"], g["betas"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32:
                raise ValueError("AdamW: an lr tensor must hold one float32")
        elif not 0.0 <= lr < math.inf:
            raise ValueError(f"AdamW: lr must be finite and not negative, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas must lie in [0, 1), got {g['betas']}")
        if g.get("amsgrad") or g.get("maximize"):  # (a loaded state dict's)
            raise ValueError("AdamW: `amsgrad` and `maximize` do not exist here")
        if g.get("decoupled_weight_decay") is False and g["weight_decay"] != 0:
            raise ValueError("AdamW: torch.optim.Adam's weight decay, a part of the gradient, does not exist here")
        if not 0.0 <= g["eps"] < math.inf or not 0.0 <= g["weight_decay"] < math.inf:
            raise ValueError(f"AdamW: eps and weight_decay must be finite and not negative, got {g['eps']}, {g['weight_decay']}")

    # ---- state
    def _length(self, p, name: str) -> int:
        blocks = -(-p.numel() // BLOCK)
        return 1 if name == "step" else p.numel() if self.state_bits == 32 else blocks if name.endswith("scale") else blocks * BLOCK

    def _new_state(self, p) -> dict:
        st = {"step": torch.zeros((), dtype=torch.int32, device=p.device)}
        for k, dt in _STATE[self.state_bits].items():
            if self.state_bits == 32:
                st[k] = torch.zeros_like(p, dtype=dt, memory_format=torch.contiguous_format)
            else:  # (a scale's exponent is 1 where all its values are zero)
                st[k] = torch.full((self._length(p, k),), int(k.endswith("scale")), dtype=torch.uint8, device=p.device).view(dt)
        return st

    def _check_state(self, p):
        """Users may write to `state`: what the kernel is given has the types and sizes it takes for granted."""
        st, want = self.state[p], {"step": torch.int32, **_STATE[self.state_bits]}
        if set(st) != set(want):
            raise ValueError(f"AdamW: state entries {sorted(st)} are not those of moments in {self.state_bits} bits")
        for k, dt in want.items():
            t, n = st[k], self._length(p, k)
            if not isinstance(t, torch.Tensor) or t.dtype != dt or t.device != p.device or t.numel() != n or not t.is_contiguous():
                got = f"{t.dtype}, {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
                raise ValueError(f"AdamW: state entry `{k}` must be a contiguous {dt} tensor of {n} elements on {p.device}; got {got}")

    def load_state_dict(self, state_dict):
        """Takes copies.  The moments must have this optimizer's width and the parameters' sizes; those of torch.optim.AdamW, and of
        torch.optim.Adam without weight decay, fit 32 bits where the parameters are fp32."""
        for g in state_dict["param_groups"]:
            self._check_group(g)
        names = _STATE[self.state_bits]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        new = {}
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i)
            if not saved:
                continue
            if set(saved) != {"step", *names}:
                raise ValueError(f"AdamW: state entries {sorted(saved)} are not those of moments in {self.state_bits} bits")
            st = self._new_state(p)
            for k, v in saved.items():
                if k == "step":
                    st[k].fill_(int(v))
                    continue
                if v.numel() != st[k].numel() or v.dtype != st[k].dtype:
                    raise ValueError(f"AdamW: `{k}` has {v.numel()} x {v.dtype}, expected {st[k].numel()} x {st[k].dtype}")
                wide = torch.uint8 if self.state_bits == 8 else v.dtype
                st[k].view(wide).copy_(v.detach().view(wide).reshape(st[k].shape))
            new[p] = st
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})  # (would cast the moments)
        self.state.update(new)
        self._tables = None

    def __setstate__(self, state):
        super().__setstate__(state)
        self._tables = None

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_grad_norm": self.max_grad_norm, "seed": self.seed,
                "grad_norm": None}

    # ---- step
    def _gather(self):
        """Tables of the parameters that have a gradient, one for each (group, device, dtype)."""
        for g in self.param_groups:
            self._check_group(g)  # (schedulers and users write to groups)
        if self._tables is not None:
            tables, rest, groups = self._tables
            if (len(groups) == len(self.param_groups)
                    and all(g is h and len(g["params"]) == len(ps) and all(map(is_, g["params"], ps)) for (h, ps), g in zip(groups, self.param_groups))
                    and all(t.holds(self.state) for t in tables) and all(p.grad is None for p in rest)):
                return tables
        tables, rest, first = [], [], 0
        for g in self.param_groups:
            sets = {}
            for i, p in enumerate(g["params"]):
                if p.grad is None:
                    rest.append(p)
                else:
                    sets.setdefault((p.device, p.dtype), []).append((p, first + i))
            first += len(g["params"])
            for (device, _), items in sets.items():
                tables.append(self._table(g, device, [p for p, _ in items], [i for _, i in items]))
        end = 0
        for at, n in sorted((p.data_ptr(), p.numel() * p.element_size()) for t in tables for p in t.params if p.numel()):
            if at < end:
                raise ValueError("AdamW: two parameters share memory")
            end = at + n
        self._tables = tables, rest, [(g, list(g["params"])) for g in self.param_groups]
        return tables

    def _table(self, group, device, params, indexes) -> _Table:
        if device.type != "cuda":
            raise RuntimeError(f"matten_amd: parameters must live on a ROCm device (no CPU fallback exists); got {device}")
        for p in params:
            if not p.is_contiguous():
                raise ValueError("AdamW: parameters must be contiguous")
            if not self.state[p]:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW: the first step allocates the state and cannot be captured; run one step before the capture")
                self.state[p].update(self._new_state(p))
            self._check_state(p)
        return _Table(group, params, [self.state[p] for p in params], indexes, self.state_bits)

    @staticmethod
    def _point_at_gradients(tables) -> Optional[list]:
        """Checks the gradients and puts their addresses into the tables.  Returns what has to live as long as these are used, or None
        where a table is out of date: the parameters' type has changed at the same addresses (memory that one type of 16 bits gave back
        and the other was handed; looked for only here, where it shows, since every step would pay for it)."""
        copies = []  # gradients that are not contiguous
        for t in tables:
            dtype, at = t.dtype, t.device.index
            lr = t.group["lr"]
            if isinstance(lr, torch.Tensor) and lr.device != t.device:
                raise RuntimeError(f"AdamW: the lr tensor is on {lr.device}, the parameters on {t.device}")
            grads = [p.grad for p in t.params]
            if set(map(_type, grads)) != {dtype} or set(map(_layout, grads)) != {torch.strided} or set(map(_device, grads)) != {at} \
                    or list(map(_numel, grads)) != t.sizes:
                if any(p.dtype != dtype for p in t.params):
                    return None
                p, g = next((p, g) for p, g, n in zip(t.params, grads, t.sizes)
                            if g.dtype != dtype or g.layout != torch.strided or g.get_device() != at or g.numel() != n)
                raise RuntimeError(f"AdamW: a gradient must be a dense {dtype} tensor of shape {tuple(p.shape)} on {t.device}; got "
                                   f"{g.dtype}, {tuple(g.shape)}, {g.layout} on {g.device}")
            if not all(map(_packed, grads)):
                grads = [g.contiguous() for g in grads]
                copies += grads
            for row, address in zip(t.each, map(_address, grads)):
                row.g = address
        return copies

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        tables = self._gather()
        copies = self._point_at_gradients(tables)
        if copies is None:
            self._tables = None
            tables = self._gather()
            copies = self._point_at_gradients(tables)  # noqa: F841 (kept until the launches are queued)
        L = _lib.lib()
        partials, n_partials = None, 0
        self.grad_norm = None
        if self.max_grad_norm is not None and tables:
            device = tables[0].device
            if any(t.device != device for t in tables):
                raise RuntimeError("AdamW: max_grad_norm needs all parameters on one device")
            counts = [L.tfc_grad_sumsq_partials(t.rows, len(t.rows)) for t in tables]
            n_partials = sum(counts)
            with ops._on(device):
                self.grad_norm = torch.empty((), dtype=torch.float32, device=device) if n_partials else torch.zeros((), device=device)
                partials = torch.empty(max(n_partials, 1), dtype=torch.float64, device=device)
                at = partials.data_ptr()
                for t, n in zip(tables, counts):
                    _lib.check(L.tfc_grad_sumsq(t.rows, len(t.rows), ops._dtype_codes[t.dtype], at, ops._stream()))
                    at += 8 * n
        for t in tables:
            g = t.group
            h = _lib.AdamwHyper(beta1=float(g["betas"][0]), beta2=float(g["betas"][1]), eps=float(g["eps"]), weight_decay=float(g["weight_decay"]),
                                max_norm=self.max_grad_norm if n_partials else 0.0, seed=self.seed)
            if isinstance(g["lr"], torch.Tensor):
                h.lr_device = g["lr"].data_ptr()
            else:
                h.lr = float(g["lr"])
            with ops._on(t.device):
                ws = torch.empty(L.tfc_adamw_workspace_bytes(len(t.rows)), dtype=torch.uint8, device=t.device)
                _lib.check(L.tfc_adamw_step(t.rows, len(t.rows), ops._dtype_codes[t.dtype], self.state_bits, C.byref(h), ops._at(partials),
                                            n_partials, ops._at(self.grad_norm), ws.data_ptr(), ws.numel(), ops._stream()))
            torch.autograd.graph.increment_version(t.params)  # (written behind torch's back: saved tensors and caches see it)
        return loss

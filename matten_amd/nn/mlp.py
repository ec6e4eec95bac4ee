"""Residual perceptron on a field of invariants, for heads that need more than the linear maps of the two target models.  Built
from two fused kernels, forward and backward: the layer norm (ops.layer_norm) and the dense product with bias, activation and
residual in its epilogue (ops.dense).  The reference's counterpart are the scalar layers of eigenn/nn/utils.py, which its two
target models do not use."""
from __future__ import annotations

import math
from typing import Dict, Optional

import torch

from .. import keys as DataKey
from .. import ops
from .._lib import DENSE_ACT
from ..irreps import Irreps
from ..module_irreps import ModuleIrreps
from .e3 import NORMALIZE2MOM, _n2m

__all__ = ["Dense", "LayerNorm", "NodewiseMLP"]


class LayerNorm(torch.nn.Module):
    """ops.layer_norm with its weight (ones) and bias (zeros)."""

    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.eps = float(eps)
        self.weight = torch.nn.Parameter(torch.ones(int(dim)))
        self.bias = torch.nn.Parameter(torch.zeros(int(dim)))

    def forward(self, x):
        return ops.layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}"


class Dense(torch.nn.Module):
    """act'(x W / sqrt(h_in) + bias) [+ residual] with W [h_in, h_out] ~ randn and the activation scaled to unit second moment, as
    in FullyConnectedNet (gelu, which has no such constant there, is taken as it is); bias zeros."""

    def __init__(self, h_in: int, h_out: int, act: str = "identity", bias: bool = True):
        super().__init__()
        if act not in DENSE_ACT:
            raise ValueError(f"matten_amd: unknown activation `{act}` (known: {sorted(DENSE_ACT)})")
        self.act, self.act_cst = act, _n2m(act) if act in NORMALIZE2MOM else 1.0
        self.weight = torch.nn.Parameter(torch.randn(int(h_in), int(h_out)))
        self.bias = torch.nn.Parameter(torch.zeros(int(h_out))) if bias else None

    def forward(self, x, residual: Optional[torch.Tensor] = None):
        alpha = 1.0 / math.sqrt(max(self.weight.shape[0], 1))
        return ops.dense(x, self.weight, self.bias, residual, act=self.act, alpha=alpha, act_cst=self.act_cst)

    def extra_repr(self):
        return f"{tuple(self.weight.shape)}, act={self.act}, bias={self.bias is not None}"


class NodewiseMLP(ModuleIrreps, torch.nn.Module):
    """num_blocks times x <- x + W2 act(W1 norm(x) + b1) + b2 on a field of invariants (irreps all 0e), then, where `irreps_out` is
    another width, a norm and a linear map to it."""

    def __init__(self, irreps_in: Dict[str, Irreps], irreps_out=None, field: str = DataKey.NODE_FEATURES, out_field: Optional[str] = None,
                 hidden: Optional[int] = None, num_blocks: int = 1, activation: str = "silu"):
        super().__init__()
        self.field = field
        self.out_field = field if out_field is None else out_field
        self.init_irreps(irreps_in, {self.out_field: irreps_in.get(field) if irreps_out is None else irreps_out},
                         required_keys_irreps_in=[field])
        for name, irreps in (("input", self.irreps_in[field]), ("output", self.irreps_out[self.out_field])):
            if any(ir.l != 0 or ir.p != 1 for _, ir in irreps) or irreps.dim == 0:
                raise ValueError(f"NodewiseMLP acts on invariants (0e), the {name} irreps are {irreps}")
        d, d_out = self.irreps_in[field].dim, self.irreps_out[self.out_field].dim
        hidden = 4 * d if hidden is None else int(hidden)
        if hidden < 1 or num_blocks < 1:
            raise ValueError(f"NodewiseMLP: hidden and num_blocks must be positive, got {hidden}, {num_blocks}")
        self.blocks = torch.nn.ModuleList(
            torch.nn.ModuleDict({"norm": LayerNorm(d), "up": Dense(d, hidden, activation), "down": Dense(hidden, d)})
            for _ in range(int(num_blocks)))
        self.out = torch.nn.ModuleDict({"norm": LayerNorm(d), "linear": Dense(d, d_out)}) if d_out != d else None

    def forward(self, data: DataKey.Type) -> DataKey.Type:
        x = data[self.field]
        for b in self.blocks:
            x = b["down"](b["up"](b["norm"](x)), x)
        data[self.out_field] = x if self.out is None else self.out["linear"](self.out["norm"](x))
        return data

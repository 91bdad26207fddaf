"""Low-rank adapters of many requests beside the projections of an FFN (no counterpart in the reference).

Every token may belong to another adapter: ``plan = kernels.adapter_plan(ids, n_adapters)`` sorts a batch's tokens once, and
``set_adapter_plan(model, plan)`` hands the plan to every ``AdapterLinear`` below ``model`` (or a call passes it along).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from .. import kernels
from .dense import DenseMLPBlock
from .mlp import _HOOKS, BlockELLLinear, MLPBlock, _plain
from .mx import MXBlockELLWeight, MXMLPBlock


def _features(base):
    """(in_features, out_features) of a projection; a 4-bit one does not hold its inputs' number."""
    out = base.out_features if hasattr(base, "out_features") else base.codes.shape[0] * base.codes.shape[2]
    return getattr(base, "in_features", None), out


class AdapterLinear(nn.Module):
    """``base(x) + scales[id] * (x a[id]^T) b[id]^T`` with each token's adapter, ``base(x)`` where there is no plan.

    ``base`` is a ``BlockELLLinear`` or an ``MXBlockELLWeight`` (its ``in_features`` to be given), frozen or not; ``a``
    [n, rank, in] starts normal with variance 1 / in, ``b`` [n, out, rank] at zero, both in ``dtype`` (rounded to the
    base's type in every call if it is another one); ``scales`` [n] is a buffer, alpha / rank.  ``dropout``: of the adapters'
    input, with the ``dropout_seed`` of a call."""

    def __init__(self, base: nn.Module, n_adapters: int, rank: int, alpha: float | None = None, dropout: float = 0.0,
                 dtype: torch.dtype = torch.bfloat16, in_features: int | None = None, device=None):
        super().__init__()
        fin, fout = _features(base)
        fin = in_features or fin
        if fin is None:
            raise ValueError("a 4-bit base does not hold its in_features: pass them")
        if fin % 8 or fout % 8:
            raise ValueError("features must be multiples of 8")
        self.base, self.n_adapters, self.rank, self.dropout = base, n_adapters, rank, dropout
        self.a = nn.Parameter(torch.randn(n_adapters, rank, fin, device=device).mul_(fin ** -0.5).to(dtype))
        self.b = nn.Parameter(torch.zeros(n_adapters, fout, rank, device=device, dtype=dtype))
        self.register_buffer("scales", torch.full((n_adapters,), (rank if alpha is None else alpha) / rank, device=device))
        self.plan = None

    def forward(self, x: torch.Tensor, plan=None, dropout_seed=None, dropout_stream: int = 0) -> torch.Tensor:
        y = self.base(x)
        plan = self.plan if plan is None else plan
        if plan is None:
            return y
        if self.dropout > 0.0 and dropout_seed is not None:
            x = kernels.dropout(x, self.dropout, dropout_seed, dropout_stream)
        x, a, b = x.to(y.dtype), self.a.to(y.dtype), self.b.to(y.dtype)
        grad = torch.is_grad_enabled() and any(t.requires_grad for t in (y, x, a, b))
        # into the base's result only where nobody else can hold it
        own = not grad and any(_plain(self.base, c) for c in (BlockELLLinear, MXBlockELLWeight))
        return kernels.adapter_add(y, x, a, b, plan, scales=self.scales, inplace=own)


def _takes_over(mlp) -> bool:
    """Whether ``mlp`` is no more than its projections and the activation that its class puts between them."""
    cls = next((c for c in (MLPBlock, MXMLPBlock, DenseMLPBlock) if isinstance(mlp, c)), None)
    own = ("forward", "swiglu_weights", "swiglu_biases")
    return (cls is not None and all(getattr(type(mlp), m, None) is getattr(cls, m, None) and m not in mlp.__dict__ for m in own)
            and not any(mlp.__dict__[h] for h in _HOOKS))


class AdapterMLPBlock(nn.Module):
    """The FFN of an ``MLPBlock`` (SwiGLU or GELU), an ``MXMLPBlock`` or a ``DenseMLPBlock`` (either activation, parameters of
    its dtype) with adapters beside each projection.  The projections run one by one, as an adapter's update comes before
    the activation.  Any other block, one whose forward is replaced and one with hooks are refused: only the projections,
    the activation and the dropout of the result are taken over.

    The result's dropout is the block's own (``MLPBlock``): with ``deterministic`` False, by torch's generator, or by
    ``kernels.dropout`` with a ``dropout_seed``, which the adapters' dropout follows too.  The projections' streams are
    ``dropout_stream`` and those behind it, in their order, the result's comes next: four of a gated block, three else."""

    def __init__(self, mlp: nn.Module, n_adapters: int, rank: int, **kw):
        super().__init__()
        if not _takes_over(mlp):
            raise ValueError("adapters go beside the projections of an MLPBlock, an MXMLPBlock or a DenseMLPBlock without hooks and "
                             f"with that class's forward, not of {type(mlp).__name__}")
        self.activation = getattr(mlp, "activation", "silu") if hasattr(mlp, "w_gate") else "gelu"
        self.dropout = getattr(mlp, "dropout", 0.0)
        self.dtype = mlp.dtype if isinstance(mlp, DenseMLPBlock) else None      # the others' projections round x
        self.names = ("w_gate", "w_up", "w_down") if hasattr(mlp, "w_gate") else ("fc1", "fc2")
        inner, last = getattr(mlp, self.names[0]), getattr(mlp, self.names[-1])
        d_model, d_ff = _features(last)[1], _features(inner)[1]
        for name in self.names:
            fin = d_ff if name == self.names[-1] else d_model
            setattr(self, name, AdapterLinear(getattr(mlp, name), n_adapters, rank, in_features=fin, **kw))

    def forward(self, x: torch.Tensor, plan=None, dropout_seed=None, dropout_stream: int = 0, deterministic: bool = True) -> torch.Tensor:
        lin = [getattr(self, n) for n in self.names]
        if self.dtype is not None:
            x = x.to(self.dtype)
        first = [m(x, plan, dropout_seed, dropout_stream + k) for k, m in enumerate(lin[:-1])]
        h = first[0].float()
        h = F.silu(h) if self.activation == "silu" else F.gelu(h, approximate="tanh")
        if len(first) == 2:
            h = h * first[1].float()
        out = lin[-1](h.to(first[0].dtype), plan, dropout_seed, dropout_stream + len(first))
        if self.dropout > 0.0 and not deterministic:
            if dropout_seed is None:
                out = F.dropout(out, p=self.dropout, training=True)
            else:
                out = kernels.dropout(out, self.dropout, dropout_seed, dropout_stream + len(lin))
        return out


def set_adapter_plan(module: nn.Module, plan) -> None:
    """Hand ``plan`` (or None) to every ``AdapterLinear`` of ``module``, for calls that pass none."""
    for m in module.modules():
        if isinstance(m, AdapterLinear):
            m.plan = plan

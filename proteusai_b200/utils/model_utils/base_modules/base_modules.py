"""``MLP`` feed-forward block with the reference's parameter names
(``utils/model_utils/base_modules/base_modules.py:6-52``): ``in_proj``, ``hidden_proj[i]``, ``out_proj``;
activation after every layer but the last, dropout after every activation; Xavier-uniform on the first
and last layer, Kaiming-uniform on hidden layers, zero biases.  ``fused=True`` (an addition to the reference's constructor) runs every layer as
one kernel with its bias, activation and residual (``fused_ops.linear``), forward and backward, where the tensors allow it.

``GatedMLP`` is the gated form of the block, ``out_proj(act(gate_proj(x)) * up_proj(x))``, its hidden layer one kernel (``fused_ops.gated_linear``).

Both take the residual of the block they stand in as ``forward(x, residual)``: ``block(x) + residual``, added in the last product's epilogue."""
import torch.nn as nn
import torch.nn.functional as F

from proteusai_b200.utils.model_utils.base_modules import fused_ops

_ACTS = {"gelu": F.gelu, "silu": F.silu, "relu": F.relu, "sigmoid": F.sigmoid}


class MLP(nn.Module):
    fused, act_name = False, None

    def __init__(self, d_in=512, d_out=512, d_hidden=1024, hidden_layers=0, dropout=0.1, act="gelu", zeros=False, fused=False):
        super().__init__()
        self.fused = fused
        self.act_name = act if act in _ACTS else None
        self.in_proj = nn.Linear(d_in, d_hidden)
        self.hidden_proj = nn.ModuleList(nn.Linear(d_hidden, d_hidden) for _ in range(hidden_layers))
        self.out_proj = nn.Linear(d_hidden, d_out)
        self.in_dropout = nn.Dropout(dropout)
        self.hidden_dropout = nn.ModuleList(nn.Dropout(dropout) for _ in range(hidden_layers))
        self.act = _ACTS.get(act, lambda x: x)
        nn.init.xavier_uniform_(self.in_proj.weight)
        nn.init.zeros_(self.in_proj.bias)
        for layer in self.hidden_proj:
            nn.init.kaiming_uniform_(layer.weight, nonlinearity="relu")
            nn.init.zeros_(layer.bias)
        if zeros:
            nn.init.zeros_(self.out_proj.weight)
        else:
            nn.init.xavier_uniform_(self.out_proj.weight)
        nn.init.zeros_(self.out_proj.bias)

    def _act(self, x):
        # bf16 inference: the erf GELU as one HBM-bound kernel, in place on the projection's output
        if self.act is F.gelu and x.numel() % 8 == 0 and fused_ops.usable(x):
            return fused_ops.gelu(x, inplace=True)
        return self.act(x)

    def _layer(self, layer, x):
        """``act(layer(x))``"""
        if self.fused and fused_ops.dense_usable(x, layer.weight, layer.bias):
            return fused_ops.linear(x, layer.weight, layer.bias, act=self.act_name)
        return self._act(layer(x))

    def forward(self, x, residual=None):
        x = self.in_dropout(self._layer(self.in_proj, x))
        for layer, drop in zip(self.hidden_proj, self.hidden_dropout):
            x = drop(self._layer(layer, x))
        if self.fused:
            return _project(x, self.out_proj, residual)
        return self.out_proj(x) if residual is None else self.out_proj(x) + residual


def _project(x, layer, residual):
    """``layer(x) + residual``, one kernel where the tensors allow it.  (Under autocast a residual of more bits keeps them: it is added outside.)"""
    if not fused_ops.dense_usable(x, layer.weight, layer.bias):
        y = layer(x)
    elif residual is not None and fused_ops.dense_usable(residual) and residual.dtype == fused_ops.dense_dtype(x):
        return fused_ops.linear(x, layer.weight, layer.bias, residual=residual)
    else:
        y = fused_ops.linear(x, layer.weight, layer.bias)
    return y if residual is None else y + residual


class GatedMLP(nn.Module):

    def __init__(self, d_in=512, d_out=512, d_hidden=1024, dropout=0.1, act="silu", bias=True):
        super().__init__()
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}, not {act!r}")
        self.gate_proj = nn.Linear(d_in, d_hidden, bias=bias)
        self.up_proj = nn.Linear(d_in, d_hidden, bias=bias)
        self.out_proj = nn.Linear(d_hidden, d_out, bias=bias)
        self.dropout = nn.Dropout(dropout)
        self.act_name = act
        for layer in (self.gate_proj, self.up_proj, self.out_proj):
            nn.init.xavier_uniform_(layer.weight)
            if bias:
                nn.init.zeros_(layer.bias)

    def forward(self, x, residual=None):
        gate, up = self.gate_proj, self.up_proj
        if fused_ops.dense_usable(x, gate.weight, up.weight, gate.bias, up.bias):
            h = fused_ops.gated_linear(x, gate.weight, up.weight, gate.bias, up.bias, act=self.act_name)
        else:
            h = _ACTS[self.act_name](gate(x)) * up(x)
        return _project(self.dropout(h), self.out_proj, residual)

"""Fused operations of the encoder block on 16-bit tensors.

Row operations (bf16, inference): ``add_layernorm`` (``LayerNorm(x + y)`` in one pass) and ``gelu`` (erf form).  The reference runs these as
PyTorch operators (``old/old_scripts/encoder.py:30-39``, ``utils/model_utils/base_modules/base_modules.py:46-52``); here they are single
HBM-bound kernels behind ``pai_add_layernorm_bf16`` / ``pai_gelu_bf16``.  They have no backward: the modules use them only when no gradient
is being recorded and fall back to the PyTorch operators otherwise.

Products of the feed-forward block (bf16 or fp16, with gradients):

``linear(x, weight, bias, act, residual)``                ``act(x W^T + b) + r`` as one kernel
``gated_linear(x, w_gate, w_up, b_gate, b_up, act)``      ``act(x Wg^T + bg) * (x Wu^T + bu)`` as one kernel

Both accumulate in fp32, apply their epilogue in fp32 and round once; the backward rounds the gradient of the pre-activation once to the
tensors' type (it is an operand of the two products that follow) and keeps the pre-activations themselves in more bits than the type has.
``act`` is ``None``, ``"gelu"`` (erf form), ``"silu"``, ``"relu"`` or ``"sigmoid"``.  There is no CPU path and no fp32 path (``TypeError``); under
``torch.autocast`` the operands are cast to its type.  Gradients are first-order only (``create_graph`` raises).
"""
import torch

from proteusai_b200 import _lib


def usable(*tensors):
    """The fused kernels apply to bf16 CUDA tensors when autograd is not recording."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return False
    return all(t.is_cuda and t.dtype == torch.bfloat16 for t in tensors)


def add_layernorm(x, y, weight, bias, eps):
    """``LayerNorm(x + y)`` over the last axis (``y`` may be ``None``); ``weight``/``bias`` bf16 or fp32."""
    d = x.shape[-1]
    x = x.contiguous()
    y = None if y is None else y.contiguous()
    fp32 = weight.dtype == torch.float32
    if weight.dtype != bias.dtype or weight.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("LayerNorm weight and bias must both be bf16 or both fp32")
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().pai_add_layernorm_bf16(
            _lib.ptr(x), _lib.ptr(y), _lib.ptr(weight.detach().contiguous()), _lib.ptr(bias.detach().contiguous()), int(fp32),
            _lib.ptr(out), x.numel() // d, d, float(eps), _lib.current_stream()), "pai_add_layernorm_bf16")
    return out


def gelu(x, inplace=False):
    """Erf GELU of a bf16 tensor whose element count is a multiple of 8."""
    x = x.contiguous()
    out = x if inplace else torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().pai_gelu_bf16(_lib.ptr(x), _lib.ptr(out), x.numel(), _lib.current_stream()), "pai_gelu_bf16")
    return out


# ---- products of the feed-forward block -------------------------------------------------------------------------------
ACTIVATIONS = {None: 0, "gelu": 1, "silu": 2, "relu": 3, "sigmoid": 4}  # enum pai_act


def dense_usable(*tensors):
    """``linear`` and ``gated_linear`` take these tensors (``None`` among them is skipped): CUDA, all bf16 or all fp16, or whatever autocast
    would make so."""
    ts = [t for t in tensors if t is not None]
    if not all(t.is_cuda and t.is_floating_point() for t in ts):
        return False
    if torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda") in (torch.bfloat16, torch.float16)
    return ts[0].dtype in (torch.bfloat16, torch.float16) and all(t.dtype == ts[0].dtype for t in ts)


def dense_dtype(x):
    """The type in which ``linear`` and ``gated_linear`` compute for an ``x`` they take."""
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype


def _act_code(what, act):
    code = ACTIVATIONS.get(act, -1)
    if code < 0:
        raise ValueError(f"{what}: act must be one of {sorted(a for a in ACTIVATIONS if a)} or None, not {act!r}")
    return code


def linear(x, weight, bias=None, act=None, residual=None):
    """``act(x weight^T + bias) + residual``: ``x`` [..., d_in], ``weight`` [d_out, d_in] (as ``nn.Linear`` keeps it), ``bias`` [d_out] of x's type or
    fp32, ``residual`` of the output's shape [..., d_out] and type.  Any strides are taken; an operand whose rows are not 16-byte aligned
    (odd widths) is copied once."""
    return _lib.torch_ops().linear(x, weight, bias, _act_code("linear", act), residual)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act="silu"):
    """``act(x w_gate^T + b_gate) * (x w_up^T + b_up)``: the hidden layer of a gated feed-forward block.  ``x`` [..., d_in], ``w_gate`` and ``w_up``
    [d_out, d_in], biases [d_out] of x's type or fp32; strides as in ``linear``."""
    return _lib.torch_ops().gated_linear(x, w_gate, w_up, b_gate, b_up, _act_code("gated_linear", act))

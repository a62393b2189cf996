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
``torch.autocast`` the operands are cast to its type.  Gradients are first-order only.
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
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}                          # enum pai_dtype


def dense_usable(*tensors):
    """``linear`` and ``gated_linear`` take these tensors (``None`` among them is skipped): CUDA, all bf16 or all fp16, or whatever autocast
    would make so."""
    ts = [t for t in tensors if t is not None]
    if not all(t.is_cuda and t.is_floating_point() for t in ts):
        return False
    if torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda") in _DTYPES
    return ts[0].dtype in _DTYPES and all(t.dtype == ts[0].dtype for t in ts)


def _addr(t):
    return None if t is None else t.data_ptr()


class _on:
    """The tensor's device as the current one; gives its current stream."""

    __slots__ = ("guard", "index")

    def __init__(self, t):
        self.index = t.device.index
        self.guard = None if self.index == torch.cuda.current_device() else torch.cuda.device(self.index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _rows(t):
    """``t`` [rows, cols], or a copy, with contiguous columns and rows that do not overlap."""
    return t if (t.stride(1) == 1 or t.size(1) == 1) and (t.stride(0) >= t.size(1) or t.size(0) == 1) else t.contiguous()


def _operand(t):
    """``t`` [rows, cols], or a copy, as the products read it: 16-byte aligned rows (``pai_copy_rows16`` makes the copy)."""
    t = _rows(t)
    if t.data_ptr() % 16 == 0 and (t.stride(0) % 8 == 0 or t.size(0) == 1):
        return t
    rows, cols = t.shape
    pitch = (cols + 7) // 8 * 8
    out = torch.empty(rows, pitch, dtype=t.dtype, device=t.device)
    with _on(t) as stream:
        _lib.check(_lib.lib().pai_copy_rows16(t.data_ptr(), t.stride(0), out.data_ptr(), pitch, rows, cols, stream), "pai_copy_rows16")
    return out[:, :cols]


def _forward(x, ws, bs, r, act, save):
    """The kernel call on 2-D tensors: ``(y, saved pre-activations or None)``; ``ws`` one weight (linear) or two (gated)."""
    (m, k), n, gated = x.shape, ws[0].shape[0], len(ws) == 2
    y = torch.empty(m, n, dtype=x.dtype, device=x.device)
    saved = None
    if m == 0:
        return y, saved
    lib = _lib.lib()
    if save and (gated or act):
        saved = torch.empty(lib.pai_dense_saved_bytes(m, n, k, gated, _DTYPES[x.dtype]), dtype=torch.uint8, device=x.device)
    fp32 = any(b is not None and b.dtype == torch.float32 for b in bs)
    with _on(x) as stream:
        if gated:
            _lib.check(lib.pai_gated_fwd(x.data_ptr(), x.stride(0), ws[0].data_ptr(), ws[0].stride(0), ws[1].data_ptr(), ws[1].stride(0),
                                         _addr(bs[0]), _addr(bs[1]), fp32, y.data_ptr(), n, _addr(saved), m, n, k, act, _DTYPES[x.dtype], stream),
                       "pai_gated_fwd")
        else:
            _lib.check(lib.pai_linear_fwd(x.data_ptr(), x.stride(0), ws[0].data_ptr(), ws[0].stride(0), _addr(bs[0]), fp32, _addr(r),
                                          0 if r is None else r.stride(0), y.data_ptr(), n, _addr(saved), m, n, k, act, _DTYPES[x.dtype], stream),
                       "pai_linear_fwd")
    return y, saved


def _backward(dy, x, ws, bs, saved, act, need_x, need_w, need_b):
    """Gradients ``(dx, [dw], [db])``, ``None`` where not needed."""
    (m, k), n, gated = x.shape, ws[0].shape[0], len(ws) == 2
    dx = torch.empty(m, k, dtype=x.dtype, device=x.device) if need_x else None
    dws = [torch.empty(n, k, dtype=x.dtype, device=x.device) if need else None for need in need_w]
    dbs = [torch.empty(n, dtype=b.dtype, device=x.device) if need else None for need, b in zip(need_b, bs)]
    if m == 0:
        for t in dws + dbs:
            if t is not None:
                t.zero_()
        return dx, dws, dbs
    dy = _rows(dy)
    if not gated and not act and (need_x or need_w[0]):
        dy = _operand(dy)
    lib = _lib.lib()
    fp32 = any(b is not None and b.dtype == torch.float32 for b in bs)
    size = lib.pai_dense_bwd_workspace_bytes(m, n, k, gated)
    ws_buf = torch.empty(size, dtype=torch.uint8, device=x.device)
    with _on(x) as stream:
        if gated:
            _lib.check(lib.pai_gated_bwd(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), ws[0].data_ptr(), ws[0].stride(0), ws[1].data_ptr(),
                                         ws[1].stride(0), _addr(saved), _addr(dx), k, _addr(dws[0]), _addr(dws[1]), _addr(dbs[0]), _addr(dbs[1]), fp32,
                                         ws_buf.data_ptr(), size, m, n, k, act, _DTYPES[x.dtype], stream), "pai_gated_bwd")
        else:
            _lib.check(lib.pai_linear_bwd(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), ws[0].data_ptr(), ws[0].stride(0), _addr(saved),
                                          _addr(dx), k, _addr(dws[0]), _addr(dbs[0]), fp32, ws_buf.data_ptr(), size, m, n, k, act, _DTYPES[x.dtype],
                                          stream), "pai_linear_bwd")
    return dx, dws, dbs


class _linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x, weight = _operand(x), _operand(weight)
        y, saved = _forward(x, (weight,), (bias,), residual, act, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, (dw,), (db,) = _backward(dy, x, (weight,), (bias,), saved, ctx.act, need[0], (need[1],), (need[2],))
        return dx, dw, db, dy if need[3] else None, None


class _gated_linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        x, w_gate, w_up = _operand(x), _operand(w_gate), _operand(w_up)
        h, saved = _forward(x, (w_gate, w_up), (b_gate, b_up), None, act, True)
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, saved)
        ctx.act = act
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up, saved = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dws, dbs = _backward(dh, x, (w_gate, w_up), (b_gate, b_up), saved, ctx.act, need[0], need[1:3], need[3:5])
        return (dx, *dws, *dbs, None)


def _checked(what, x, ws, bs, act):
    """The arguments with autocast applied, after the checks both operators share; weights first, then biases."""
    if act not in ACTIVATIONS:
        raise ValueError(f"{what}: act must be one of {sorted(a for a in ACTIVATIONS if a)} or None, not {act!r}")
    for t in (x, *ws, *bs):
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{what} needs CUDA tensors: there is no CPU path")
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, ws = x.to(dt), [w.to(dt) for w in ws]
        bs = [b if b is None or b.dtype == torch.float32 else b.to(dt) for b in bs]
    if x.dtype not in _DTYPES or any(w.dtype != x.dtype for w in ws):
        raise TypeError(f"{what}: x and weights must all be bfloat16 or all float16, not {x.dtype} and {', '.join(str(w.dtype) for w in ws)}")
    if x.dim() < 1 or any(w.dim() != 2 for w in ws) or any(w.shape != ws[0].shape for w in ws) or ws[0].shape[1] != x.shape[-1]:
        raise ValueError(f"{what}: x [..., d_in] and weights [d_out, d_in] do not fit: {tuple(x.shape)}, {', '.join(str(tuple(w.shape)) for w in ws)}")
    if 0 in ws[0].shape:
        raise ValueError(f"{what}: weights must not be empty: {tuple(ws[0].shape)}")
    given = [b for b in bs if b is not None]
    for b in given:
        if b.shape != ws[0].shape[:1]:
            raise ValueError(f"{what}: a bias must have shape {tuple(ws[0].shape[:1])}, not {tuple(b.shape)}")
        if b.dtype not in (x.dtype, torch.float32) or b.dtype != given[0].dtype:
            raise TypeError(f"{what}: biases must be {x.dtype} or float32, not {', '.join(str(b.dtype) for b in given)}")
    if any(t is not None and t.device != x.device for t in (*ws, *bs)):
        raise RuntimeError(f"{what}: all tensors must be on one device")
    return x, ws, [b if b is None or b.is_contiguous() else b.contiguous() for b in bs]


def _flat(t):
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _recording(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def linear(x, weight, bias=None, act=None, residual=None):
    """``act(x weight^T + bias) + residual``: ``x`` [..., d_in], ``weight`` [d_out, d_in] (as ``nn.Linear`` keeps it), ``bias`` [d_out] of x's type or
    fp32, ``residual`` of the output's shape [..., d_out] and type.  Any strides are taken; an operand whose rows are not 16-byte aligned
    (odd widths) is copied once."""
    shape = x.shape
    x, (weight,), (bias,) = _checked("linear", x, (weight,), (bias,), act)
    if residual is not None:
        if not residual.is_cuda or residual.device != x.device:
            raise RuntimeError("linear: all tensors must be on one CUDA device")
        if torch.is_autocast_enabled("cuda"):
            residual = residual.to(x.dtype)
        if residual.dtype != x.dtype:
            raise TypeError(f"linear: residual must be {x.dtype}, not {residual.dtype}")
        if residual.shape != (*shape[:-1], weight.shape[0]):
            raise ValueError(f"linear: residual must have the output's shape {(*shape[:-1], weight.shape[0])}, not {tuple(residual.shape)}")
        residual = _flat(residual)
        if not (residual.stride(1) == 1 or residual.size(1) == 1):
            residual = residual.contiguous()
    x = _flat(x)
    if _recording(x, weight, bias, residual):
        y = _linear.apply(x, weight, bias, residual, ACTIVATIONS[act])
    else:
        y, _ = _forward(_operand(x), (_operand(weight),), (bias,), residual, ACTIVATIONS[act], False)
    return y if len(shape) == 2 else y.view(*shape[:-1], y.shape[1])


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act="silu"):
    """``act(x w_gate^T + b_gate) * (x w_up^T + b_up)``: the hidden layer of a gated feed-forward block.  ``x`` [..., d_in], ``w_gate`` and ``w_up``
    [d_out, d_in], biases [d_out] of x's type or fp32; strides as in ``linear``."""
    shape = x.shape
    x, (w_gate, w_up), (b_gate, b_up) = _checked("gated_linear", x, (w_gate, w_up), (b_gate, b_up), act)
    x = _flat(x)
    if _recording(x, w_gate, w_up, b_gate, b_up):
        h = _gated_linear.apply(x, w_gate, w_up, b_gate, b_up, ACTIVATIONS[act])
    else:
        h, _ = _forward(_operand(x), (_operand(w_gate), _operand(w_up)), (b_gate, b_up), None, ACTIVATIONS[act], False)
    return h if len(shape) == 2 else h.view(*shape[:-1], h.shape[1])

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


def _on(t):
    """``(current stream of t's device, guard)``; the guard, if not ``None``, makes that device the current one for the call."""
    index = t.get_device()
    return torch._C._cuda_getCurrentRawStream(index), None if index == torch.cuda.current_device() else torch.cuda.device(index)


def _call(name, guard, args):
    fn = getattr(_lib.lib(), name)
    if guard is None:
        status = fn(*args)
    else:
        with guard:
            status = fn(*args)
    if status:
        _lib.check(status, name)


def _rows(t):
    """``t`` [rows, cols], or a copy, with contiguous columns and rows that do not overlap."""
    if t.is_contiguous() or ((t.stride(1) == 1 or t.size(1) == 1) and (t.stride(0) >= t.size(1) or t.size(0) == 1)):
        return t
    return t.contiguous()


def _operand(t):
    """``t`` [rows, cols], or a copy, as the products read it: 16-byte aligned rows (``pai_copy_rows16`` makes the copy)."""
    t = _rows(t)
    if not (t.data_ptr() & 15 or (t.stride(0) & 7 and t.size(0) != 1)):
        return t
    rows, cols = t.shape
    pitch = (cols + 7) // 8 * 8
    out = torch.empty(rows, pitch, dtype=t.dtype, device=t.device)
    stream, guard = _on(t)
    _call("pai_copy_rows16", guard, (t.data_ptr(), t.stride(0), out.data_ptr(), pitch, rows, cols, stream))
    return out[:, :cols]


def _forward(x, w, w2, b, b2, r, act, save):
    """The kernel call on 2-D tensors: ``(y, saved pre-activations or None)``; ``w2`` not ``None``: gated."""
    (m, k), n, dtype = x.shape, w.shape[0], _DTYPES[x.dtype]
    y = torch.empty(m, n, dtype=x.dtype, device=x.device)
    if m == 0:
        return y, None
    saved, at = None, None
    if save and (act or w2 is not None):
        saved = torch.empty(_lib.lib().pai_dense_saved_bytes(m, n, k, w2 is not None, dtype), dtype=torch.uint8, device=x.device)
        at = saved.data_ptr()
    fp32 = (b is not None and b.dtype is torch.float32) or (b2 is not None and b2.dtype is torch.float32)
    stream, guard = _on(x)
    if w2 is None:
        _call("pai_linear_fwd", guard, (x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), None if b is None else b.data_ptr(), fp32,
                                        None if r is None else r.data_ptr(), 0 if r is None else r.stride(0), y.data_ptr(), n, at, m, n, k, act,
                                        dtype, stream))
    else:
        _call("pai_gated_fwd", guard, (x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), w2.data_ptr(), w2.stride(0),
                                       None if b is None else b.data_ptr(), None if b2 is None else b2.data_ptr(), fp32, y.data_ptr(), n, at, m, n, k,
                                       act, dtype, stream))
    return y, saved


def _gradient(like, rows, *shape):
    """An output buffer of the backward call and its address (zeros where there are no rows to sum)."""
    t = (torch.empty if rows else torch.zeros)(*shape, dtype=like.dtype, device=like.device)
    return t, t.data_ptr()


class _linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x, weight = _operand(x), _operand(weight)
        need = ctx.needs_input_grad
        y, saved = _forward(x, weight, None, bias, None, residual, act, need[0] or need[1] or need[2])
        ctx.save_for_backward(x, weight, bias, saved)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        if not (need_x or need_w or need_b):
            return None, None, None, dy, None
        x, weight, bias, saved = ctx.saved_tensors
        (m, k), n, act = x.shape, weight.shape[0], ctx.act
        dx = dw = db = px = pw = pb = None
        if need_x:
            dx, px = _gradient(x, 1, m, k)
        if need_w:
            dw, pw = _gradient(weight, m, n, k)
        if need_b:
            db, pb = _gradient(bias, m, n)
        if m:
            d = _operand(dy) if not act and (need_x or need_w) else _rows(dy)
            size = _lib.lib().pai_dense_bwd_workspace_bytes(m, n, k, 0)
            buf = torch.empty(size, dtype=torch.uint8, device=x.device)
            stream, guard = _on(x)
            _call("pai_linear_bwd", guard, (d.data_ptr(), d.stride(0), x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0),
                                            None if saved is None else saved.data_ptr(), px, k, pw, pb, need_b and bias.dtype is torch.float32,
                                            buf.data_ptr(), size, m, n, k, act, _DTYPES[x.dtype], stream))
        return dx, dw, db, dy if need_r else None, None


class _gated_linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        x, w_gate, w_up = _operand(x), _operand(w_gate), _operand(w_up)
        h, saved = _forward(x, w_gate, w_up, b_gate, b_up, None, act, True)
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, saved)
        ctx.act = act
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        need_x, need_wg, need_wu, need_bg, need_bu, _ = ctx.needs_input_grad
        x, w_gate, w_up, b_gate, b_up, saved = ctx.saved_tensors
        (m, k), n = x.shape, w_gate.shape[0]
        dx = dwg = dwu = dbg = dbu = px = pwg = pwu = pbg = pbu = None
        if need_x:
            dx, px = _gradient(x, 1, m, k)
        if need_wg:
            dwg, pwg = _gradient(w_gate, m, n, k)
        if need_wu:
            dwu, pwu = _gradient(w_up, m, n, k)
        if need_bg:
            dbg, pbg = _gradient(b_gate, m, n)
        if need_bu:
            dbu, pbu = _gradient(b_up, m, n)
        if m:
            d = _rows(dh)
            fp32 = (need_bg and b_gate.dtype is torch.float32) or (need_bu and b_up.dtype is torch.float32)
            size = _lib.lib().pai_dense_bwd_workspace_bytes(m, n, k, 1)
            buf = torch.empty(size, dtype=torch.uint8, device=x.device)
            stream, guard = _on(x)
            _call("pai_gated_bwd", guard, (d.data_ptr(), d.stride(0), x.data_ptr(), x.stride(0), w_gate.data_ptr(), w_gate.stride(0), w_up.data_ptr(),
                                           w_up.stride(0), saved.data_ptr(), px, k, pwg, pwu, pbg, pbu, fp32, buf.data_ptr(), size, m, n, k, ctx.act,
                                           _DTYPES[x.dtype], stream))
        return dx, dwg, dwu, dbg, dbu, None


def _refuse(what, x, ws, bs, r):
    """The error for arguments that do not fit, or ``None``.  (Called when the quick test of ``_fits`` fails.)"""
    given = [t for t in (x, *ws, *bs, r) if t is not None]
    if not all(t.is_cuda for t in given):
        return RuntimeError(f"{what} needs CUDA tensors: there is no CPU path")
    if any(t.device != x.device for t in given):
        return RuntimeError(f"{what}: all tensors must be on one device")
    if x.dtype not in _DTYPES or any(w.dtype != x.dtype for w in ws):
        return TypeError(f"{what}: x and weights must all be bfloat16 or all float16, not {x.dtype} and {', '.join(str(w.dtype) for w in ws)}")
    if x.dim() < 1 or any(w.dim() != 2 or w.shape != ws[0].shape for w in ws) or ws[0].shape[1] != x.shape[-1]:
        return ValueError(f"{what}: x [..., d_in] and weights [d_out, d_in] do not fit: {tuple(x.shape)}, {', '.join(str(tuple(w.shape)) for w in ws)}")
    if 0 in ws[0].shape:
        return ValueError(f"{what}: weights must not be empty: {tuple(ws[0].shape)}")
    biases = [b for b in bs if b is not None]
    for b in biases:
        if b.shape != ws[0].shape[:1]:
            return ValueError(f"{what}: a bias must have shape {tuple(ws[0].shape[:1])}, not {tuple(b.shape)}")
        if b.dtype not in (x.dtype, torch.float32) or b.dtype != biases[0].dtype:
            return TypeError(f"{what}: biases must all be {x.dtype} or all float32, not {', '.join(str(b.dtype) for b in biases)}")
    if r is not None:
        if r.dtype != x.dtype:
            return TypeError(f"{what}: residual must be {x.dtype}, not {r.dtype}")
        if r.shape != (*x.shape[:-1], ws[0].shape[0]):
            return ValueError(f"{what}: residual must have the output's shape {(*x.shape[:-1], ws[0].shape[0])}, not {tuple(r.shape)}")
    return None


def _fits(x, w, b):
    """x [rows, d_in], one weight and its bias, all of one 16-bit type on one device: what most calls are."""
    if not (x.is_cuda and w.is_cuda and x.dim() == 2 and w.dim() == 2) or x.dtype not in _DTYPES or w.dtype is not x.dtype:
        return False
    (n, k), index = w.shape, x.get_device()
    if x.size(1) != k or n == 0 or k == 0 or w.get_device() != index:
        return False
    return b is None or (b.dtype is x.dtype and b.is_cuda and b.dim() == 1 and b.size(0) == n and b.get_device() == index and b.is_contiguous())


def _cast(t, dtype, keep_fp32=False):
    return t if t is None or t.dtype is dtype or (keep_fp32 and t.dtype is torch.float32) else t.to(dtype)


def _contiguous(b):
    return b if b is None or b.is_contiguous() else b.contiguous()


def linear(x, weight, bias=None, act=None, residual=None):
    """``act(x weight^T + bias) + residual``: ``x`` [..., d_in], ``weight`` [d_out, d_in] (as ``nn.Linear`` keeps it), ``bias`` [d_out] of x's type or
    fp32, ``residual`` of the output's shape [..., d_out] and type.  Any strides are taken; an operand whose rows are not 16-byte aligned
    (odd widths) is copied once."""
    code = ACTIVATIONS.get(act, -1)
    if code < 0:
        raise ValueError(f"linear: act must be one of {sorted(a for a in ACTIVATIONS if a)} or None, not {act!r}")
    shape = None
    if residual is not None or torch.is_autocast_enabled("cuda") or not _fits(x, weight, bias):
        if torch.is_autocast_enabled("cuda"):
            dt = torch.get_autocast_dtype("cuda")
            x, weight, bias, residual = _cast(x, dt), _cast(weight, dt), _cast(bias, dt, True), _cast(residual, dt)
        error = _refuse("linear", x, (weight,), (bias,), residual)
        if error is not None:
            raise error
        if x.dim() != 2:
            shape = x.shape
            x = x.reshape(-1, shape[-1])
        bias = _contiguous(bias)
        if residual is not None:
            residual = residual if residual.dim() == 2 else residual.reshape(-1, residual.shape[-1])
            if residual.stride(1) != 1 and residual.size(1) != 1:
                residual = residual.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        y = _linear.apply(x, weight, bias, residual, code)
    else:
        y, _ = _forward(_operand(x), _operand(weight), None, bias, None, residual, code, False)
    return y if shape is None else y.view(*shape[:-1], y.shape[1])


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act="silu"):
    """``act(x w_gate^T + b_gate) * (x w_up^T + b_up)``: the hidden layer of a gated feed-forward block.  ``x`` [..., d_in], ``w_gate`` and ``w_up``
    [d_out, d_in], biases [d_out] of x's type or fp32; strides as in ``linear``."""
    code = ACTIVATIONS.get(act, -1)
    if code < 0:
        raise ValueError(f"gated_linear: act must be one of {sorted(a for a in ACTIVATIONS if a)} or None, not {act!r}")
    shape = None
    if torch.is_autocast_enabled("cuda") or not (_fits(x, w_gate, b_gate) and _fits(x, w_up, b_up) and w_gate.shape == w_up.shape):
        if torch.is_autocast_enabled("cuda"):
            dt = torch.get_autocast_dtype("cuda")
            x, w_gate, w_up, b_gate, b_up = _cast(x, dt), _cast(w_gate, dt), _cast(w_up, dt), _cast(b_gate, dt, True), _cast(b_up, dt, True)
        error = _refuse("gated_linear", x, (w_gate, w_up), (b_gate, b_up), None)
        if error is not None:
            raise error
        if x.dim() != 2:
            shape = x.shape
            x = x.reshape(-1, shape[-1])
        b_gate, b_up = _contiguous(b_gate), _contiguous(b_up)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or (b_gate is not None and b_gate.requires_grad) or
                                    (b_up is not None and b_up.requires_grad)):
        h = _gated_linear.apply(x, w_gate, w_up, b_gate, b_up, code)
    else:
        h, _ = _forward(_operand(x), _operand(w_gate), _operand(w_up), b_gate, b_up, None, code, False)
    return h if shape is None else h.view(*shape[:-1], h.shape[1])

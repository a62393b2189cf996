"""Measured cases of the feed-forward operators of the encoder block: the matrix product with bias, activation and residual in its
epilogue (``fused_ops.linear``) and the gated product of two projections (``fused_ops.gated_linear``), forward alone (inference) and
forward + backward (training).

    linear          y = act(x W^T + b) + r                              x [M, K], W [N, K], b [N], r [M, N]
    gated_linear    h = act(x Wg^T + bg) * (x Wu^T + bu)                x [M, K], Wg, Wu [N, K], bg, bu [N]

``run`` computes them from elementary torch operations in 32 bits where ``own`` is false, and through the framework's public calls where it is
true.  A training pass returns the output and the gradients of every floating input that has one.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_ACTS = ("none", "gelu", "silu", "relu", "sigmoid")
_MAX_FLOPS = 2.0 * 16384 * 4096 * 4096   # the largest listed case
_MAX_BYTES = 600e6


def _case(name, op, train, dtype, rows, d_in, d_out, act, bias, residual, lead):
    """``lead``: columns of a wider buffer in front of x's own (0: x is contiguous), so that its rows start off the alignment of a tensor."""
    c = {"op": op, "train": train, "dtype": dtype, "rows": rows, "d_in": d_in, "d_out": d_out, "act": act, "bias": bias,
         "residual": residual, "lead": lead}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one residue through the first projection of the encoder's MLP (decoding one position at a time): latency
        _case("linear_one_residue", "linear", False, "bf16", 1, 512, 2048, "gelu", True, False, 0),
        # one chain of 256 residues through the second projection, added to the block's input
        _case("linear_one_chain", "linear", False, "bf16", 256, 2048, 512, "none", True, True, 0),
        # 64 chains padded to 1024: the first projection of the encoder inference configuration
        _case("linear_batch_in", "linear", False, "bf16", 65536, 512, 2048, "gelu", True, False, 0),
        # 8 chains of 1024, second projection with the residual, training
        _case("linear_train_out", "linear", True, "bf16", 8192, 2048, 512, "none", True, True, 0),
        # 8 chains of 1024, the head to 20 amino-acid logits, training
        _case("linear_train_head", "linear", True, "bf16", 8192, 512, 20, "none", True, False, 0),
        # valid residues of a packed ragged batch, odd widths, x a column slice of a wider buffer, training in fp16
        _case("linear_train_ragged", "linear", True, "fp16", 3001, 1001, 1357, "silu", True, True, 3),
        # a wide model: the rate of the matrix product itself
        _case("linear_wide", "linear", False, "bf16", 16384, 4096, 4096, "none", True, False, 0),
        # one residue through the gated projections: latency
        _case("gated_one_residue", "gated", False, "bf16", 1, 512, 2048, "silu", False, False, 0),
        # one chain of 131 residues, fp16 inference
        _case("gated_one_chain", "gated", False, "fp16", 131, 512, 1024, "gelu", True, False, 0),
        # 64 chains padded to 1024: the gated form of the encoder inference configuration
        _case("gated_batch", "gated", False, "bf16", 65536, 512, 2048, "silu", False, False, 0),
        # 16 chains of 1024, training
        _case("gated_train", "gated", True, "bf16", 16384, 512, 2048, "silu", True, False, 0),
        # ragged rows and odd widths, training
        _case("gated_train_ragged", "gated", True, "bf16", 777, 250, 1023, "gelu", True, False, 0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    """A width of 16 to 4096: half of them multiples of 64 or 8, the others as they come, odd ones among them."""
    w = _log_int(rng, 16, 4096)
    step = rng.choice((1, 1, 8, 64))
    return max(16, (w // step) * step)


def draw(rng):
    op = rng.choice(("linear", "gated"))
    train = rng.random() < 0.5
    act = rng.choice(_ACTS if op == "linear" else _ACTS[1:])
    c = _case(None, op, train, rng.choice(("bf16", "bf16", "fp16")), _log_int(rng, 1, 65536), _width(rng), _width(rng), act,
              rng.random() < 0.7, op == "linear" and rng.random() < 0.5, rng.choice((0, 0, 0, 1, 8)))
    w = work(c)
    while w["flops"] > _MAX_FLOPS or w["bytes"] > _MAX_BYTES:
        c["rows"] = max(1, int(c["rows"] / 1.37))
        w = work(c)
    return c


def work(case):
    m, k, n = case["rows"], case["d_in"], case["d_out"]
    mats = 2 if case["op"] == "gated" else 1
    elements = m * k + mats * n * k + m * n                     # x, the weights, the output
    elements += mats * n if case["bias"] else 0
    elements += m * n if case["residual"] else 0
    flops = 2.0 * m * k * n * mats
    if case["train"]:
        elements += m * n + m * k + mats * n * k                # the output's gradient; dx and the weights' gradients
        elements += mats * n if case["bias"] else 0
        flops *= 3
    return {"bytes": 2 * elements, "flops": flops}


def _tensors(case, seed):
    """The inputs: rows as a LayerNorm leaves them, Xavier-uniform weights, small biases, a unit gradient of the output."""
    dt = _DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    m, k, n = case["rows"], case["d_in"], case["d_out"]
    mats = 2 if case["op"] == "gated" else 1
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    wide = randn(m, k + case["lead"]).to(dt)
    x = wide[:, case["lead"]:]
    bound = math.sqrt(6.0 / (k + n))
    ws = [((torch.rand(n, k, generator=g, device="cuda") * 2 - 1) * bound).to(dt) for _ in range(mats)]
    bs = [(0.1 * randn(n)).to(dt) if case["bias"] else None for _ in range(mats)]
    r = randn(m, n).to(dt) if case["residual"] else None
    dy = randn(m, n).to(dt) if case["train"] else None
    return x, ws, bs, r, dy


def prepare(case, seed):
    x, ws, bs, r, dy = _tensors(case, seed)
    leaves = [t for t in (x, *ws, *bs, r) if t is not None] if case["train"] else []
    for t in leaves:
        t.requires_grad_(True)
    return {"gated": case["op"] == "gated", "act": case["act"], "x": x, "ws": ws, "bs": bs, "r": r, "dy": dy, "leaves": leaves}


def run(state):
    if own:
        from proteusai_b200.utils.model_utils.base_modules import fused_ops
        act = None if state["act"] == "none" else state["act"]
        with torch.set_grad_enabled(state["dy"] is not None):
            if state["gated"]:
                y = fused_ops.gated_linear(state["x"], *state["ws"], *state["bs"], act=act)
            else:
                y = fused_ops.linear(state["x"], state["ws"][0], state["bs"][0], act=act, residual=state["r"])
        if state["dy"] is None:
            return y
        return (y.detach(), *torch.autograd.grad(y, state["leaves"], state["dy"]))
    with torch.no_grad():
        return _plain_gated(state) if state["gated"] else _plain_linear(state)


def _act(z, name):
    """The activation and its derivative, elementwise."""
    if name == "gelu":
        phi = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if name == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s, s * (1.0 - s)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    return z, torch.ones_like(z)


def _affine(x, w, b):
    z = x @ w.float().t()
    return z if b is None else z + b.float()


def _plain_linear(s):
    dt, x, w, b = s["x"].dtype, s["x"].float(), s["ws"][0], s["bs"][0]
    z = _affine(x, w, b)
    a, da = _act(z, s["act"])
    y = a if s["r"] is None else a + s["r"].float()
    if s["dy"] is None:
        return y.to(dt)
    dz = s["dy"].float() * da
    out = [y, dz @ w.float(), dz.t() @ x]
    out += [] if b is None else [dz.sum(0)]
    out += [] if s["r"] is None else [s["dy"]]
    return tuple(t.to(dt) for t in out)


def _plain_gated(s):
    dt, x, (wg, wu), (bg, bu) = s["x"].dtype, s["x"].float(), s["ws"], s["bs"]
    zg, u = _affine(x, wg, bg), _affine(x, wu, bu)
    a, da = _act(zg, s["act"])
    h = a * u
    if s["dy"] is None:
        return h.to(dt)
    dh = s["dy"].float()
    dg, du = dh * u * da, dh * a
    out = [h, dg @ wg.float() + du @ wu.float(), dg.t() @ x, du.t() @ x]
    out += [] if bg is None else [dg.sum(0), du.sum(0)]
    return tuple(t.to(dt) for t in out)


def exact(case, seed):
    """The definition in 64 bits: torch's own activations and its differentiation of them."""
    x, ws, bs, r, dy = _tensors(case, seed)
    f = torch.nn.functional
    fn = {"none": lambda t: t, "gelu": f.gelu, "silu": f.silu, "relu": f.relu, "sigmoid": torch.sigmoid}[case["act"]]
    leaves = [t.detach().double().requires_grad_(case["train"]) if t is not None else None for t in (x, *ws, *bs, r)]
    given = [t for t in leaves if t is not None]
    mats = len(ws)
    x64, w64, b64, r64 = leaves[0], leaves[1:1 + mats], leaves[1 + mats:1 + 2 * mats], leaves[-1]
    with torch.set_grad_enabled(case["train"]):
        z = [f.linear(x64, w, b) for w, b in zip(w64, b64)]
        y = fn(z[0]) * z[1] if mats == 2 else fn(z[0])
        y = y if r64 is None else y + r64
    if not case["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, given, dy.double()))

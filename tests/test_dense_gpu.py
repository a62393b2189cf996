"""The feed-forward products (``fused_ops.linear``, ``fused_ops.gated_linear``) against their definitions in 64 bits.

Tolerances, from the arithmetic.  u = finfo(dtype).eps / 2 is half a rounding step relative to the value.  A product over K terms summed in
fp32 is off by at most K 2^-23 sum|x||w| (every addition rounded or truncated to 24 bits); call that d.  The activations are Lipschitz with a
constant below 1.2 and evaluated to 1e-5 relative and 1e-6 absolute.  So an output is within

    u |y| + 1.2 d + 1e-5 |a| + 1e-6,

a gradient of a pre-activation (rounded once, its slope off by at most max|act''| d <= d and 1e-5) within E = u |dz| + |dy| (d + 1e-5), with
|dy| added where a ReLU's z is within d of its kink, and a product with it within E |w| + (its own sum's) N 2^-23 |dz||w| + u |dx|.  These bounds
hold element by element and are loose for long sums, where rounding errors cancel: there the 2-norm is held too, the error of independent
roundings (dz and the output, each below u / sqrt 3 in the mean) being below u for any long sum; 2 u is allowed.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = (None, "gelu", "silu", "relu", "sigmoid")
DTYPES = (torch.bfloat16, torch.float16)
# rows, d_in, d_out: single tokens, single columns, odd widths, tile borders (16, 32, 64, 128, 256 rows; 64 and 128 columns), ragged batches
SHAPES = [(1, 1, 1), (1, 512, 2048), (2, 8, 16), (3, 7, 5), (4, 2056, 33), (8, 300, 77), (9, 300, 77), (16, 64, 128), (17, 65, 129), (33, 1000, 20), (64, 130, 66), (131, 512, 1024),
          (256, 2048, 512), (300, 96, 1), (777, 250, 1023), (1025, 72, 136)]


def _f(name):
    f = torch.nn.functional
    return {None: lambda t: t, "gelu": f.gelu, "silu": f.silu, "relu": f.relu, "sigmoid": torch.sigmoid}[name]


def _inputs(m, k, n, dtype, mats=1, bias=True, residual=False, seed=0, bias_dtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * m + 11 * k + 13 * n)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    bound = math.sqrt(6.0 / (k + n))
    x = rnd(m, k).to(dtype)
    ws = [((torch.rand(n, k, generator=g, device="cuda") * 2 - 1) * bound).to(dtype) for _ in range(mats)]
    bs = [(0.3 * rnd(n)).to(bias_dtype or dtype) if bias else None for _ in range(mats)]
    r = rnd(m, n).to(dtype) if residual else None
    return x, ws, bs, r, rnd(m, n).to(dtype)


def _expected(x, ws, bs, r, dy, act):
    """Outputs and gradients in 64 bits and the bound of each: a list of (name, value, bound)."""
    u = torch.finfo(x.dtype).eps / 2
    step = 2.0 ** -23
    k, n, m = x.shape[1], ws[0].shape[0], x.shape[0]
    x64, dy64 = x.double(), dy.double()
    z, d = [], []
    for w, b in zip(ws, bs):
        b64 = 0.0 if b is None else b.double()
        z.append(x64 @ w.double().t() + b64)
        d.append((k + 1) * step * (x64.abs() @ w.double().abs().t() + (0.0 if b is None else b64.abs())))
    z0 = z[0].clone().requires_grad_(True)
    a = _f(act)(z0)
    slope, = torch.autograd.grad(a.sum(), z0)
    a = a.detach()
    ea = 1.2 * d[0] + 1e-5 * a.abs() + 1e-6
    es = d[0] + 1e-5 + (z[0].abs() <= d[0]).double() * (act == "relu")
    if len(ws) == 2:
        y = a * z[1]
        ey = ea * (z[1].abs() + d[1]) + a.abs() * d[1]
        dzs = [dy64 * z[1] * slope, dy64 * a]
        eds = [dy64.abs() * (es * (z[1].abs() + d[1]) + slope.abs() * d[1]), dy64.abs() * ea]
    else:
        y, ey = a + (0.0 if r is None else r.double()), ea
        dzs, eds = [dy64 * slope], [dy64.abs() * es if act else torch.zeros_like(dy64)]
    out = [("y", y, ey + u * y.abs())]
    rounded = 0.0 if len(ws) == 1 and act is None else u
    eds = [e + rounded * (dz.abs() + e) for e, dz in zip(eds, dzs)]
    dx = sum(dz @ w.double() for dz, w in zip(dzs, ws))
    ex = sum((e + n * len(ws) * step * (dz.abs() + e)) @ w.double().abs() for e, dz, w in zip(eds, dzs, ws))
    out.append(("dx", dx, ex + u * (dx.abs() + ex)))
    for i, (dz, e) in enumerate(zip(dzs, eds)):
        dw, ew = dz.t() @ x64, (e + m * step * (dz.abs() + e)).t() @ x64.abs()
        out.append((f"dw{i}", dw, ew + u * (dw.abs() + ew)))
    for i, (dz, e, b) in enumerate(zip(dzs, eds, bs)):
        if b is not None:
            ub = torch.finfo(b.dtype).eps / 2
            db, eb = dz.sum(0), (e + m * step * (dz.abs() + e)).sum(0)
            out.append((f"db{i}", db, eb + ub * (db.abs() + eb)))
    if r is not None:
        out.append(("dr", dy64, torch.zeros_like(dy64)))
    return out


def _check(got, expected, dtype, what=""):
    u = torch.finfo(dtype).eps / 2
    assert len(got) == len(expected)
    for t, (name, ref, bound) in zip(got, expected):
        assert t.shape == ref.shape, (what, name)
        err = (t.double() - ref).abs()
        tiny = torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps  # results below the normal range
        worst = (err - bound - tiny).max().item() if err.numel() else 0.0
        assert worst <= 0, f"{what} {name}: {worst:.3e} beyond its bound, error {err.max().item():.3e}"
        if err.numel() >= 64:
            rel = (err.norm() / ref.norm().clamp_min(1e-30)).item()
            assert rel <= 2 * u + 1e-5, f"{what} {name}: 2-norm {rel:.3e}"


def _run(x, ws, bs, r, dy, act):
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    leaves = [t.detach().requires_grad_(True) for t in (x, *ws, *[b for b in bs if b is not None], *([] if r is None else [r]))]
    it = iter(leaves)
    xl, wl = next(it), [next(it) for _ in ws]
    bl = [None if b is None else next(it) for b in bs]
    rl = None if r is None else next(it)
    if len(ws) == 2:
        y = fused_ops.gated_linear(xl, *wl, *bl, act=act)
    else:
        y = fused_ops.linear(xl, wl[0], bl[0], act=act, residual=rl)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_and_gradients(m, k, n, dtype):
    for i, act in enumerate(ACTS):
        bias, residual = (m + i) % 3 != 0, (m + i) % 2 == 0
        x, ws, bs, r, dy = _inputs(m, k, n, dtype, 1, bias, residual, seed=i)
        _check(_run(x, ws, bs, r, dy, act), _expected(x, ws, bs, r, dy, act), dtype, f"{act}")


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_gated_linear_and_gradients(m, k, n, dtype):
    for i, act in enumerate(ACTS):
        x, ws, bs, _, dy = _inputs(m, k, n, dtype, 2, (m + i) % 3 != 0, False, seed=20 + i)
        _check(_run(x, ws, bs, None, dy, act), _expected(x, ws, bs, None, dy, act), dtype, f"{act}")


@pytest.fixture
def tuned():
    from proteusai_b200 import _lib
    yield _lib.tune
    _lib.tune_reset()


# Every kernel and shape at sizes that cross its borders, whichever the library would have chosen: a tile, less than one, several.
VARIANTS = [("tile", w, s) for w in (16, 64, 128, 256) for s in (1, 8)] + [("pair", 128, 1), ("pair", 256, 1), ("pair", 256, 3)]


@pytest.mark.parametrize("kernel,width,splits", VARIANTS)
@pytest.mark.parametrize("m,k,n", [(5, 40, 24), (256, 64, 256), (333, 321, 263), (700, 520, 640)])
def test_kernel_variants(tuned, kernel, width, splits, m, k, n):
    tuned(dense_kernel=1 if kernel == "tile" else 2, dense_width=width, dense_splits=splits)
    for dtype in DTYPES:
        for act, residual in ((None, True), ("gelu", False), ("silu", True)):
            x, ws, bs, r, dy = _inputs(m, k, n, dtype, 1, True, residual, seed=3)
            _check(_run(x, ws, bs, r, dy, act), _expected(x, ws, bs, r, dy, act), dtype, f"{act}")
        x, ws, bs, _, dy = _inputs(m, k, n, dtype, 2, True, False, seed=4)
        _check(_run(x, ws, bs, None, dy, "gelu"), _expected(x, ws, bs, None, dy, "gelu"), dtype, "gated")

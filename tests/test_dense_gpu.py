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


def test_many_tiles_per_pair(tuned):
    """More tiles than pairs of SMs: the persistent kernel's second and later rounds, both accumulators, both staging buffers."""
    for width in (128, 256):
        tuned(dense_kernel=2, dense_width=width)
        for act, residual, dtype in (("gelu", True, torch.bfloat16), (None, True, torch.float16), ("silu", False, torch.bfloat16)):
            x, ws, bs, r, dy = _inputs(9000, 72, 1160, dtype, 1, True, residual, seed=5)
            _check(_run(x, ws, bs, r, dy, act), _expected(x, ws, bs, r, dy, act), dtype, f"{width} {act}")
        x, ws, bs, _, dy = _inputs(9000, 72, 1160, torch.bfloat16, 2, False, seed=6)
        _check(_run(x, ws, bs, None, dy, "silu"), _expected(x, ws, bs, None, dy, "silu"), torch.bfloat16, "gated")


@pytest.mark.parametrize("m", [1, 5, 40, 700])
def test_strides_and_alignments(m):
    """Slices of wider buffers at odd offsets, transposed weights, expanded and strided gradients and residuals, three and one axes."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    k, n = 136, 72
    x, ws, bs, r, dy = _inputs(m, k, n, torch.bfloat16, 2, True, True, seed=7)
    want1, want2 = _expected(x, ws[:1], bs[:1], r, dy, "gelu"), _expected(x, ws, bs, None, dy, "silu")

    def inside(t, lead, tail):
        wide = torch.full((t.shape[0], t.shape[1] + lead + tail), float("nan"), dtype=t.dtype, device=t.device)
        wide[:, lead:lead + t.shape[1]] = t
        return wide[:, lead:lead + t.shape[1]]

    forms = [lambda t: inside(t, 3, 2), lambda t: inside(t, 8, 0), lambda t: inside(t, 0, 5), lambda t: t.t().contiguous().t()]
    for form in forms:
        got = _run(form(x), [form(w) for w in ws[:1]], bs[:1], form(r), form(dy), "gelu")
        _check(got, want1, torch.bfloat16, "linear")
        _check(_run(form(x), [form(w) for w in ws], bs, None, form(dy), "silu"), want2, torch.bfloat16, "gated")
    bias = torch.stack([bs[0], bs[1]], 1)[:, 0]  # every other element
    assert torch.equal(fused_ops.linear(x, ws[0], bias), fused_ops.linear(x, ws[0], bs[0]))
    # a gradient broadcast from one row, a residual broadcast to all rows: its gradient is the sum over them
    xl, rl = x.clone().requires_grad_(True), r[:1].clone().requires_grad_(True)
    y = fused_ops.linear(xl, ws[0], bs[0], act="gelu", residual=rl.expand(m, n))
    gx, gr = torch.autograd.grad(y, (xl, rl), dy[:1].expand(m, n))
    want = _expected(x, ws[:1], bs[:1], r[:1].expand(m, n).contiguous(), dy[:1].expand(m, n).contiguous(), "gelu")
    _check([y.detach(), gx], want[:2], torch.bfloat16, "broadcast")
    assert torch.allclose(gr.float(), (dy[:1].double() * m).float(), rtol=2.0 ** -7)
    # leading axes
    x3 = x.view(1, m, k).expand(2, m, k)
    assert torch.equal(fused_ops.linear(x3, ws[0], act="relu")[1], fused_ops.linear(torch.cat([x, x]), ws[0], act="relu")[m:])
    assert fused_ops.gated_linear(x[0], *ws).shape == (n,)
    assert fused_ops.linear(x.view(m, 1, k), ws[0], residual=r.view(m, 1, n)).shape == (m, 1, n)


def test_no_rows():
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x = torch.empty(0, 3, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, u = (torch.randn(8, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    b = torch.zeros(8, device="cuda", requires_grad=True)
    y = fused_ops.linear(x, w, b, act="gelu")
    assert y.shape == (0, 3, 8)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert gx.shape == x.shape and not gw.any() and not gb.any() and gb.dtype == torch.float32
    h = fused_ops.gated_linear(x, w, u, b, b)
    assert h.shape == (0, 3, 8) and not any(g.any() for g in torch.autograd.grad(h, (w, u, b), torch.empty_like(h)))


def test_only_the_gradients_asked_for():
    """Every subset of the inputs, each gradient the same bits as with all of them."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x, ws, bs, r, dy = _inputs(130, 96, 80, torch.bfloat16, 2, True, True, seed=8)
    for act in (None, "silu"):
        full = _run(x, ws[:1], bs[:1], r, dy, act)[1:]
        gfull = _run(x, ws, bs, None, dy, act)[1:]
        for mask in range(1, 16):
            ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, ws[0], bs[0], r))]
            y = fused_ops.linear(ts[0], ts[1], ts[2], act=act, residual=ts[3])
            want = [i for i in range(4) if mask >> i & 1]
            for i, g in zip(want, torch.autograd.grad(y, [ts[i] for i in want], dy)):
                assert torch.equal(g, full[i]), (act, mask, i)
        for mask in range(1, 32):
            ts = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, *ws, *bs))]
            h = fused_ops.gated_linear(*ts, act=act)
            want = [i for i in range(5) if mask >> i & 1]
            for i, g in zip(want, torch.autograd.grad(h, [ts[i] for i in want], dy)):
                assert torch.equal(g, gfull[i]), (act, mask, i)
    # biases on one side only, and none
    for b0, b1 in ((bs[0], None), (None, bs[1])):
        leaves = [t.clone().requires_grad_(True) for t in (x, *ws, b0 if b0 is not None else b1)]
        h = fused_ops.gated_linear(*leaves[:3], *((leaves[3], None) if b0 is not None else (None, leaves[3])), act="silu")
        zero = torch.zeros_like(bs[0])
        full = _run(x, ws, [b0 if b0 is not None else zero, b1 if b1 is not None else zero], None, dy, "silu")
        got = [h.detach(), *torch.autograd.grad(h, leaves, dy)]
        for g, f in zip(got, (full[0], *full[1:4], full[4] if b0 is not None else full[5])):
            assert torch.equal(g, f)


def test_inference_and_training_give_the_same_output_and_repeat():
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    for m, k, n in ((1, 512, 256), (7, 100, 64), (130, 96, 80), (5000, 512, 1024)):
        x, ws, bs, r, dy = _inputs(m, k, n, torch.bfloat16, 2, True, True, seed=9)
        first, again = _run(x, ws[:1], bs[:1], r, dy, "gelu"), _run(x, ws[:1], bs[:1], r, dy, "gelu")
        gfirst, gagain = _run(x, ws, bs, None, dy, "gelu"), _run(x, ws, bs, None, dy, "gelu")
        assert all(torch.equal(a, b) for a, b in zip(first + gfirst, again + gagain))
        with torch.no_grad():
            assert torch.equal(first[0], fused_ops.linear(x, ws[0], bs[0], act="gelu", residual=r))
            assert torch.equal(gfirst[0], fused_ops.gated_linear(x, *ws, *bs, act="gelu"))


def test_fp32_biases_and_shared_tensors():
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x, ws, bs, r, dy = _inputs(200, 64, 64, torch.float16, 2, True, False, seed=10, bias_dtype=torch.float32)
    _check(_run(x, ws[:1], bs[:1], None, dy, "silu"), _expected(x, ws[:1], bs[:1], None, dy, "silu"), torch.float16, "fp32 bias")
    _check(_run(x, ws, bs, None, dy, "gelu"), _expected(x, ws, bs, None, dy, "gelu"), torch.float16, "fp32 biases")
    # one tensor as both weights; x as its own residual
    w = ws[0].clone().requires_grad_(True)
    h = fused_ops.gated_linear(x, w, w, act=None)
    gw, = torch.autograd.grad(h, w, dy)
    z = x.double() @ ws[0].double().t()
    ref = (2 * dy.double() * z).t() @ x.double()
    u = torch.finfo(torch.float16).eps / 2
    assert ((h.double() - z * z).norm() / (z * z).norm()).item() <= u + 1e-5
    assert ((gw.double() - ref).norm() / ref.norm()).item() <= 3 * u  # two gradients, each rounded, and their sum
    xl = x.clone().requires_grad_(True)
    y = fused_ops.linear(xl, ws[0], residual=xl)
    gx, = torch.autograd.grad(y, xl, dy)
    ref = dy.double() @ ws[0].double() + dy.double()
    assert ((gx.double() - ref).norm() / ref.norm()).item() <= 3 * u


def test_refusals():
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    bf = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)
    x, w = bf(4, 16), bf(8, 16)
    for error, f in ((TypeError, lambda: fused_ops.linear(x.float(), w.float())), (TypeError, lambda: fused_ops.linear(x, w.half())),
                     (TypeError, lambda: fused_ops.linear(x, w, bf(8).half())), (TypeError, lambda: fused_ops.linear(x, w, residual=bf(4, 8).float())),
                     (TypeError, lambda: fused_ops.gated_linear(x, w, w, bf(8), bf(8).float())),
                     (TypeError, lambda: fused_ops.linear(x.double(), w)),
                     (ValueError, lambda: fused_ops.linear(x, bf(8, 15))), (ValueError, lambda: fused_ops.linear(x, bf(16))),
                     (ValueError, lambda: fused_ops.linear(x, w, bf(7))), (ValueError, lambda: fused_ops.linear(x, w, bf(8, 1))),
                     (ValueError, lambda: fused_ops.linear(x, w, residual=bf(8))), (ValueError, lambda: fused_ops.linear(x, w, residual=bf(3, 8))),
                     (ValueError, lambda: fused_ops.linear(x, w, residual=bf(4, 16))), (ValueError, lambda: fused_ops.gated_linear(x, w, bf(9, 16))),
                     (ValueError, lambda: fused_ops.linear(bf(4, 0), bf(8, 0))), (ValueError, lambda: fused_ops.linear(x, bf(0, 16))),
                     (RuntimeError, lambda: fused_ops.linear(x, w.cpu())), (RuntimeError, lambda: fused_ops.linear(x, w, residual=bf(4, 8).cpu())),
                     (RuntimeError, lambda: fused_ops.gated_linear(x.cpu(), w, w))):
        with pytest.raises(error):
            f()
    xl = x.clone().requires_grad_(True)
    y = fused_ops.linear(xl, w, act="gelu")
    with pytest.raises(RuntimeError, match="first-order"):
        torch.autograd.grad(y.sum(), xl, create_graph=True)


def test_rows_and_columns_keep_to_themselves():
    """NaN and infinities in a token reach its row alone, in a row of the weights its column alone; rows of a gradient that are zero add nothing."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    for m, k, n in ((3, 64, 40), (100, 72, 136), (3000, 136, 520)):
        x, ws, bs, r, dy = _inputs(m, k, n, torch.bfloat16, 2, True, True, seed=11)
        clean = fused_ops.linear(x, ws[0], bs[0], act="gelu", residual=r), fused_ops.gated_linear(x, *ws, *bs)
        xb, wb = x.clone(), ws[0].clone()
        xb[1, 5], xb[2, 0] = float("nan"), float("inf")
        wb[7] = float("nan")
        for got, ref in zip((fused_ops.linear(xb, wb, bs[0], act="gelu", residual=r), fused_ops.gated_linear(xb, wb, ws[1], *bs)), clean):
            rows = torch.ones(m, dtype=torch.bool, device="cuda")
            cols = torch.ones(n, dtype=torch.bool, device="cuda")
            rows[1:3], cols[7] = False, False
            assert torch.equal(got[rows][:, cols], ref[rows][:, cols])
            assert got[1].isnan().all() and got[:, 7].isnan().all()
    big = torch.full((2, 16), 3e38, device="cuda", dtype=torch.bfloat16)  # z overflows to +inf and -inf
    eye = torch.zeros(2, 16, device="cuda", dtype=torch.bfloat16)
    eye[0, :2], eye[1, :2] = 1.0, -1.0
    for act, hi, lo in (("gelu", float("inf"), 0.0), ("relu", float("inf"), 0.0), ("sigmoid", 1.0, 0.0), (None, float("inf"), float("-inf"))):
        y = fused_ops.linear(big, eye, act=act).float()
        assert (y[:, 0] == hi).all() and (y[:, 1] == lo).all(), act


def test_wide_ranges_of_saved_pre_activations(tuned):
    """Pre-activations from 1e-30 to 1e30 in one tensor, far outside fp16: the saved form scales them by runs of 16 columns."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    m, k, n = 300, 64, 256
    tuned(dense_kernel=2, dense_width=256)
    x, ws, bs, _, dy = _inputs(m, k, n, torch.bfloat16, 2, False, seed=12)
    scale = (10.0 ** torch.linspace(-15, 15, n // 16, device="cuda")).repeat_interleave(16)[:, None]
    ws = [(w.float() * scale).to(torch.bfloat16) for w in ws]
    got, want = _run(x, ws, [None, None], None, dy, "relu"), _expected(x, ws, [None, None], None, dy, "relu")
    u = torch.finfo(torch.bfloat16).eps / 2
    for g, (name, ref, _) in zip(got, want):
        parts = [(g.double(), ref)] if name == "dx" else list(zip(g.double().split(16, 1 if name == "y" else 0), ref.split(16, 1 if name == "y" else 0)))
        for a, b in parts:  # each run of columns (rows of dw) by its own norm
            assert ((a - b).norm() / b.norm()).item() <= 2 * u, name


def test_more_than_two_to_the_31_elements():
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    m, k, n = 1100000, 64, 2048
    x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(n, k, device="cuda", dtype=torch.bfloat16) * 0.1
    for out, ref in ((fused_ops.linear(x, w, act="silu"), lambda t: torch.nn.functional.silu(t @ w.double().t())),
                     (fused_ops.gated_linear(x, w, w, act="silu"), lambda t: torch.nn.functional.silu(t @ w.double().t()) * (t @ w.double().t()))):
        assert m * n > 2 ** 31
        for at in (0, 1048570, m - 40):
            r = ref(x[at:at + 40].double())
            assert ((out[at:at + 40].double() - r).norm() / r.norm()).item() <= 2.0 ** -8
        del out
    torch.cuda.empty_cache()


def test_neighbours_of_strided_outputs_stay(tuned):
    """The C entry points write their own columns and rows of a wider buffer and nothing else, whichever kernel runs."""
    from proteusai_b200 import _lib
    lib = _lib.lib()
    for kernel, m in ((0, 5), (1, 70), (2, 300)):
        if kernel:
            tuned(dense_kernel=kernel)
        for n, lead, tail in ((72, 8, 8), (72, 3, 5), (65, 1, 6)):
            k = 64
            x, ws, bs, r, dy = _inputs(m, k, n, torch.bfloat16, 1, True, False, seed=13)
            wide = torch.full((m + 2, lead + n + tail), 7.0, device="cuda", dtype=torch.bfloat16)
            at = wide.data_ptr() + 2 * (wide.stride(0) + lead)
            _lib.check(lib.pai_linear_fwd(x.data_ptr(), k, ws[0].data_ptr(), k, bs[0].data_ptr(), 0, None, 0, at, wide.stride(0), None, m, n, k, 3, 0,
                                          torch.cuda.current_stream().cuda_stream), "pai_linear_fwd")
            ref = torch.relu(x.double() @ ws[0].double().t() + bs[0].double())
            got = wide[1:m + 1, lead:lead + n].double()
            assert ((got - ref).norm() / ref.norm()).item() <= 2.0 ** -8
            wide[1:m + 1, lead:lead + n] = 7.0
            assert (wide == 7.0).all(), (kernel, n, lead)


def test_streams_and_concurrent_calls():
    """Calls on two streams at once, and from a stream other than the inputs' own, give what they give alone."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    sets = [_inputs(700 + 300 * i, 256, 264, torch.bfloat16, 2, True, False, seed=14 + i) for i in range(2)]
    alone = [_run(x, ws, bs, None, dy, "gelu") for x, ws, bs, _, dy in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, (x, ws, bs, _, dy) in zip(streams, sets):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_run(x, ws, bs, None, dy, "gelu"))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_steps_replay():
    """Two training steps captured as graphs (their workspaces come from the graphs' pools), replayed in both orders and at once on new inputs."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    sets = [_inputs(m, 136, 264, torch.bfloat16, 2, True, False, seed=16 + m) for m in (3, 900)]
    news = [_inputs(m, 136, 264, torch.bfloat16, 2, True, False, seed=99 + m) for m in (3, 900)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for x, ws, bs, _, dy in sets:
        with torch.cuda.stream(side):
            _run(x, ws, bs, None, dy, "silu")  # (warm-up outside the capture)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(_run(x, ws, bs, None, dy, "silu"))
        graphs.append(g)
    for s, f in zip(sets, news):
        for a, b in zip((s[0], *s[1], *s[2], s[4]), (f[0], *f[1], *f[2], f[4])):
            a.copy_(b)
    expected = [_run(x, ws, bs, None, dy, "silu") for x, ws, bs, _, dy in news]
    torch.cuda.synchronize()
    lanes = [torch.cuda.Stream() for _ in graphs]
    for order in ((0, 1), (1, 0)):
        for i in order:
            with torch.cuda.stream(lanes[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip(expected, outs):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_other_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x, ws, bs, r, dy = _inputs(300, 64, 72, torch.bfloat16, 1, True, True, seed=20)
    there = [t.to("cuda:1") for t in (x, ws[0], bs[0], r)]
    y = fused_ops.linear(*there[:3], act="gelu", residual=there[3])  # the current device is cuda:0
    assert y.device.index == 1 and torch.equal(y.cpu(), fused_ops.linear(x, ws[0], bs[0], act="gelu", residual=r).cpu())


def test_autocast():
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x, ws, bs, r, _ = _inputs(50, 64, 72, torch.float32, 2, True, True, seed=21)
    lo = [t.to(torch.bfloat16) for t in (x, *ws, r)]
    xl = x.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = fused_ops.linear(xl, ws[0], bs[0], act="gelu", residual=r)
        h = fused_ops.gated_linear(x, *ws, *bs)
    assert y.dtype == torch.bfloat16 and torch.equal(y.detach(), fused_ops.linear(lo[0], lo[1], bs[0], act="gelu", residual=lo[3]))
    assert torch.equal(h, fused_ops.gated_linear(lo[0], lo[1], lo[2], *bs))
    gx, = torch.autograd.grad(y.float().sum(), xl)
    assert gx.dtype == torch.float32 and torch.isfinite(gx).all()


def test_gradients_against_differences():
    """Central differences of the operators themselves along random directions, in fp16 with a step that its rounding allows: the output is
    off by u |y| at most, so the quotient by u sum|dy y| / step, and by the step's square for the curvature."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x, ws, bs, r, dy = _inputs(60, 48, 56, torch.float16, 2, True, False, seed=22)
    dy = dy.float()
    u, step = torch.finfo(torch.float16).eps / 2, 2.0 ** -4
    calls = {"linear": (lambda t: fused_ops.linear(t[0], t[1], t[3], act="gelu"), [x, ws[0], None, bs[0]]),
             "gated": (lambda t: fused_ops.gated_linear(t[0], t[1], t[2], t[3], None, act="silu"), [x, ws[0], ws[1], bs[0]])}
    for name, (call, args) in calls.items():
        leaves = [None if t is None else t.clone().requires_grad_(True) for t in args]
        live = [t for t in leaves if t is not None]
        y = call(leaves)
        grads = torch.autograd.grad(y, live, dy.to(torch.float16))
        for t, g in zip(live, grads):
            d = torch.where(torch.rand(t.shape, generator=torch.Generator("cuda").manual_seed(3), device="cuda") < 0.1, 1.0, 0.0).to(torch.float16)
            with torch.no_grad():
                moved = []
                for s in (step, -step):
                    # (t + s d is rounded: the step that was made is the difference of what was given)
                    given = [None if a is None else (a + s * d if a is t else a) for a in leaves]
                    moved.append((call(given).double(), next(b for a, b in zip(leaves, given) if a is t).double()))
                made = (moved[0][1] - moved[1][1]) / (2 * step)
            quotient = ((moved[0][0] - moved[1][0]) * dy.double()).sum() / (2 * step)
            slope = (g.double() * made).sum()
            noise = u * (dy.double().abs() * y.double().abs()).sum() / step / math.sqrt(y.numel()) * 8   # (independent roundings)
            curve = 0.2 * step ** 2 * g.double().abs().sum() + 3 * u * (g.double().abs() * made.abs()).sum()
            assert abs(quotient - slope).item() <= (noise + curve).item(), (name, t.shape, quotient.item(), slope.item())


# ---- the block and the model that use them -----------------------------------------------------------------------------
def _block_reference(block, x, residual):
    """The feed-forward block in 64 bits on the weights it has."""
    f = lambda lin, t: t @ lin.weight.double().t() + (0.0 if lin.bias is None else lin.bias.double())
    from proteusai_b200.utils.model_utils.base_modules.base_modules import GatedMLP
    if isinstance(block, GatedMLP):
        h = _f(block.act_name)(f(block.gate_proj, x)) * f(block.up_proj, x)
    else:
        h = _f(block.act_name)(f(block.in_proj, x))
        for lin in block.hidden_proj:
            h = _f(block.act_name)(f(lin, h))
    return f(block.out_proj, h) + residual


@pytest.mark.parametrize("dtype", DTYPES, ids=("bf16", "fp16"))
@pytest.mark.parametrize("kind", ("fused", "gated"))
def test_block_forward_and_backward(kind, dtype):
    """The whole block as the encoder calls it: hidden layer, second product with the residual, gradients of all parameters.  Against 64 bits on the
    same weights: a rounding (u) each of the hidden layer, its gradient, its pre-activations' gradient and the result stack to below 4 u."""
    from proteusai_b200.utils.model_utils.base_modules.base_modules import MLP, GatedMLP
    torch.manual_seed(23)
    u = torch.finfo(dtype).eps / 2
    for shape in ((1, 128), (3, 41, 128), (2, 700, 128)):
        block = (MLP(128, 128, 320, 1, 0.0, fused=True) if kind == "fused" else GatedMLP(128, 128, 320, dropout=0.0)).cuda().to(dtype)
        x = torch.randn(*shape, device="cuda").to(dtype).requires_grad_(True)
        dy = torch.randn(*shape, device="cuda").to(dtype)
        y = block(x, residual=x)
        params = list(block.parameters())
        grads = torch.autograd.grad(y, [x, *params], dy)
        ref = type(block)(128, 128, 320, **({"hidden_layers": 1} if kind == "fused" else {}), dropout=0.0).cuda().double()
        ref.load_state_dict({k: v.double() for k, v in block.state_dict().items()})
        xr = x.detach().double().requires_grad_(True)
        yr = _block_reference(ref, xr, xr)
        want = torch.autograd.grad(yr, [xr, *ref.parameters()], dy.double())
        assert ((y.double() - yr).norm() / yr.norm()).item() <= 2 * u
        for (name, _), g, w in zip([("x", x), *block.named_parameters()], grads, want):
            assert ((g.double() - w).norm() / w.norm()).item() <= 4 * u, (shape, name)


@pytest.mark.parametrize("ffn", ("fused", "gated"))
def test_encoder_model_inference_and_training(ffn):
    """The encoder model with the products of this library in its feed-forward blocks: bf16 inference beside the oracle composition, and a
    training step with a gradient for every parameter."""
    from oracle import chains
    from oracle.encoder_ref import encoder_forward_ref
    from proteusai_b200.utils.model_utils.base_modules.encoder import ProteusEncoderModel
    torch.manual_seed(24)
    model = ProteusEncoderModel(d_model=128, heads=2, layers=2, d_hidden=256, ffn=ffn).cuda().eval()
    c, m = chains.chain_batch([200, 64, 131], 200, seed=25)
    c, m = torch.from_numpy(c), torch.from_numpy(m)
    tokens = torch.randint(0, 33, (3, 200), generator=torch.Generator().manual_seed(26))
    with torch.no_grad():
        ref = None
        if ffn == "fused":
            ref = encoder_forward_ref(model, tokens, c, m)
        else:
            full = model(tokens.cuda(), c.cuda(), m.cuda()).float().cpu()  # fp32: the plain operators
        model.to_compute_dtype_(torch.bfloat16)
        logits = model(tokens.cuda(), c.cuda(), m.cuda()).float().cpu()
    ref = full if ref is None else ref
    assert (logits[~m] - ref[~m]).abs().max().item() < 1e-1
    model.train()
    out = model(tokens.cuda(), c.cuda(), m.cuda())
    torch.nn.functional.cross_entropy(out[~m.cuda()].float(), tokens[~m].cuda() % 20).backward()
    for name, p in ((n, p) for n, p in model.named_parameters() if p.requires_grad):
        if "beta_weights" not in name:
            assert p.grad is not None and torch.isfinite(p.grad).all(), name


@pytest.mark.parametrize("m,k,n", [(65536, 64, 64), (40000, 512, 20), (20001, 72, 136)])
def test_long_reductions_in_many_splits(m, k, n):
    """Few tiles of weight gradient under a long batch: the reduction is split over many pairs of SMs and joined in order, the same bits every time."""
    for mats, act in ((1, "silu"), (1, None), (2, "gelu")):
        x, ws, bs, _, dy = _inputs(m, k, n, torch.bfloat16, mats, True, False, seed=30)
        got, again = _run(x, ws, bs, None, dy, act), _run(x, ws, bs, None, dy, act)
        _check(got, _expected(x, ws, bs, None, dy, act), torch.bfloat16, f"{mats} {act}")
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("kernel", (1, 2))
def test_an_infinity_beside_finite_pre_activations(tuned, kernel):
    """A pre-activation that overflows does not cost its neighbours in the same saved run their bits: their gradients are as without it."""
    m, k, n = 256, 64, 256
    tuned(dense_kernel=kernel)
    x, ws, _, _, dy = _inputs(m, k, n, torch.bfloat16, 2, False, seed=31)
    x[:, 0] = 1e38
    ws = [w.clone() for w in ws]
    for w in ws:
        w[:, 0] = 0.0
    clean = _run(x, ws, [None, None], None, dy, "relu")
    ws[1][5, 0] = 1e30                               # u is +inf in column 5, z is as before
    got = _run(x, ws, [None, None], None, dy, "relu")
    others = torch.arange(n, device="cuda") != 5
    assert torch.equal(got[0][:, others], clean[0][:, others])
    for a, b in zip(got[2:], clean[2:]):
        assert torch.equal(a[others], b[others])


def test_a_backward_pass_under_another_tuning_is_refused(tuned):
    """The saved pre-activations have the form of the kernel that wrote them."""
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x, ws, _, _, dy = _inputs(512, 64, 256, torch.bfloat16, 2, False, seed=32)
    for gated in (False, True):
        tuned(dense_kernel=2)
        xl = x.clone().requires_grad_(True)
        y = fused_ops.gated_linear(xl, *ws) if gated else fused_ops.linear(xl, ws[0], act="silu")
        tuned(dense_kernel=1)
        with pytest.raises(RuntimeError, match="tuning changed"):
            y.backward(dy)
        assert xl.grad is None


def test_capture_beside_a_graph_of_the_default_stream_is_refused():
    from proteusai_b200.utils.model_utils.base_modules import fused_ops
    x, ws, _, _, dy = _inputs(40, 64, 72, torch.bfloat16, 1, False, seed=33)
    w = ws[0].clone().requires_grad_(True)
    alive = fused_ops.linear(x, w)                   # keeps w's accumulator, which belongs to the default stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="being captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            fused_ops.linear(x, w).backward(dy)
    assert w.grad is None
    alive.backward(dy)                               # neither graph nor device came to harm
    ref = dy.double().t() @ x.double()
    assert ((w.grad.double() - ref).norm() / ref.norm()).item() <= 2 * 2.0 ** -8
    del alive
    w.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        fused_ops.linear(x, w).backward(dy)
    g.replay()
    torch.cuda.synchronize()
    assert ((w.grad.double() - ref).norm() / ref.norm()).item() <= 2 * 2.0 ** -8


def test_waits_never_ran_out():
    from proteusai_b200 import _lib
    _lib.device_status()

"""RMS norm with the residual's addition, its gradient and its 8-bit output against the
formulas in 64 bits.

Tolerances: a result rounded to type t is off by at most eps(t) / 2 of itself; the
fp32 statistics behind it are sums of at most 16 terms a lane and a tree over the
lanes, under 64 roundings of 2^-24 each, and a handful of products: 2^-17 of the sum
of the terms' magnitudes covers them.  Values below the type's normal range: half its
smallest step."""
import pytest
import torch

from oracle import fa2_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
STAT = 2.0 ** -17


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def within(got, ref, bound, what):
    got, ref = got.double(), ref.double()
    assert torch.isfinite(got).all(), what
    worst = ((got - ref).abs() - bound).max().item()
    assert worst <= 0, f"{what}: over its bound by {worst:.3e} (largest error {(got - ref).abs().max().item():.3e})"


def keep_of(seed, rows, cols, p):
    import numpy as np
    r, c = np.arange(rows)[:, None], np.arange(cols)[None, :]
    return torch.from_numpy(orc.dropout_keep(seed, r, c, 0, p)).to(DEV)


def data(rows, cols, xt, rt, wt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g).to(xt).to(DEV)
    r = (torch.randn(rows, cols, generator=g) * 3).to(rt).to(DEV)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(wt).to(DEV)
    dy = torch.randn(rows, cols, generator=g).to(xt).to(DEV)
    dh = torch.randn(rows, cols, generator=g).to(rt).to(DEV)
    return x, r, w, dy, dh


def check_all(fa, x, r, w, dy, dh, eps, p=0.0, seed=7, rows_of=None):
    cols = x.shape[-1]
    rows = x.numel() // cols
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    if r is not None:
        r = r.requires_grad_(True)
        y, h = fa.add_rms_norm(x, r, w, eps=eps, dropout_p=p, seed=seed)
        gx, gr, gw = torch.autograd.grad((y, h), (x, r, w), (dy, dh))
    else:
        y = fa.rms_norm(x, w, eps=eps)
        gx, gw = torch.autograd.grad(y, (x, w), dy)
    f = 1.0
    if p > 0:
        f = keep_of(seed, rows, cols, p).view(x.shape).double() / (1.0 - p)
    xd, wd = x.detach().double(), w.detach().double()
    if r is not None:
        href = r.detach().double() + xd * f
        mag = r.detach().double().abs() + (xd * f).abs()
        within(h, href, half_step(h.dtype) * href.abs() + 2.0 ** -23 * mag + least(h.dtype), "h")
        a = h.detach().double()
    else:
        a = xd
    s = 1.0 / torch.sqrt((a * a).mean(-1, keepdim=True) + eps)
    n = a * s
    yref = n * wd
    within(y, yref, (half_step(y.dtype) + STAT) * yref.abs() + least(y.dtype), "y")
    gwd = dy.double() * wd
    dot = (gwd * n).mean(-1, keepdim=True)
    total = s * (gwd - n * dot)
    bound = STAT * s * (gwd.abs() + n.abs() * (dot.abs() + (gwd * n).abs().mean(-1, keepdim=True)))
    if r is not None:
        total = total + dh.double()
        bound = bound + 2.0 ** -23 * dh.double().abs()
        within(gr, total, half_step(gr.dtype) * total.abs() + bound + least(gr.dtype), "dresidual")
    within(gx, total * f, half_step(gx.dtype) * (total * f).abs() + bound * f + least(gx.dtype), "dx")
    terms = (dy.double() * n).reshape(rows, cols)
    # rows are added one after the other in at most 512 workgroups' parts, and those in order
    order = (rows + 512) * 2.0 ** -24
    within(gw, terms.sum(0), half_step(gw.dtype) * terms.sum(0).abs() + (STAT + order) * terms.abs().sum(0) + least(gw.dtype), "dw")


@pytest.mark.parametrize("cols", [1, 2, 3, 4, 63, 64, 65, 255, 256, 257, 512, 768, 771, 1000, 1024, 1025, 2048, 2049, 4096,
                                  4100, 6000, 8191, 8192])
@pytest.mark.parametrize("xt,rt", [(F16, F32), (BF16, BF16)])
def test_widths(fa, cols, xt, rt):
    check_all(fa, *data(5, cols, xt, rt, rt, cols), eps=1e-6, p=0.1)


@pytest.mark.parametrize("xt,rt,wt", [(F16, F16, F16), (F16, F16, F32), (F16, F32, F16), (BF16, BF16, F32), (BF16, F32, BF16),
                                      (F32, F32, F32), (F32, F32, F16)])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_types(fa, xt, rt, wt, p):
    check_all(fa, *data(33, 768, xt, rt, wt, 3), eps=1e-5, p=p)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 2047, 2048, 2049, 4099])
def test_rows(fa, rows):
    check_all(fa, *data(rows, 100, F16, F32, F32, rows), eps=1e-6, p=0.1)
    x, _, w, dy, _ = data(rows, 100, BF16, F32, F32, rows)
    check_all(fa, x, None, w, dy, None, eps=1e-6)


@pytest.mark.parametrize("out", [F16, BF16, F32])
def test_fp32_rows_to_other_types(fa, out):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(7, 300, generator=g).to(DEV).requires_grad_(True)
    w = torch.rand(300, generator=g).to(DEV)
    dy = torch.randn(7, 300, generator=g).to(out).to(DEV)
    y = fa.rms_norm(x, w, out_dtype=out)
    assert y.dtype == out
    (gx,) = torch.autograd.grad(y, x, dy)
    xd = x.detach().double().requires_grad_(True)
    ref = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + 1e-6) * w.double()
    (rx,) = torch.autograd.grad(ref, xd, dy.double())
    within(y, ref.detach(), (half_step(out) + STAT) * ref.detach().abs() + least(out), "y")
    within(gx, rx, STAT * 8 * dy.double().abs().amax(-1, keepdim=True), "dx")


def test_layouts_and_shapes(fa):
    """Leading dimensions, rows with a stride, a transposed batch, an expanded residual, an offset base."""
    x, r, w, dy, dh = data(24, 128, F16, F32, F32, 5)
    y0, h0 = fa.add_rms_norm(x, r, w)
    for view in (lambda t: t.view(2, 3, 4, 128), lambda t: torch.cat([t, t], 1)[:, :128],
                 lambda t: t.view(4, 6, 128).transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(24, 128)):
        y, h = fa.add_rms_norm(view(x), view(r), w)
        assert y.shape == view(x).shape and torch.equal(y.reshape(24, 128), y0) and torch.equal(h.reshape(24, 128), h0)
    one = r[:1].clone().requires_grad_(True)
    y, h = fa.add_rms_norm(x, one.expand(24, 128), w)
    (g,) = torch.autograd.grad(h.sum(), one)
    assert g.shape == one.shape and torch.allclose(g, torch.full_like(g, 24.0))
    v = x[0].clone().requires_grad_(True)
    assert torch.equal(fa.rms_norm(v, w), fa.rms_norm(x, w)[0])
    e = fa.rms_norm(x[:0], w)
    assert e.shape == (0, 128)
    w0 = w.clone().requires_grad_(True)
    fa.rms_norm(x[:0], w0).sum().backward()
    assert torch.equal(w0.grad, torch.zeros_like(w0))


def test_partial_gradients(fa):
    """Only y, only h, or only some inputs need a gradient."""
    x, r, w, dy, dh = data(9, 130, BF16, F32, F32, 8)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = fa.add_rms_norm(*leaves, dropout_p=0.2, seed=5)
    both = torch.autograd.grad((y, h), leaves, (dy, dh), retain_graph=True)
    only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    only_h = torch.autograd.grad(h, leaves, dh, allow_unused=True, retain_graph=True)
    assert torch.equal(only_h[1], dh) and not only_h[2].any()
    assert torch.equal(only_h[0], fa.dropout(dh, 0.2, seed=5).to(BF16))
    assert torch.allclose(both[1], only_y[1] + dh, atol=1e-6) and torch.equal(both[2], only_y[2])
    for i in range(3):
        some = [t.clone().requires_grad_(i == k) for k, t in enumerate((x, r, w))]
        y, h = fa.add_rms_norm(*some, dropout_p=0.2, seed=5)
        (g,) = torch.autograd.grad((y, h) if i < 2 else y, some[i], (dy, dh) if i < 2 else dy)
        assert torch.equal(g, both[i]), i
    with pytest.raises(RuntimeError):   # no second derivative
        y, h = fa.add_rms_norm(*leaves)
        g = torch.autograd.grad(y, leaves[0], dy, create_graph=True)[0]
        g.float().sum().backward()


def test_gradient_against_differences(fa):
    """fp32: the central difference of sum(dy * y) + sum(dh * h) along a direction v.  Its own
    error is eps^2 / 6 of the third derivative (under 2^-8 of the first here, eps = 1/16 with |v| << |h|) and the
    forwards' rounding over eps."""
    x, r, w, dy, dh = (t.double().float() for t in data(3, 64, F32, F32, F32, 11))
    g = torch.Generator().manual_seed(2)
    vx, vr, vw = (torch.randn(t.shape, generator=g).to(DEV) * 0.1 for t in (x, r, w))
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    grads = torch.autograd.grad(fa.add_rms_norm(*leaves), leaves, (dy, dh))
    slope = sum((a.double() * b.double()).sum() for a, b in zip(grads, (vx, vr, vw)))

    def value(e):
        y, h = fa.add_rms_norm(x + e * vx, r + e * vr, w + e * vw)
        return (y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()

    diff = (value(1 / 16) - value(-1 / 16)) * 8
    assert abs(diff - slope) <= 2.0 ** -8 * abs(slope) + 1e-3, (diff.item(), slope.item())


def test_extreme_values(fa):
    """Rows of zeros, of the smallest and of large values; inf and NaN stay in their row."""
    x = torch.randn(6, 96, generator=torch.Generator().manual_seed(4)).to(DEV)
    x[1] = 0
    x[2] *= 1e-20
    x[3] *= 1e15
    x[4, 7] = float("inf")
    x[5, 9] = float("nan")
    w = torch.ones(96, device=DEV)
    y = fa.rms_norm(x, w)
    xd = x[:4].double()
    ref = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + 1e-6)
    within(y[:4], ref, STAT * ref.abs(), "y")
    assert torch.isnan(y[4, 7]) and torch.isnan(y[5]).all()
    q, s = fa.rms_norm_fp8(x, w)
    assert torch.isfinite(s[:4]).all() and (s[:4] > 0).all() and not q[1].float().any()
    assert torch.isnan(q[5].float()).all() and torch.isnan(s[5]).all()


def e4m3(v):
    e = torch.frexp(v)[1].double() - 1
    step = torch.exp2(torch.clamp_min(e, -6.0) - 3)
    return torch.round(v / step) * step


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 768), (8, 768), (5, 771), (3, 1025), (2, 5000), (1, 8192), (300, 256)])
@pytest.mark.parametrize("xt,rt", [(F16, F16), (BF16, F32), (F32, F32), (F16, None), (F32, None)])
def test_fp8(fa, rows, cols, xt, rt):
    x, r, w, _, _ = data(rows, cols, xt, rt or F32, F32, rows + cols)
    if rt is None:
        q, scale = fa.rms_norm_fp8(x, w)
        a = x.double()
    else:
        q, scale, h = fa.rms_norm_fp8(x, w, residual=r)
        within(h, r.double() + x.double(), half_step(rt) * (r.double() + x.double()).abs() + 2.0 ** -23 * (r.double().abs() + x.double().abs()), "h")
        a = h.double()
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows, 1) and q.shape == x.shape
    y = a / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-6) * w.double()
    ref = y.abs().amax(-1, keepdim=True) / 448
    within(scale, ref, (STAT + 2.0 ** -23) * ref, "scale")
    # half a step of e4m3 (2^-4 of the value, at least 2^-10), of a value that is itself STAT off
    v = y / scale.double()
    within(q.float(), v, 2.0 ** -4 * v.abs() * (1 + STAT) + STAT * v.abs() + 2.0 ** -10, "q")
    assert q.float().abs().amax() <= 448
    # away from the middle between two steps it is the nearest one
    lo, hi = e4m3(v * (1 - STAT)), e4m3(v * (1 + STAT))
    sure = lo == hi
    assert sure.double().mean() > 0.9 or rows * cols < 10
    assert torch.equal(q.double()[sure], lo[sure])


def test_repeats_bit_for_bit(fa):
    x, r, w, dy, dh = data(3000, 257, F16, F32, F32, 9)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    runs = [torch.autograd.grad(fa.add_rms_norm(*leaves, dropout_p=0.1, seed=3), leaves, (dy, dh)) for _ in range(3)]
    for a in runs[1:]:
        assert all(torch.equal(u, v) for u, v in zip(a, runs[0]))


def test_refusals_on_gpu(fa):
    x, r, w, _, _ = data(4, 64, F16, F32, F32, 1)
    for call in (lambda: fa.rms_norm(x.double(), w), lambda: fa.rms_norm(x, w[:5]), lambda: fa.rms_norm(x, w.cpu()),
                 lambda: fa.add_rms_norm(x, r[:2], w), lambda: fa.add_rms_norm(x, r.bfloat16(), w),
                 lambda: fa.add_rms_norm(x, None, w), lambda: fa.add_rms_norm(x, r, w, dropout_p=1.0),
                 lambda: fa.rms_norm(x, w, out_dtype=F32), lambda: fa.rms_norm(x, w, eps=-1.0),
                 lambda: fa.rms_norm(torch.zeros(2, 8193, device=DEV), torch.zeros(8193, device=DEV))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        fa.rms_norm_fp8(x.requires_grad_(True), w)

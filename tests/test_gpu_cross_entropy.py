"""Language model head with cross entropy against the formulas in 64 bits.

Tolerances, element by element.  A logit is a sum of d exact products in fp32: off by
at most (d + 8) 2^-24 of the products' magnitudes, S.  The loss adds the exponential's
and the logarithm's own errors (2^-20 of 1 + |z|, the argument of exp2 being rounded).
P = softmax - onehot inherits the logits' errors (relative, so e = 2 (d + 8) 2^-24 S +
2^-20 (1 + |z|)) and is rounded to the type: half a step of each term of dx and dW;
fp16 values of P under its normal range lose at most 2^-25 of a scale of 2^15.  The sums
over up to V or N terms are fp32: 2^-24 of the magnitudes a term, in blocks of 16: under
2^-13 here.  The result is rounded once more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def data(n, d, V, t, seed, wstd=0.1, ignored=0.0, ignore=-100):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g).to(t).to(DEV)
    w = (torch.randn(V, d, generator=g) * wstd).to(t).to(DEV)
    target = torch.randint(0, V, (n,), generator=g)
    target[torch.rand(n, generator=g) < ignored] = ignore
    return x, w, target.to(DEV)


def run(fa, x, w, target, reduction="mean", g=None, ignore=-100):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = fa.linear_cross_entropy(x, w, target, ignore_index=ignore, reduction=reduction)
    g = torch.ones_like(loss) if g is None else g
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), g))


def check(fa, x, w, target, reduction="mean", g=None, ignore=-100):
    t = x.dtype
    loss, dx, dw = run(fa, x, w, target, reduction, g, ignore)
    xd, wd = x.double().reshape(-1, x.shape[-1]), w.double()
    tg = target.reshape(-1)
    n, d = xd.shape
    rows = (tg != ignore).nonzero()[:, 0]
    z = xd[rows] @ wd.T
    S = (xd[rows].abs() @ wd.abs().T).amax(1)
    zmax = z.abs().amax(1)
    e = 2 * (d + 8) * 2.0 ** -24 * S + 2.0 ** -20 * (1 + zmax)
    lse = torch.logsumexp(z, 1)
    per = lse - z[torch.arange(len(rows), device=DEV), tg[rows]]
    count = len(rows)
    gone = torch.ones((), device=DEV) if g is None else g
    if reduction == "none":
        got = loss.reshape(-1)
        assert not got[tg == ignore].any()
        assert ((got[rows].double() - per).abs() <= e + 2.0 ** -23 * per.abs()).all(), (got[rows] - per).abs().max()
        c = gone.reshape(-1)[rows].double() if gone.numel() > 1 else gone.double().expand(count)
    else:
        ref = per.sum() if reduction == "sum" else per.mean()
        tol = e.sum() if reduction == "sum" else e.mean()
        assert abs(loss.double() - ref) <= tol + 2.0 ** -23 * abs(ref), (loss.item(), ref.item())
        c = (gone.double() / (count if reduction == "mean" else 1)).expand(count)
    prob = torch.softmax(z, 1)
    G = prob.clone()
    G[torch.arange(count, device=DEV), tg[rows]] -= 1
    top = c.abs().max() if count else torch.zeros((), dtype=torch.float64, device=DEV)
    # error of an element of c P: relative (rounding), through the logits, and below fp16's normal range
    eP = c.abs()[:, None] * (half_step(t) * G.abs() + e[:, None] * prob + 2.0 ** -23) + (top * 2.0 ** -40 if t == F16 else 0)
    G = c[:, None] * G
    rdx = torch.zeros(n, d, dtype=torch.float64, device=DEV)
    rdx[rows] = G @ wd
    bdx = torch.zeros_like(rdx)
    bdx[rows] = eP @ wd.abs() + 2.0 ** -13 * (G.abs() @ wd.abs())
    rdw = G.T @ xd[rows]
    bdw = eP.T @ xd[rows].abs() + 2.0 ** -13 * (G.abs().T @ xd[rows].abs())
    for name, got, ref, b in (("dx", dx.reshape(n, d), rdx, bdx), ("dw", dw, rdw, bdw)):
        assert got.dtype == t and torch.isfinite(got).all(), name
        over = ((got.double() - ref).abs() - (half_step(t) * ref.abs() + b + least(t))).max().item()
        assert over <= 0, f"{name}: over its bound by {over:.3e}, largest {(got.double() - ref).abs().max().item():.3e}"
    assert not dx.reshape(n, d)[tg == ignore].any()


@pytest.mark.parametrize("n,d,V", [(1, 64, 2), (1, 8, 1), (2, 64, 127), (3, 128, 128), (5, 64, 129), (63, 192, 255), (64, 64, 256),
                                   (65, 64, 257), (127, 320, 300), (128, 256, 1000), (129, 64, 513), (255, 128, 512),
                                   (256, 512, 777), (257, 768, 1500), (510, 256, 1000), (700, 64, 5003)])
@pytest.mark.parametrize("t", [F16, BF16])
def test_sizes(fa, n, d, V, t):
    check(fa, *data(n, d, V, t, n + V), g=torch.tensor(1024.0 if t == F16 else 1.0, device=DEV))


@pytest.mark.parametrize("d", [1, 3, 7, 8, 63, 65, 72, 100, 127, 771])
@pytest.mark.parametrize("t", [F16, BF16])
def test_hidden_sizes_that_no_tile_divides(fa, d, t):
    check(fa, *data(70, d, 300, t, d, wstd=0.3), g=torch.tensor(512.0 if t == F16 else 1.0, device=DEV))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("ignored", [0.0, 0.4, 0.97])
def test_reductions_and_ignored(fa, reduction, ignored):
    x, w, target = data(333, 128, 600, F16, 5, ignored=ignored)
    target[7] = 3
    g = None
    if reduction == "none":   # gradients of very different sizes, zeros among them
        g = torch.randn(333, generator=torch.Generator().manual_seed(3)).to(DEV)
        g[::5] *= 1e-3
        g[::7] = 0
    elif reduction == "mean":
        g = torch.tensor(333.0, device=DEV)
    check(fa, x, w, target, reduction, g)
    check(fa, x, w, torch.where(target == -100, 5, target), reduction, g, ignore=5)


@pytest.mark.parametrize("wstd", [0.0, 0.01, 1.0, 8.0])
def test_flat_and_peaked(fa, wstd):
    """From uniform logits to rows whose largest logit takes all."""
    x, w, target = data(200, 256, 900, BF16, 6, wstd=wstd)
    check(fa, x, w, target)
    with torch.no_grad():
        target = (x.float() @ w.float().T).argmax(1)   # the model is right
    check(fa, x, w, target)


def test_matches_torch_on_cross_entropy(fa):
    """F.cross_entropy in fp64 on the same numbers, leading dimensions and a shifted view as the decoder makes it."""
    x, w, _ = data(4 * 65, 128, 1000, F16, 8)
    x = x.view(4, 65, 128)
    ids = torch.randint(0, 1000, (4, 65), generator=torch.Generator().manual_seed(1)).to(DEV)
    loss = fa.linear_cross_entropy(x[:, :-1], w, ids[:, 1:])
    ref = torch.nn.functional.cross_entropy((x[:, :-1].double() @ w.double().T).flatten(0, 1), ids[:, 1:].flatten())
    assert abs(loss.item() - ref.item()) < 1e-5
    check(fa, x[:, :-1], w, ids[:, 1:])
    each = fa.linear_cross_entropy(x[:, :-1], w, ids[:, 1:], reduction="none")
    assert each.shape == (4, 64) and abs(each.double().mean() - ref) < 1e-5


def test_nothing_counts(fa):
    x, w, target = data(20, 64, 100, F16, 2)
    target[:] = -100
    loss, dx, dw = run(fa, x, w, target)
    assert math.isnan(loss.item()) and not dx.any() and not dw.any()
    loss, dx, dw = run(fa, x, w, target, "sum")
    assert loss.item() == 0 and not dx.any() and not dw.any()
    loss, dx, dw = run(fa, x, w, target, "none")
    assert not loss.any() and not dx.any() and not dw.any()
    loss, dx, dw = run(fa, x[:0], w, target[:0], "sum")
    assert loss.item() == 0 and dx.shape == (0, 64) and not dw.any()
    assert run(fa, x[:0], w, target[:0], "none")[0].shape == (0,)


def test_garbage_in_ignored_tokens(fa):
    """States of tokens that do not count may hold anything, inf and NaN included."""
    x, w, target = data(300, 128, 500, BF16, 4, ignored=0.3)
    clean = run(fa, x, w, target)
    bad = x.clone()
    rows = (target == -100).nonzero()[:, 0]
    bad[rows[::2]] = float("nan")
    bad[rows[1::2]] = float("inf")
    for a, b in zip(run(fa, bad, w, target), clean):
        assert torch.equal(a, b)


def test_targets_outside_the_vocabulary(fa):
    x, w, target = data(40, 64, 100, F16, 4)
    target[3], target[9] = 100, -1
    each, dx, _ = run(fa, x, w, target, "none", torch.ones(40, device=DEV))
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 9]] = True
    assert torch.isnan(each[bad]).all() and torch.isfinite(each[~bad]).all()
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    assert math.isnan(run(fa, x, w, target)[0].item())


def test_infinite_logits(fa):
    """A vocabulary row that no token can produce (logit -inf), and NaN states of a token that counts."""
    x, w, target = data(30, 64, 200, BF16, 4)
    x = x.abs()
    w[17] = float("-inf")
    target[target == 17] = 18
    loss = fa.linear_cross_entropy(x, w, target, reduction="none")
    z = x.double() @ w.double().T
    assert torch.allclose(loss.double(), torch.nn.functional.cross_entropy(z, target, reduction="none"), atol=1e-5)
    x[5, 3] = float("nan")
    loss = fa.linear_cross_entropy(x, w, target, reduction="none")
    assert torch.isnan(loss[5]) and torch.isfinite(torch.cat([loss[:5], loss[6:]])).all()


def test_layouts(fa):
    x, w, target = data(50, 128, 300, F16, 3)
    ref = run(fa, x, w, target)
    wide = torch.cat([x, x], 1)[:, :128]
    wwide = torch.cat([w, w], 1)[:, :128]
    off = torch.cat([w.flatten()[:1], w.flatten()])[1:].view(300, 128)
    for xx, ww in ((wide, w), (x, wwide), (x, off), (x, w.t().contiguous().t()), (x.t().contiguous().t(), w)):
        for a, b in zip(run(fa, xx, ww, target), ref):
            assert torch.equal(a, b)
    one = x[:1].clone().requires_grad_(True)   # a broadcast state: its gradient is the sum of all rows'
    (g,) = torch.autograd.grad(fa.linear_cross_entropy(one.expand(50, 128), w, target, reduction="sum"), one)
    rows = run(fa, one.detach().expand(50, 128), w, target, "sum")[1]
    assert torch.allclose(g.float(), rows.float().sum(0, keepdim=True), rtol=1e-2, atol=1e-2)


def test_one_gradient_at_a_time(fa):
    x, w, target = data(150, 64, 400, BF16, 3)
    ref = run(fa, x, w, target)
    (dx,) = torch.autograd.grad(fa.linear_cross_entropy(x.requires_grad_(True), w, target), x)
    (dw,) = torch.autograd.grad(fa.linear_cross_entropy(x.detach(), w.requires_grad_(True), target), w)
    assert torch.equal(dx, ref[1]) and torch.equal(dw, ref[2])
    with torch.no_grad():
        assert torch.equal(fa.linear_cross_entropy(x, w, target), ref[0])


def test_gradient_against_differences(fa):
    """The central difference of the summed loss along a direction that fp16 holds exactly: its error is eps^2 / 6 of the
    third derivative, small beside the slope, and the losses' own rounding over eps."""
    g = torch.Generator().manual_seed(9)
    x = (torch.randint(-64, 64, (40, 64), generator=g).float() / 64).half().to(DEV)
    w = (torch.randint(-64, 64, (90, 64), generator=g).float() / 256).half().to(DEV)
    target = torch.randint(0, 90, (40,), generator=g).to(DEV)
    v = (torch.randint(-1, 2, (40, 64), generator=g).float() / 64).half().to(DEV)
    u = (torch.randint(-1, 2, (90, 64), generator=g).float() / 256).half().to(DEV)
    _, dx, dw = run(fa, x, w, target, "sum")
    slope = (dx.double() * v.double()).sum() + (dw.double() * u.double()).sum()

    def value(s):
        with torch.no_grad():
            return fa.linear_cross_entropy(x + s * v, w + s * u, target, reduction="none").double().sum()

    diff = (value(1) - value(-1)) / 2
    assert abs(diff - slope) < 0.02 * abs(slope) + 1e-2, (diff.item(), slope.item())


def test_autocast_and_types(fa):
    x, w, target = data(60, 128, 200, F16, 3)
    wf = w.float().requires_grad_(True)
    xf = x.float().requires_grad_(True)
    with torch.autocast("cuda", dtype=F16):
        loss = fa.linear_cross_entropy(xf, wf, target)
    loss.backward()
    ref = run(fa, x, w, target)
    assert torch.equal(loss.detach(), ref[0])
    assert wf.grad.dtype == torch.float32 and torch.equal(wf.grad, ref[2].float()) and torch.equal(xf.grad, ref[1].float())
    for call in (lambda: fa.linear_cross_entropy(xf, wf, target), lambda: fa.linear_cross_entropy(x, w.bfloat16(), target),
                 lambda: fa.linear_cross_entropy(x, w[:, :64], target), lambda: fa.linear_cross_entropy(x, w, target[:5]),
                 lambda: fa.linear_cross_entropy(x, w, target.int()), lambda: fa.linear_cross_entropy(x, w, target, reduction="max"),
                 lambda: fa.linear_cross_entropy(x, w[:0], target), lambda: fa.linear_cross_entropy(x, w, target.cpu())):
        with pytest.raises(ValueError):
            call()


def test_many_pieces_and_slices(fa):
    """Enough tokens that the vocabulary goes in several pieces: 16384 tokens leave 4096 columns a piece."""
    x, w, target = data(16300, 64, 9001, F16, 1, ignored=0.1)
    check(fa, x, w, target, g=torch.tensor(65536.0, device=DEV))
    runs = [run(fa, x, w, target) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_large_vocabulary_few_tokens(fa):
    check(fa, *data(9, 128, 131072, BF16, 1))


@pytest.mark.parametrize("n,d,V", [(1, 64, 1), (3, 64, 130), (64, 128, 4000), (65, 768, 16500), (199, 128, 20001), (256, 64, 32000),
                                   (257, 64, 9000), (300, 192, 40000), (1000, 64, 33000), (5000, 64, 3001), (40, 100, 500)])
@pytest.mark.parametrize("t", [F16, BF16])
def test_forward_only(fa, n, d, V, t):
    """Scoring: no gradient, one loss a token, states read where they are or packed; garbage in ignored tokens; a
    strided and a misaligned view."""
    x, w, target = data(n, d, V, t, n, ignored=0.2)
    target[0] = V - 1
    ref = run(fa, x, w, target, "none")[0]
    z = x.double() @ w.double().T
    S = (x.double().abs() @ w.double().abs().T).amax(1)
    e = 2 * (d + 8) * 2.0 ** -24 * S + 2.0 ** -20 * (1 + z.abs().amax(1))
    exact = torch.nn.functional.cross_entropy(z, target, reduction="none")
    bad = x.clone()
    bad[target == -100] = float("nan")
    wide = torch.cat([bad, bad], 1)[:, :d]
    off = torch.cat([bad.flatten()[:1], bad.flatten()])[1:].view(n, d)
    with torch.no_grad():
        for xx in (x, bad, wide, off):
            got = fa.linear_cross_entropy(xx, w, target, reduction="none")
            assert ((got.double() - exact).abs() <= e + 2.0 ** -23 * exact.abs()).all()
            assert not got[target == -100].any()
        total = fa.linear_cross_entropy(bad, w, target, reduction="sum")
        assert abs(total.double() - ref.double().sum()) <= 2 * e.sum()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("t", [F16, BF16])
def test_a_gradient_that_is_not_finite_stays_in_its_row(fa, bad, t):
    x, w, target = data(70, 128, 300, t, 12)
    g = torch.rand(70, generator=torch.Generator().manual_seed(3)).to(DEV) + 0.5
    g[11], g[40] = 0.0, 0.0
    _, dx0, dw0 = run(fa, x, w, target, "none", g)
    g[11], g[40] = bad, 0.0
    _, dx1, dw1 = run(fa, x, w, target, "none", g)
    others = torch.arange(70, device=DEV) != 11
    assert torch.equal(dx1[others], dx0[others]) and not dx1[40].any()
    assert not torch.isfinite(dx1[11]).any() and not torch.isfinite(dw1).any()
    assert torch.isfinite(dw0).all()


@pytest.mark.parametrize("n,d,V", [(1, 8, 5), (40, 72, 300), (130, 200, 4000), (300, 328, 2000), (300, 1160, 700), (700, 56, 1030),
                                   (9000, 136, 20000)])
@pytest.mark.parametrize("t", [F16, BF16])
def test_rows_of_wider_matrices_whose_rest_is_nan(fa, n, d, V, t):
    """Hidden sizes that are multiples of 8 only: tiles end inside the row, and what lies behind it is not taken."""
    x, w, target = data(n, d, V, t, n + d)
    wide_x = torch.full((n, d + 64), float("nan"), dtype=t, device=DEV)
    wide_w = torch.full((V, d + 64), float("nan"), dtype=t, device=DEV)
    wide_x[:, :d], wide_w[:, :d] = x, w
    xs, ws = wide_x[:, :d], wide_w[:, :d]
    with torch.no_grad():
        assert torch.equal(fa.linear_cross_entropy(xs, ws, target, reduction="none"),
                           fa.linear_cross_entropy(x, w, target, reduction="none"))
    check(fa, x, w, target, g=torch.tensor(1024.0 if t == F16 else 1.0, device=DEV))
    a = run(fa, x, w, target)
    xs, ws = xs.detach().requires_grad_(True), ws.detach().requires_grad_(True)
    loss = fa.linear_cross_entropy(xs, ws, target)
    for got, want in zip((loss, *torch.autograd.grad(loss, (xs, ws))), a):
        assert torch.equal(got, want)

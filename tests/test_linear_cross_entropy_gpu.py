"""linear_cross_entropy against the definition in 64 bits, on the GPU.

Tolerances, from the arithmetic (u = 2^-24, r = half a step of the 16-bit type):
* a logit is a sum of `hidden` exact products in fp32: off by at most
  dz = hidden * 2u * sum_k |x_k w_k| (2u per addition, whatever the order);
* lse moves by at most the largest dz; sums of exponentials add fewer than 256
  roundings on any path, exp and log a few ulp;
* numbers under 2^-126, the smallest normal one of fp32 and bf16, may be taken as 0 by
  the exponential, by a matrix instruction or by a product of two: each such step is
  off by less than 2^-126, so d and d times its token's gradient are, besides all else;
* a logit's gradient d is off by |d| (r + its exponent's error) after its rounding to
  16 bits, and the products that use it add one 2u per term and one r at the end.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = 2.0**-24


def _inputs(t, h, v, dtype, seed=0, ignore=0.2, ignore_index=-100):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, h, generator=g).to(dtype).cuda()
    w = (torch.randn(v, h, generator=g) * 2.0 / h**0.5).to(dtype).cuda()
    y = torch.randint(v, (t,), generator=g)
    if ignore:
        y = torch.where(torch.rand(t, generator=g) < ignore, ignore_index, y)
    return x, w, y.cuda()


def _expected(x, w, y, grad, reduction, ignore_index=-100, path=256):
    """Everything in 64 bits, and the tolerances; ``path``: roundings on the way of an
    exponential into its sum."""
    r = torch.finfo(x.dtype).eps / 2
    hidden = x.shape[1]
    used = y != ignore_index
    x, w = torch.where(used[:, None], x.double(), 0.0), w.double()
    z = x @ w.t().contiguous()
    dz = (x.abs() @ w.abs().t().contiguous()).amax(1) * hidden * 2 * U  # per token
    lse = torch.logsumexp(z, 1)
    at = torch.where(used, y, 0)[:, None]
    each = (lse - z.gather(1, at)[:, 0]) * used
    tol = (2 * dz + path * U + 8 * U * (lse.abs() + z.abs().amax(1))) * used
    n = used.sum()
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / n}[reduction]
    t_sum = tol.sum() + each.abs().sum() * (len(y) + 8) * U
    loss_tol = {"none": tol, "sum": t_sum, "mean": t_sum / n}[reduction]
    up = (grad.double() / n if reduction == "mean" else grad.double()) * used
    d = torch.exp(z - lse[:, None])
    d.scatter_add_(1, at, torch.full_like(d[:, :1], -1.0))
    # what p = exp(z - lse) is off by before the 1 is taken off, relative to p
    rel = (dz * 2 + path * U + 16 * U * (lse.abs() + z.abs().amax(1)))[:, None]
    p = torch.exp(z - lse[:, None])
    err = (p * rel + d.abs() * (r + 2 * U)) + 2.0**-126  # of d, rounded
    if x.numel() and r == 2.0**-11:  # smallest fp16 step, under the lift of 2^15
        err = err + 2.0**-40
    v, t = w.shape[0], x.shape[0]
    up_abs = up.abs()[:, None]
    dx = (d * up[:, None]) @ w
    dx_tol = (up_abs * ((err + d.abs() * (v + 8) * 2 * U) @ w.abs())) + dx.abs() * r
    e = err * up_abs + 2.0**-126
    if r == 2.0**-11:
        # d under its lift, and x times a power of two: fp16's smallest step is 2^-24
        e = e + 2.0**-40 * up.abs().max()
        small_x = 2.0**-25 * d.abs().sum(0)[:, None] * up.abs().max()
    dw = (d * up[:, None]).t().contiguous() @ x
    dw_tol = (e + (d * up[:, None]).abs() * (t + 8) * 2 * U).t().contiguous() @ x.abs()
    dw_tol = dw_tol + dw.abs() * r + (small_x if r == 2.0**-11 else 0.0)
    tiny = torch.finfo(torch.float16).smallest_normal * 2.0**-10 if r == 2.0**-11 else 0.0
    return (loss, loss_tol), (dx, dx_tol + tiny), (dw, dw_tol + tiny)


def _run(x, w, y, grad, **kw):
    from offload_adam_amd import linear_cross_entropy

    x = x.detach().requires_grad_(True)
    w = w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, y, **kw)
    dx, dw = torch.autograd.grad(loss, (x, w), grad)
    return loss.detach(), dx, dw


def _close(got, want, what):
    value, tol = want
    off = (got.double() - value).abs() - tol
    assert torch.isfinite(got).all(), what
    assert bool((off <= 0).all()), f"{what}: over by {float(off.max())}"


def _grad_for(reduction, t, seed=5):
    g = torch.Generator().manual_seed(seed)
    shape = (t,) if reduction == "none" else ()
    return (torch.rand(shape, generator=g) * 2 - 0.7).cuda()


SHAPES = [(1, 8, 1), (1, 64, 300), (3, 24, 5), (64, 256, 1024), (65, 72, 257), (128, 128, 128),
          (130, 200, 1000), (257, 64, 513), (17, 2048, 9001), (300, 1000, 3001)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradients(shape, dtype):
    t, h, v = shape
    for reduction in ("mean", "sum", "none"):
        x, w, y = _inputs(t, h, v, dtype, seed=t + h + v)
        if bool((y == -100).all()):
            y[0] = v - 1
        grad = _grad_for(reduction, t)
        got = _run(x, w, y, grad, reduction=reduction)
        for g, want, what in zip(got, _expected(x, w, y, grad, reduction), ("loss", "dx", "dw")):
            _close(g, want, f"{shape} {reduction} {what}")
        assert got[0].dtype == torch.float32 and got[1].dtype == dtype and got[2].dtype == dtype


@pytest.mark.parametrize("shape", [(8192, 64, 20011), (2048, 520, 33000), (6000, 256, 12345)])
def test_many_pieces_and_large_tiles(shape):
    """Several pieces of the vocabulary, the last one short; tiles of both sizes."""
    x, w, y = _inputs(*shape, BF16, seed=1)
    grad = _grad_for("mean", shape[0])
    got = _run(x, w, y, grad)
    for g, want, what in zip(got, _expected(x, w, y, grad, "mean"), ("loss", "dx", "dw")):
        _close(g, want, f"{shape} {what}")


@pytest.mark.parametrize("shape", [(1, 64, 70001), (4, 80, 60001), (9, 8, 33000)])
def test_few_tokens_of_a_large_vocabulary(shape):
    """Hundreds of tiles to join per token, and dx in many slices."""
    x, w, y = _inputs(*shape, BF16, seed=2, ignore=0.0)
    for reduction in ("sum", "none"):
        grad = _grad_for(reduction, shape[0])
        got = _run(x, w, y, grad, reduction=reduction)
        want = _expected(x, w, y, grad, reduction)
        for g, e, what in zip(got, want, ("loss", "dx", "dw")):
            _close(g, e, f"{shape} {reduction} {what}")


def test_more_rows_than_32_bits_address_in_lines():
    """64 lines of the logits' gradient of 13 million rows are over 2^30 bytes.  A lane joins
    13e6 / 128 / 32 pairs, at most 6 roundings each."""
    x, w, y = _inputs(2, 8, 13_000_000, BF16, seed=2, ignore=0.0)
    y[1] = 12_999_999
    grad = _grad_for("none", 2)
    got = _run(x, w, y, grad, reduction="none")
    want = _expected(x, w, y, grad, "none", path=6 * 13_000_000 // 128 // 32)
    for g, e, what in zip(got, want, ("loss", "dx", "dw")):
        _close(g, e, what)


def test_large_logits_and_confident_rows():
    """Logits of some hundreds: exponentials that vanish, probabilities of 1."""
    t, h, v = 70, 64, 700
    x, w, y = _inputs(t, h, v, BF16, seed=3, ignore=0.0)
    x = x * 60
    z = x.double() @ w.double().t().contiguous()
    y = torch.where(torch.arange(t, device="cuda") % 2 == 0, z.argmax(1), y)
    grad = _grad_for("none", t)
    got = _run(x, w, y, grad, reduction="none")
    for g, want, what in zip(got, _expected(x, w, y, grad, "none"), ("loss", "dx", "dw")):
        _close(g, want, what)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_exact_logits_of_thousands(dtype):
    """Logits up to 6000 that fp32 holds exactly, so that all that is left is the exponentials'
    exponents (under 64 in base 2 where they count: 2^-24 of 64 each way, and as much again
    for log2 e), the sum and the logarithm.  First the target far above all others: loss and
    gradients 0 but for two exponentials and a product of 1 +- 2^-23.  Then 16 equal logits at
    the top and the others 1 to 40 below."""
    t, v, h = 130, 300, 16
    g = torch.Generator().manual_seed(11)
    top = torch.randint(33, 96, (t,), generator=g).float()  # times 64: 2112 to 6080
    x = torch.zeros(t, h)
    x[:, 0], x[:, 1] = top, 1.0
    w = torch.zeros(v, h)
    w[:, 0] = 64.0
    for far in (True, False):
        w[:, 1] = -torch.randint(200, 250, (v,), generator=g) if far else \
            -torch.randint(1, 41, (v,), generator=g)
        same = 1 if far else 16
        w[100:100 + same, 1] = 0.0
        y = torch.full((t,), 100)
        a, b = x.to(dtype).cuda(), w.to(dtype).cuda()
        loss, dx, dw = _run(a, b, y.cuda(), torch.ones(t, device="cuda"), reduction="none")
        z = (x.double() @ w.double().t())
        want = torch.logsumexp(z, 1) - z[:, 100]
        tol = 2.0**-16 if not far else 2.0**-21
        assert float((loss.cpu().double() - want).abs().max()) <= tol
        if far:
            assert float(dx[:, 0].abs().max()) <= 2.0**-21 * 64
            assert float(dw[100, 0].abs()) <= 2.0**-21 * float(top.sum())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_ignored_rows_may_hold_anything(dtype):
    t, h, v = 150, 88, 400
    x, w, y = _inputs(t, h, v, dtype, seed=4, ignore_index=7)
    y[::5] = 7
    grad = _grad_for("none", t)
    clean = _run(x, w, y, grad, reduction="none", ignore_index=7)
    dirty = x.clone()
    dirty[::5] = float("nan")
    dirty[5::10] = float("inf")
    for a, b in zip(clean, _run(dirty, w, y, grad, reduction="none", ignore_index=7)):
        assert torch.equal(a, b)
    assert not clean[0][::5].any() and not clean[1][::5].any()


def test_nothing_takes_part():
    x, w, y = _inputs(33, 40, 100, BF16)
    y[:] = -100
    one = torch.ones((), device="cuda")
    loss, dx, dw = _run(x, w, y, one)
    assert torch.isnan(loss) and not dx.any() and not dw.any()
    loss, dx, dw = _run(x, w, y, one, reduction="sum")
    assert loss == 0 and not dx.any() and not dw.any()
    empty = _run(x[:0], w, y[:0], one, reduction="sum")
    assert empty[0] == 0 and empty[1].shape == (0, 40) and not empty[2].any()
    assert torch.isnan(_run(x[:0], w, y[:0], one)[0])
    none = _run(x[:0], w, y[:0], torch.ones(0, device="cuda"), reduction="none")
    assert none[0].shape == (0,)


def test_targets_outside_the_vocabulary_give_nan():
    for bad in (-1, 100, 2**40, -(2**62)):
        x, w, y = _inputs(40, 40, 100, BF16, ignore=0.0)
        y[3] = bad
        loss, dx, dw = _run(x, w, y, torch.ones(40, device="cuda"), reduction="none")
        assert torch.isnan(loss[3]) and torch.isfinite(loss[:3]).all()
        assert torch.isfinite(loss[4:]).all()
        assert torch.isnan(dx[3]).all() and torch.isfinite(dx[4:]).all()
        assert torch.isnan(dw).all()


def test_non_finite_logits_show():
    x, w, y = _inputs(40, 40, 100, BF16, ignore=0.0)
    x[5, 0] = float("nan")
    x[6, 0] = float("inf")
    loss, dx, dw = _run(x, w, y, torch.ones(40, device="cuda"), reduction="none")
    assert torch.isnan(loss[5]) and not torch.isfinite(loss[6])
    assert torch.isfinite(loss[7:]).all() and torch.isfinite(dx[7:]).all()


def test_strides_shapes_and_odd_hidden():
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(6, 11, 96, generator=g).to(BF16).cuda()
    head = torch.randn(50, 128, generator=g).to(BF16).cuda() * 0.1
    y = torch.randint(50, (6, 11), generator=g).cuda()
    cases = {
        "column slice, unaligned": (wide[..., 3:67], head[:, 5:69]),
        "row slice": (wide[..., 8:72], head[:, 64:]),
        "odd width": (wide[..., :17], head[:, :17]),
        "transposed": (wide.transpose(0, 1)[..., :64], head.t().contiguous().t()[:, :64]),
        "every other row": (wide[::2, :, :64], head[::2, :64]),
        "broadcast": (wide[:1, :1, :64].expand(6, 11, 64), head[:, :64]),
    }
    for name, (x, w) in cases.items():
        t = y % w.shape[0]
        t = t.t() if name == "transposed" else t[::2] if name == "every other row" else t
        grad = _grad_for("none", t.numel()).reshape(t.shape)
        got = _run(x, w, t, grad, reduction="none")
        assert got[0].shape == t.shape and got[1].shape == x.shape and got[2].shape == w.shape
        flat = x.reshape(-1, x.shape[-1])
        want = _expected(flat, w, t.reshape(-1), grad.reshape(-1), "none")
        for a, b, what in zip(got, want, ("loss", "dx", "dw")):
            _close(a.reshape(b[0].shape), b, f"{name} {what}")


def test_one_gradient_at_a_time_gives_the_same_bits():
    from offload_adam_amd import linear_cross_entropy

    x, w, y = _inputs(200, 136, 900, BF16)
    one = torch.ones((), device="cuda")
    _, dx, dw = _run(x, w, y, one)
    a = x.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, y), a)[0], dx)
    b = w.detach().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, b, y), b)[0], dw)
    with torch.no_grad():
        assert not linear_cross_entropy(a, b, y).requires_grad


def test_second_derivatives_are_refused():
    from offload_adam_amd import linear_cross_entropy

    x, w, y = _inputs(20, 64, 100, BF16)
    one = torch.ones((), device="cuda")
    want = _run(x, w, y, one)
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w), create_graph=True)
    assert torch.equal(dx.detach(), want[1]) and torch.equal(dw.detach(), want[2])
    for penalty, by in ((dx, w), (dw, x), (loss + dx.float().square().sum(), x)):
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(penalty.sum(), by, retain_graph=True, allow_unused=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.functional.jvp(lambda t: linear_cross_entropy(t, w, y), (x.detach(),),
                                      (torch.ones_like(x),))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_tokens_whose_gradient_is_zero(dtype, reduction):
    """As a caller's own mask makes them: nothing flows, whatever their rows hold."""
    x, w, y = _inputs(140, 72, 500, dtype, seed=6, ignore=0.0)
    grad = _grad_for(reduction, 140)
    if reduction == "none":
        grad[::3] = 0.0
        clean = _run(x, w, y, grad, reduction=reduction)
        x[::3] = float("nan")
        for a, b in zip(clean[1:], _run(x, w, y, grad, reduction=reduction)[1:]):
            assert torch.equal(a, b)
        assert not clean[1][::3].any() and clean[1][1::3].any()
    else:
        _, dx, dw = _run(x, w, y, torch.zeros_like(grad), reduction=reduction)
        assert not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_that_are_not_finite_stay_in_their_rows(dtype):
    x, w, y = _inputs(140, 72, 500, dtype, seed=7, ignore_index=7)
    y[:4] = 3
    grad = _grad_for("none", 140)
    clean = _run(x, w, y, grad, reduction="none", ignore_index=7)
    for bad in (float("inf"), -float("inf"), float("nan")):
        grad[[1, 3]] = bad
        loss, dx, dw = _run(x, w, y, grad, reduction="none", ignore_index=7)
        assert torch.equal(loss, clean[0])
        assert not torch.isfinite(dx[[1, 3]]).all(1).any() and not torch.isfinite(dw).all()
        # the largest gradient of the others is the same: so is what it scales
        rest = grad.clone()
        rest[[1, 3]] = 0.0
        want = _run(x, w, y, rest, reduction="none", ignore_index=7)[1]
        keep = torch.ones(140, dtype=torch.bool, device="cuda")
        keep[[1, 3]] = False
        assert torch.equal(dx[keep], want[keep]) and torch.isfinite(want).all()
    grad[:] = float("inf")  # nothing finite to scale by
    assert not torch.isfinite(_run(x, w, y, grad, reduction="none", ignore_index=7)[2]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("shape", [(140, 72, 500), (300, 512, 400), (3, 64, 9000)])
def test_tokens_that_take_no_part_meet_a_head_that_is_not_finite(shape, reduction, dtype):
    x, w, y = _inputs(*shape, dtype, seed=8, ignore=0.5)
    y[0], y[-1] = -100, 0
    w[3, 5], w[7, 0] = float("inf"), float("nan")
    grad = _grad_for(reduction, shape[0])
    out = y == -100
    if reduction == "none":
        grad[1] = 0.0
        out[1] = True
    loss, dx, _ = _run(x, w, y, grad, reduction=reduction)
    assert not dx[out].any() and not torch.isfinite(dx[~out]).all(1).any()
    if reduction == "none":
        assert not loss[y == -100].any()


@pytest.mark.parametrize("low", [-4, -8, -13, -20])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gradients_of_very_different_size(dtype, low):
    """Words that only tokens of small gradients know of: their rows of dw, and those tokens'
    rows of dx, as exact as the large ones.  fp16 holds d under a lift of 2^15, of which a
    small gradient takes up to 2^12, and x times 2^-8 or more: half of its smallest step, 2^-25,
    is 2^-40 of d (small gradients: 2^-28) and 2^-17 of x."""
    t, h, v = 96, 64, 300
    g = torch.Generator().manual_seed(3)
    x = torch.randn(t, h, generator=g)
    w = torch.randn(v, h, generator=g) / 4
    x[:, 0] = torch.where(torch.arange(t) < t // 2, 8.0, -8.0)
    w[:, 0] = torch.where(torch.arange(v) < v // 2, 8.0, -8.0)  # the other half: e^-128 less
    x, w = x.to(dtype).cuda(), w.to(dtype).cuda()
    y = torch.cat((torch.randint(v // 2, (t // 2,), generator=g),
                   torch.randint(v // 2, v, (t // 2,), generator=g))).cuda()
    grad = (torch.rand(t, generator=g) + 0.5).cuda() * 2.0**12
    grad[t // 2:] *= 2.0**low
    _, dx, dw = _run(x, w, y, grad, reduction="none")
    r = torch.finfo(dtype).eps / 2
    xd, wd, up = x.double(), w.double(), grad.double()[:, None]
    z = xd @ wd.t().contiguous()
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    d = p.scatter_add(1, y[:, None], torch.full_like(p[:, :1], -1.0))
    dz = (xd.abs() @ wd.abs().t().contiguous()).amax(1, keepdim=True) * h * 2 * U
    rel = 2 * dz + 256 * U + 16 * U * (lse.abs() + z.abs().amax(1, keepdim=True))
    err = p * rel + d.abs() * (r + 2 * U) + 2.0**-126
    off_x = torch.zeros(())
    if dtype == F16:
        err = err + torch.where(torch.arange(t) < t // 2, 2.0**-40, 2.0**-28)[:, None].cuda()
        off_x = 2.0**-17 * (d.abs() * up).sum(0)[:, None]
    floor = 2.0**-24 if dtype == F16 else 2.0**-126
    want = (d * up) @ wd
    tol = up * ((err + d.abs() * (v + 8) * 2 * U) @ wd.abs()) + want.abs() * r + floor
    _close(dx, (want, tol), "dx")
    du = (d * up).t().contiguous()
    want = du @ xd
    tol = (err * up).t().contiguous() @ xd.abs() + du.abs() @ xd.abs() * (t + 8) * 2 * U
    tol = tol + off_x.cuda() + want.abs() * r + floor
    # two tokens of one word: 2 * 8 * 6144 = 98304 in column 0, over fp16's 65504
    fits = want.abs() + tol < torch.finfo(dtype).max
    assert fits[:, 1:].all() and torch.equal(torch.isinf(dw), ~fits)
    _close(dw[fits], (want[fits], tol[fits]), "dw")


def test_gradient_against_differences():
    """Along a direction s of +-1 with steps that 16-bit numbers hold exactly.  The
    third derivative along s is a third cumulant of the logits' direction, at most the
    cube of its range, so a central difference is off by at most h^2 / 6 of that."""
    from offload_adam_amd import linear_cross_entropy

    t, h, v, step = 48, 32, 90, 2.0**-5
    g = torch.Generator().manual_seed(2)
    x = (torch.randint(-32, 33, (t, h), generator=g) / 16.0).to(BF16).cuda()
    w = (torch.randint(-8, 9, (v, h), generator=g) / 32.0).to(BF16).cuda()
    y = torch.randint(v, (t,), generator=g).cuda()
    s = (torch.randint(0, 2, (t, h), generator=g) * 2 - 1).to(BF16).cuda()

    def loss(x, w):
        return float(linear_cross_entropy(x, w, y, reduction="sum"))

    _, dx, dw = _run(x, w, y, torch.ones((), device="cuda"), reduction="sum")
    diff = (loss(x + s * step, w) - loss(x - s * step, w)) / (2 * step)
    reach = (s.double() @ w.double().t().contiguous())
    third = ((reach.amax(1) - reach.amin(1)) ** 3).sum() * step**2 / 6
    want = _expected(x, w, y, torch.ones((), device="cuda"), "sum")
    noise = 2 * float(want[0][1]) / (2 * step)
    assert abs(float((dx.double() * s.double()).sum()) - diff) <= float(
        third + want[1][1].sum() + noise)
    sw = (torch.randint(0, 2, (v, h), generator=g) * 2 - 1).to(BF16).cuda()
    diff = (loss(x, w + sw * step) - loss(x, w - sw * step)) / (2 * step)
    reach = x.double() @ sw.double().t().contiguous()
    third = ((reach.amax(1) - reach.amin(1)) ** 3).sum() * step**2 / 6
    assert abs(float((dw.double() * sw.double()).sum()) - diff) <= float(
        third + want[2][1].sum() + noise)


def test_quantised_head():
    from offload_adam_amd import linear_cross_entropy
    from offload_adam_amd.qweight import Int8QWeight

    x, w, y = _inputs(100, 128, 300, BF16)
    q = torch.nn.Parameter(Int8QWeight.from_float(w))
    plain = q.dequantize().detach().requires_grad_(True)
    a = x.detach().requires_grad_(True)
    got = torch.autograd.grad(linear_cross_entropy(a, q, y), (a, q))
    want = torch.autograd.grad(linear_cross_entropy(a, plain, y), (a, plain))
    assert all(torch.equal(i, j) for i, j in zip(got, want))


@pytest.mark.parametrize("quantised", [False, True])
def test_autocast_casts_as_for_plain_logits(quantised):
    from offload_adam_amd import linear_cross_entropy
    from offload_adam_amd.qweight import FP8QWeight

    x, w, y = _inputs(70, 128, 300, BF16)
    x = x.float().requires_grad_(True)
    w = torch.nn.Parameter(FP8QWeight.from_float(w.float()) if quantised else w.float())
    for low in (BF16, F16):
        c = x.detach().to(low).requires_grad_(True)
        plain = w.detach().dequantize(low) if quantised else w.detach().to(low)
        plain.requires_grad_(True)
        want = linear_cross_entropy(c, plain, y)
        want = (want, *torch.autograd.grad(want, (c, plain)))
        with torch.autocast("cuda", dtype=low):
            loss = linear_cross_entropy(x, w, y)
        got = (loss, *torch.autograd.grad(loss, (x, w)))
        assert all(v.dtype == torch.float32 for v in got)
        assert all(torch.equal(i.float(), j.float()) for i, j in zip(got, want))


def test_another_stream_and_repeated_calls():
    x, w, y = _inputs(300, 264, 2000, F16)
    one = torch.ones((), device="cuda")
    want = _run(x, w, y, one)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [_run(x, w, y, one) for _ in range(3)]
    side.synchronize()
    for g in got:
        assert all(torch.equal(i, j) for i, j in zip(g, want))


def test_captured_and_replayed():
    """Forward and backward in one graph, replayed on changing inputs with eager calls
    in between; two graphs side by side do not share anything."""
    from offload_adam_amd import linear_cross_entropy

    sets = [_inputs(90, 128, 700, BF16, seed=s) for s in range(4)]
    one = torch.ones((), device="cuda")
    want = [_run(*s, one) for s in sets]

    def capture(s):
        x = s[0].clone().requires_grad_(True)
        w = s[1].clone().requires_grad_(True)
        y = s[2].clone()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            torch.autograd.grad(linear_cross_entropy(x, w, y), (x, w))
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = linear_cross_entropy(x, w, y)
            dx, dw = torch.autograd.grad(loss, (x, w))
        return graph, (x, w, y), (loss, dx, dw)

    graphs = [capture(sets[0]), capture(sets[1])]
    for turn in range(4):
        for k, (graph, held, _) in enumerate(graphs):
            s = sets[(turn + k) % 4]
            with torch.no_grad():
                for a, b in zip(held, s):
                    a.copy_(b)
            graph.replay()
        eager = _run(*sets[turn], one)
        torch.cuda.synchronize()
        assert all(torch.equal(i, j) for i, j in zip(eager, want[turn]))
        for k, (_, _, out) in enumerate(graphs):
            ref = want[(turn + k) % 4]
            assert all(torch.equal(i.detach(), j) for i, j in zip(out, ref)), (turn, k)

"""Losses of a large-vocabulary head against their definitions in 64 bits.

Tolerances follow the arithmetic.  A logit is a sum of exact 16-bit products; the tensor core adds at most 96 partial sums
between drains, each off by at most 2^-23 of sum |x_k w_k|, and the drains are added with 2^-24 each, so a logit is off by
delta = (128 + D / 256) 2^-23 sum |x_k w_k|.  exp and log add 2^-20 of their arguments at most.  A gradient element is a sum of
|dZ| |W| (or |dZ| |X|): dZ is rounded by u (half a step of the 16-bit type; float32 carries 2^-24), its probability by
2 delta, the sum again by (128 + length / 256) 2^-23, the result by u."""
import math

import pytest
import torch

import tensorcomprehensions_b200 as tc

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make_ce(cuda, n, d, v, dtype, ignored=0.0, index=torch.int64, seed=0, scale=1.5):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn(n, d, generator=g, device=cuda).to(dtype)
    w = (torch.randn(v, d, generator=g, device=cuda) * (scale / math.sqrt(d))).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device=cuda).to(index)
    t[torch.rand(n, generator=g, device=cuda) < ignored] = -100
    up = torch.rand(n, generator=g, device=cuda) / max(n, 1)
    return x, w, t, up


def reference_ce(x, w, t, up, ignore=-100):
    """loss, dX, dW and what their tolerances are made of, in 64 bits."""
    live = t != ignore
    X, W = x.detach().double() * live[:, None], w.detach().double()
    X = torch.where(live[:, None], x.detach().double(), torch.zeros_like(X))
    z = X @ W.t()
    lse = torch.logsumexp(z, 1)
    at = torch.where(live, t.long(), torch.zeros_like(t.long()))[:, None]
    loss = torch.where(live, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    dz = torch.exp(z - lse[:, None])
    dz.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    dz *= torch.where(live, up.double(), torch.zeros_like(lse))[:, None]
    delta = (128 + x.shape[1] / 256) * 2.0**-23 * (X.abs() @ W.abs().t()).amax(1)
    return loss, dz @ W, dz.t() @ X, dz, delta


def check_ce(x, w, t, up, loss, dx=None, dw=None, ignore=-100):
    rl, rx, rw, dz, delta = reference_ce(x, w, t, up, ignore)
    assert loss.dtype == torch.float32 and loss.shape == (x.shape[0],)
    tol = 2 * delta + 2.0**-20 * (1 + rl.abs())
    assert ((loss.double() - rl).abs() <= tol).all(), "loss off by %g of its tolerance" % ((loss.double() - rl).abs() / tol).max()
    u = half_step(x.dtype)
    # the probabilities' own error, next to what rounding dZ adds: p is below |dZ| / g except at the target, where 1 - p is
    p = dz.abs()
    hot = torch.nonzero(t != ignore)[:, 0]
    if hot.numel():
        p[hot, t.long()[hot]] += up.double()[hot]
    rel = (2 * delta + 2.0**-18)[:, None]
    tiny = torch.finfo(x.dtype).tiny  # below the smallest normal number a type's steps no longer shrink
    X, W = torch.where((t != ignore)[:, None], x.detach().double(), torch.zeros((), dtype=torch.float64, device=x.device)).abs(), w.detach().double().abs()
    if dx is not None:
        assert dx.dtype == x.dtype and dx.shape == x.shape
        err = (dz.abs() * (u + (128 + w.shape[0] / 256) * 2.0**-23) + p * rel) @ W + u * rx.abs() + u * tiny
        assert ((dx.double() - rx).abs() <= err).all(), "dX off by %g of its tolerance" % ((dx.double() - rx).abs() / err).max()
        assert (dx[t == ignore] == 0).all()
    if dw is not None:
        assert dw.dtype == w.dtype and dw.shape == w.shape
        err = (dz.abs() * (u + (128 + x.shape[0] / 256) * 2.0**-23) + p * rel).t() @ X + u * rw.abs() + u * tiny
        assert ((dw.double() - rw).abs() <= err).all(), "dW off by %g of its tolerance" % ((dw.double() - rw).abs() / err).max()


def step_ce(x, w, t, up, **kw):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = tc.linear_cross_entropy(x, w, t, **kw)
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    return loss.detach(), dx, dw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v,ignored", [
    (1, 64, 256, 0), (1, 1, 1, 0), (1, 8, 2, 0), (3, 7, 5, 0), (2, 1000, 300, 0), (130, 65, 257, 0.3), (128, 64, 128, 0), (256, 256, 512, 0),
    (257, 513, 1000, 0.2), (300, 136, 5000, 0.5), (64, 520, 1003, 0), (515, 24, 777, 0.9), (40, 2056, 640, 0),
    (140, 112, 300, 0.1), (140, 60, 300, 0), (140, 700, 300, 0), (140, 1100, 300, 0), (2000, 256, 6000, 0.97), (1500, 512, 9000, 0.5), (1000, 1032, 2000, 0.1)])
def test_linear_cross_entropy(cuda, dtype, n, d, v, ignored):
    x, w, t, up = make_ce(cuda, n, d, v, dtype, ignored, seed=n + d + v)
    check_ce(x, w, t, up, *step_ce(x, w, t, up))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v,ignored", [
    (1, 1024, 32000, 0), (1, 20000, 300, 0), (2, 96, 31, 0), (4, 1000, 3001, 0.3), (5, 77, 40000, 0), (8, 512, 9999, 0.3), (8, 2500, 700, 0),
    (8, 4096, 500, 0), (3, 8200, 257, 0), (7, 333, 33, 0.5), (9, 1000, 3001, 0), (16, 705, 4000, 0.2), (13, 64, 130, 0), (17, 100, 300, 0)])
def test_few_rows(cuda, dtype, n, d, v, ignored):
    x, w, t, up = make_ce(cuda, n, d, v, dtype, ignored, seed=n * d + v)
    t[n // 2] = v - 1
    got = step_ce(x, w, t, up)
    check_ce(x, w, t, up, *got)
    # rows of W off the 16-byte boundaries: the same products in another order
    ws = torch.full((v, d + 1), float("nan"), device=cuda, dtype=dtype)[:, 1:]
    ws.copy_(w)
    check_ce(x, ws, t, up, *step_ce(x, ws, t, up))
    # masked rows hold anything; a target outside is NaN
    if (t == -100).any():
        x2, up2 = x.clone(), up.clone()
        x2[t == -100] = float("inf")
        up2[t == -100] = float("nan")
        for a, b in zip(got, step_ce(x2, w, t, up2)):
            assert torch.equal(a, b)
    t2 = t.clone()
    t2[0] = v
    loss, dx, dw = step_ce(x, w, t2, up)
    assert loss[0].isnan() and dx[0].isnan().all() and dw.isnan().all() and dx[1:].isfinite().all()


@pytest.mark.parametrize("dtype,n,d,v", [(torch.bfloat16, 4000, 40, 40000), (torch.float32, 1000, 33, 50000), (torch.float16, 2050, 41, 70001)])
def test_several_pieces_of_the_vocabulary(cuda, dtype, n, d, v):
    x, w, t, up = make_ce(cuda, n, d, v, dtype, 0.1, seed=5)
    check_ce(x, w, t, up, *step_ce(x, w, t, up))


@pytest.mark.parametrize("dtype", TYPES)
def test_long_reduction_and_wide_logits(cuda, dtype):
    x, w, t, up = make_ce(cuda, 100, 8192, 600, dtype, scale=6.0)
    check_ce(x, w, t, up, *step_ce(x, w, t, up))
    # a sum that only grows: the drift of the tensor core's truncation shows here first
    x, w = x.abs(), w.abs() / 50
    check_ce(x, w, t, up, *step_ce(x, w, t, up))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_int32_targets_strided_rows_and_unaligned_weights(cuda, dtype):
    n, d, v = 70, 48, 300
    x, w, t, up = make_ce(cuda, n, d, v, dtype, 0.2, index=torch.int32)
    xs = torch.full((n, d + 3), float("nan"), device=cuda, dtype=dtype)[:, 2:2 + d]
    xs.copy_(x)
    ws = torch.full((v, d + 5), float("nan"), device=cuda, dtype=dtype)[:, 3:3 + d]
    ws.copy_(w)
    wide = torch.full((v, 2 * d), float("nan"), device=cuda, dtype=dtype)[:, d:]
    wide.copy_(w)
    ts = torch.stack([t, t + 1], 1)[:, 0]
    want = step_ce(x, w, t, up)
    check_ce(x, w, t, up, *want)
    for weights in (ws, wide):
        got = step_ce(xs, weights, ts, up)
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_rows_without_a_target_are_never_read(cuda):
    x, w, t, up = make_ce(cuda, 333, 72, 500, torch.bfloat16, 0.4)
    want = step_ce(x, w, t, up)
    x2, up2 = x.clone(), up.clone()
    x2[t == -100] = float("nan")
    up2[t == -100] = float("inf")
    got = step_ce(x2, w, t, up2)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    # all rows
    none = torch.full_like(t, 7)
    loss, dx, dw = step_ce(x2, w, none, up2, ignore_index=7)
    assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all()


def test_a_target_outside_the_vocabulary_is_nan(cuda):
    x, w, t, up = make_ce(cuda, 20, 32, 100, torch.float16)
    for bad in (100, 1 << 40, -1, -(1 << 40)):
        t2 = t.clone()
        t2[3] = bad
        loss, dx, dw = step_ce(x, w, t2, up)
        assert loss[3].isnan() and dx[3].isnan().all() and dw.isnan().all()
        rest = torch.arange(20, device=cuda) != 3
        assert torch.equal(loss[rest], tc.linear_cross_entropy(x, w, t)[rest]) and dx[rest].isfinite().all()


def test_one_gradient_for_all_rows_and_one_input_only(cuda):
    x, w, t, _ = make_ce(cuda, 200, 64, 300, torch.bfloat16, 0.25)
    live = int((t != -100).sum())
    x.requires_grad_()
    (tc.linear_cross_entropy(x, w, t).sum() / live).backward()   # an expanded gradient: stride 0
    up = torch.full((200,), 1.0 / live, device=cuda)
    check_ce(x, w, t, up, tc.linear_cross_entropy(x, w, t).detach(), dx=x.grad)
    w.requires_grad_()
    x = x.detach()
    tc.linear_cross_entropy(x, w, t).mean().backward()
    check_ce(x, w, t, torch.full_like(up, 1 / 200), tc.linear_cross_entropy(x, w, t).detach(), dw=w.grad)


def test_gradient_scales_far_from_one(cuda):
    for scale in (1e-30, 1e-6, 1e6):
        x, w, t, up = make_ce(cuda, 60, 64, 300, torch.bfloat16)
        up = up * scale
        check_ce(x, w, t, up, *step_ce(x, w, t, up))
    x, w, t, up = make_ce(cuda, 60, 64, 300, torch.bfloat16)
    loss, dx, dw = step_ce(x, w, t, torch.zeros_like(up))
    assert (dx == 0).all() and (dw == 0).all()


def test_gradient_against_differences(cuda):
    x, w, t, up = make_ce(cuda, 5, 16, 40, torch.float32, 0.2)
    _, dx, dw = step_ce(x, w, t, up)
    h = 2.0**-6  # truncation h^2 |f'''| / 6 is below 2^-14 here, rounding 2^-21 |loss| / h below 2^-13
    for tensor, grad in ((x, dx), (w, dw)):
        for at in ((0, 0), (1, 3), (4, 15)):
            lo, hi = tensor.clone(), tensor.clone()
            lo[at] -= h
            hi[at] += h
            a, b = ((lo, w), (hi, w)) if tensor is x else ((x, lo), (x, hi))
            f = [(tc.linear_cross_entropy(*p, t).double() * up.double()).sum() for p in (a, b)]
            assert abs((f[1] - f[0]).item() / (2 * h) - grad[at].item()) < 2.0**-12


def test_empty_batch(cuda):
    for dtype in TYPES:
        x = torch.empty(0, 32, device=cuda, dtype=dtype)
        w = torch.randn(100, 32, device=cuda).to(dtype)
        t = torch.empty(0, device=cuda, dtype=torch.int64)
        loss, dx, dw = step_ce(x, w, t, torch.empty(0, device=cuda))
        assert loss.shape == (0,) and dx.shape == (0, 32) and (dw == 0).all()


def test_strided_gradient_and_saved_inputs(cuda):
    x, w, t, up = make_ce(cuda, 50, 40, 90, torch.float32)
    want = step_ce(x, w, t, up)
    wide = torch.full((50, 3), float("nan"), device=cuda)
    wide[:, 1] = up
    for a, b in zip(want, step_ce(x, w, t, wide[:, 1])):
        assert torch.equal(a, b)
    x.requires_grad_()
    loss = tc.linear_cross_entropy(x, w, t)
    w.mul_(2)  # the backward pass would read another W than the forward did
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()
    # no second derivative
    (dx,) = torch.autograd.grad(tc.linear_cross_entropy(x, w, t).sum(), x, retain_graph=True)
    assert not dx.requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(tc.linear_cross_entropy(x, w, t).sum(), x, create_graph=True)
    z, i, s, _ = make_kd(cuda, 4, 50, 3, torch.float32)
    z.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(tc.topk_distillation(z, i, s).sum(), z, create_graph=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(1, 64, 100), (3, 33, 65), (20, 72, 300), (300, 45, 513), (257, 264, 1000)])
@pytest.mark.parametrize("shift", [0, 1])
def test_nothing_is_written_outside_the_outputs(cuda, dtype, n, d, v, shift):
    """The C entry points with every buffer between two guards, dX and dW on and off their 16-byte boundaries."""
    import ctypes
    from tensorcomprehensions_b200 import cabi
    x, w, t, up = make_ce(cuda, n, d, v, dtype, 0.2)
    size = x.element_size()
    code = {torch.float32: cabi.F32, torch.float16: cabi.F16, torch.bfloat16: cabi.BF16}[dtype]
    p = cabi.LinearCe(n, d, v, d, d, -100, code, 8, int(d * size % 16 != 0), 0)
    f, b = ctypes.c_int64(), ctypes.c_int64()
    cabi.check(cabi.lib().tcb200_linear_ce_workspace(ctypes.byref(p), ctypes.byref(f), ctypes.byref(b)), "workspace")
    GUARD = 4096

    def guarded(nbytes, offset=0):
        buf = torch.full((GUARD + offset + nbytes + GUARD,), 0xCD, device=cuda, dtype=torch.uint8)
        return buf, GUARD + offset, nbytes

    def untouched(g):
        buf, at, nbytes = g
        return bool((buf[:at] == 0xCD).all()) and bool((buf[at + nbytes:] == 0xCD).all())

    def ptr(g):
        return ctypes.c_void_p(g[0].data_ptr() + g[1])

    def values(g, dt, shape):
        return g[0][g[1]:g[1] + g[2]].clone().view(dt).view(shape)

    loss, lse, wf, wb = guarded(4 * n), guarded(4 * n), guarded(f.value), guarded(b.value)
    dx, dw = guarded(n * d * size, shift * size), guarded(v * d * size, shift * size)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    P = lambda a: ctypes.c_void_p(a.data_ptr())  # noqa: E731
    cabi.check(cabi.lib().tcb200_linear_ce_forward(ctypes.byref(p), P(x), P(w), P(t), ptr(loss), ptr(lse), ptr(wf), f.value, st, None), "forward")
    cabi.check(cabi.lib().tcb200_linear_ce_backward(ctypes.byref(p), P(x), P(w), P(t), ptr(lse), P(up), 1, ptr(dx), ptr(dw), ptr(wb), b.value, st, None), "backward")
    torch.cuda.synchronize()
    assert all(untouched(g) for g in (loss, lse, wf, wb, dx, dw))
    check_ce(x, w, t, up, values(loss, torch.float32, (n,)), values(dx, dtype, (n, d)), values(dw, dtype, (v, d)))


@pytest.mark.parametrize("n", [3, 40])
def test_offsets_behind_32_bits(cuda, n):
    """W and dW of 2.4e9 elements: single entries behind the 2^31st against 64 bits."""
    d, v = 4096, 590000
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(n, d, generator=g, device=cuda).bfloat16()
    w = torch.empty(v, d, device=cuda, dtype=torch.bfloat16).normal_(0, 1 / 64, generator=g)
    t = torch.randint(v - 1000, v, (n,), generator=g, device=cuda)
    up = torch.rand(n, generator=g, device=cuda)
    loss, dx, dw = step_ce(x, w, t, up)
    X = x.double()
    z = torch.cat([X @ w[a:a + 50000].double().t() for a in range(0, v, 50000)], 1)
    lse = torch.logsumexp(z, 1)
    rl = lse - z[torch.arange(n, device=cuda), t]
    assert ((loss.double() - rl).abs() <= 2.0**-14 * (1 + rl)).all()
    dz = torch.exp(z - lse[:, None])
    dz[torch.arange(n, device=cuda), t] -= 1
    dz *= up.double()[:, None]
    rows = torch.cat([t, torch.tensor([0, v // 2, v - 1], device=cuda)])
    rw = dz[:, rows].t() @ X
    # dZ and dW are rounded to bfloat16, half a step 2^-8 each; the probabilities are off by 2^-10
    tol = dz[:, rows].abs().t() @ X.abs() * (2.0**-8 + 2.0**-10) + 2.0**-8 * rw.abs()
    assert ((dw[rows].double() - rw).abs() <= tol).all()
    rx = sum(dz[:, a:a + 50000] @ w[a:a + 50000].double() for a in range(0, v, 50000))
    tol = sum(dz[:, a:a + 50000].abs() @ w[a:a + 50000].double().abs() for a in range(0, v, 50000)) * (2.0**-8 + 2.0**-10) + 2.0**-8 * rx.abs()
    assert ((dx.double() - rx).abs() <= tol).all()


# ---------------------------------------------------------------------------------- distillation
def make_kd(cuda, n, v, k, dtype, ragged=False, index=torch.int64, seed=0, teacher_dtype=None):
    g = torch.Generator(device=cuda).manual_seed(seed)
    z = (torch.randn(n, v, generator=g, device=cuda) * 2.5).to(dtype)
    i = torch.rand(n, v, generator=g, device=cuda).argsort(1)[:, :k] if k <= v else torch.randint(0, v, (n, k), generator=g, device=cuda)
    s = (torch.randn(n, k, generator=g, device=cuda) * 3).to(teacher_dtype or dtype)
    if ragged:
        lengths = torch.randint(0, k + 1, (n, 1), generator=g, device=cuda)
        i = torch.where(torch.arange(k, device=cuda) < lengths, i, torch.full_like(i, -1))
    up = torch.rand(n, generator=g, device=cuda) / max(n, 1)
    return z, i.to(index).contiguous(), s, up


def reference_kd(z, i, s, up, temperature):
    z, s, i, t = z.detach().double() / temperature, s.double() / temperature, i.long(), temperature
    there = (i >= 0) & (s > -math.inf)
    some = there.any(1)
    s = s.masked_fill(~there, -math.inf)
    s[~some] = 0
    logq = torch.log_softmax(s, 1)
    q = torch.exp(logq).masked_fill(~there, 0)
    logp = torch.log_softmax(z, 1)
    at = i.clamp(min=0)
    loss = t * t * (q * (logq - logp.gather(1, at))).masked_fill(q == 0, 0).sum(1)
    spread = torch.zeros_like(z).scatter_add_(1, at, q)
    p = torch.exp(logp)
    k = (t * up.double() * some)[:, None]
    return torch.where(some, loss, torch.zeros_like(loss)), torch.where(some[:, None], k * (p - spread), torch.zeros_like(z)), k.abs() * p, k.abs() * spread, some


def check_kd(z, i, s, up, temperature, loss, dz):
    rl, rz, p, q, some = reference_kd(z, i, s, up, temperature)
    # exp and log are off by 2^-22 of their arguments, which are differences of logits / T
    span = (2 * z.detach().double().abs().amax(1) + 2 * torch.where(s.isfinite(), s, torch.zeros_like(s)).double().abs().amax(1)) / temperature
    tol = temperature**2 * 2.0**-20 * (4 + span)
    assert loss.dtype == torch.float32
    assert ((loss.double() - rl).abs() <= tol).all(), "loss off by %g of its tolerance" % ((loss.double() - rl).abs() / tol).max()
    u = half_step(z.dtype)
    tol = u * rz.abs() + (p + q) * (2.0**-20 * (4 + span))[:, None] + u * torch.finfo(z.dtype).tiny
    assert dz.dtype == z.dtype and dz.shape == z.shape
    assert ((dz.double() - rz).abs() <= tol).all(), "gradient off by %g of its tolerance" % ((dz.double() - rz).abs() / tol).max()
    assert (loss[~some] == 0).all() and (dz[~some] == 0).all()


def step_kd(z, i, s, up, temperature=1.0):
    z = z.detach().requires_grad_()
    loss = tc.topk_distillation(z, i, s, temperature)
    (dz,) = torch.autograd.grad(loss, (z,), up)
    return loss.detach(), dz


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k,ragged,temperature", [
    (1, 1, 1, False, 1.0), (1, 2, 2, False, 2.0), (1, 32000, 8, False, 1.0), (1, 40001, 100, False, 4.0), (3, 7, 3, True, 1.0), (5, 9001, 1, False, 0.5),
    (200, 1000, 20, True, 2.0), (33, 30011, 64, True, 1.0), (700, 515, 128, False, 3.0), (2, 100000, 4096, True, 1.0), (17, 16385, 600, False, 1.0)])
def test_topk_distillation(cuda, dtype, n, v, k, ragged, temperature):
    z, i, s, up = make_kd(cuda, n, v, k, dtype, ragged, seed=n + v + k)
    check_kd(z, i, s, up, temperature, *step_kd(z, i, s, up, temperature))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k,ragged", [
    (1200, 515, 5, True), (1300, 90, 120, False), (1184, 4099, 33, True), (1250, 8192, 128, False), (1250, 8193, 65, False), (2500, 31, 1, True),
    (1300, 600, 129, True), (40, 500, 2000, False), (3, 70001, 4096, False)])
def test_distillation_many_short_rows_and_equal_indices(cuda, dtype, n, v, k, ragged):
    """Rows enough for small blocks, and (K > V, and every third entry a copy of the first) places that many entries share."""
    z, i, s, up = make_kd(cuda, n, v, k, dtype, ragged, seed=n + v + k)
    i[::2, ::3] = i[::2, :1]
    got = step_kd(z, i, s, up, 2.0)
    check_kd(z, i, s, up, 2.0, *got)
    again = step_kd(z, i, s, up, 2.0)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_distillation_other_types_and_strides(cuda):
    n, v, k = 37, 5003, 24
    z, i, s, up = make_kd(cuda, n, v, k, torch.bfloat16, True, index=torch.int32, teacher_dtype=torch.float32)
    want = step_kd(z, i, s, up, 2.0)
    check_kd(z, i, s, up, 2.0, *want)
    for offset in (1, 3, 8):
        zs = torch.full((n, v + 9), float("nan"), device=cuda, dtype=z.dtype)[:, offset:offset + v]
        zs.copy_(z)
        it = torch.full((n, 2 * k), 1 << 20, device=cuda, dtype=torch.int32)[:, k:]
        it.copy_(i)
        st = torch.full((n, k + 1), float("nan"), device=cuda)[:, 1:]
        st.copy_(s)
        got = step_kd(zs, it, st, up, 2.0)
        # another alignment is another order of a row's sum
        check_kd(zs, it, st, up, 2.0, *got)
    check_kd(z, i, s, up, 2.0, *step_kd(z, i.long(), s, up, 2.0))


def test_distillation_same_index_twice_and_masked_values(cuda):
    z, i, s, up = make_kd(cuda, 40, 3000, 12, torch.float32)
    i[:, 5] = i[:, 2]
    i[:, 11] = i[:, 2]
    check_kd(z, i, s, up, 1.0, *step_kd(z, i, s, up))
    # masked vocabulary (-inf logits) away from the entries, teacher logits of -inf, the type's lowest value
    z[:, 2999] = -math.inf
    z[:, 2998] = torch.finfo(z.dtype).min
    i[(i == 2999) | (i == 2998)] = -1
    s[:, 3] = -math.inf
    s[7] = -math.inf       # a row that keeps nothing
    i[8] = -1
    loss, dz = step_kd(z, i, s, up)
    finite = z.clone()
    finite[:, 2998:] = -200  # the same probabilities
    check_kd(finite, i, s, up, 1.0, loss, dz)
    assert loss[7] == 0 and loss[8] == 0
    # a row without entries is 0 whatever its logits hold; NaN elsewhere stays in its row
    z[8] = math.nan
    z[9, 17] = math.nan
    l2, d2 = step_kd(z, i, s, up)
    assert l2[8] == 0 and (d2[8] == 0).all() and l2[9].isnan() and d2[9].isnan().all()
    rest = torch.tensor([r for r in range(40) if r not in (8, 9)], device=cuda)
    assert torch.equal(l2[rest], loss[rest]) and torch.equal(d2[rest], dz[rest])
    # a place the student gives nothing: infinite loss, finite gradient
    z[0, i[0, 0]] = -math.inf
    l3, d3 = step_kd(z, i, s, up)
    assert l3[0] == math.inf and d3[0].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_rows_of_the_lowest_value(cuda, dtype):
    """A row masked with its type's lowest value throughout is uniform; large logits lose nothing against their differences."""
    z, i, s, up = make_kd(cuda, 6, 4003, 9, dtype, seed=11)
    z[1] = torch.finfo(dtype).min
    z[2, 100:] = torch.finfo(dtype).min
    i[2] = torch.arange(9, device=cuda)
    z[3] = (torch.randint(0, 8, (4003,), device=cuda) + 16000).to(dtype)   # whole numbers: exact in every type but bfloat16, where they are 16000 + 0 or 64
    z[4] = -z[3]
    for temperature in (1.0, 3.0):
        rl, rz, p, q, _ = reference_kd(z, i, s, up, temperature)
        loss, dz = step_kd(z, i, s, up, temperature)
        # the tolerances of differences alone: they are at most 64 / T here, or the masked ones' exp is 0 on both sides
        tol = temperature**2 * 2.0**-20 * (4 + (64 + 32) / temperature)
        assert ((loss.double() - rl).abs() <= tol).all()
        u = half_step(dtype)
        assert ((dz.double() - rz).abs() <= u * rz.abs() + (p + q) * 2.0**-20 * (4 + 96 / temperature) + u * torch.finfo(dtype).tiny).all()


def test_distillation_index_outside_the_vocabulary_is_nan(cuda):
    z, i, s, up = make_kd(cuda, 10, 5000, 6, torch.bfloat16)
    want = step_kd(z, i, s, up)
    for bad in (5000, 1 << 40):
        j = i.clone()
        j[4, 2] = bad
        loss, dz = step_kd(z, j, s, up)
        assert loss[4].isnan() and dz[4].isnan().all()
        rest = torch.arange(10, device=cuda) != 4
        assert torch.equal(loss[rest], want[0][rest]) and torch.equal(dz[rest], want[1][rest])


def test_distillation_one_gradient_for_all_rows_and_differences(cuda):
    z, i, s, _ = make_kd(cuda, 6, 50, 5, torch.float32)
    z.requires_grad_()
    tc.topk_distillation(z, i, s, 2.0).mean().backward()
    up = torch.full((6,), 1 / 6, device=cuda)
    check_kd(z, i, s, up, 2.0, tc.topk_distillation(z, i, s, 2.0).detach(), z.grad)
    h = 2.0**-5
    for at in ((0, int(i[0, 0])), (3, 7), (5, 49)):
        f = []
        for d in (-h, h):
            y = z.detach().clone()
            y[at] += d
            f.append(tc.topk_distillation(y, i, s, 2.0).double().mean())
        assert abs((f[1] - f[0]).item() / (2 * h) - z.grad[at].item()) < 2.0**-11


def test_distillation_empty_batch(cuda):
    z = torch.empty(0, 100, device=cuda)
    loss, dz = step_kd(z, torch.empty(0, 3, device=cuda, dtype=torch.int64), torch.empty(0, 3, device=cuda), torch.empty(0, device=cuda))
    assert loss.shape == (0,) and dz.shape == (0, 100)


def test_distillation_offsets_behind_32_bits(cuda):
    n, v, k = 17000, 131072, 5
    g = torch.Generator(device=cuda).manual_seed(4)
    z = torch.empty(n, v, device=cuda, dtype=torch.bfloat16).normal_(0, 2, generator=g)
    i = torch.randint(0, v, (n, k), generator=g, device=cuda)
    s = torch.randn(n, k, generator=g, device=cuda)
    up = torch.rand(n, generator=g, device=cuda)
    loss, dz = step_kd(z, i, s, up)
    rows = torch.tensor([0, 8191, 16383, 16384, 16999], device=cuda)
    check_kd(z[rows], i[rows], s[rows], up[rows], 1.0, loss[rows], dz[rows])


def test_distillation_writes_nothing_outside_its_output(cuda):
    import ctypes
    from tensorcomprehensions_b200 import cabi
    for dtype, code in ((torch.float32, cabi.F32), (torch.bfloat16, cabi.BF16)):
        for n, v, k, shift in ((3, 5001, 7, 0), (3, 5001, 7, 1), (1, 40000, 300, 0), (9, 17, 4, 1)):
            z, i, s, up = make_kd(cuda, n, v, k, dtype, True)
            p = cabi.TopkDistill(n, v, k, v, k, k, 2.0, code, code, 8)
            size, P = z.element_size(), (lambda a: ctypes.c_void_p(a.data_ptr()))
            st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
            bufs = [torch.full((4096 + o + b + 4096,), 0xCD, device=cuda, dtype=torch.uint8) for o, b in ((0, 4 * n), (0, 12 * n), (shift * size, n * v * size))]
            loss, stats, dz = (ctypes.c_void_p(b.data_ptr() + 4096 + o) for b, o in zip(bufs, (0, 0, shift * size)))
            cabi.check(cabi.lib().tcb200_topk_distill_forward(ctypes.byref(p), P(z), P(i), P(s), loss, stats, st), "forward")
            cabi.check(cabi.lib().tcb200_topk_distill_backward(ctypes.byref(p), P(z), P(i), P(s), stats, P(up), 1, dz, st), "backward")
            torch.cuda.synchronize()
            for b, o, nb in zip(bufs, (0, 0, shift * size), (4 * n, 12 * n, n * v * size)):
                assert (b[:4096 + o] == 0xCD).all() and (b[4096 + o + nb:] == 0xCD).all()
            got = [b[4096 + o:4096 + o + nb].clone() for b, o, nb in zip(bufs, (0, 0, shift * size), (4 * n, 12 * n, n * v * size))]
            check_kd(z, i, s, up, 2.0, got[0].view(torch.float32), got[2].view(dtype).view(n, v))


# ---------------------------------------------------------------------------------- together, as they are used
MATMUL = """
def logits(float(N, D) X, float(V, D) W) -> (Z) { Z(n, v) +=! X(n, r_d) * W(v, r_d) }
def dx(float(N, V) G, float(V, D) W) -> (O) { O(n, d) +=! G(n, r_v) * W(r_v, d) }
def dw(float(N, V) G, float(N, D) X) -> (O) { O(v, d) +=! G(r_n, v) * X(r_n, d) }
"""


def test_both_losses_on_one_head_made_of_comprehensions(cuda):
    """A student's step: the logits come from a comprehension, its gradients from two more; the distillation loss takes the
    logits, the cross entropy the same X and W."""
    n, d, v, k = 96, 64, 512, 16
    x, w, t, _ = make_ce(cuda, n, d, v, torch.float32, 0.2)
    _, i, s, _ = make_kd(cuda, n, v, k, torch.float32, True)
    T = tc.define(MATMUL, tc.make_naive_options_factory())
    head = tc.make_autograd(lambda a, b: T.logits(a, b), lambda a, b, g: (T.dx(g, b), T.dw(g, a)))
    x, w = x.requires_grad_(), w.requires_grad_()
    live = (t != -100).sum()
    loss = 0.5 * tc.linear_cross_entropy(x, w, t).sum() / live + 0.5 * tc.topk_distillation(head(x, w), i, s, 2.0).mean()
    loss.backward()
    X, W = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    z = X @ W.t()
    ce = torch.nn.functional.cross_entropy(z, t, ignore_index=-100, reduction="sum") / live
    there = i >= 0
    q = torch.softmax((s.double() / 2).masked_fill(~there, -1e300), 1).masked_fill(~there, 0)
    kd = 4 * (q * (torch.log(q.clamp(min=1e-300)) - torch.log_softmax(z / 2, 1).gather(1, i.clamp(min=0)))).sum(1)
    want = 0.5 * ce + 0.5 * kd.mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 2.0**-17 * (1 + abs(want.item()))
    # the comprehensions' products keep 1e-5 of the sum of magnitudes (their own criterion); so do the losses' gradients
    for got, ref, mag in ((x.grad, X.grad, W.abs().sum(0).max()), (w.grad, W.grad, X.abs().sum(0).max())):
        assert (got.double() - ref).abs().max() <= 1e-5 * mag


def test_another_stream_and_a_captured_step(cuda):
    x, w, t, up = make_ce(cuda, 300, 96, 1000, torch.bfloat16, 0.1)
    z, i, s, uk = make_kd(cuda, 50, 6000, 10, torch.bfloat16, True)
    want = step_ce(x, w, t, up) + step_kd(z, i, s, uk, 2.0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step_ce(x, w, t, up) + step_kd(z, i, s, uk, 2.0)
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    # two graphs of the same inputs, replayed at the same time: each has scratch memory of its own
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step_ce(x, w, t, up) + step_kd(z, i, s, uk, 2.0))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(want, o):
            assert torch.equal(a, b)
    # new inputs in the captured tensors
    x2, w2, t2, _ = make_ce(cuda, 300, 96, 1000, torch.bfloat16, 0.6, seed=9)
    x.copy_(x2), w.copy_(w2), t.copy_(t2)
    graphs[0].replay()
    torch.cuda.synchronize()
    check_ce(x, w, t, up, *outs[0][:3])


def test_the_first_calls_of_a_process_may_be_captured(cuda):
    """Nothing has to run before a capture: no kernel needs a warm-up, nothing allocates outside ATen's pools."""
    import subprocess
    import sys
    code = """
import torch, tensorcomprehensions_b200 as tc
x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_(); w = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_()
xf = torch.randn(2, 64, device="cuda").requires_grad_(); wf = torch.randn(300, 64, device="cuda")
t = torch.randint(0, 300, (40,), device="cuda"); up = torch.rand(40, device="cuda")
z = torch.randn(5, 4000, device="cuda").requires_grad_(); i = torch.randint(0, 4000, (5, 7), device="cuda"); s = torch.randn(5, 7, device="cuda"); uk = torch.rand(5, device="cuda")
def step():
    a = tc.linear_cross_entropy(x, w, t); b = tc.linear_cross_entropy(xf, wf, t[:2]); c = tc.topk_distillation(z, i, s)
    return [a.detach(), b.detach(), c.detach(), *torch.autograd.grad(a, (x, w), up), *torch.autograd.grad(b, (xf,), up[:2]), *torch.autograd.grad(c, (z,), uk)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay(); torch.cuda.synchronize()
want = step(); torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, want))
print("captured ok")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured ok" in r.stdout, r.stdout + r.stderr


def test_the_same_bits_on_every_run(cuda):
    for dtype in TYPES:
        x, w, t, up = make_ce(cuda, 600, 264, 3001, dtype, 0.2)
        z, i, s, uk = make_kd(cuda, 3, 50000, 32, dtype)
        want = step_ce(x, w, t, up) + step_kd(z, i, s, uk)
        for _ in range(3):
            for a, b in zip(want, step_ce(x, w, t, up) + step_kd(z, i, s, uk)):
                assert torch.equal(a, b)


def test_another_device_than_the_current_one(cuda):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    other = torch.device("cuda:1")
    x, w, t, up = make_ce(other, 30, 64, 200, torch.bfloat16)
    check_ce(x, w, t, up, *step_ce(x, w, t, up))
    z, i, s, uk = make_kd(other, 5, 3000, 4, torch.bfloat16)
    check_kd(z, i, s, uk, 1.0, *step_kd(z, i, s, uk))


def test_refusals_on_the_device(cuda):
    x, w, t, _ = make_ce(cuda, 4, 8, 16, torch.float32)
    z, i, s, _ = make_kd(cuda, 4, 16, 3, torch.float32)
    bad_ce = [(x.half(), w, t), (x.double(), w.double(), t), (x, w[:, :4], t), (x[0], w, t), (x, w, t[:3]), (x, w, t.float()), (x, w, t.cpu()),
              (x.cpu(), w, t), (x, w.cpu(), t), (x.t().contiguous().t(), w, t), (x, w.t().contiguous().t(), t), (x[:1].expand(4, 8), w, t), (x, w[:0], t)]
    for args in bad_ce:
        with pytest.raises(RuntimeError):
            tc.linear_cross_entropy(*args)
    bad_kd = [(z, i, s[:, :2]), (z, i[:3], s[:3]), (z.double(), i, s), (z, i.float(), s), (z, i.short(), s), (z, i.cpu(), s), (z.cpu(), i, s),
              (z, i[:, :0], s[:, :0]), (z[:, :0], i, s), (z.t().contiguous().t(), i, s), (z[0], i, s)]
    for args in bad_kd:
        with pytest.raises(RuntimeError):
            tc.topk_distillation(*args)
    for temperature in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError):
            tc.topk_distillation(z, i, s, temperature)
    with pytest.raises(RuntimeError):
        tc.topk_distillation(z, i, s.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        tc.topk_distillation(z, torch.zeros(4, 4097, device=cuda, dtype=torch.int64), torch.zeros(4, 4097, device=cuda))


@pytest.mark.parametrize("v,parts", [(4096, 2), (8191, 2), (8192, 4), (16384, 8), (40000, 8)])
def test_distillation_of_rows_split_over_clusters(cuda, v, parts):
    """Clusters of every size with the shortest stretches they take, from a single one to more than the device holds at a time: CTAs of a
    cluster that start apart leave the same bits."""
    for n in (1, 3, 1183 // parts):
        z, i, s, up = make_kd(cuda, n, v, 6, torch.float32, seed=v + n)
        want = step_kd(z, i, s, up, 2.0)
        check_kd(z, i, s, up, 2.0, *want)
        for _ in range(20):
            got = step_kd(z, i, s, up, 2.0)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("n,v,k", [(9, 4003, 9), (9, 20000, 700), (1300, 90, 40)])
def test_distillation_teacher_rows_of_the_lowest_value_and_large_ones(cuda, dtype, temperature, n, v, k):
    """The teacher's distribution follows from differences of its logits alone, in the loss and in the gradient: rows of the type's
    lowest value are uniform, rows of large whole numbers are what the small differences between them say."""
    z, i, s, up = make_kd(cuda, n, v, k, dtype, seed=n + k)
    top = 60000 if dtype == torch.float16 else 2.0**20
    s[0] = torch.finfo(dtype).min
    s[1] = torch.finfo(dtype).min
    s[1, 0] = 3
    s[2] = (torch.randint(0, 8, (k,), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda) + 16000).to(dtype)  # exact, but 16000 + 0 or 64 in bfloat16
    s[3] = -s[2]
    s[4] = top
    s[5] = -top
    s[6] = torch.finfo(dtype).max
    s[7, ::2] = -math.inf
    s[7, 1::2] = top
    i[7, 1::3] = -1
    rl, rz, p, q, _ = reference_kd(z, i, s, up, temperature)
    loss, dz = step_kd(z, i, s, up, temperature)
    # differences of the teacher's logits are at most 64 / T where their exp is not 0 on both sides, the student's (deviation 2.5) 30 / T
    rel = 2.0**-20 * (4 + 94 / temperature)
    assert ((loss.double() - rl).abs() <= temperature**2 * rel).all()
    u = half_step(dtype)
    tol = u * rz.abs() + (p + q) * rel + u * torch.finfo(dtype).tiny
    assert ((dz.double() - rz).abs() <= tol).all(), "gradient off by %g of its tolerance" % ((dz.double() - rz).abs() / tol).max()


def test_tangents_are_refused_on_the_device(cuda):
    """Forward mode over a loss, and over its gradient."""
    import torch.autograd.forward_ad as fwd
    x, w, t, up = make_ce(cuda, 4, 8, 16, torch.float32)
    z, i, s, uk = make_kd(cuda, 4, 16, 3, torch.float32)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: tc.linear_cross_entropy(a, w, t), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: tc.topk_distillation(z, i, a), (s,), (s,))
    x.requires_grad_(), z.requires_grad_()
    with fwd.dual_level():
        for loss, leaf, g in ((tc.linear_cross_entropy(x, w, t), x, up), (tc.topk_distillation(z, i, s), z, uk)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(loss, leaf, fwd.make_dual(g, g))


def test_distillation_extreme_temperatures(cuda):
    z, i, s, up = make_kd(cuda, 4, 300, 3, torch.float32)
    for temperature in (1e-39, 1e-20, 1e20):
        with pytest.raises(RuntimeError, match="square must be a normal float32 number"):
            tc.topk_distillation(z, i, s, temperature)
    # the coldest one accepted: each side puts all of itself on its largest logit
    z[:, 0], z[:, 1] = 20, 20.5
    i[:, 0], i[:, 1], i[:, 2] = 1, 5, 6
    s[:, 0], s[:, 1], s[:, 2] = 4, 3, 2
    loss, dz = step_kd(z, i, s, up, 2.0**-63)
    assert (loss == 0).all() and (dz == 0).all()
    # the hottest: both are uniform over their places, p is 1 / 300 and q 1 / 3
    _, dz = step_kd(z, i, s, up, 1e19)
    want = torch.full((4, 300), 1 / 300, device=cuda, dtype=torch.float64)
    want[:, [1, 5, 6]] -= 1 / 3
    want *= 1e19 * up.double()[:, None]
    assert ((dz.double() - want).abs() <= 2.0**-18 * want.abs()).all()


@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("n,v", [(5, 2003), (1300, 515)])
def test_distillation_small_probabilities_keep_float32_accuracy(cuda, temperature, n, v):
    """Differences of logits are exact here and the row's sum is its largest element's 1 and almost nothing else, so that a probability far
    from the maximum is off by expf's two units (2^-22) and three roundings (2^-24 each) alone, however far it is."""
    g = torch.Generator(device=cuda).manual_seed(2)
    z = -torch.randint(20 * 64, 80 * 64, (n, v), generator=g, device=cuda).float() / 64 * temperature
    z[:, 7] = 0
    i = torch.tensor([7, 9, 11], device=cuda).expand(n, 3).contiguous()
    s = torch.randn(n, 3, generator=g, device=cuda)
    up = torch.rand(n, generator=g, device=cuda) + 0.5
    _, want, _, _, _ = reference_kd(z, i, s, up, temperature)
    _, dz = step_kd(z, i, s, up, temperature)
    rest = [k for k in range(v) if k not in (7, 9, 11)]
    assert ((dz.double() - want).abs()[:, rest] <= 2.0**-21 * want.abs()[:, rest]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(60, 64, 3000), (300, 72, 1003)])
def test_gradient_scales_far_from_each_other(cuda, dtype, n, d, v):
    """Rows whose gradients lie far apart, as of weights under a loss scale: each row of dX as near as any other."""
    x, w, t, _ = make_ce(cuda, n, d, v, dtype, 0.1)
    for top, bottom in ((17, -24), (10, -2), (0, -16), (-10, -40)):
        up = torch.exp2(torch.linspace(top, bottom, n, device=cuda)) * torch.where(torch.arange(n, device=cuda) % 3 == 0, -1.3, 1.0)
        up[n // 2] = 0
        loss, dx, dw = step_ce(x, w, t, up)
        # the bounds of check_ce with p itself, which holds for gradients of either sign; what lies above a type's largest value
        # (65504, under the scales of 2^17) is infinite in it
        _, rx, rw, dz, delta = reference_ce(x, w, t, up)
        u, most, tiny = half_step(dtype), torch.finfo(dtype).max, torch.finfo(dtype).tiny
        live = (t != -100)[:, None]
        p = torch.softmax((x.double() * live) @ w.double().t(), 1) * up.double().abs()[:, None] * live * (2 * delta + 2.0**-18)[:, None]
        for got, ref, err in ((dx, rx, (dz.abs() * (u + (128 + v / 256) * 2.0**-23) + p) @ w.double().abs()),
                              (dw, rw, (dz.abs() * (u + (128 + n / 256) * 2.0**-23) + p).t() @ (x.double() * live).abs())):
            err = err + u * ref.abs() + u * tiny
            over = ref.abs() + err > most
            assert ((got.double() - ref).abs() <= err)[~over].all(), "off by %g of its tolerance" % ((got.double() - ref).abs() / err)[~over].max()
            assert ((got.double() * ref.sign())[over] >= (ref.abs() - err).clamp(max=most)[over]).all()
        xs = x.detach().requires_grad_()
        (only,) = torch.autograd.grad(tc.linear_cross_entropy(xs, w, t), xs, up)
        assert torch.equal(only, dx)
        ws = w.detach().requires_grad_()
        (only,) = torch.autograd.grad(tc.linear_cross_entropy(x, ws, t), ws, up)
        assert torch.equal(only, dw)
        # a row's own scale changes nothing for the others
        big = up.abs() >= up.abs().max() * 2.0**-16
        alone = torch.where(big, up, torch.zeros_like(up))
        assert torch.equal(step_ce(x, w, t, alone)[1][big], dx[big])


def test_a_gradient_that_is_a_negated_view(cuda):
    """Behind complex arithmetic autograd hands on views that stand for the negative of what memory holds."""
    x, w, t, up = make_ce(cuda, 40, 64, 300, torch.float32)
    z, i, s, uk = make_kd(cuda, 40, 300, 5, torch.float32)
    for want, leaf, loss, g in ((step_ce(x, w, t, up)[1], x, lambda a: tc.linear_cross_entropy(a, w, t), up),
                                (step_kd(z, i, s, uk)[1], z, lambda a: tc.topk_distillation(a, i, s), uk)):
        leaf = leaf.detach().requires_grad_()
        view = torch.imag(torch.complex(g, -g).conj())
        assert view.is_neg() and torch.equal(view, g)
        (got,) = torch.autograd.grad(loss(leaf), leaf, view)
        assert torch.equal(got, want)
        # the imaginary part's gradient of a conjugate: -g
        (got,) = torch.autograd.grad(torch.complex(torch.zeros_like(g), loss(leaf)).conj(), leaf, torch.complex(g, g))
        assert torch.equal(got, -want)


@pytest.mark.parametrize("outlier", [2.0**10, 2.0**20, 2.0**24, 2.0**28])
@pytest.mark.parametrize("n,d,v", [(200, 256, 1000), (300, 1030, 700)])
def test_float32_rows_with_an_outlier(cuda, n, d, v, outlier):
    """A value far above the rest of its row of X (or of W) that meets zeros of W (or X) costs the other products nothing.  A logit's operands are
    off by 2^-22 each, the dropped product is 2^-22, values below 2^-29 of the row's largest keep 2^-50 of it, and the tensor core adds
    48 partial sums between drains with 2^-23 each."""
    x, w, t, up = make_ce(cuda, n, d, v, torch.float32, 0.1)
    x[:, 3], w[:, 3] = outlier, 0
    x[:, d - 2], w[:, d - 2] = 0, -outlier
    loss, dx, dw = step_ce(x, w, t, up)
    check_ce(x, w, t, up, loss, dx, dw)
    X, W = x.double().abs(), w.double().abs()
    X[:, 3], W[:, d - 2] = 0, 0  # (they meet zeros)
    delta = ((48 + d / 256 + 6) * 2.0**-23 * (X @ W.t()) + 2.0**-50 * outlier * (X.sum(1, keepdim=True) + W.sum(1))).amax(1)
    rl = reference_ce(x, w, t, up)[0]
    assert ((loss.double() - rl).abs() <= 2 * delta + 2.0**-20 * (1 + rl.abs())).all()

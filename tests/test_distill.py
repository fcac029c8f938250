"""Distillation from a teacher's top logits (ops/distill.py): the reference
against hand-written 64-bit formulas and differences on the CPU, the kernels
against the reference in 64 bits on the GPU."""
import math

import pytest
import torch

from lstm_tensorspark_amd.ops import distill
from lstm_tensorspark_amd.ops.distill import _ref_distill, distill_loss


def make(N, V, K, seed=0, dtype=torch.float64, dev="cpu", holes=True,
         index=torch.int64):
    g = torch.Generator().manual_seed(seed)
    z = 3.0 * torch.randn(N, V, generator=g)
    i = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(N)]) \
        if N else torch.zeros(0, K)
    t = 3.0 * torch.randn(N, K, generator=g)
    y = torch.randint(0, V, (N,), generator=g)
    if holes:
        drop = torch.rand(N, K, generator=g) < 0.2
        i = torch.where(drop, torch.where(torch.rand(N, K, generator=g) < .5,
                                          -1, V + 3), i)
        t[torch.rand(N, K, generator=g) < 0.1] = -math.inf
        for n in range(0, N, 5):
            i[n] = -1                      # rows without a teacher
        for n in range(0, N, 3):
            y[n] = (-100, -1, V)[n % 3]    # rows without a label
    return (z.to(dtype).to(dev), i.to(index).to(dev), t.to(dtype).to(dev),
            y.to(dev))


def by_hand(z, i, t, y, alpha, tau):
    """Loss and gradient of the definition, row by row."""
    z, t = z.double().cpu(), t.double().cpu()
    i, N, V = i.cpu(), z.shape[0], z.shape[1]
    total, count, d = 0.0, 0, torch.zeros(N, V, dtype=torch.float64)
    for n in range(N):
        ok = [(int(a), float(b)) for a, b in zip(i[n], t[n])
              if 0 <= int(a) < V and float(b) != -math.inf]
        label = y is not None and 0 <= int(y[n]) < V
        count += bool(ok) or label
        if ok and alpha != 0:
            q = torch.softmax(torch.tensor([b for _, b in ok],
                                           dtype=torch.float64) / tau, 0)
            lp = torch.log_softmax(z[n] / tau, 0)
            d[n] += alpha * tau * lp.exp()
            for (a, _), w in zip(ok, q):
                if w > 0:
                    total += float(alpha * tau * tau * w * (w.log() - lp[a]))
                d[n, a] -= alpha * tau * w
        if label and alpha != 1:
            lp = torch.log_softmax(z[n], 0)
            total -= float((1 - alpha) * lp[int(y[n])])
            d[n] += (1 - alpha) * lp.exp()
            d[n, int(y[n])] -= 1 - alpha
    return total / max(1, count), d / max(1, count)


SETTINGS = [(1.0, 1.0), (1.0, 2.0), (0.5, 1.0), (0.3, 4.0), (0.0, 2.0)]


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("alpha,tau", SETTINGS)
def test_reference_matches_the_definition(alpha, tau):
    z, i, t, y = make(11, 23, 7)
    z.requires_grad_()
    loss = distill_loss(z, i, t, y, alpha=alpha, temperature=tau)
    loss.backward()
    want, d = by_hand(z.detach(), i, t, y, alpha, tau)
    assert abs(float(loss.detach()) - want) < 1e-12 * max(1, abs(want))
    assert (z.grad - d).abs().max() < 1e-13


def test_reference_gradient_by_differences():
    z, i, t, y = make(6, 9, 4, seed=3)
    z.requires_grad_()
    assert torch.autograd.gradcheck(
        lambda a: distill_loss(a, i, t, y, alpha=0.4, temperature=2.0), (z,))


def test_same_index_twice_counts_twice():
    z = torch.randn(1, 5, dtype=torch.float64)
    t = torch.tensor([[1.0, 2.0, 0.5]], dtype=torch.float64)
    i = torch.tensor([[3, 3, 1]])
    want, _ = by_hand(z, i, t, None, 1.0, 1.5)
    assert abs(float(distill_loss(z, i, t, temperature=1.5)) - want) < 1e-13


def test_equal_distributions_lose_nothing():
    z = torch.randn(4, 8, dtype=torch.float64, requires_grad=True)
    i = torch.arange(8).repeat(4, 1)
    loss = distill_loss(z, i, z.detach(), temperature=3.0)
    loss.backward()
    assert abs(float(loss.detach())) < 1e-14 and z.grad.abs().max() < 1e-15


def test_rows_of_padding_are_not_counted():
    z, i, t, y = make(4, 10, 3, holes=False)
    full = distill_loss(z, i, t, y, alpha=0.5)
    zz = torch.cat([z, torch.full((3, 10), math.nan, dtype=z.dtype)])
    zz.requires_grad_()
    loss = distill_loss(zz, torch.cat([i, torch.full((3, 3), -1)]),
                        torch.cat([t, torch.zeros(3, 3, dtype=t.dtype)]),
                        torch.cat([y, torch.full((3,), -100)]), alpha=0.5)
    loss.backward()
    assert abs(float(loss.detach()) - float(full)) < 1e-14
    assert (zz.grad[4:] == 0).all()


def test_nothing_to_learn_from():
    z = torch.randn(3, 6, requires_grad=True)
    loss = distill_loss(z, torch.full((3, 2), -1), torch.zeros(3, 2))
    loss.backward()
    assert float(loss.detach()) == 0.0 and (z.grad == 0).all()
    assert float(distill_loss(torch.zeros(0, 6),
                              torch.zeros(0, 2, dtype=torch.long),
                              torch.zeros(0, 2))) == 0.0
    assert float(distill_loss(torch.randn(3, 6),
                              torch.zeros(3, 0, dtype=torch.long),
                              torch.zeros(3, 0))) == 0.0


def test_refusals():
    z, i, t, y = make(4, 10, 3)
    ok = dict(alpha=0.5)
    distill_loss(z, i, t, y, **ok)
    for args, kw in [
            ((z[0], i, t, y), ok), ((z, i[:2], t, y), ok),
            ((z, i, t[:, :2], y), ok), ((z, i.double(), t, y), ok),
            ((z, i, t.long(), y), ok), ((z.long(), i, t, y), ok),
            ((z, i, t, y[:2]), ok), ((z, i, t, y.int()), ok),
            ((z, i, t), ok), ((z, i, t, y), dict(alpha=1.5)),
            ((z, i, t, y), dict(alpha=math.nan)),
            ((z, i, t, y), dict(temperature=0.0)),
            ((z, i, t, y), dict(temperature=math.inf)),
            ((z, i, t, y), dict(temperature=1e-39)),
            ((z, i, t, y), dict(temperature=1e20)),
            ((z, i, t, y), dict(weight=math.nan)),
            ((z[:, :0], i, t, y), ok)]:
        with pytest.raises(ValueError):
            distill_loss(*args, **kw)


# ------------------------------------------------------------------- GPU
def check_on_gpu(z, i, t, y, alpha, tau, scale=1.0):
    """Kernel against the reference in 64 bits, on the same inputs.

    Loss: an fp32 sum of V/256 terms a thread and a tree behind it is off by
    (V/256 + 16) 2^-24 relative, which the logarithm turns into an absolute
    error; the terms themselves (|z| / tau, log q) are rounded about 8 times.
    Gradient: p and q are exp2 of an argument of at most ~64 that carries 3
    roundings, over a sum with the error above; then one rounding to the type,
    half a subnormal step where the value is that small.  The hardware's exp2
    gives zero for what lies below the smallest normal number, 2^-126: p and
    q are off by that much at most, whatever the type."""
    V = z.shape[1]
    n = max(1, int((((i >= 0) & (i < V) & (t != -math.inf)).any(1)
                    | (torch.zeros_like(i[:, 0] if i.shape[1] else z[:, 0])
                       .bool() if y is None else (y >= 0) & (y < V))).sum()))
    zk = z.detach().clone().requires_grad_()
    loss = distill_loss(zk, i, t, y, alpha=alpha, temperature=tau)
    (loss * scale).backward()
    zr = z.detach().double().requires_grad_()
    want = _ref_distill(zr, i, t.double(), y, alpha, tau)
    (want * scale).backward()
    u = 2.0 ** -24
    sums = (V / 256 + 16) * u
    big = 1 + float(z.detach().double().nan_to_num(0, 0, 0).abs().max()) / \
        min(1.0, tau)           # of padding rows nothing is computed
    assert loss.dtype == torch.float32
    tol = max(1.0, tau * tau) * (sums + 8 * big * u)
    assert abs(float(loss.detach()) - float(want.detach())) <= tol
    p = (torch.softmax(zr.detach() / tau, 1)
         + torch.softmax(zr.detach(), 1)).nan_to_num(0)
    q = (zr.grad / scale).abs() * n
    exps = 3 * 64 * u + sums
    eps = torch.finfo(z.dtype).eps / 2
    tiny = torch.finfo(z.dtype).smallest_normal * eps * 2
    bound = eps * zr.grad.abs() * (1 + 1e-3) + tiny + \
        abs(scale) / n * max(1.0, tau) * (4 * exps * (p + q) + 2.0 ** -125)
    off = (zk.grad.double() - zr.grad).abs()
    assert zk.grad.dtype == z.dtype
    assert (off <= bound).all(), float((off - bound).max())
    return loss.detach(), zk.grad


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (1, 7, 3), (3, 257, 16),
                                   (37, 2049, 33), (5, 50000, 64),
                                   (600, 1001, 20), (513, 4096, 4096),
                                   (2, 70001, 300)])
def test_kernel_sizes(dtype, N, V, K):
    z, i, t, y = make(N, V, K, seed=N + V, dtype=dtype, dev="cuda")
    for alpha, tau in ((1.0, 1.0), (0.6, 2.0)):
        check_on_gpu(z, i, t, y, alpha, tau)


@pytest.mark.gpu
@pytest.mark.parametrize("alpha,tau", SETTINGS)
def test_kernel_settings(alpha, tau):
    z, i, t, y = make(29, 1003, 17, seed=5, dtype=torch.bfloat16, dev="cuda",
                      index=torch.int32)
    check_on_gpu(z, i, t.float(), y, alpha, tau, scale=0.125)
    check_on_gpu(z, i, t.half(), y, alpha, tau, scale=-3.0)
    if alpha == 1.0:
        check_on_gpu(z, i, t, None, alpha, tau)


@pytest.mark.gpu
def test_kernel_large_logits():
    z, i, t, y = make(16, 999, 9, seed=6, dtype=torch.float32, dev="cuda")
    check_on_gpu(z * 300, i, t, y, 0.5, 2.0)


@pytest.mark.gpu
def test_kernel_strides_and_duplicates():
    z, i, t, y = make(12, 640, 8, seed=7, dtype=torch.bfloat16, dev="cuda")
    wide = torch.randn(12, 999, device="cuda").bfloat16()
    wide[:, 13:653] = z
    i[:, 3] = i[:, 1]
    i[:, 5] = i[:, 1]
    i[4, :] = 17
    y[4] = 17
    y[1] = i[1].clamp(0, 639)[2]
    i2 = torch.empty(12, 16, dtype=torch.long, device="cuda")[:, ::2]
    i2.copy_(i)
    a = check_on_gpu(z, i, t, y, 0.5, 2.0)
    b = check_on_gpu(wide[:, 13:653], i2, t.t().contiguous().t(), y, 0.5, 2.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = distill_loss(z.t().contiguous().t(), i, t, y, alpha=.5, temperature=2.)
    assert torch.equal(a[0], c)


@pytest.mark.gpu
def test_kernel_infinities_and_padding():
    z, i, t, y = make(6, 500, 5, seed=8, dtype=torch.bfloat16, dev="cuda",
                      holes=False)
    z[0, ::3] = -math.inf               # masked places of the student
    i[0] = torch.tensor([1, 2, 4, 5, 7])
    y[0] = 10
    i[1], y[1] = -1, -100               # padding: NaN and inf inside
    z[1] = math.nan
    i[2], y[2] = 500, 500
    z[2] = math.inf
    t[3] = -math.inf                    # nothing left of the teacher's list
    _, d = check_on_gpu(z, i, t, y, 0.5, 2.0)
    assert (d[1:3] == 0).all() and (d[0, ::3] == 0).all()
    low = torch.finfo(torch.bfloat16).min     # masked by the lowest value
    a, b = z.clone(), z.clone()
    a[4, 7:20], b[4, 7:20] = low, -math.inf
    i[4] = torch.tensor([1, 2, 30, 40, 50])
    y[4] = 2
    got = [distill_loss(x.requires_grad_(), i, t, y, alpha=.5) for x in (a, b)]
    ga, gb = (torch.autograd.grad(f, x)[0] for f, x in zip(got, (a, b)))
    assert torch.equal(*got) and torch.equal(ga, gb)
    # a row that holds the lowest value everywhere is uniform
    a = torch.full((1, 500), low, device="cuda").bfloat16()
    want = math.log(500) - math.log(5)
    for tau in (0.01, 1.0):
        f = distill_loss(a, i[4:5], torch.zeros_like(t[:1]), temperature=tau)
        assert abs(float(f) / tau ** 2 - want) < 1e-5
    bad = z.clone()
    bad[5] = math.nan
    zr = bad.clone().requires_grad_()
    loss = distill_loss(zr, i, t, y, alpha=0.5)
    loss.backward()
    assert torch.isnan(loss) and torch.isnan(zr.grad[5]).all()
    assert torch.isfinite(zr.grad[:5]).all()
    # an entry that the student rules out costs infinitely much
    bad = z.clone()
    bad[4, int(i[4, 0])] = -math.inf
    assert float(distill_loss(bad, i, t, y, alpha=0.5)) == math.inf


@pytest.mark.gpu
def test_kernel_empty():
    z = torch.zeros(0, 9, device="cuda", requires_grad=True)
    loss = distill_loss(z, torch.zeros(0, 2, dtype=torch.long, device="cuda"),
                        torch.zeros(0, 2, device="cuda"))
    loss.backward()
    assert float(loss.detach()) == 0 and z.grad.shape == (0, 9)
    z = torch.randn(3, 9, device="cuda", requires_grad=True)
    loss = distill_loss(z, torch.zeros(3, 0, dtype=torch.long, device="cuda"),
                        torch.zeros(3, 0, device="cuda"))
    loss.backward()
    assert float(loss.detach()) == 0 and (z.grad == 0).all()


@pytest.mark.gpu
def test_kernel_gradient_by_differences():
    """Along a direction d: (f(z + h d) - f(z - h d)) / 2h is off by h^2/6
    times a third derivative (of order |d|^3 <= 1 here) and by the loss's own
    rounding, 2 * 30 * 2^-24 over 2h."""
    z, i, t, y = make(7, 300, 11, seed=9, dtype=torch.float32, dev="cuda")
    z.requires_grad_()
    f = lambda a: distill_loss(a, i, t, y, alpha=0.5, temperature=2.0)  # noqa: E731
    g, = torch.autograd.grad(f(z), z)
    d = torch.randn(z.shape, device="cuda")
    d /= d.norm()
    h = 0.02
    with torch.no_grad():
        diff = (f(z + h * d) - f(z - h * d)) / (2 * h)
    assert abs(float(diff) - float((g * d).sum())) < h * h / 6 + 2 * 30 * 2 ** -24 / h


@pytest.mark.gpu
def test_kernel_repeats_bitwise_on_another_stream():
    z, i, t, y = make(300, 5000, 31, seed=10, dtype=torch.bfloat16, dev="cuda")
    a = check_on_gpu(z, i, t, y, 0.5, 2.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        zz = z.clone().requires_grad_()
        loss = distill_loss(zz, i, t, y, alpha=0.5, temperature=2.0)
        g, = torch.autograd.grad(loss, zz)
    s.synchronize()
    assert torch.equal(a[0], loss.detach()) and torch.equal(a[1], g)


@pytest.mark.gpu
def test_kernel_captured_and_replayed():
    N, V, K = 40, 3000, 8
    z, i, t, y = make(N, V, K, seed=11, dtype=torch.bfloat16, dev="cuda")
    zs = z.clone().requires_grad_()
    step = lambda: distill_loss(zs, i, t, y, alpha=0.5, temperature=2.0)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(step(), zs)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
        g, = torch.autograd.grad(loss, zs)
    for seed in (12, 13, 14):
        z2, i2, t2, y2 = make(N, V, K, seed=seed, dtype=torch.bfloat16,
                              dev="cuda")
        with torch.no_grad():
            zs.copy_(z2)
        i.copy_(i2), t.copy_(t2), y.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        want = check_on_gpu(z2, i2, t2, y2, 0.5, 2.0)
        assert torch.equal(loss.detach(), want[0]) and torch.equal(g, want[1])


@pytest.mark.gpu
def test_kernel_backward_captured_apart():
    """A backward pass in a graph of its own writes its gradient at every
    replay, also where the forward in another graph had left it."""
    z, i, t, y = make(40, 3000, 8, seed=15, dtype=torch.bfloat16, dev="cuda")
    zs = z.clone().requires_grad_()
    step = lambda: distill_loss(zs, i, t, y, alpha=0.5, temperature=2.0)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(step(), zs)
    torch.cuda.current_stream().wait_stream(s)
    fwd, bwd = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(fwd, stream=s):
        loss = step()
    with torch.cuda.graph(bwd, stream=s, pool=fwd.pool()):
        g, = torch.autograd.grad(loss, zs)
    for seed in (16, 17):
        z2 = make(40, 3000, 8, seed=seed, dtype=torch.bfloat16, dev="cuda")[0]
        with torch.no_grad():
            zs.copy_(z2)
        fwd.replay()
        want = check_on_gpu(z2, i, t, y, 0.5, 2.0)
        for _ in range(3):
            g.zero_()
            bwd.replay()
            torch.cuda.synchronize()
            # from the logits again: the same numbers, in another kernel
            assert torch.equal(loss.detach(), want[0])
            off = (g.double() - want[1].double()).abs()
            assert (off <= 2.0 ** -7 * want[1].double().abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 9000, 40000, 57344, 57345])
def test_kernel_weight_and_incoming_gradients(V, dtype):
    """The gradient that the forward leaves (g = 1), the one that the backward
    computes anew, and a kept graph's second and third pass."""
    z, i, t, y = make(9, V, 12, seed=15, dtype=dtype, dev="cuda")
    i[4, 1] = i[4, 0]
    for tau in (1.0, 2.0, 3.0, 4.0):
        _, one = check_on_gpu(z, i, t, y, 0.5, tau)
        _, quarter = check_on_gpu(z, i, t, y, 0.5, tau, scale=0.25)
        zs = z.clone().requires_grad_()
        kw = dict(alpha=0.5, temperature=tau)
        loss = distill_loss(zs, i, t, y, weight=0.25, **kw)
        g = [torch.autograd.grad(loss, zs, retain_graph=True)[0]
             for _ in range(2)]
        full, = torch.autograd.grad(4.0 * loss, zs)
        plain = distill_loss(z, i, t, y, **kw)
        with torch.no_grad():
            assert torch.equal(plain, distill_loss(zs, i, t, y, **kw))
        assert abs(float(loss.detach()) - float(plain) / 4) <= \
            2 ** -23 * abs(float(plain))
        # the sums are the same: a factor of 4 moves only subnormal roundings
        tiny = torch.finfo(dtype).smallest_normal
        for a, b in ((g[0], quarter), (g[1], quarter), (full, one)):
            assert ((a == b) | ((a - b).abs() <= tiny)).all()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(distill_loss(zs, i, t, y, alpha=0.5), zs,
                            create_graph=True)


@pytest.mark.gpu
def test_kernel_is_what_runs(monkeypatch):
    z, i, t, y = make(4, 50, 3, dtype=torch.bfloat16, dev="cuda")
    monkeypatch.setattr(distill, "_ref_distill", None)
    distill_loss(z, i, t, y, alpha=0.5)


@pytest.mark.gpu
def test_kernel_refusals(monkeypatch):
    """The same refusals, raised before anything is launched."""
    plain = make
    monkeypatch.setitem(globals(), "make", lambda *a: plain(
        *a, dtype=torch.bfloat16, dev="cuda"))
    test_refusals()


@pytest.mark.gpu
def test_kernel_teacher_gets_no_gradient():
    z, i, t, y = make(6, 300, 5, dtype=torch.bfloat16, dev="cuda")
    want = distill_loss(z, i, t.double(), y, alpha=0.5)
    t = t.double().requires_grad_()
    loss = distill_loss(z, i, t, y, alpha=0.5)
    assert torch.equal(loss, want) and not loss.requires_grad
    z.requires_grad_()
    distill_loss(z, i, t, y, alpha=0.5).backward()
    assert t.grad is None and z.grad is not None


@pytest.mark.gpu
def test_kernel_refuses_forward_mode():
    fw = torch.autograd.forward_ad
    z, i, t, y = make(4, 50, 3, dtype=torch.bfloat16, dev="cuda")
    with fw.dual_level():
        with pytest.raises(RuntimeError):
            distill_loss(fw.make_dual(z, torch.ones_like(z)), i, t, y,
                         alpha=0.5)


def seconds(f):
    """The least of three runs on the GPU, after one."""
    f()
    times = []
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,K", [(300, 250), (9000, 4096), (40000, 5000),
                                 (60000, 5000)])
def test_kernel_long_lists_with_repeats(V, K, dtype):
    """One index twice, and few indices a hundred times each: their entries
    are summed in fp32, at most 128 of them, within the bound of
    `check_on_gpu` (four times 192 roundings of q)."""
    for few in (None, max(2, K // 40), 2 * WIDE):
        z, i, t, y = make(3, V, K, seed=K, dtype=dtype, dev="cuda")
        if few is None:
            i[:, K // 3] = i[:, K - 1]
        elif few >= V:
            continue
        else:
            i = (torch.arange(K, device="cuda") * 7 % few * (V // few)) \
                .repeat(3, 1)
            i[1] = torch.where(i[1] < V // 2, i[1], -1)
        y[0], y[1] = i[0, K - 1].clamp(0, V - 1), V - 1
        a = check_on_gpu(z, i, t, y, 0.5, 2.0)
        check_on_gpu(z, i, t, y, 1.0, 1.0, scale=0.5)
        b = check_on_gpu(z, i, t, y, 0.5, 2.0)
        assert torch.equal(a[1], b[1])


WIDE = 256      # columns that one wave sums repeated entries of at once


@pytest.mark.gpu
def test_kernel_one_repeat_costs_no_walk_an_entry():
    """Work is linear in the list's length, with repeats or without: a walk
    through 20000 entries for each of them took five hundred times as long."""
    z, i, t, _ = make(2, 50000, 20000, dtype=torch.bfloat16, dev="cuda",
                      holes=False)
    z.requires_grad_()
    for scale in (1.0, 2.0):
        def go():
            (scale * distill_loss(z, i, t)).backward()
        plain = seconds(go)
        old = i[:, 777].clone()
        i[:, 777] = i[:, 19000]
        assert seconds(go) < 20 * plain
        i[:, 777] = old

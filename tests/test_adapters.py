"""Low-rank adapters by row (ops/adapters.py): the reference against row by
row products and differences on the CPU, the kernels against products in 64
bits, with error bounds carried through them, on the GPU."""
import pytest
import torch

from lstm_tensorspark_amd.ops import adapters as mod
from lstm_tensorspark_amd.ops.adapters import (AdapterRows, lowrank_add,
                                               lowrank_add_)


def make(T, B, K, M, R, L, seed=0, dtype=torch.float64, dev="cpu", idle=0.25,
         index=None):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g)

    if index is None:
        index = torch.randint(0, L, (B,), generator=g)
        index[torch.rand(B, generator=g) < idle] = -1
        index = index.tolist()
    t = dict(y=r(T, B, M), x=r(T, B, K), a=r(L, K, R) / K ** 0.5,
             b=r(L, R, M) / R ** 0.5)
    t = {n: v.to(dtype).to(dev) for n, v in t.items()}
    return t, AdapterRows(index, L, device=dev), \
        (0.5 + torch.rand(L, generator=g)).to(dev)


def by_hand(t, rows, scale):
    out = t["y"].clone()
    for c, l in enumerate(rows.index):
        if l >= 0:
            s = float(scale[l]) if isinstance(scale, torch.Tensor) else scale
            out[:, c] += s * (t["x"][:, c] @ t["a"][l]) @ t["b"][l]
    return out


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("T,B,K,M,R,L", [(1, 1, 3, 2, 1, 1), (4, 7, 9, 5, 2, 3),
                                         (3, 5, 8, 8, 4, 9)])
def test_reference_matches_row_by_row(T, B, K, M, R, L):
    t, rows, scale = make(T, B, K, M, R, L)
    scale = scale.double()
    for s in (scale, 0.7):
        assert (lowrank_add(**t, rows=rows, scale=s)
                - by_hand(t, rows, s)).abs().max() < 1e-13
    y = t.pop("y")
    want = lowrank_add(y, **t, rows=rows, scale=scale)
    assert lowrank_add_(y, **t, rows=rows, scale=scale) is y
    assert torch.equal(y, want)


def test_reference_gradients_by_differences():
    t, rows, scale = make(2, 4, 3, 5, 2, 3, seed=1)
    v = [t[n].requires_grad_() for n in ("y", "x", "a", "b")]
    assert torch.autograd.gradcheck(
        lambda *v: lowrank_add(*v, rows=rows, scale=scale.double()), v)


def test_grouping():
    r = AdapterRows([2, -1, 0, 2, 0, 2], 4)
    assert r.order.tolist() == [1, 2, 4, 0, 3, 5]
    assert r.segs.view(-1, 4).tolist() == [[-1, 0, 1, 0], [0, 1, 2, 0],
                                           [2, 3, 3, 0]]
    assert r.counts == [1, 2, 3] and r.adapter.tolist() == list(r.index)
    assert AdapterRows(torch.tensor([0, -1]), 1).index == (0, -1)
    for bad in ([], [4], [-2]):
        with pytest.raises(ValueError):
            AdapterRows(bad, 4)
    with pytest.raises(ValueError):
        AdapterRows([0], 0)
    with pytest.raises(ValueError):
        AdapterRows(torch.tensor([0.0]), 1)


def test_rows_without_an_adapter_and_empty_sequences():
    t, _, _ = make(3, 4, 5, 6, 2, 2)
    rows = AdapterRows([-1] * 4, 2)
    assert torch.equal(lowrank_add(**t, rows=rows), t["y"])
    z = {n: v[:0] if n in "xy" else v for n, v in t.items()}
    assert lowrank_add(**z, rows=rows).shape == (0, 4, 6)


def test_refusals():
    t, rows, scale = make(2, 4, 5, 6, 2, 3)
    scale = scale.double()
    lowrank_add(**t, rows=rows, scale=scale)
    for over in [dict(a=t["a"][0]), dict(a=t["a"][:2]),
                 dict(b=t["b"][:, :1]), dict(x=t["x"][:, :3]),
                 dict(x=t["x"][..., :4]), dict(y=t["y"][..., :4]),
                 dict(y=t["y"].float()), dict(rows=[0, 1, 2, 0]),
                 dict(rows=AdapterRows([0] * 5, 3)),
                 dict(rows=AdapterRows([0] * 4, 2)),
                 dict(scale=scale[:2]), dict(scale=float("nan")),
                 dict(scale=torch.ones(3, dtype=torch.long)),
                 dict(scale=scale.clone().requires_grad_()),
                 dict(a=t["a"][..., :0], b=t["b"][:, :0]),
                 dict(a=torch.zeros(3, 5, 129, dtype=torch.float64),
                      b=torch.zeros(3, 129, 6, dtype=torch.float64)),
                 dict(x=t["x"][0, 0], y=t["y"][0, 0])]:
        args = {**t, "rows": rows, "scale": scale, **over}
        with pytest.raises(ValueError):
            lowrank_add(**args)
        with pytest.raises(ValueError):
            lowrank_add_(**args)
    with pytest.raises(ValueError):
        lowrank_add_(**{**t, "y": t["y"].transpose(0, 1).contiguous()
                        .transpose(0, 1)}, rows=rows)


# ------------------------------------------------------------------- GPU
def bounds(t, dy, rows, scale):
    """Results in 64 bits and how far rounding may put the kernels off them.

    A sum of n products in fp32 is off by at most n 2^-24 of the sum of
    magnitudes; v = s x A and u = s dy B^T are rounded to the type once, and
    that error passes through the next product; each result is rounded once."""
    dt = t["x"].dtype
    eps, w = torch.finfo(dt).eps / 2, 2.0 ** -24
    tiny = torch.finfo(dt).smallest_normal * eps * 2
    y, x, a, b = (t[n].double().cpu() for n in ("y", "x", "a", "b"))
    dy = dy.double().cpu()
    T, B, K = x.shape
    M, R = b.shape[2], b.shape[1]
    r = dict(out=y.clone(), x=torch.zeros_like(x), a=torch.zeros_like(a),
             b=torch.zeros_like(b))
    e = {n: torch.zeros_like(v) for n, v in r.items()}
    for l in sorted(set(rows.index) - {-1}):
        c = [i for i, k in enumerate(rows.index) if k == l]
        s = float(scale[l]) if isinstance(scale, torch.Tensor) else scale
        xs, ds = x[:, c].reshape(-1, K), dy[:, c].reshape(-1, M)
        n = xs.shape[0]
        v, u = s * xs @ a[l], s * ds @ b[l].t()
        ev = (K + 8) * w * abs(s) * xs.abs() @ a[l].abs()
        ev += eps * (v.abs() + ev) + tiny
        eu = (M + 8) * w * abs(s) * ds.abs() @ b[l].abs().t()
        eu += eps * (u.abs() + eu) + tiny

        def put(name, value, err, shape):
            r[name][:, c] += value.reshape(T, len(c), shape)
            e[name][:, c] += err.reshape(T, len(c), shape)

        put("out", v @ b[l],
            (ev + R * w * (v.abs() + ev)) @ b[l].abs(), M)
        put("x", u @ a[l].t(), (eu + R * w * (u.abs() + eu)) @ a[l].abs().t(), K)
        r["a"][l] = xs.t() @ u
        e["a"][l] = xs.abs().t() @ (eu + (n + 8) * w * (u.abs() + eu))
        r["b"][l] = v.t() @ ds
        e["b"][l] = (ev + (n + 8) * w * (v.abs() + ev)).t() @ ds.abs()
    for k in r:
        e[k] = e[k] * (1 + 1e-3) + (eps + 2 * w) * r[k].abs() + \
            eps * e[k] + tiny
    return r, e


def check_on_gpu(t, rows, scale, grad=True):
    g = torch.Generator().manual_seed(99)
    dy = torch.randn(t["y"].shape, generator=g).to(t["y"])
    want, err = bounds(t, dy, rows, scale)
    v = {n: p.detach().clone().requires_grad_() for n, p in t.items()}
    out = lowrank_add(**v, rows=rows, scale=scale)
    got = {"out": out}
    if grad:
        gy, got["x"], got["a"], got["b"] = torch.autograd.grad(
            out, [v[n] for n in ("y", "x", "a", "b")], dy)
        assert torch.equal(gy, dy)
    for n, p in got.items():
        assert p.dtype == t["x"].dtype and p.shape == want[n].shape
        off = (p.detach().double().cpu() - want[n]).abs()
        assert (off <= err[n]).all(), (n, float((off / err[n]).max()))
    with torch.no_grad():       # nothing kept for a backward pass
        plain = lowrank_add(**t, rows=rows, scale=scale)
    assert (plain.double().cpu() - want["out"]).abs().le(err["out"]).all()
    y = t["y"].detach().clone()
    lowrank_add_(y, *(t[n] for n in "xab"), rows=rows, scale=scale)
    assert (y.double().cpu() - want["out"]).abs().le(err["out"]).all()
    for c, l in enumerate(rows.index):
        if l < 0:       # untouched
            assert torch.equal(y[:, c], t["y"][:, c])
            assert torch.equal(out[:, c], t["y"][:, c])
    return {n: p.detach() for n, p in got.items()}


SHAPES = [
    # T, B, K, M, R, L
    (1, 1, 8, 8, 1, 1), (1, 1, 1, 1, 1, 1), (1, 1, 1024, 4096, 16, 8),
    (1, 3, 37, 41, 5, 2), (1, 64, 256, 1000, 16, 24), (1, 17, 129, 257, 33, 3),
    (1, 33, 1000, 777, 100, 5), (5, 7, 100, 300, 12, 4), (1, 70, 64, 64, 8, 70),
    (64, 3, 128, 513, 16, 2), (37, 29, 101, 259, 12, 6), (130, 9, 65, 70, 128, 2),
    (300, 1, 520, 136, 64, 1), (3, 200, 300, 90, 32, 100), (1, 1, 9000, 9001, 24, 1),
    (1, 5, 2050, 50, 3, 5),
    # u in wide shares of columns, few and many of them
    (64, 70, 40, 8001, 16, 2), (20, 53, 33, 16901, 20, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_kernel_sizes(shape, dtype):
    t, rows, scale = make(*shape, seed=sum(shape), dtype=dtype, dev="cuda")
    check_on_gpu(t, rows, scale)
    t, rows, _ = make(*shape, seed=1, dtype=dtype, dev="cuda", idle=0.0)
    check_on_gpu(t, rows, -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 32, 33, 63,
                               64, 65, 127, 129])
def test_kernel_group_sizes(n):
    """One adapter with n rows beside others with one, in mixed order."""
    index = [1] * n + [0, 2, -1, 3]
    index = [index[(i * 7) % len(index)] if len(index) % 7 else index[i]
             for i in range(len(index))]
    for T in (1, 3):
        t, rows, scale = make(T, len(index), 72, 200, 16, 4, seed=n,
                              dtype=torch.bfloat16, dev="cuda", index=index)
        check_on_gpu(t, rows, scale)


@pytest.mark.gpu
def test_kernel_no_row_has_an_adapter():
    t, rows, scale = make(3, 5, 40, 50, 4, 3, dtype=torch.bfloat16,
                          dev="cuda", index=[-1] * 5)
    g = check_on_gpu(t, rows, scale)
    assert all((g[n] == 0).all() for n in "xab")


@pytest.mark.gpu
def test_kernel_other_rows_do_not_leak():
    """NaN and inf in one sequence stay in it, and in its adapter."""
    t, rows, scale = make(4, 6, 64, 300, 8, 4, dtype=torch.bfloat16,
                          dev="cuda", index=[0, 1, 2, -1, 1, 0])
    clean = check_on_gpu(t, rows, scale)
    t["x"][:, 2] = float("nan")
    t["x"][1, 3] = float("inf")
    t["y"][0, 3] = float("nan")
    t["a"][3] = float("nan")
    t["b"][3] = float("inf")
    v = {n: p.clone().requires_grad_() for n, p in t.items()}
    out = lowrank_add(**v, rows=rows, scale=scale)
    keep = [0, 1, 4, 5]
    assert torch.equal(out[:, keep], clean["out"][:, keep])
    g = torch.Generator().manual_seed(99)
    dy = torch.randn(t["y"].shape, generator=g).to(t["y"])
    dx, da, db = torch.autograd.grad(out, [v[n] for n in "xab"], dy)
    assert torch.equal(dx, clean["x"])
    assert torch.equal(da[:2], clean["a"][:2]) and (da[3] == 0).all()
    assert torch.equal(db[:2], clean["b"][:2]) and (db[3] == 0).all()
    assert torch.isnan(db[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 5, 16, 31, 33, 100])
@pytest.mark.parametrize("K", [40, 2000])
def test_kernel_an_infinity_stays_one(K, R):
    """An overflow is not turned into NaN by ranks that fill no tile."""
    t, rows, _ = make(1, 70, K, 90, R, 2, dtype=torch.bfloat16, dev="cuda",
                      index=[0] * 70)
    t = {n: p.abs() + 0.01 for n, p in t.items()}
    t["x"][0, 3, 1] = float("inf")
    with torch.no_grad():
        few = lowrank_add(t["y"][:, :4], t["x"][:, :4], t["a"], t["b"],
                          AdapterRows([0] * 4, 2, device="cuda"))
    assert (few[0, 3] == float("inf")).all()
    v = {n: p.clone().requires_grad_() for n, p in t.items()}
    out = lowrank_add(**v, rows=rows)
    dy = torch.ones_like(out)
    dy[0, 5, 7] = float("inf")
    dx, = torch.autograd.grad(out, [v["x"]], dy)
    assert (out[0, 3] == float("inf")).all()
    assert (dx[0, 5] == float("inf")).all()
    rest = [i for i in range(70) if i not in (3, 5)]
    assert out[0, rest].isfinite().all() and dx[0, rest].isfinite().all()


@pytest.mark.gpu
def test_kernel_strides():
    t, rows, scale = make(1, 9, 50, 70, 6, 3, dtype=torch.bfloat16, dev="cuda")
    want = check_on_gpu(t, rows, scale)["out"]
    wide = torch.randn(9, 131, device="cuda").bfloat16()
    wide[:, 3:53] = t["x"][0]
    wide_y = torch.randn(9, 171, device="cuda").bfloat16()
    wide_y[:, 1:71] = t["y"][0]
    a = t["a"].transpose(1, 2).contiguous().transpose(1, 2)
    got = lowrank_add(wide_y[:, 1:71], wide[:, 3:53], a, t["b"], rows, scale)
    assert torch.equal(got, want[0])
    got = lowrank_add(t["y"][0].t().contiguous().t(),
                      t["x"][0].t().contiguous().t(), a, t["b"], rows, scale)
    assert torch.equal(got, want[0])
    # one row for all: a broadcast input's gradient is the rows' sum
    x1 = t["x"][:, :1].clone().requires_grad_()
    out = lowrank_add(t["y"], x1.expand(1, 9, 50), t["a"], t["b"], rows, scale)
    g1, = torch.autograd.grad(out.float().sum(), x1)
    x2 = t["x"][:, :1].expand(1, 9, 50).contiguous().requires_grad_()
    out2 = lowrank_add(t["y"], x2, t["a"], t["b"], rows, scale)
    g2, = torch.autograd.grad(out2.float().sum(), x2)
    assert torch.equal(out, out2) and torch.equal(g1, g2.sum(1, keepdim=True))


@pytest.mark.gpu
@pytest.mark.parametrize("B,K,M,R", [(64, 70, 300, 16), (128, 257, 257, 5),
                                     (100, 33, 1031, 40), (65, 9, 511, 128),
                                     (3, 300, 1025, 16)])
def test_kernel_what_lies_behind_the_rows_is_not_used(B, K, M, R):
    """Rows inside wider ones whose other columns hold NaN: the same bits."""
    t, rows, scale = make(1, B, K, M, R, 3, dtype=torch.bfloat16, dev="cuda")
    g = torch.Generator().manual_seed(5)
    t["dy"] = torch.randn(1, B, M, generator=g).to(t["y"])

    def inside(p):
        wide = torch.full((1, B, p.shape[-1] + 19), float("nan"),
                          device="cuda", dtype=p.dtype)
        wide[..., 6:6 + p.shape[-1]] = p
        return wide[..., 6:6 + p.shape[-1]]

    got = []
    for put in (lambda p: p, inside):
        v = {n: put(t[n]).detach().requires_grad_() for n in "yx"}
        v.update({n: t[n].clone().requires_grad_() for n in "ab"})
        out = lowrank_add(**v, rows=rows, scale=scale)
        got.append((out, *torch.autograd.grad(out, list(v.values()),
                                              put(t["dy"]))))
        with torch.no_grad():
            got[-1] += (lowrank_add(**v, rows=rows, scale=scale),)
    assert all(torch.equal(p, q) for p, q in zip(*got))
    assert all(p.isfinite().all() for p in got[0])


@pytest.mark.gpu
def test_kernel_some_gradients_only():
    for R in (8, 40):
        t, rows, scale = make(20, 6, 80, 90, R, 3, dtype=torch.bfloat16,
                              dev="cuda")
        g = torch.Generator().manual_seed(99)
        dy = torch.randn(t["y"].shape, generator=g).to(t["y"])
        want, err = bounds(t, dy, rows, scale)
        for names in ("x", "a", "b", "xa", "xb", "ab"):
            v = {n: p.clone().requires_grad_(n in names)
                 for n, p in t.items()}
            out = lowrank_add(**v, rows=rows, scale=scale)
            got = torch.autograd.grad(out, [v[n] for n in names], dy)
            for n, p in zip(names, got):
                assert ((p.double().cpu() - want[n]).abs() <= err[n]).all()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(lowrank_add(**v, rows=rows, scale=scale),
                                v["a"], dy, create_graph=True)


@pytest.mark.gpu
def test_kernel_repeats_bitwise_on_another_stream():
    t, rows, scale = make(40, 50, 300, 700, 16, 7, dtype=torch.bfloat16,
                          dev="cuda")
    want = check_on_gpu(t, rows, scale)
    g = torch.Generator().manual_seed(99)
    dy = torch.randn(t["y"].shape, generator=g).to(t["y"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        v = {n: p.clone().requires_grad_() for n, p in t.items()}
        out = lowrank_add(**v, rows=rows, scale=scale)
        grads = torch.autograd.grad(out, [v[n] for n in "xab"], dy)
    s.synchronize()
    assert torch.equal(out, want["out"])
    assert all(torch.equal(p, want[n]) for n, p in zip("xab", grads))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_kernel_rows_may_end_before_another_stream_does(grad):
    """Rows that nobody keeps, used on a stream that is not theirs: their
    memory is not given away while that stream has work to do."""
    t, rows, _ = make(4, 40, 64, 300, 8, 3, dtype=torch.bfloat16, dev="cuda")
    index = list(rows.index)
    want = lowrank_add(**t, rows=rows)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    if grad:
        t["x"].requires_grad_()
    dy = torch.ones_like(want)
    for _ in range(3):
        rows = AdapterRows(index, 3, device="cuda")
        at = rows.segs.data_ptr()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.cuda._sleep(20_000_000)
            out = lowrank_add(**t, rows=rows)
            if grad:
                torch.cuda._sleep(20_000_000)
                torch.autograd.grad(out, t["x"], dy)
        del rows
        out = out.detach()
        again = [AdapterRows(index, 3, device="cuda") for _ in range(4)]
        assert all(r.segs.data_ptr() != at for r in again)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 30])
def test_kernel_captured_and_replayed(T):
    shape = (T, 12, 200, 330, 16, 5)
    t, rows, scale = make(*shape, dtype=torch.bfloat16, dev="cuda")
    v = {n: p.clone().requires_grad_() for n, p in t.items()}
    g = torch.Generator().manual_seed(99)
    dy = torch.randn(t["y"].shape, generator=g).to(t["y"])

    def step():
        out = lowrank_add(**v, rows=rows, scale=scale)
        return out, torch.autograd.grad(out, [v[n] for n in "xab"], dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = step()
    for seed in (3, 4, 5):
        t2, _, _ = make(*shape, seed=seed, dtype=torch.bfloat16, dev="cuda",
                        index=list(rows.index))
        with torch.no_grad():
            for n in v:
                v[n].copy_(t2[n])
        graph.replay()
        torch.cuda.synchronize()
        want = check_on_gpu(t2, rows, scale)
        assert torch.equal(out, want["out"])
        assert all(torch.equal(p, want[n]) for n, p in zip("xab", grads))


@pytest.mark.gpu
def test_kernel_in_place_is_seen_by_autograd():
    t, rows, scale = make(1, 3, 16, 24, 4, 2, dtype=torch.bfloat16, dev="cuda",
                          index=[0, 1, -1])
    w = torch.randn(24, device="cuda").bfloat16().requires_grad_()
    out = (t["y"] * w).sum()            # keeps y for its backward pass
    lowrank_add_(t["y"], t["x"], t["a"], t["b"], rows, scale)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.backward()


@pytest.mark.gpu
def test_kernel_input_and_output_are_one_tensor():
    t, rows, scale = make(2, 5, 48, 48, 6, 2, dtype=torch.bfloat16, dev="cuda")
    t["x"] = t["y"].clone()
    want, err = bounds(t, torch.zeros_like(t["y"]), rows, scale)
    y = t["y"].clone()
    lowrank_add_(y, y, t["a"], t["b"], rows, scale)
    assert ((y.double().cpu() - want["out"]).abs() <= err["out"]).all()


@pytest.mark.gpu
def test_kernel_is_what_runs(monkeypatch):
    t, rows, scale = make(1, 4, 16, 16, 4, 2, dtype=torch.bfloat16, dev="cuda")
    monkeypatch.setattr(mod, "_ref_lowrank", None)
    lowrank_add(**t, rows=rows, scale=scale)


@pytest.mark.gpu
def test_kernel_refusals(monkeypatch):
    """The same refusals, raised before anything is launched."""
    plain = make
    monkeypatch.setitem(globals(), "make", lambda *a: plain(
        *a, dtype=torch.bfloat16, dev="cuda"))
    test_refusals()


def bounds32(t, dy, rows, scale):
    """As `bounds`, of kernels that hold v = s x A and u = s dy B^T in fp32.

    What they multiply is off from v by 2^-22 of it at most and 2^-37 of the
    largest v (two fp16 parts of 11 digits, of numbers scaled to at most 2^15
    and rounded or raised by 2^-24 + 2^-25; three bf16 parts are better than
    both), and the sums have three times as many products.

    A matrix instruction adds eight products at 2^-24 of the largest, in which
    a subnormal operand counts with the exponent of the smallest normal number
    (fp16: 2^-24 * 2^14 beside 2^-25 loses the latter).  So n products are off
    by at most n 2^-24 of the sum of magnitudes, none taken below that number;
    v's parts, scaled to 2^14, none below 2^-28 of the largest."""
    dt = t["x"].dtype
    eps, w = torch.finfo(dt).eps / 2, 2.0 ** -24
    tiny = torch.finfo(dt).smallest_normal * eps * 2
    y, x, a, b = (t[n].double().cpu() for n in ("y", "x", "a", "b"))
    dy = dy.double().cpu()
    K, M, R = x.shape[2], b.shape[2], b.shape[1]
    r = dict(out=y.clone(), x=torch.zeros_like(x), a=torch.zeros_like(a),
             b=torch.zeros_like(b))
    e = {n: torch.zeros_like(v) for n, v in r.items()}

    def size(p):
        return p.abs().clamp_min(torch.finfo(dt).smallest_normal)

    def inner(n, left, right, s):
        v = s * left @ right
        off = (n + 8) * w * abs(s) * size(left) @ size(right)
        off += 2.0 ** -22 * v.abs() + 2.0 ** -37 * v.abs().max()
        return v, off, v.abs().clamp_min(2.0 ** -28 * float(v.abs().max()))

    for l in sorted(set(rows.index) - {-1}):
        c = [i for i, k in enumerate(rows.index) if k == l]
        s = float(scale[l]) if isinstance(scale, torch.Tensor) else scale
        xs, ds = x[:, c].reshape(-1, K), dy[:, c].reshape(-1, M)
        n = xs.shape[0]
        v, ev, av = inner(K, xs, a[l], s)
        u, eu, au = inner(M, ds, b[l].t(), s)
        for name, value, err in (
                ("out", v @ b[l],
                 (ev + (3 * R + 8) * w * (av + ev)) @ size(b[l])),
                ("x", u @ a[l].t(),
                 (eu + (3 * R + 8) * w * (au + eu)) @ size(a[l]).t())):
            r[name][:, c] += value.reshape(x.shape[0], len(c), -1)
            e[name][:, c] += err.reshape(x.shape[0], len(c), -1)
        r["a"][l] = xs.t() @ u
        e["a"][l] = size(xs).t() @ (eu + (3 * n + 8) * w * (au + eu))
        r["b"][l] = v.t() @ ds
        e["b"][l] = (ev + (3 * n + 8) * w * (av + ev)).t() @ size(ds)
    for k in r:
        e[k] = e[k] * (1 + eps) + (eps + 2 * w) * r[k].abs() + tiny
    return r, e


def held_in_32_bits(t, rows, scale, dy):
    want, err = bounds32(t, dy, rows, scale)
    v = {n: p.detach().clone().requires_grad_() for n, p in t.items()}
    out = lowrank_add(**v, rows=rows, scale=scale)
    got = [("out", out), *zip("xab", torch.autograd.grad(
        out, [v[n] for n in "xab"], dy))]
    with torch.no_grad():
        got.append(("out", lowrank_add(**t, rows=rows, scale=scale)))
    for n, p in got:
        off = (p.detach().double().cpu() - want[n]).abs()
        assert (off <= err[n]).all(), (n, float((off / err[n]).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_kernel_intermediates_are_32_bits(shape, dtype):
    t, rows, scale = make(*shape, seed=3, dtype=dtype, dev="cuda")
    g = torch.Generator().manual_seed(4)
    held_in_32_bits(t, rows, scale,
                    torch.randn(t["y"].shape, generator=g).to(t["y"]))


@pytest.mark.gpu
@pytest.mark.parametrize("R", [3, 16, 32, 60, 128])
@pytest.mark.parametrize("T,B", [(1, 3), (50, 7)])
def test_kernel_intermediates_past_fp16(T, B, R):
    """x A beyond 65504 and dy B^T below 2^-24, results within the type."""
    t, rows, scale = make(T, B, 90, 300, R, 2, seed=R, dtype=torch.float16,
                          dev="cuda")
    t["x"] *= 300
    t["a"] *= 1000
    t["b"] *= 1e-4
    g = torch.Generator().manual_seed(4)
    dy = (1e-3 * torch.randn(t["y"].shape, generator=g)).to(t["y"])
    assert (t["x"].float()[:, :, None].abs().amax(0) * 1000).max() > 65504
    held_in_32_bits(t, rows, scale, dy)
    # columns of one gradient far apart: the large one takes no digits
    t["a"][..., 0] *= 30
    t["a"][..., 1:] /= 1000
    held_in_32_bits(t, rows, scale, dy / 30)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R", [2, 16, 40, 128])
def test_kernel_infinite_weights_and_gradients(R, dtype):
    """Infinities where the sums in 64 bits have them, of the same sign."""
    t, rows, _ = make(9, 6, 70, 90, R, 2, dtype=dtype, dev="cuda",
                      index=[0, 1, -1, 0, 1, 0])
    g = torch.Generator().manual_seed(4)
    dy = torch.randn(t["y"].shape, generator=g).to(t["y"])
    inf = float("inf")
    for n, at, f in (("b", (0, 1, 5), inf), ("b", (1, 0, 88), -inf),
                     ("a", (1, 60, 1), inf), ("dy", (2, 3, 7), -inf),
                     ("x", (4, 4, 8), inf)):
        c = {m: p.clone() for m, p in t.items()}
        d = dy.clone()
        (d if n == "dy" else c[n])[at] = f
        both = []
        for dev, to in (("cuda", dtype), ("cpu", torch.float64)):
            v = {m: p.to(dev, to).requires_grad_() for m, p in c.items()}
            out = lowrank_add(**v, rows=AdapterRows(rows.index, 2, device=dev))
            both.append([out.detach(), *torch.autograd.grad(
                out, [v[m] for m in "xab"], d.to(dev, to))])
            with torch.no_grad():
                both[-1].append(lowrank_add(**v, rows=AdapterRows(
                    rows.index, 2, device=dev)))
        for p, q in zip(*both):
            p = p.double().cpu()
            assert torch.equal(p.isnan(), q.isnan())
            assert torch.equal(p == inf, q == inf)
            assert torch.equal(p == -inf, q == -inf)


def along(t, rows, scale, name, d, f):
    """f's derivative along d of one of its tensors, forward mode."""
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        out = f(**{**t, name: fw.make_dual(t[name], d)}, rows=rows,
                scale=scale)
        return fw.unpack_dual(out).tangent


@pytest.mark.parametrize("name", ["y", "x", "a", "b"])
def test_reference_forward_mode(name):
    t, rows, scale = make(2, 4, 3, 5, 2, 3, seed=1)
    d = torch.randn_like(t[name])
    got = along(t, rows, scale.double(), name, d, lowrank_add)
    v = t[name].clone().requires_grad_()
    w = torch.randn_like(t["y"])
    g, = torch.autograd.grad(
        lowrank_add(**{**t, name: v}, rows=rows, scale=scale.double()), v, w)
    assert abs(float((got * w).sum() - (g * d).sum())) < 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["y", "x", "a", "b"])
def test_kernel_refuses_forward_mode(name):
    t, rows, scale = make(2, 4, 30, 50, 2, 3, dtype=torch.bfloat16, dev="cuda")
    for f in (lowrank_add, lowrank_add_):
        with pytest.raises(NotImplementedError):
            along(t, rows, scale, name, torch.randn_like(t[name]), f)
    with torch.no_grad(), pytest.raises(NotImplementedError):
        along(t, rows, scale, name, torch.randn_like(t[name]), lowrank_add)

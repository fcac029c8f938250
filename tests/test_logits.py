"""Penalties, biases and masks on decode logits (ops/logits.py): the
reference against the definition token by token on the CPU, the kernel
against the reference in 64 bits on the GPU."""
import math

import pytest
import torch

from lstm_tensorspark_amd.ops import logits as mod
from lstm_tensorspark_amd.ops.logits import (_ref_adjust, adjust_logits,
                                             pack_allowed)


def make(B, V, L, K, seed=0, dtype=torch.float64, dev="cpu",
         index=torch.int64, masked=True):
    g = torch.Generator().manual_seed(seed)
    z = 3 * torch.randn(B, V, generator=g)
    h = torch.randint(-2, V + 2, (B, L), generator=g)
    h = torch.where(torch.rand(B, L, generator=g) < .5, h % 5, h)
    n = torch.randint(0, L + 3, (B,), generator=g)      # past L: all of it
    p = torch.randint(0, L + 3, (B,), generator=g)
    bi = torch.randint(-1, V + 1, (B, K), generator=g)  # now and then twice
    args = dict(
        lengths=n.to(index).to(dev), prompt_lengths=p.to(index).to(dev),
        repetition=(0.6 + torch.rand(B, generator=g)).to(dev),
        presence=torch.randn(B, generator=g).to(dev),
        frequency=torch.randn(B, generator=g).to(dev),
        bias_index=bi.to(index).to(dev) if K else None,
        bias=4 * torch.randn(B, K, generator=g).to(dev) if K else None,
        allowed=pack_allowed(torch.rand(B, V, generator=g) < .6).to(dev)
        if masked else None)
    return z.to(dtype).to(dev), h.to(index).to(dev), args


def by_hand(z, h, lengths, prompt_lengths, repetition, presence, frequency,
            bias_index, bias, allowed):
    out = z.double().clone()
    B, V = z.shape
    for b in range(B):
        n = min(int(lengths[b]), h.shape[1])
        seq = [int(t) for t in h[b][:n]]
        fresh = seq[int(prompt_lengths[b]):]
        for v in range(V):
            x = float(out[b, v])
            if v in seq:
                r = float(repetition[b])
                x = x / r if x > 0 else x * r
                c = fresh.count(v)
                if c:
                    x -= float(frequency[b]) * c + float(presence[b])
            for i, f in zip(bias_index[b], bias[b]):
                x += float(f) if int(i) == v else 0.0
            if not int(allowed[b, v // 32]) >> (v % 32) & 1:
                x = -math.inf
            out[b, v] = x
    return out


def test_reference_matches_the_definition():
    z, h, a = make(7, 37, 12, 6)
    want = by_hand(z, h, **a)
    got = adjust_logits(z, h, **a)
    assert torch.equal(torch.isinf(want), torch.isinf(got))
    f = torch.isfinite(want)
    assert (got - want)[f].abs().max() < 1e-13


def test_pack_allowed():
    for V in (1, 31, 32, 33, 100):
        m = torch.rand(3, V) < .5
        w = pack_allowed(m)
        assert w.shape == (3, (V + 31) // 32) and w.dtype == torch.int32
        back = torch.tensor([[bool(int(w[b, v // 32]) >> (v % 32) & 1)
                              for v in range(V)] for b in range(3)])
        assert torch.equal(back, m)
    with pytest.raises(ValueError):
        pack_allowed(torch.ones(2, 3))


def test_parts_alone_and_neutral_values():
    z, h, _ = make(3, 20, 6, 0)
    assert torch.equal(adjust_logits(z), z)
    assert torch.equal(adjust_logits(z, h), z)
    assert torch.equal(adjust_logits(z, h, repetition=1.0, presence=0.0,
                                     frequency=0.0), z)
    d = adjust_logits(z, h.clamp(0, 19), presence=1.0) - z
    assert ((d == 0) | ((d + 1).abs() < 1e-12)).all()
    assert adjust_logits(z[:0], h[:0]).shape == (0, 20)
    assert torch.equal(adjust_logits(z, h[:, :0], presence=1.0), z)


def test_refusals():
    z, h, a = make(3, 40, 6, 4)
    adjust_logits(z, h, **a)
    for over in [dict(lengths=a["lengths"][:2]),
                 dict(lengths=a["lengths"].float()),
                 dict(prompt_lengths=a["prompt_lengths"][None]),
                 dict(repetition=0.0), dict(repetition=-1.0),
                 dict(repetition=math.nan), dict(presence=math.inf),
                 dict(repetition=a["repetition"][:2]),
                 dict(frequency=a["lengths"]),
                 dict(bias=None), dict(bias_index=None),
                 dict(bias=a["bias"][:, :2]),
                 dict(bias_index=a["bias_index"].double()),
                 dict(allowed=a["allowed"].long()),
                 dict(allowed=a["allowed"][:, :1])]:
        with pytest.raises(ValueError):
            adjust_logits(z, h, **{**a, **over})
    for args in [(z[0], h), (z.long(), h), (z, h[:2]), (z, h.float()),
                 (z, h[0])]:
        with pytest.raises(ValueError):
            adjust_logits(*args)
    with pytest.raises(ValueError):
        adjust_logits(z, presence=1.0)
    with pytest.raises(ValueError):
        adjust_logits(z, lengths=a["lengths"])


# ------------------------------------------------------------------- GPU
def check_on_gpu(z, h, a):
    """fp32: a division or product, a product with the count, three sums and
    the list of biases: at most 6 + K roundings of values no larger than the
    sum of all magnitudes; then one rounding to the type."""
    got = adjust_logits(z, h, **a)
    names = ("lengths", "prompt_lengths", "repetition", "presence",
             "frequency", "bias_index", "bias", "allowed")
    pos = {n: a.get(n) for n in names}
    for n, none in (("repetition", 1.0), ("presence", 0.0),
                    ("frequency", 0.0)):
        if pos[n] is None:
            pos[n] = none
    want = _ref_adjust(z.double(), h, *(pos[n] for n in names))
    assert got.dtype == z.dtype and got.shape == z.shape
    fine = torch.isfinite(want.to(z.dtype))     # past the type's range: inf
    assert torch.equal(got[~fine].nan_to_num(7),
                       want.to(z.dtype)[~fine].nan_to_num(7))
    K = 0 if a.get("bias") is None else a["bias"].shape[1]
    L = 0 if h is None else h.shape[1]
    rho = a.get("repetition", 1.0)
    rho = rho.max().item() if isinstance(rho, torch.Tensor) else rho or 1.0
    size = z.double().nan_to_num(0, 0, 0).abs() * max(rho, 2) + 4 * (L + 1) + \
        (a["bias"].abs().sum(1, keepdim=True) if K else 0)
    eps = torch.finfo(z.dtype).eps / 2
    tiny = torch.finfo(z.dtype).smallest_normal * eps * 2
    bound = eps * want.abs() * (1 + 1e-3) + (6 + K) * 2 ** -24 * size + tiny
    assert ((got.double() - want).abs() <= bound)[fine].all()
    return got


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,V,L,K", [(1, 1, 1, 1), (1, 7, 3, 2),
                                     (2, 2047, 100, 5), (3, 2049, 1, 40),
                                     (1, 50000, 300, 8), (17, 4097, 700, 0),
                                     (300, 1000, 20, 3), (5, 70001, 4096, 300),
                                     (3, 8193, 5001, 9), (2, 100, 4100, 2),
                                     (1, 20000, 40000, 0)])
def test_kernel_sizes(dtype, B, V, L, K):
    for masked in (True, False):
        z, h, a = make(B, V, L, K, seed=V + B, dtype=dtype, dev="cuda",
                       masked=masked)
        check_on_gpu(z, h, a)


@pytest.mark.gpu
def test_kernel_types_of_indexes_and_strides():
    z, h, a = make(9, 3001, 64, 12, seed=1, dtype=torch.bfloat16, dev="cuda")
    want = check_on_gpu(z, h, a)
    z2, h2, a2 = make(9, 3001, 64, 12, seed=1, dtype=torch.bfloat16,
                      dev="cuda", index=torch.int32)
    assert torch.equal(want, adjust_logits(z2, h2, **a2))
    wide = torch.zeros(9, 3333, device="cuda").bfloat16()
    wide[:, 5:3006] = z
    hh = torch.zeros(9, 200, dtype=torch.long, device="cuda")
    hh[:, 3:67] = h
    aa = dict(a, bias=a["bias"].t().contiguous().t(),
              bias_index=a["bias_index"].t().contiguous().t(),
              repetition=a["repetition"].double())
    assert torch.equal(want, adjust_logits(wide[:, 5:3006], hh[:, 3:67], **aa))
    # one mask, one list of biases and one row of logits for all requests
    one = dict(a, allowed=a["allowed"][:1].expand(9, -1),
               bias=a["bias"][:1].expand(9, -1),
               bias_index=a["bias_index"][:1].expand(9, -1))
    check_on_gpu(z[:1].expand(9, -1), h, one)


@pytest.mark.gpu
def test_kernel_numbers_for_all_rows_and_parts_alone():
    z, h, a = make(4, 900, 50, 7, seed=2, dtype=torch.float32, dev="cuda")
    check_on_gpu(z, h, dict(repetition=1.3, presence=0.5, frequency=0.25))
    check_on_gpu(z, h, dict(repetition=1.3))
    check_on_gpu(z, None, dict(allowed=a["allowed"]))
    check_on_gpu(z, None, dict(bias_index=a["bias_index"], bias=a["bias"]))
    assert torch.equal(adjust_logits(z), z)
    assert torch.equal(adjust_logits(z, h[:, :0], presence=1.0), z)
    assert torch.equal(adjust_logits(z, bias_index=a["bias_index"][:, :0],
                                     bias=a["bias"][:, :0]), z)
    assert adjust_logits(z[:0]).shape == (0, 900)
    assert adjust_logits(z[:, :0]).shape == (4, 0)


@pytest.mark.gpu
def test_kernel_infinities_and_empty_masks():
    z, h, a = make(6, 500, 30, 4, seed=3, dtype=torch.bfloat16, dev="cuda")
    z[0, :200] = math.nan
    z[1, :200] = -math.inf
    z[2, :200] = math.inf
    z[3] = torch.finfo(torch.bfloat16).min
    a["allowed"][4] = 0
    a["bias"][5] = -math.inf
    got = check_on_gpu(z, h, a)
    assert (got[4] == -math.inf).all()


@pytest.mark.gpu
def test_kernel_many_biases_for_one_token_repeat_bitwise():
    z = torch.randn(3, 100, device="cuda")
    i = torch.full((3, 64), 11, device="cuda")
    b = torch.randn(3, 64, device="cuda") * torch.logspace(
        -6, 6, 64, device="cuda")
    want = z[:, 11].clone()
    s = b[:, 0].clone()
    for k in range(1, 64):
        s = s + b[:, k]
    for _ in range(3):
        got = adjust_logits(z, bias_index=i, bias=b)
        assert torch.equal(got[:, 11], want + s)


@pytest.mark.gpu
def test_kernel_captured_replayed_and_on_another_stream():
    z, h, a = make(5, 5000, 40, 6, seed=4, dtype=torch.bfloat16, dev="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = adjust_logits(z, h, **a)
    s.synchronize()
    assert torch.equal(first, check_on_gpu(z, h, a))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = adjust_logits(z, h, **a)
    for seed in (5, 6, 7):
        z2, h2, a2 = make(5, 5000, 40, 6, seed=seed, dtype=torch.bfloat16,
                          dev="cuda")
        z.copy_(z2), h.copy_(h2)
        for n in a:
            a[n].copy_(a2[n])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check_on_gpu(z2, h2, a2))


@pytest.mark.gpu
def test_kernel_is_what_runs(monkeypatch):
    z, h, a = make(2, 50, 4, 2, dtype=torch.bfloat16, dev="cuda")
    monkeypatch.setattr(mod, "_ref_adjust", None)
    adjust_logits(z, h, **a)


@pytest.mark.gpu
def test_kernel_refusals(monkeypatch):
    """The same refusals, raised before anything is launched."""
    plain = make
    monkeypatch.setitem(globals(), "make", lambda *a: plain(
        *a, dtype=torch.bfloat16, dev="cuda"))
    test_refusals()


@pytest.mark.gpu
def test_kernel_refuses_forward_mode():
    fw = torch.autograd.forward_ad
    z, h, a = make(3, 50, 6, 4, dtype=torch.bfloat16, dev="cuda")
    with fw.dual_level():
        with pytest.raises(NotImplementedError):
            adjust_logits(fw.make_dual(z, torch.ones_like(z)), h, **a)
        for n in ("repetition", "presence", "frequency", "bias"):
            with pytest.raises(NotImplementedError):
                adjust_logits(z, h, **{**a, n: fw.make_dual(
                    a[n], torch.ones_like(a[n]))})
        adjust_logits(z, h, **a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,L,K", [(300, 5, 250), (9000, 50, 4000),
                                   (20001, 4100, 4000)])
def test_kernel_long_lists_of_biases_with_repeats(V, L, K, dtype):
    for few in (None, 1, 30, 700):
        z, h, a = make(3, V, L, K, seed=K, dtype=dtype, dev="cuda")
        if few is None:         # one token twice
            a["bias_index"] = torch.stack(
                [torch.randperm(V, device="cuda")[:K] for _ in range(3)])
            a["bias_index"][:, K // 3] = a["bias_index"][:, K - 1]
        else:
            a["bias_index"] = (torch.arange(K, device="cuda") * 7
                               % min(few, V) * (V // min(few, V))).repeat(3, 1)
            a["bias_index"][1, ::3] = -1
        got = check_on_gpu(z, h, a)
        assert torch.equal(got, adjust_logits(z, h, **a))


@pytest.mark.gpu
def test_kernel_one_repeat_costs_no_walk_an_entry():
    """Work is linear in the list's length, with repeats or without: a walk
    through 20000 biases for each of them took four thousand times as long."""
    z = torch.randn(2, 50000, device="cuda")
    i = torch.stack([torch.randperm(50000, device="cuda")[:20000]
                     for _ in range(2)])
    f = torch.randn(2, 20000, device="cuda")

    def least():
        times = []
        for _ in range(4):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            torch.cuda.synchronize()
            a.record()
            for _ in range(5):
                adjust_logits(z, bias_index=i, bias=f)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    plain = least()
    i[:, 777] = i[:, 19000]
    assert least() < 50 * plain

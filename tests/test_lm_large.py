"""The operators around the language-model head where element offsets pass
31 bits: the far end of a large tensor against the same rows alone."""
import pytest
import torch

from lstm_tensorspark_amd.ops.adapters import AdapterRows, lowrank_add
from lstm_tensorspark_amd.ops.distill import distill_loss
from lstm_tensorspark_amd.ops.logits import adjust_logits

pytestmark = pytest.mark.gpu

N, V = 43000, 50000             # 2.15e9 elements, 4.3 GB in bf16


def big(rows=N, cols=V):
    t = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for i in range(0, rows, 8192):
        t[i:i + 8192].normal_(std=2.0)
    return t


@pytest.fixture(autouse=True)
def room():
    torch.manual_seed(0)
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("g", [1.0, 2.0])
def test_distill_far_rows(g):
    z = big().requires_grad_()
    i = torch.randint(0, V, (N, 8), device="cuda")
    t = torch.randn(N, 8, device="cuda")
    y = torch.randint(0, V, (N,), device="cuda")
    kw = dict(alpha=0.5, temperature=2.0)
    loss = distill_loss(z, i, t, y, weight=N / g, **kw)
    d, = torch.autograd.grad(loss, z, torch.full_like(loss, g))
    for s in (slice(0, 3), slice(N - 3, N)):
        zs = z.detach()[s].clone().requires_grad_()
        part = distill_loss(zs, i[s], t[s], y[s], weight=3.0, **kw)
        want, = torch.autograd.grad(part, zs)
        # the factors N / N and 3 / 3 may be rounded apart
        off = (d[s].float() - want.float()).abs()
        assert (off <= 2 ** -7 * want.float().abs()).all()
    assert torch.isfinite(loss)


def test_adjust_far_rows():
    z = big()
    h = torch.randint(0, V, (N, 12), device="cuda")
    kw = dict(repetition=1.5, presence=0.5, frequency=0.25)
    out = adjust_logits(z, h, **kw)
    for s in (slice(0, 3), slice(N - 3, N)):
        assert torch.equal(out[s], adjust_logits(z[s].clone(), h[s], **kw))


def test_adjust_more_rows_than_large_workgroups_fit():
    """2^22 rows with long histories: 1024 threads each are 2^32."""
    n = 1 << 22
    z = torch.randn(64, 3, device="cuda").bfloat16()
    h = (torch.arange(4096, device="cuda") % 5)[None]
    kw = dict(repetition=1.5, presence=0.5, frequency=0.25)
    want = adjust_logits(z, h.expand(64, -1), **kw)
    out = adjust_logits(z.repeat(n // 64, 1), h.expand(n, -1), **kw)
    assert (out.view(-1, 64, 3) == want).all()


def test_adapters_far_rows():
    y = big()
    x = torch.randn(N, 64, device="cuda").bfloat16()
    a = torch.randn(2, 64, 8, device="cuda").bfloat16()
    b = torch.randn(2, 8, V, device="cuda").bfloat16()
    index = [i % 2 for i in range(N)]
    rows = AdapterRows(index, 2, device="cuda")
    with torch.no_grad():
        out = lowrank_add(y, x, a, b, rows)
    for s in (slice(0, 4), slice(N - 4, N)):
        want = y[s].float()
        for k, c in enumerate(range(s.start, s.stop)):
            v = (x[c].float() @ a[index[c]].float()).bfloat16().float()
            want[k] += v @ b[index[c]].float()
        # v may be rounded to the neighbour, the result is rounded once
        size = want.abs() + (x[s].float().abs() @ a.float().abs().amax(0)
                             @ b.float().abs().amax(0))
        assert ((out[s].float() - want).abs() <= 2 ** -8 * size).all()
    # gradients that reach across the whole of it
    xs = x.clone().requires_grad_()
    o = lowrank_add(y, xs, a, b, rows)
    dx, = torch.autograd.grad(o, xs, y)
    for c in (0, 1, N - 2, N - 1):
        u = y[c].float() @ b[index[c]].float().t()
        want = u @ a[index[c]].float().t()
        size = (y[c].float().abs() @ b[index[c]].float().abs().t()) @ \
            a[index[c]].float().abs().t()
        assert ((dx[c].float() - want).abs() <= 2 ** -7 * size).all()


def test_adapters_refuse_more_rows_than_a_launch_holds():
    """Rows that are one and the same in memory: 2^30 / 64 workgroups of 256
    threads are 2^32."""
    one = torch.ones(1, 1, 1, device="cuda").bfloat16()
    rows = AdapterRows([0], 1, device="cuda")
    wide = one.expand(1 << 30, 1, 1)
    with pytest.raises(ValueError, match="too many rows"):
        lowrank_add(wide, wide, one, one, rows)
    many = one.expand(1 << 22, 1, 1)
    out = lowrank_add(many, many, one, one, rows)
    assert (out == 2).all()


def test_adapters_many_columns():
    """One group of every column of a wide batch, and an odd split of it."""
    n = 70001
    x = torch.randn(n, 40, device="cuda").bfloat16()
    y = torch.randn(n, 24, device="cuda").bfloat16()
    a = torch.randn(3, 40, 8, device="cuda").bfloat16()
    b = torch.randn(3, 8, 24, device="cuda").bfloat16()
    for index in ([1] * n, [(i * i) % 3 if i % 5 else -1 for i in range(n)]):
        out = lowrank_add(y, x, a, b, AdapterRows(index, 3, device="cuda"))
        i = torch.tensor(index, device="cuda")
        for l in range(3):
            m = i == l
            v = (x[m].float() @ a[l].float()).bfloat16().float()
            want = y[m].float() + v @ b[l].float()
            size = want.abs() + (x[m].float().abs() @ a[l].float().abs()
                                 @ b[l].float().abs())
            assert ((out[m].float() - want).abs() <= 2 ** -8 * size).all()
        assert torch.equal(out[i < 0], y[i < 0])

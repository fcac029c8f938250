"""The operators around the language-model head as the framework's own paths
call them: adapters in LSTMModel, rules and adapters in generate() and the
ContinuousBatcher, a teacher in the Trainer, and all of them together."""
import math

import pytest
import torch

from lstm_tensorspark_amd import (AdapterSet, Config, ContinuousBatcher,
                                  LogitRules, LSTMModel, Trainer)
from lstm_tensorspark_amd.config import DataConfig, ModelConfig, TrainConfig

gpu = pytest.mark.gpu


def make_cfg(head="lm", bidirectional=False, hidden=16, vocab=30, layers=2):
    return ModelConfig(input_size=12, hidden_size=hidden, num_layers=layers,
                       head=head, vocab_size=vocab if head == "lm" else 0,
                       num_classes=7, bidirectional=bidirectional)


def make_set(cfg, rank=3, count=3, seed=1, alpha=6.0):
    torch.manual_seed(seed)
    s = AdapterSet(cfg, rank, count, alpha=alpha)
    for n, p in s.weight_dict().items():
        if n.endswith("/B"):
            torch.nn.init.normal_(p, std=0.3)
    return s


def merged(model, adapters, l):
    """A model with adapter l inside its weights."""
    m = LSTMModel(model.cfg).to(next(model.parameters()).dtype)
    m.load_state_dict(model.state_dict())
    w = adapters.weight_dict()
    with torch.no_grad():
        for n in {n.split("/")[0] for n in w}:
            at = n + ("/W" if n == "head" else "/W_x")
            m.weight(at).add_(adapters.scale * w[n + "/A"][l] @ w[n + "/B"][l])
    return m


HEADS = [("lm", False), ("classifier", False), ("seq_classifier", True),
         ("none", True)]


# ------------------------------------------------------------------- CPU
@pytest.mark.parametrize("head,bidi", HEADS)
def test_new_adapters_change_nothing(head, bidi):
    cfg = make_cfg(head, bidi)
    m, s = LSTMModel(cfg).double(), AdapterSet(cfg, 4, 2).double()
    x = torch.randint(0, 30, (5, 3)) if head == "lm" else \
        torch.randn(5, 3, 12, dtype=torch.float64)
    want, _ = m(x)
    got, _ = m(x, None, s.rows([0, 1, -1]))
    assert torch.equal(got, want)


@pytest.mark.parametrize("head,bidi", HEADS)
def test_adapters_equal_merged_weights(head, bidi):
    """Values and gradients: with W = W0 + s A B, dA = s dW B^T and dB = s
    A^T dW, and a column without an adapter sees the base."""
    cfg = make_cfg(head, bidi)
    torch.manual_seed(0)
    m, s = LSTMModel(cfg).double(), make_set(cfg).double()
    m.requires_grad_(False)
    T, index = 6, [1, -1, 2, 1]
    x = torch.randint(0, 30, (T, 4)) if head == "lm" else \
        torch.randn(T, 4, 12, dtype=torch.float64)
    out, state = m(x, None, s.rows(index))
    weigh = torch.randn_like(out)
    (out * weigh).sum().backward()
    grads = {n: torch.zeros_like(p) for n, p in s.weight_dict().items()}
    for c, l in enumerate(index):
        one = m if l < 0 else merged(m, s, l)
        one.requires_grad_(True)
        o, st = one(x[:, c:c + 1])
        ref = out[c] if head == "classifier" else out[:, c]
        assert (ref - (o[0] if head == "classifier" else o[:, 0])).abs() \
            .max() < 1e-12
        for (h, k), (h1, k1) in zip(state, st):
            assert (h[c] - h1[0]).abs().max() < 1e-12
        if l < 0:
            one.requires_grad_(False)
            continue
        w = weigh[c:c + 1] if head == "classifier" else weigh[:, c:c + 1]
        (o * w).sum().backward()
        for n in {n.split("/")[0] for n in grads}:
            dw = one.weight(n + ("/W" if n == "head" else "/W_x")).grad
            A, B = s.weight_dict()[n + "/A"][l], s.weight_dict()[n + "/B"][l]
            grads[n + "/A"][l] += s.scale * dw @ B.t()
            grads[n + "/B"][l] += s.scale * A.t() @ dw
    for n, p in s.weight_dict().items():
        assert (p.grad - grads[n]).abs().max() < 1e-10
        assert (p.grad[0] == 0).all()           # nobody used adapter 0
    assert all(p.grad is None for p in m.parameters())


def test_base_and_adapters_train_together():
    """Gradients of the base's weights beside adapters, by differences (in 64
    bits: error h^2 = 1e-10 and 2^-52 / h = 2e-11, times a few units)."""
    cfg = make_cfg()
    torch.manual_seed(0)
    m, s = LSTMModel(cfg).double(), make_set(cfg).double()
    x, y = torch.randint(0, 30, (4, 2)), torch.randint(0, 30, (4, 2, 1))

    def loss():
        out, _ = m(x, None, s.rows([0, 2]))
        return -torch.log_softmax(out, dim=2).gather(2, y).mean()

    loss().backward()
    h = 1e-5
    for n, p in {**m.weight_dict(), **s.weight_dict()}.items():
        i = (int(x[0, 0]), 3) if n == "embed/W" else \
            (0,) * (p.dim() == 3) + tuple(int(k) // 2 for k in p.shape[-2:])
        with torch.no_grad():
            p[i] += h
            up = float(loss())
            p[i] -= 2 * h
            down = float(loss())
            p[i] += h
        assert abs((up - down) / (2 * h) - float(p.grad[i])) < 1e-8, n


def even_after_odd(tokens):
    ok = torch.zeros(30, dtype=torch.bool)
    ok[1 - tokens[-1] % 2::2] = True
    return ok


RULES = [None, LogitRules(repetition=1.8),
         LogitRules(presence=1.0, frequency=0.5),
         LogitRules(bias={3: 4.0, 5: -math.inf, 0: 1.5}),
         LogitRules(grammar=even_after_odd),
         LogitRules(1.3, 0.2, 0.1, {7: 2.0}, even_after_odd)]


def solo(m, tokens, steps, rules=None, adapters=None, l=-1, **kw):
    dev = next(m.parameters()).device
    prompt = torch.tensor(tokens, device=dev).unsqueeze(1)
    rows = adapters.rows([l]) if adapters is not None and l >= 0 else None
    return m.generate(prompt, steps=steps, rules=rules, adapters=rows,
                      use_graph=False, **kw)[:, 0].tolist()


def batcher_parity(m, s):
    eng = ContinuousBatcher(m, max_batch=5, adapters=s)
    reqs = [([1 + i, 2, 9], 4 + 3 * i, r, i % (s.count + 1) - 1)
            for i, r in enumerate(RULES)] + [([4], 9, RULES[5], 1)]
    rids = [eng.submit(t, n, rules=r, adapter=l) for t, n, r, l in reqs[:4]]
    for _ in range(3):
        eng.step()
    rids += [eng.submit(t, n, rules=r, adapter=l) for t, n, r, l in reqs[4:]]
    seeded = eng.submit([8, 8], 6, rules=RULES[1], adapter=0, seed=5,
                        temperature=0.8, top_k=9)
    eng.drain()
    got = [eng.result(r, timeout=0) for r in rids]
    return reqs, got, eng.result(seeded, timeout=0)


def test_batcher_matches_solo_with_rules_and_adapters():
    cfg = make_cfg()
    torch.manual_seed(2)
    m, s = LSTMModel(cfg), make_set(cfg)
    reqs, got, seeded = batcher_parity(m, s)
    for (t, n, r, l), g in zip(reqs, got):
        assert g == solo(m, t, n, r, s, l)
    assert seeded == solo(m, [8, 8], 6, RULES[1], s, 0, temperature=0.8,
                          top_k=9,
                          generator=torch.Generator().manual_seed(5))


def test_rules_do_what_they_say():
    torch.manual_seed(3)
    m = LSTMModel(make_cfg())
    t = solo(m, [1], 12, LogitRules(grammar=even_after_odd))
    assert all((a + b) % 2 for a, b in zip(t, t[1:]))
    t = solo(m, [1], 12, LogitRules(presence=1e4))
    assert len(set(t[1:])) == 12            # nothing twice
    t = solo(m, [1], 5, LogitRules(bias={11: 1e4}))
    assert t[1:] == [11] * 5
    plain = solo(m, [1], 8)
    assert solo(m, [1], 8, LogitRules()) == plain
    two = m.generate(torch.tensor([[1, 2], [3, 4]]), 6,
                     rules=LogitRules(presence=1e4))
    assert all(len(set(two[2:, c].tolist())) == 6 for c in (0, 1))


def test_grammars_that_fail_end_their_request_only():
    m = LSTMModel(make_cfg())

    def nothing(tokens):
        return torch.zeros(30, dtype=torch.bool)

    def later(tokens):
        return torch.full((30,), len(tokens) < 5)

    def wrong(tokens):
        return [True] * 30

    def raises(tokens):
        raise KeyError("no rule")

    def only_banned(tokens):
        return torch.arange(30) == 5

    eng = ContinuousBatcher(m)
    good = eng.submit([1, 2], 6)
    bad = [eng.submit([1, 2], 6, rules=LogitRules(grammar=g))
           for g in (nothing, later, wrong, raises)]
    bad.append(eng.submit([1, 2], 6, rules=LogitRules(
        bias={5: -math.inf}, grammar=only_banned), temperature=1.0))
    eng.drain()
    assert eng.result(good, timeout=0) == solo(m, [1, 2], 6)
    for rid, kind in zip(bad, (ValueError, ValueError, ValueError, KeyError,
                               ValueError)):
        with pytest.raises(kind):
            eng.peek(rid)
        with pytest.raises(kind):
            eng.result(rid, timeout=0)
    assert eng.try_result(bad[0]) is None
    with pytest.raises(ValueError):
        solo(m, [1, 2], 6, LogitRules(grammar=later))


def test_a_request_keeps_the_rules_it_was_submitted_with():
    torch.manual_seed(3)
    m = LSTMModel(make_cfg())
    eng = ContinuousBatcher(m)
    rules = LogitRules(bias={11: 1e4})
    first = eng.submit([1], 6, rules=rules)
    eng.step()
    rules.bias[11] = -1e4
    rules.bias[12] = 2e4
    rules.presence = 1e4
    other = eng.submit([2], 6)          # a new batch reads its rules again
    eng.drain()
    assert eng.result(first, timeout=0)[1:] == [11] * 6
    assert eng.result(other, timeout=0) == solo(m, [2], 6)


def test_bias_tokens_are_whole_numbers():
    m = LSTMModel(make_cfg())
    eng = ContinuousBatcher(m)
    for bad in (1.5, "3", None, 2.0):
        with pytest.raises(ValueError):
            eng.submit([1], 3, rules=LogitRules(bias={bad: 1.0}))
        with pytest.raises(ValueError):
            solo(m, [1], 3, LogitRules(bias={bad: 1.0}))


class OneBuffer:
    """A grammar that allows a request's first token alone, and answers with
    one and the same tensor for every request."""

    def __init__(self, dev="cpu"):
        self.ok = torch.zeros(30, dtype=torch.bool, device=dev)

    def __call__(self, tokens):
        self.ok.fill_(False)
        self.ok[tokens[0]] = True
        return self.ok


def grammars_with_one_buffer(m, dev):
    rules = LogitRules(grammar=OneBuffer(dev))
    out = m.generate(torch.tensor([[3, 9, 4]], device=dev), 5, rules=rules)
    assert out.t().tolist() == [[3] * 6, [9] * 6, [4] * 6]
    eng = ContinuousBatcher(m)
    rids = [eng.submit([t], 5, rules=rules) for t in (3, 9, 4)]
    eng.drain()
    assert [eng.result(r, timeout=0) for r in rids] == [
        [3] * 6, [9] * 6, [4] * 6]


def test_grammars_may_answer_with_one_buffer():
    grammars_with_one_buffer(LSTMModel(make_cfg()), "cpu")


def test_grammar_is_not_asked_about_finished_columns():
    """Columns of one batch end at different steps."""
    m = LSTMModel(make_cfg())
    ends = 7

    def grammar(tokens):
        if ends in tokens:
            raise KeyError("asked behind the end")
        ok = torch.zeros(30, dtype=torch.bool)
        ok[ends if len(tokens) > tokens[0] else 1] = True
        return ok

    out = m.generate(torch.tensor([[2, 4, 3]]), 6, eos_token=ends,
                     rules=LogitRules(grammar=grammar))
    # the token behind as many as the first one says is the end
    assert out[:6].t().tolist() == [[2, 1, 1, 7, 7, 7], [4, 1, 1, 1, 1, 7],
                                    [3, 1, 1, 1, 7, 7]]


def test_workflow_refusals():
    cfg = make_cfg()
    m, s = LSTMModel(cfg), make_set(cfg)
    with pytest.raises(ValueError):
        AdapterSet(cfg, 0)
    with pytest.raises(ValueError):
        AdapterSet(cfg, 129)
    with pytest.raises(ValueError):
        AdapterSet(cfg, 4, 0)
    with pytest.raises(ValueError):
        s.rows([3])
    with pytest.raises(ValueError):
        m(torch.zeros(2, 3).long(), None, s.rows([0, 1]))
    eng = ContinuousBatcher(m, adapters=s)
    for kw in (dict(adapter=3), dict(adapter=-2),
               dict(rules=LogitRules(repetition=0.0)),
               dict(rules=LogitRules(repetition=math.nan)),
               dict(rules=LogitRules(presence=math.inf)),
               dict(rules=LogitRules(frequency=2e4)),
               dict(rules=LogitRules(bias={30: 1.0})),
               dict(rules=LogitRules(bias={3: math.inf})),
               dict(rules=LogitRules(bias={3: math.nan})),
               dict(rules=LogitRules(bias=dict.fromkeys(range(30),
                                                        -math.inf)))):
        with pytest.raises(ValueError):
            eng.submit([1], 3, **kw)
    with pytest.raises(ValueError):
        ContinuousBatcher(m).submit([1], 3, adapter=0)
    with pytest.raises(ValueError):
        ContinuousBatcher(m, adapters=make_set(cfg).double())
    with pytest.raises(AssertionError):
        m.generate(torch.zeros(1, 1).long(), 2, use_graph=True,
                   rules=LogitRules())
    with pytest.raises(ValueError):
        m.distill_loss(torch.zeros(2, 3, 30), torch.zeros(2, 3, 31), None)
    with pytest.raises(ValueError):
        Trainer(Config(model=cfg), teacher=LSTMModel(make_cfg(vocab=31)))
    with pytest.raises(ValueError):
        Trainer(Config(model=cfg), model=m, teacher=m)


def test_a_teacher_without_entries_is_refused():
    """top_k = 0 would leave (1 - alpha) of the label loss alone."""
    m = LSTMModel(make_cfg())
    z, y = torch.zeros(2, 3, 30), torch.zeros(2, 3).long()
    for k in (0, -1):
        with pytest.raises(ValueError):
            m.distill_loss(z, z, y, top_k=k)
    assert torch.isfinite(m.distill_loss(z, z, y, top_k=31))


def test_a_refused_generate_keeps_the_training_mode():
    m = LSTMModel(make_cfg())
    prompt = torch.zeros(1, 1).long()
    for training in (True, False):
        m.train(training)
        for kind, kw in ((ValueError, dict(rules=LogitRules(repetition=0.0))),
                         (ValueError, dict(rules=LogitRules(bias={30: 1.0}))),
                         (ValueError, dict(rules=LogitRules(
                             grammar=lambda t: torch.zeros(30).bool()))),
                         (AssertionError, dict(use_graph=True, eos_token=1)),
                         (AssertionError, dict(use_graph=True,
                                               temperature=1.0)),
                         (AssertionError, dict(use_graph=True,
                                               rules=LogitRules()))):
            with pytest.raises(kind):
                m.generate(prompt, 3, **kw)
            assert m.training is training


def rules_at_their_limits(m, dev):
    """Sampling in fp16 where the adjusted logits pass its range."""
    torch.manual_seed(11)
    for r in (LogitRules(frequency=-1e4), LogitRules(presence=-1e4),
              LogitRules(frequency=1e4, presence=1e4),
              LogitRules(repetition=100.0), LogitRules(repetition=0.01),
              LogitRules(repetition=0.01, frequency=-1e4, presence=-1e4,
                         bias={t: 1e4 for t in range(30)})):
        prompt = torch.tensor([[1, 2]] * 9, device=dev)
        prompt[:, 1] = torch.arange(9)
        out = m.generate(prompt, 12, temperature=1.0, rules=r)
        assert out.shape == (21, 2) and (out < 30).all()
        if r == LogitRules(frequency=-1e4):     # what came first comes again
            assert (out[9:, 0] == out[9, 0]).all()
        eng = ContinuousBatcher(m)
        rids = [eng.submit([1] * 9, 12, temperature=1.0, rules=r),
                eng.submit([1] * 9, 12)]
        eng.drain()
        assert len(eng.result(rids[0], timeout=0)) == 21
        assert eng.result(rids[1], timeout=0) == solo(m, [1] * 9, 12)


def test_rules_at_their_limits_in_fp16():
    torch.manual_seed(10)
    m = LSTMModel(make_cfg()).half()
    with torch.no_grad():
        m.weight("head/b").mul_(0).add_(torch.linspace(-700, 700, 30))
    rules_at_their_limits(m, "cpu")


def distill_config(dtype="fp32", bptt=4):
    return Config(model=make_cfg(),
                  train=TrainConfig(batch_size=6, seq_len=8, bptt=bptt, lr=0.1,
                                    momentum=0.0, log_interval=0, dtype=dtype,
                                    distill_alpha=0.7, distill_top_k=5),
                  data=DataConfig(task="lm"))


def test_trainer_with_a_teacher():
    torch.manual_seed(4)
    teacher = LSTMModel(make_cfg(hidden=20, layers=1))
    before = {n: p.detach().clone() for n, p in teacher.weight_dict().items()}
    t = Trainer(distill_config(), teacher=teacher)
    twin = LSTMModel(t.model.cfg)
    twin.load_state_dict(t.model.state_dict())
    x, y = t.data.batch(0)
    info = t.train_step((x, y))
    want, state, t_state = 0.0, None, None
    for w in (slice(0, 4), slice(4, 8)):
        out, state = twin(x[w], state)
        state = twin.detach_state(state)
        with torch.no_grad():
            ref, t_state = teacher(x[w], t_state)
        top = ref.reshape(-1, 30).topk(5, dim=1)
        q = torch.softmax(top.values / 2.0, 1)
        logp = torch.log_softmax(out.reshape(-1, 30) / 2.0, 1)
        kl = (q * (q.log() - logp.gather(1, top.indices))).sum(1).mean()
        ce = torch.nn.functional.cross_entropy(out.reshape(-1, 30),
                                               y[w].reshape(-1))
        loss = (0.7 * 4.0 * kl + 0.3 * ce) / 2
        loss.backward()
        want += float(loss.detach())
    assert abs(info["loss"] - want) < 1e-5
    for n, p in twin.weight_dict().items():
        moved = t.model.weight(n).detach()
        assert (moved - (p.detach() - 0.1 * p.grad)).abs().max() < 1e-6
    for n, p in teacher.weight_dict().items():
        assert torch.equal(p, before[n]) and p.grad is None


def distil_adapters(dev, dtype):
    """Two teachers distilled into two adapters of one frozen base, in one
    batch."""
    torch.manual_seed(5)
    cfg = make_cfg(hidden=64, vocab=200)
    base = LSTMModel(cfg).to(dev, dtype).requires_grad_(False)
    teachers = [LSTMModel(cfg).to(dev, dtype) for _ in range(2)]
    s = AdapterSet(cfg, rank=4, count=2).to(dev, dtype)
    x = torch.randint(0, 200, (7, 4), device=dev)
    y = torch.randint(0, 200, (7, 4), device=dev)
    rows = s.rows([0, 1, 1, -1])
    with torch.no_grad():
        ref = torch.cat([teachers[i](x[:, c:c + 1])[0]
                         for c, i in enumerate((0, 1, 1, 0))], dim=1)
    opt = torch.optim.SGD(s.parameters(), lr=0.1)
    for _ in range(2):
        opt.zero_grad()
        out, _ = base(x, None, rows)
        loss = base.distill_loss(out, ref, y, top_k=16)
        loss.backward()
        opt.step()
    return base, s, loss.detach(), x, y, ref


def serve_them(base, s):
    eng = ContinuousBatcher(base, adapters=s)
    rules = LogitRules(repetition=1.2, frequency=0.3, bias={4: 0.5},
                       grammar=lambda t: torch.arange(200) % 3 != t[-1] % 3)
    rids = [eng.submit([1, 2, 3], 10, rules=rules if l != 0 else None,
                       adapter=l) for l in (-1, 0, 1)]
    eng.drain()
    out = [eng.result(r, timeout=0) for r in rids]
    for t, l in zip(out, (-1, 0, 1)):
        assert len(t) == 13 and all(0 <= k < 200 for k in t)
        if l != 0:
            assert all(b % 3 != a % 3 for a, b in zip(t[2:], t[3:]))
    return out


def test_distil_into_adapters_and_serve_them():
    base, s, loss, *_ = distil_adapters("cpu", torch.float32)
    assert math.isfinite(float(loss))
    assert all(float(p.grad.abs().sum()) > 0 for n, p in
               s.weight_dict().items())
    assert all(p.grad is None for p in base.parameters())
    serve_them(base, s)


@pytest.mark.parametrize("batched", [False, True])
def test_served_requests_have_penalties(batched, monkeypatch):
    import os
    monkeypatch.syspath_prepend(os.path.join(os.path.dirname(
        os.path.dirname(os.path.abspath(__file__))), "examples"))
    import serve
    from starlette.testclient import TestClient
    torch.manual_seed(9)
    m = LSTMModel(make_cfg()).eval()
    eng = ContinuousBatcher(m) if batched else None
    if eng:
        eng.start()
    try:
        c = TestClient(serve.build_app(m, torch.device("cpu"), batcher=eng))
        ask = {"tokens": [1, 2], "steps": 9}
        plain = c.post("/generate", json=ask).json()["generated"]
        assert plain == solo(m, [1, 2], 9)[2:]
        got = c.post("/generate", json={**ask, "presence_penalty": 1e4})
        assert len(set(got.json()["generated"])) == 9
        got = c.post("/generate", json={**ask, "logit_bias": {"7": 1e4}})
        assert got.json()["generated"] == [7] * 9
        for bad in ({"repetition_penalty": 0.0}, {"logit_bias": {"30": 1.0}},
                    {"presence_penalty": 1.0, "beam_size": 2}):
            assert c.post("/generate", json={**ask, **bad}).status_code == 400
    finally:
        if eng:
            eng.stop()


# ------------------------------------------------------------------- GPU
@gpu
@pytest.mark.parametrize("head,bidi", [("lm", False), ("seq_classifier", True)])
def test_gpu_adapters_track_the_reference(head, bidi):
    """bf16 kernels against the same bf16 weights in fp32 on the CPU: the
    outputs are rounded at about ten places along two layers (bf16, 2^-8)."""
    cfg = make_cfg(head, bidi, hidden=64)
    torch.manual_seed(6)
    m, s = LSTMModel(cfg).bfloat16(), make_set(cfg, alpha=1.0).bfloat16()
    x = torch.randint(0, 30, (6, 4)) if head == "lm" else \
        torch.randn(6, 4, 12).bfloat16()
    mg, sg = LSTMModel(cfg).bfloat16().cuda(), make_set(cfg, alpha=1.0).bfloat16().cuda()
    mg.load_state_dict(m.state_dict())
    sg.load_state_dict(s.state_dict())
    m, s = m.float(), s.float()
    want, _ = m(x if head == "lm" else x.float(), None, s.rows([1, -1, 2, 1]))
    got, _ = mg(x.cuda(), None, sg.rows([1, -1, 2, 1]))
    size = float(want.detach().abs().max())
    assert (got.detach().float().cpu() - want.detach()).abs().max() < \
        10 * 2 ** -8 * max(1.0, size)
    w = torch.randn(want.shape)
    (want * w).sum().backward()
    (got * w.cuda().bfloat16()).sum().backward()
    for n, p in sg.weight_dict().items():
        ref = s.weight_dict()[n].grad
        off = (p.grad.float().cpu() - ref).norm() / ref.norm()
        assert off < 0.05, (n, float(off))
        assert (p.grad[0] == 0).all()


@gpu
def test_gpu_grammars_may_answer_with_one_buffer():
    m = LSTMModel(make_cfg(hidden=64)).bfloat16().cuda()
    grammars_with_one_buffer(m, "cuda")


@gpu
def test_gpu_rules_at_their_limits_in_fp16():
    torch.manual_seed(10)
    m = LSTMModel(make_cfg(hidden=64)).half().cuda()
    with torch.no_grad():
        m.weight("head/b").mul_(0).add_(torch.linspace(
            -700, 700, 30, device="cuda").half())
    rules_at_their_limits(m, "cuda")


@gpu
def test_gpu_distil_into_adapters_and_serve_them():
    base, s, loss, x, y, ref = distil_adapters("cuda", torch.bfloat16)
    assert math.isfinite(float(loss))
    assert all(float(p.grad.abs().sum()) > 0 for n, p in
               s.weight_dict().items())
    out = serve_them(base, s)
    again = serve_them(base, s)
    assert out == again


@gpu
def test_gpu_batcher_with_rules_and_adapters():
    """Every request alone in the engine gives what it gives in a batch as
    long as the base's logits do; held here to the rules alone."""
    cfg = make_cfg(hidden=64)
    torch.manual_seed(7)
    m, s = LSTMModel(cfg).bfloat16().cuda(), make_set(cfg).bfloat16().cuda()
    reqs, got, seeded = batcher_parity(m, s)
    for (t, n, r, l), g in zip(reqs, got):
        assert g[:len(t)] == t and len(g) == len(t) + n
        if r is not None and r.grammar:
            assert all((a + b) % 2 for a, b in zip(g[len(t) - 1:], g[len(t):]))
        if r is not None and r.bias and 5 in r.bias:
            assert 5 not in g[len(t):]
    assert len(seeded) == 8


@gpu
def test_gpu_trainer_with_a_teacher():
    torch.manual_seed(8)
    cfg = distill_config("bf16")
    cfg.model = make_cfg(hidden=64)
    t = Trainer(cfg, teacher=LSTMModel(make_cfg(hidden=128, layers=1)),
                device="cuda:0")
    twin = LSTMModel(cfg.model)
    twin.load_state_dict({n: p.float().cpu() for n, p in
                          t.model.state_dict().items()})
    big = LSTMModel(t.teacher.cfg)
    big.load_state_dict({n: p.float().cpu() for n, p in
                         t.teacher.state_dict().items()})
    x, y = t.data.batch(0)
    info = t.train_step((x, y))
    state = ts = None
    want = 0.0
    with torch.no_grad():
        for w in (slice(0, 4), slice(4, 8)):
            out, state = twin(x[w].cpu(), state)
            ref, ts = big(x[w].cpu(), ts)
            want += float(twin.distill_loss(out, ref, y[w].cpu(), 5, 0.7)) / 2
    # logits rounded to bf16 on both sides: 2 x 2^-8 of a few units
    assert abs(info["loss"] - want) < 0.1

"""The operators that stand around the language-model head, case by case: distillation from a
teacher's top logits, low-rank adapters of many requests beside a shared projection, and the
penalties, biases and grammar masks on the logits of a decode step.

`run` computes them from elementary torch operations in 32 bits where `own` is false, and through
the package's public entry points where it is true."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the last, short micro-batch of a distillation run: launches count, not bytes
        {"name": "distill 24 rows", "op": "distill", "n": 24, "v": 50000, "k": 32, "dtype": "bf16",
         "temperature": 2.0, "alpha": 0.5, "targets": True, "padded": 0.0, "grad": True},
        # a debug run in fp32 on an odd vocabulary, soft targets alone, a fifth of the rows padding
        {"name": "distill 1021 rows fp32 odd", "op": "distill", "n": 1021, "v": 32001, "k": 50,
         "dtype": "fp32", "temperature": 1.0, "alpha": 1.0, "targets": False, "padded": 0.2,
         "grad": True},
        # held-out evaluation of the student: the loss alone
        {"name": "distill 8192 rows eval", "op": "distill", "n": 8192, "v": 50000, "k": 64,
         "dtype": "bf16", "temperature": 1.0, "alpha": 0.5, "targets": True, "padded": 0.0,
         "grad": False},
        # a window of 64 steps at batch 256 of the 50k-vocabulary model: loss and gradient
        {"name": "distill 16384 rows", "op": "distill", "n": 16384, "v": 50000, "k": 64,
         "dtype": "bf16", "temperature": 2.0, "alpha": 0.7, "targets": True, "padded": 0.05,
         "grad": True},
        # one request decoding, one layer's input projection
        {"name": "adapter 1 row", "op": "adapter", "t": 1, "b": 1, "k": 1024, "m": 4096, "r": 16,
         "adapters": 8, "idle": 0.0, "dtype": "bf16", "grad": False},
        # a full decode batch of many tenants at the vocabulary head, some without an adapter
        {"name": "adapter 64 rows head", "op": "adapter", "t": 1, "b": 64, "k": 1024, "m": 50000,
         "r": 16, "adapters": 24, "idle": 0.15, "dtype": "bf16", "grad": False},
        # several tenants' fine-tuning in one small batch, nothing a multiple of anything, fp16
        {"name": "adapter training fp16 odd", "op": "adapter", "t": 37, "b": 29, "k": 1001,
         "m": 2049, "r": 12, "adapters": 6, "idle": 0.1, "dtype": "fp16", "grad": True},
        # fine-tuning one adapter on a layer's input projection
        {"name": "adapter training W_x", "op": "adapter", "t": 128, "b": 512, "k": 1024, "m": 4096,
         "r": 16, "adapters": 1, "idle": 0.0, "dtype": "bf16", "grad": True},
        # fine-tuning four adapters at once on the vocabulary head
        {"name": "adapter training head", "op": "adapter", "t": 32, "b": 256, "k": 1024,
         "m": 50000, "r": 32, "adapters": 4, "idle": 0.0, "dtype": "bf16", "grad": True},
        # one request decoding with penalties and a few biases
        {"name": "logits 1 row", "op": "logits", "b": 1, "v": 50000, "history": 256, "bias": 16,
         "masked": False, "dtype": "bf16"},
        # a full decode batch, penalties, biases and a grammar for every request
        {"name": "logits 64 rows grammar", "op": "logits", "b": 64, "v": 50000, "history": 1024,
         "bias": 32, "masked": True, "dtype": "bf16"},
        # a large batch in fp32 on an odd vocabulary with long histories
        {"name": "logits 257 rows fp32 odd", "op": "logits", "b": 257, "v": 32001,
         "history": 2048, "bias": 300, "masked": True, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["distill", "adapter", "logits"])
    if op == "distill":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        v = _log(rng, 100, 60000)
        n = _log(rng, 1, max(2, min(16384, int(4e8 / v))))
        targets = rng.random() < 0.7
        return {"op": op, "n": n, "v": v, "k": min(v, _log(rng, 1, 128)), "dtype": dtype,
                "temperature": rng.choice([1.0, 1.5, 2.0, 4.0]),
                "alpha": round(rng.uniform(0.1, 0.9), 3) if targets else 1.0,
                "targets": targets, "padded": rng.choice([0.0, 0.1, 0.3]),
                "grad": rng.random() < 0.7}
    if op == "adapter":
        grad = rng.random() < 0.5
        k, r = _log(rng, 64, 4096), _log(rng, 2, 64)
        m = _log(rng, 64, 50000)
        b = _log(rng, 1, 256)
        t = _log(rng, 1, max(2, min(256, int(2e8 / (m + k) / b)))) if rng.random() < 0.7 else 1
        return {"op": op, "t": t, "b": b, "k": k, "m": m, "r": r,
                "adapters": rng.randint(1, max(1, min(24, 384 // r))),
                "idle": rng.choice([0.0, 0.2]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
                "grad": grad}
    return {"op": op, "b": _log(rng, 1, 256), "v": _log(rng, 100, 60000),
            "history": _log(rng, 1, 4096), "bias": rng.choice([0, 1, 24, 300]),
            "masked": rng.random() < 0.6, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}


# ------------------------------------------------------------------ inputs
def _distinct(g, rows, count, n, dev):
    """(rows, count) whole numbers below n, no two of a row alike."""
    start = torch.randint(0, n, (rows, 1), generator=g, device=dev)
    room = max(1, n // max(1, count))
    step = torch.randint(1, room + 1, (rows, 1), generator=g, device=dev)
    return (start + step * torch.arange(count, device=dev)) % n


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(shape, generator=g, device=dev)

    s = {"case": case}
    if case["op"] == "distill":
        n, v, k = case["n"], case["v"], case["k"]
        z = randn(n, v).mul_(2.0)
        index = _distinct(g, n, k, v, dev)
        # a teacher's top logits, the student a noisy step behind
        teacher = (5.0 + 2.5 * randn(n, k)).sort(dim=1, descending=True).values
        z.scatter_(1, index, 0.7 * teacher + randn(n, k))
        y = index.gather(1, torch.randint(0, k, (n, 1), generator=g, device=dev)).squeeze(1)
        pad = rand(n) < case["padded"]          # rows behind the end of a sequence
        pad[0] = False
        index = index.masked_fill(pad[:, None], -1)
        short = torch.randint(1, k + 1, (n, 1), generator=g, device=dev)
        some = rand(n, 1) < case["padded"]      # and rows with fewer entries than the others
        index = index.masked_fill(some & (torch.arange(k, device=dev) >= short), -1)
        y = y.masked_fill(pad, -100)
        s.update(logits=z.to(dt).requires_grad_(case["grad"]), index=index,
                 teacher=teacher.to(dt), targets=y if case["targets"] else None)
    elif case["op"] == "adapter":
        t, b, k, m, r, ads = (case[c] for c in ("t", "b", "k", "m", "r", "adapters"))
        x = randn(t, b, k).to(dt)
        y = randn(t, b, m).to(dt)
        a = (randn(ads, k, r) / math.sqrt(k)).to(dt)
        w = (randn(ads, r, m) / math.sqrt(r)).to(dt)
        index = torch.randint(0, ads, (b,), generator=g, device=dev)
        index = index.masked_fill(rand(b) < case["idle"], -1)
        s.update(x=x, y=y, a=a, b=w, index=index,
                 scale=(0.5 + rand(ads)).to(torch.float32))
        if case["grad"]:
            s["dy"] = randn(t, b, m).to(dt)
            for name in ("x", "y", "a", "b"):
                s[name].requires_grad_()
        if own:  # who shares a batch is known on the host, and changes less often than the tokens
            from lstm_tensorspark_amd.ops.adapters import AdapterRows
            s["rows"] = AdapterRows(index.tolist(), ads, device=dev)
    else:
        b, v, h, nb = case["b"], case["v"], case["history"], case["bias"]
        # text repeats itself: most tokens come from a small part of the vocabulary
        common = torch.randint(0, max(1, v // 50), (b, h), generator=g, device=dev)
        rare = torch.randint(0, v, (b, h), generator=g, device=dev)
        lengths = torch.randint(max(1, h // 2), h + 1, (b,), generator=g, device=dev)
        s.update(logits=(3.0 * randn(b, v)).to(dt), history=torch.where(rand(b, h) < 0.8, common,
                                                                        rare),
                 lengths=lengths, prompt_lengths=(lengths * rand(b)).long(),
                 repetition=1.0 + 0.5 * rand(b), presence=rand(b), frequency=0.5 * rand(b),
                 bias_index=_distinct(g, b, min(nb, v), v, dev) if nb else None,
                 bias=4.0 * randn(b, min(nb, v)) if nb else None, allowed=None)
        if case["masked"]:
            words = (v + 31) // 32
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (b, words), generator=g, device=dev,
                                         dtype=torch.int64).to(torch.int32)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"distill": _distill, "adapter": _adapter, "logits": _logits}[s["case"]["op"]](s)


def _distill(s):
    c, z = s["case"], s["logits"]
    if own:
        from lstm_tensorspark_amd.ops.distill import distill_loss
        loss = distill_loss(z, s["index"], s["teacher"], s["targets"], alpha=c["alpha"],
                            temperature=c["temperature"])
    else:
        loss = _plain_distill(z, s["index"], s["teacher"], s["targets"], c["alpha"],
                              c["temperature"])
    if not c["grad"]:
        return loss
    return loss.detach(), torch.autograd.grad(loss, z)[0]


def _log_softmax(z):
    z = z - z.amax(dim=1, keepdim=True).detach()
    return z - z.exp().sum(dim=1, keepdim=True).log()


def _plain_distill(z, index, teacher, targets, alpha, tau):
    z = z.float()
    given = index >= 0
    q = (teacher.float() / tau).masked_fill(~given, -math.inf)
    has = given.any(dim=1)
    q = q - q.amax(dim=1, keepdim=True).masked_fill(~has[:, None], 0.0)
    total = q.exp().sum(dim=1, keepdim=True)
    logq = q - total.masked_fill(~has[:, None], 1.0).log()
    logp = _log_softmax(z / tau).gather(1, index.clamp_min(0))
    rows = torch.where(given, logq.exp() * (logq.masked_fill(~given, 0.0) - logp), 0.0).sum(dim=1)
    rows = alpha * tau * tau * rows
    if targets is not None:
        counted = targets >= 0
        hard = -_log_softmax(z).gather(1, targets.clamp_min(0)[:, None]).squeeze(1)
        rows = rows + (1.0 - alpha) * torch.where(counted, hard, 0.0)
        has = has | counted
    return rows.sum() / has.sum().clamp_min(1)


def _adapter(s):
    c = s["case"]
    x, y, a, b = s["x"], s["y"], s["a"], s["b"]
    if own:
        from lstm_tensorspark_amd.ops.adapters import lowrank_add
        out = lowrank_add(y, x, a, b, s["rows"], scale=s["scale"])
    else:
        out = _plain_adapter(y, x, a, b, s["index"], s["scale"])
    if not c["grad"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, (y, x, a, b), s["dy"]))


def _plain_adapter(y, x, a, b, index, scale):
    """Every row through every adapter at once, all but its own set to zero between the two."""
    ads, k, r = a.shape
    wide = x.float() @ a.float().permute(1, 0, 2).reshape(k, ads * r)
    mine = (index[:, None] == torch.arange(ads, device=index.device)).float() * scale
    wide = wide * mine.repeat_interleave(r, dim=1)
    return (y.float() + wide @ b.float().reshape(ads * r, -1)).to(y.dtype)


def _logits(s):
    names = ("repetition", "presence", "frequency", "bias_index", "bias", "allowed")
    if own:
        from lstm_tensorspark_amd.ops.logits import adjust_logits
        return adjust_logits(s["logits"], s["history"], s["lengths"], s["prompt_lengths"],
                             **{n: s[n] for n in names})
    return _plain_logits(s["logits"], s["history"], s["lengths"], s["prompt_lengths"],
                         *(s[n] for n in names))


def _plain_logits(logits, history, lengths, prompt_lengths, repetition, presence, frequency,
                  bias_index, bias, allowed):
    z = logits.float()
    at = torch.arange(history.shape[1], device=z.device)
    inside = (at < lengths[:, None]).float()
    fresh = inside * (at >= prompt_lengths[:, None]).float()
    seen = torch.zeros_like(z).scatter_add_(1, history, inside) > 0
    count = torch.zeros_like(z).scatter_add_(1, history, fresh)
    rho = repetition[:, None]
    z = torch.where(seen, torch.where(z > 0, z / rho, z * rho), z)
    z = z - frequency[:, None] * count - presence[:, None] * (count > 0).float()
    if bias_index is not None:
        z = z.scatter_add(1, bias_index, bias)
    if allowed is not None:
        v = torch.arange(z.shape[1], device=z.device)
        bit = (allowed[:, v // 32] >> (v % 32).to(torch.int32)) & 1
        z = z.masked_fill(bit == 0, -math.inf)
    return z.to(logits.dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "distill":
        n, v, k = case["n"], case["v"], case["k"]
        lists = n * k * (8 + e) + (8 * n if case["targets"] else 0)
        sums = 2 if case["targets"] and case["temperature"] != 1.0 else 1
        grad = 1 if case["grad"] else 0
        return {"bytes": n * v * e * (1 + grad) + lists + 4,
                "flops": n * v * (3 * sums + grad * (3 * sums + 2)) + 6 * n * k}
    if case["op"] == "adapter":
        n, k, m, r = case["t"] * case["b"], case["k"], case["m"], case["r"]
        used = min(case["adapters"], case["b"])     # at most so many have a row
        weights = used * r * (k + m) * e
        fwd = n * (k + 2 * m) * e + weights
        if not case["grad"]:
            return {"bytes": fwd, "flops": 2 * n * r * (k + m)}
        return {"bytes": fwd + n * (m + k) * e + case["adapters"] * r * (k + m) * e,
                "flops": 6 * n * r * (k + m)}
    b, v, h = case["b"], case["v"], case["history"]
    mask = b * ((v + 31) // 32) * 4 if case["masked"] else 0
    return {"bytes": 2 * b * v * e + b * h * 8 + mask + b * case["bias"] * 12 + 28 * b,
            "flops": 6 * b * v}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"distill": _exact_distill, "adapter": _exact_adapter,
            "logits": _exact_logits}[case["op"]](s)


def _exact_distill(s):
    c, z = s["case"], s["logits"].detach()
    n, tau, alpha = z.shape[0], c["temperature"], c["alpha"]
    entry = s["index"] >= 0
    carries = entry.any(dim=1)
    if s["targets"] is not None:
        carries = carries | (s["targets"] >= 0)
    count = max(1, int(carries.sum()))
    total = torch.zeros((), dtype=torch.float64, device=z.device)
    grad = torch.empty(z.shape, dtype=torch.float64, device=z.device) if c["grad"] else None
    for i in range(0, n, 512):
        cut = slice(i, min(n, i + 512))
        part, e = z[cut].double(), entry[cut]
        at = s["index"][cut].clamp_min(0)
        has = e.any(dim=1, keepdim=True)
        lse = torch.logsumexp(part / tau, dim=1, keepdim=True)
        t = s["teacher"][cut].double() / tau
        t = torch.where(e, t, torch.full_like(t, -math.inf))
        q = torch.where(has, torch.softmax(torch.where(has, t, 0.0), dim=1), 0.0)
        lq = torch.where(q > 0, q.clamp_min(1e-300).log(), 0.0)
        total += alpha * tau * tau * (q * (lq - (part / tau).gather(1, at) + lse)).sum()
        d = torch.exp(part / tau - lse) * has
        d = alpha * tau * d.scatter_add(1, at, -q)
        if s["targets"] is not None:
            y = s["targets"][cut]
            ok = y >= 0
            one = torch.logsumexp(part, dim=1, keepdim=True)
            hit = y.clamp_min(0)[:, None]
            total += (1 - alpha) * ((one - part.gather(1, hit)).squeeze(1) * ok).sum()
            h = torch.exp(part - one).scatter_add(
                1, hit, torch.full_like(one, -1.0)) * ok[:, None]
            d = d + (1 - alpha) * h
        if grad is not None:
            grad[cut] = d / count
    return (total / count, grad) if c["grad"] else total / count


def _exact_adapter(s):
    x, y, a, b = (s[n].detach().double() for n in ("x", "y", "a", "b"))
    out = y.clone()
    if s["case"]["grad"]:
        dy = s["dy"].double()
        dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for l, f in enumerate(s["scale"].double().tolist()):
        at = (s["index"] == l).nonzero().squeeze(1)
        if not len(at):
            continue
        xl = x[:, at].reshape(-1, x.shape[2])
        vl = xl @ a[l]
        out[:, at] += f * (vl @ b[l]).reshape(x.shape[0], len(at), -1)
        if s["case"]["grad"]:
            g = dy[:, at].reshape(-1, y.shape[2])
            dv = f * (g @ b[l].t().contiguous())
            dx[:, at] = (dv @ a[l].t().contiguous()).reshape(x.shape[0], len(at), -1)
            da[l] = xl.t().contiguous() @ dv
            db[l] = f * (vl.t().contiguous() @ g)
    return (out, dy, dx, da, db) if s["case"]["grad"] else out


def _exact_logits(s):
    z = s["logits"].double()
    b, v = z.shape
    h = s["history"].shape[1]
    row = torch.arange(b, device=z.device)[:, None].expand(b, h)
    place = torch.arange(h, device=z.device).expand(b, h)
    keep = place < s["lengths"][:, None]
    flat = row * v + s["history"]
    seen = torch.bincount(flat[keep], minlength=b * v).reshape(b, v)
    late = torch.bincount(flat[keep & (place >= s["prompt_lengths"][:, None])],
                          minlength=b * v).reshape(b, v)
    rho = s["repetition"].double()[:, None]
    z = z * torch.where(seen > 0, torch.where(z > 0, 1.0 / rho, rho), 1.0)
    z = z - late * s["frequency"].double()[:, None] - late.clamp_max(1) * \
        s["presence"].double()[:, None]
    if s["bias_index"] is not None:
        rows = torch.arange(b, device=z.device)[:, None]
        z.index_put_((rows, s["bias_index"]), s["bias"].double(), accumulate=True)
    if s["allowed"] is not None:
        bits = torch.stack([(s["allowed"] >> k) & 1 for k in range(32)], dim=2)
        z[bits.reshape(b, -1)[:, :v] == 0] = -math.inf
    return z

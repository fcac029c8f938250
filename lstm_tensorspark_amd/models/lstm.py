"""Stacked (optionally bidirectional) LSTM model with task heads.

Replaces the reference's hand-rolled TF-graph LSTM cell/model module
(SURVEY.md §2.1 "LSTM model / cell": weights 4 gates x {W_x, W_h, b},
stepped over the sequence, truncated BPTT, loss, optimizer update).

Inter-layer dropout is applied with torch's native dropout on the layer
OUTPUT (never on the recurrent path -- standard LSTM practice, and the
reason it is NOT fused into the cell kernels: the recurrent chain consumes
the un-dropped h_t, so fusing would require writing a second, dropped copy
of h -- MORE HBM traffic than the separate elementwise kernel, not less).

Weight naming follows the checkpoint layout contract (SURVEY.md §5
Checkpoint row): a flat named-weight dict with keys
    layer{i}/W_x, layer{i}/W_h, layer{i}/b           (forward direction)
    layer{i}_rev/W_x, ...                            (reverse direction)
    embed/W, head/W, head/b                          (task head)
Gate order along the 4H axis is blocked [i|f|g|o].
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..config import ModelConfig
from ..ops.lstm_layer import lstm_layer
from ..ops import xent
from ..ops.distill import distill_loss
from ..ops.logits import LogitRules, RowRules


def _pname(layer: int, rev: bool, which: str) -> str:
    return f"layer{layer}{'_rev' if rev else ''}/{which}"


# fp8 LM-head projection: +12.5% lm-50k step throughput BUT measurably
# hurts learning on the 50k-way next-token task (loss stalls at ~10.5
# where bf16 reaches 6.9 by step 150 -- e4m3 logits blur the fine logit
# differences a large-vocab head must resolve).  Default OFF; the fp8
# mode proper (recurrent + input GEMMs) converges identically to bf16.
_FP8_HEAD = False


def enable_fp8_head(on: bool):
    global _FP8_HEAD
    _FP8_HEAD = bool(on)


_REV_STREAM = None


def _rev_stream():
    """Second HIP stream for the reverse direction of bidirectional layers."""
    global _REV_STREAM
    if _REV_STREAM is None:
        _REV_STREAM = torch.cuda.Stream()
    return _REV_STREAM


class _Fp8HeadFn(torch.autograd.Function):
    """LM-head projection with the forward GEMM in e4m3 (feats are
    tanh-bounded -> FIXED scale 448; W amax-scaled).  Backward stays bf16:
    dW = feats^T·dlogits and dfeats = dlogits·W^T at full precision, so
    only the forward logits carry fp8 quantization error."""

    @staticmethod
    def forward(ctx, feats, w, b):
        # r2: ROWWISE scales (probe-verified supported by _scaled_mm on
        # ROCm torch 2.10) -- per-token amax for feats and PER-COLUMN amax
        # for W.  The r1 global-amax version measurably stalled 50k-way
        # learning (loss 10.5 vs 6.9 @150 steps): W's per-vocab-column
        # norms vary widely, so one global scale wastes e4m3 range on most
        # columns.  Falls back to global scales if rowwise is rejected.
        f8t = torch.float8_e4m3fn
        try:
            sa = feats.abs().amax(dim=1, keepdim=True).float() \
                     .clamp_min(1e-6) / 448.0
            sb = w.abs().amax(dim=0, keepdim=True).float() \
                  .clamp_min(1e-8) / 448.0
            q8 = (feats / sa).to(f8t)
            w8 = (w / sb).to(f8t).t().contiguous().t()
            out = torch._scaled_mm(q8, w8, scale_a=sa, scale_b=sb,
                                   out_dtype=torch.bfloat16)
            out += b.to(torch.bfloat16)
        except RuntimeError:
            sw = w.abs().amax().float().clamp_min(1e-8) / 448.0
            q8 = (feats * 320.0).to(f8t)
            w8 = (w * (1.0 / sw)).to(f8t).t().contiguous().t()
            sa = torch.full((), 1.0 / 320.0, device=feats.device)
            out = torch._scaled_mm(q8, w8, scale_a=sa, scale_b=sw,
                                   bias=b.to(torch.bfloat16),
                                   out_dtype=torch.bfloat16)
        ctx.save_for_backward(feats, w)
        return out

    @staticmethod
    def backward(ctx, dlogits):
        feats, w = ctx.saved_tensors
        dl = dlogits.contiguous()
        dfeats = dl @ w.t()
        dw = feats.t() @ dl
        db = dl.sum(dim=0, dtype=torch.float32).to(w.dtype)
        return dfeats, dw, db


class LSTMModel(nn.Module):
    """Multi-layer (bi)LSTM + head. Compute dtype follows parameter dtype;
    cell state is always fp32."""

    def __init__(self, cfg: ModelConfig):
        super().__init__()
        self.cfg = cfg
        H = cfg.hidden_size
        D = cfg.num_directions
        self._params: dict[str, nn.Parameter] = {}
        self._zero_state: dict = {}   # (B, device, dtype) -> (h0, c0)

        if cfg.head == "lm":
            assert cfg.vocab_size > 0
            self._register("embed/W", torch.empty(cfg.vocab_size, cfg.input_size))

        for l in range(cfg.num_layers):
            in_size = cfg.input_size if l == 0 else H * D
            for rev in ([False, True] if cfg.bidirectional else [False]):
                self._register(_pname(l, rev, "W_x"), torch.empty(in_size, 4 * H))
                self._register(_pname(l, rev, "W_h"), torch.empty(H, 4 * H))
                self._register(_pname(l, rev, "b"), torch.empty(4 * H))

        feat = H * D
        if cfg.head in ("classifier", "seq_classifier"):
            self._register("head/W", torch.empty(feat, cfg.num_classes))
            self._register("head/b", torch.empty(cfg.num_classes))
        elif cfg.head == "lm":
            self._register("head/W", torch.empty(feat, cfg.vocab_size))
            self._register("head/b", torch.empty(cfg.vocab_size))
        self.reset_parameters()

    # -- flat named-weight dict plumbing ----------------------------------
    def _register(self, name: str, t: torch.Tensor):
        p = nn.Parameter(t)
        self.register_parameter(name.replace("/", "__"), p)
        self._params[name] = p

    def weight(self, name: str) -> nn.Parameter:
        return self._params[name]

    def weight_dict(self) -> dict[str, nn.Parameter]:
        """The flat named-weight dict (checkpoint layout contract)."""
        return dict(self._params)

    def reset_parameters(self, seed: Optional[int] = None):
        g = None
        if seed is not None:
            g = torch.Generator(device="cpu")
            g.manual_seed(seed)
        H = self.cfg.hidden_size
        std = 1.0 / math.sqrt(H)
        with torch.no_grad():
            for name, p in self._params.items():
                if name == "embed/W":
                    src = torch.randn(p.shape, generator=g) * 0.02
                elif name.endswith("/b"):
                    src = torch.zeros(p.shape)
                    if name.startswith("layer"):
                        # forget-gate bias = 1 (standard LSTM practice)
                        src[H : 2 * H] = 1.0
                else:
                    src = (torch.rand(p.shape, generator=g) * 2 - 1) * std
                p.copy_(src)

    # -- forward -----------------------------------------------------------
    def _layer_io(self, x, layer: int, rev: bool, state=None, adapters=None):
        B = x.shape[1]
        H = self.cfg.hidden_size
        w_x = self.weight(_pname(layer, rev, "W_x"))
        w_h = self.weight(_pname(layer, rev, "W_h"))
        b = self.weight(_pname(layer, rev, "b"))
        if state is None:
            # cached zero states: the per-call torch.zeros pair cost
            # ~2 ms/step at the headline shape (200 MB/step of zero-fill
            # for 2 layers); these are read-only inputs everywhere (the
            # kernels never write h0/c0 and autograd saves, not mutates),
            # so one cached pair per (B, device, dtype) is safe -- and
            # address-stable, which hipGraph capture likes.
            key = (B, x.device, x.dtype)
            zs = self._zero_state.get(key)
            if zs is None:
                zs = (torch.zeros(B, H, dtype=x.dtype, device=x.device),
                      torch.zeros(B, H, dtype=torch.float32, device=x.device))
                self._zero_state[key] = zs
            h0, c0 = zs
        else:
            h0, c0 = state
        add = None
        if adapters is not None:
            site = f"layer{layer}{'_rev' if rev else ''}"
            add = lambda pre, x: adapters.add(pre, x, site)  # noqa: E731
        return lstm_layer(x, h0, c0, w_x, w_h, b, reverse=rev, add=add)

    def backbone(self, x: torch.Tensor, state: Optional[list] = None,
                 adapters=None):
        """Run embedding (if LM) + all LSTM layers.

        x: (T,B,input_size) features, or (T,B) long tokens for LM
           (TIME-MAJOR -- the engine's native layout, see ops/functional.py).
        state: per-(layer,dir) list of (h0, c0) carry (truncated BPTT), or
               None for zero state.
        adapters: AdapterSet.rows(...) of the batch's columns, or None.
        Returns (features (T,B,H*D), new_state list).
        """
        cfg = self.cfg
        if cfg.head == "lm":
            x = F.embedding(x, self.weight("embed/W"))
        new_state = []
        si = 0
        for l in range(cfg.num_layers):
            if cfg.bidirectional and x.is_cuda:
                # The two directions are independent: run the REVERSE pass
                # on a second HIP stream so its sequential recurrence
                # overlaps the forward direction's (SURVEY.md §7 hard part
                # 5).  Autograd records each op's stream, so the two
                # backward recurrences overlap the same way; the engine
                # inserts the cross-stream grad syncs itself.
                cur = torch.cuda.current_stream()
                s2 = _rev_stream()
                s2.wait_stream(cur)            # x (and carries) are ready
                st = state[si + 1] if state is not None else None
                with torch.cuda.stream(s2):
                    x.record_stream(s2)
                    h_rev, hT_r, cT_r = self._layer_io(x, l, True, st,
                                                     adapters)
                st = state[si] if state is not None else None
                h_fwd, hT_f, cT_f = self._layer_io(x, l, False, st,
                                                 adapters)
                cur.wait_stream(s2)            # before the concat reads
                new_state += [(hT_f, cT_f), (hT_r, cT_r)]
                si += 2
                x = torch.cat([h_fwd, h_rev], dim=2)
            else:
                outs = []
                for rev in ([False, True] if cfg.bidirectional else [False]):
                    st = state[si] if state is not None else None
                    h_seq, hT, cT = self._layer_io(x, l, rev, st, adapters)
                    outs.append(h_seq)
                    new_state.append((hT, cT))
                    si += 1
                x = outs[0] if len(outs) == 1 else torch.cat(outs, dim=2)
            if cfg.dropout > 0 and self.training and l < cfg.num_layers - 1:
                x = F.dropout(x, p=cfg.dropout)
        return x, new_state

    def forward(self, x, state: Optional[list] = None, adapters=None):
        """Returns (output, new_state).

        output: logits -- (B,C) for "classifier", (T,B,C) for
        "seq_classifier", (T,B,V) for "lm", features (T,B,H*D) for "none".
        """
        feats, new_state = self.backbone(x, state, adapters)
        cfg = self.cfg
        if cfg.head == "none":
            return feats, new_state
        w, b = self.weight("head/W"), self.weight("head/b")
        if cfg.head == "classifier":
            out = torch.addmm(b, feats[-1], w)
            if adapters is not None:
                out = adapters.add(out, feats[-1], "head")
            return out, new_state
        T, B, F_ = feats.shape
        flat = feats.reshape(T * B, F_)
        if (cfg.head == "lm" and feats.is_cuda
                and feats.dtype == torch.bfloat16 and self._fp8_head()
                and (T * B) % 16 == 0 and F_ % 16 == 0
                and w.shape[1] % 16 == 0):
            logits = _Fp8HeadFn.apply(flat, w, b).view(T, B, -1)
        else:
            logits = torch.addmm(b, flat, w).view(T, B, -1)
        if adapters is not None:
            logits = adapters.add(logits, feats, "head")
        return logits, new_state

    @staticmethod
    def _fp8_head() -> bool:
        # r2: independent of the fp8 RECURRENT switch -- the r1 "fp8 head
        # quality failure" was misattributed: isolation runs showed the
        # fp8 recurrent path stalls 50k-way LM learning (loss stuck at
        # ~10.3 vs bf16's 0.29 @120 steps on lm_assoc) while bf16
        # recurrent + fp8 head converges cleanly (profiles/r02_fp8_lm.md).
        from ..ops import extension
        return _FP8_HEAD and extension.extension_available()

    def loss(self, output: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        head = self.cfg.head
        if head == "classifier":
            return xent.cross_entropy(output, y)
        if head in ("seq_classifier", "lm"):
            C = output.shape[-1]
            # fused K3 kernel on GPU bf16 (one online-softmax pass, no fp32
            # (N,V) intermediate); torch CE elsewhere
            return xent.cross_entropy(output.reshape(-1, C), y.reshape(-1))
        # regression on features
        return F.mse_loss(output.float(), y.float())

    def distill_loss(self, output: torch.Tensor, teacher: torch.Tensor,
                     y: Optional[torch.Tensor], top_k: int = 64,
                     alpha: float = 0.5, temperature: float = 2.0,
                     weight: float = 1.0) -> torch.Tensor:
        """Loss against a teacher's logits (same shape as `output`): its
        top_k of every position at `temperature`, weighed by alpha against
        the labels y, the whole multiplied by weight (ops/distill.py)."""
        if self.cfg.head == "none":
            raise ValueError("distillation needs a head with logits")
        if teacher.shape != output.shape:
            raise ValueError(f"teacher's logits {tuple(teacher.shape)} and "
                             f"the model's {tuple(output.shape)} differ")
        if top_k < 1:
            raise ValueError(f"top_k must be positive, got {top_k}")
        C = output.shape[-1]
        top = teacher.detach().reshape(-1, C).topk(min(top_k, C), dim=1)
        return distill_loss(output.reshape(-1, C), top.indices, top.values,
                            None if y is None else y.reshape(-1),
                            alpha=alpha, temperature=temperature,
                            weight=weight)

    def detach_state(self, state):
        """Detach the (h, c) carry for truncated BPTT."""
        if state is None:
            return None
        return [(h.detach(), c.detach()) for h, c in state]

    @torch.no_grad()
    def generate(self, prompt: torch.Tensor, steps: int,
                 temperature: float = 0.0,
                 generator: "Optional[torch.Generator]" = None,
                 use_graph: Optional[bool] = None,
                 use_gemv: Optional[bool] = None,
                 top_k: int = 0, top_p: float = 0.0,
                 eos_token: int = -1,
                 rules: "Optional[LogitRules]" = None,
                 adapters=None) -> torch.Tensor:
        """Autoregressive decode for the LM head (the serving path).

        prompt: (Tp, B) long tokens (time-major).  Returns (Tp+steps, B):
        the prompt followed by `steps` generated tokens.  temperature 0 =
        greedy argmax; >0 = softmax sampling.  The recurrent (h, c) state
        is carried across steps, so each decode step is one T=1 pass.
        top_k / top_p restrict sampling to the k most likely tokens /
        the smallest nucleus with mass >= top_p (sampling path only).
        eos_token >= 0 stops a sequence at that token (a finished column
        keeps emitting eos); decode ends early once EVERY column is done
        (eager path only -- the graphed decode runs fixed steps).
        rules: penalties, biases and a grammar for every column
        (ops/logits.py); adapters: AdapterSet.rows(...) of the B columns
        (both on the eager path only).

        use_graph (default: auto = greedy + CUDA + steps >= 16): capture
        ONE decode step as a hipGraph whose body copies its outputs back
        into its own static inputs and appends the token to a device
        buffer, then replay it per token -- removes ALL per-token launch
        and Python overhead (small-B decode is launch-latency bound).
        """
        assert self.cfg.head == "lm", "generate() requires the LM head"
        assert not self.cfg.bidirectional, "decode is causal: fwd-only"
        assert prompt.dim() == 2 and prompt.dtype == torch.long
        if use_graph is None:
            use_graph = (temperature <= 0 and prompt.is_cuda and steps >= 16
                         and eos_token < 0 and rules is None
                         and adapters is None)
        assert not (use_graph and temperature > 0), \
            "the graphed decode step is greedy-only"
        assert not (use_graph and eos_token >= 0), \
            "eos early-stop needs the eager path (use_graph=False)"
        assert not (use_graph and (rules is not None
                                   or adapters is not None)), \
            "rules and adapters need the eager path (use_graph=False)"
        Tp, B = prompt.shape
        if rules is not None:
            rules.check(self.cfg.vocab_size)
            every = RowRules([rules] * B, [Tp] * B, self.cfg.vocab_size,
                             prompt.device)
            seen = torch.zeros(B, Tp + max(steps, 1), dtype=torch.long,
                               device=prompt.device)
            seen[:, :Tp] = prompt.t()

        done = None

        def ruled(logits, length):
            if rules is None:
                return logits
            past = seen[:, :length]
            allowed = ()
            if rules.grammar:       # not asked about a finished column
                ended = [False] * B if done is None else done.tolist()
                allowed = [None if e else rules.allows(t, logits.shape[1])
                           for t, e in zip(past.tolist(), ended)]
            return every.apply(logits, past, None, allowed)

        # behind every refusal: a refused call leaves the mode as it was
        was_training = self.training
        self.eval()
        try:
            out, state = self.forward(prompt, None, adapters)  # (Tp, B, V)
            cur = self._sample(ruled(out[-1], Tp), temperature, generator,
                               top_k, top_p)
            if use_graph:
                return torch.cat(
                    [prompt, self._graph_decode(cur, state, steps, use_gemv)],
                    dim=0)
            toks = [prompt]
            done = (cur == eos_token) if eos_token >= 0 else None
            for i in range(steps - 1):
                toks.append(cur.unsqueeze(0))
                if done is not None and bool(done.all()):
                    break
                if rules is not None:
                    seen[:, Tp + i] = cur
                out, state = self.forward(cur.unsqueeze(0), state, adapters)
                cur = self._sample(ruled(out[-1], Tp + i + 1), temperature,
                                   generator, top_k, top_p)
                if done is not None:
                    cur = torch.where(done, torch.full_like(cur, eos_token),
                                      cur)
                    done = done | (cur == eos_token)
            else:
                toks.append(cur.unsqueeze(0))
            return torch.cat(toks, dim=0)
        finally:
            if was_training:
                self.train()

    @torch.no_grad()
    def generate_beam(self, prompt: torch.Tensor, steps: int,
                      beam_size: int = 4, eos_token: int = -1):
        """Beam-search decode for a single prompt (B=1): the beams ride the
        BATCH dimension, so every decode step is ONE batched forward (the
        same kernels that serve batched greedy decode -- no per-beam loop).

        Keeps the `beam_size` highest-sum-logprob prefixes each step.  If
        `eos_token` >= 0, a beam that emits it is frozen (it keeps emitting
        eos at no score change) so finished hypotheses compete with live
        ones on equal footing.  Returns (tokens (Tp+steps, 1), score) --
        the best beam and its total log-probability.
        """
        assert self.cfg.head == "lm", "beam search requires the LM head"
        assert not self.cfg.bidirectional, "decode is causal: fwd-only"
        assert prompt.dim() == 2 and prompt.shape[1] == 1, \
            "generate_beam takes a single prompt (Tp, 1)"
        assert beam_size >= 1
        V = self.cfg.vocab_size
        was_training = self.training
        self.eval()
        try:
            out, state = self.forward(prompt)               # (Tp, 1, V)
            logp = torch.log_softmax(out[-1, 0].float(), dim=-1)
            k = min(beam_size, V)
            if k == 1:
                # argmax guarantees first-index tie-breaking (topk does
                # not), making beam_size=1 identical to greedy decode by
                # construction -- including on bf16 logit ties
                tok = logp.argmax().unsqueeze(0)
                scores = logp[tok]
            else:
                scores, tok = logp.topk(k)                  # (k,)
            state = [(h.expand(k, -1).contiguous(),
                      c.expand(k, -1).contiguous()) for h, c in state]
            seqs = tok.unsqueeze(0)                         # (t, k)
            frozen = (tok == eos_token)
            for _ in range(steps - 1):
                out, state = self.forward(seqs[-1:].contiguous(), state)
                lp = torch.log_softmax(out[-1].float(), dim=-1)  # (k, V)
                if frozen.any():
                    # frozen beams only extend with eos at zero cost
                    lp[frozen] = float("-inf")
                    lp[frozen, eos_token] = 0.0
                cand = (scores.unsqueeze(1) + lp).reshape(-1)    # (k*V,)
                if k == 1:
                    idx = cand.argmax().unsqueeze(0)
                    scores = cand[idx]
                else:
                    scores, idx = cand.topk(k)
                parent = torch.div(idx, V, rounding_mode="floor")
                tok = idx % V
                state = [(h[parent], c[parent]) for h, c in state]
                seqs = torch.cat([seqs[:, parent], tok.unsqueeze(0)], dim=0)
                frozen = frozen[parent] | (tok == eos_token)
            best = int(scores.argmax())
            seq = torch.cat([prompt, seqs[:, best:best + 1]], dim=0)
            return seq, float(scores[best])
        finally:
            if was_training:
                self.train()

    _DECODE_CAP = 8192  # tokens per replay series (out ring capacity)

    def _gemv_cache(self):
        """Serving weight layout: pre-transposed [W_x;W_h]^T per layer and
        head W^T (doubles head-weight memory -- a serving cache, not a
        training cost).  Rebuilt whenever the weights version changes
        (Trainer bumps `_weights_version` after every optimizer step), so
        train -> generate -> train -> generate serves CURRENT weights."""
        gc = getattr(self, "_gemv_weights", None)
        ver = getattr(self, "_weights_version", 0)
        if gc is not None and gc.get("version") == ver:
            return gc
        cfg = self.cfg
        layers = []
        for l in range(cfg.num_layers):
            w_x = self.weight(_pname(l, False, "W_x"))
            w_h = self.weight(_pname(l, False, "W_h"))
            b = self.weight(_pname(l, False, "b"))
            wcat_t = torch.cat([w_x.detach(), w_h.detach()], dim=0).t().contiguous()
            layers.append((wcat_t, b.detach().float()))
        head_t = self.weight("head/W").detach().t().contiguous()
        head_b = self.weight("head/b").detach().float()
        gc = {"layers": layers, "head_t": head_t, "head_b": head_b,
              "version": ver}
        self._gemv_weights = gc
        # the captured decode graph reads the gemv cache tensors by
        # address: a rebuilt cache means new tensors, so drop the graph too
        if getattr(self, "_dec_cache", None) is not None \
                and self._dec_cache.get("gemv"):
            self._dec_cache = None
        return gc

    def _gemv_step(self, cur, g_state):
        """One greedy decode step through the streaming-GEMV kernels
        (updates g_state in place, returns the next token)."""
        from ..ops.extension import get_extension
        ext = get_extension()
        gc = self._gemv_cache()
        x = F.embedding(cur, self.weight("embed/W"))
        for l, (wcat_t, b) in enumerate(gc["layers"]):
            h, c = g_state[l]
            xcat = torch.cat([x, h], dim=1)
            raw = ext.decode_gemv(wcat_t, xcat, b)
            ext.decode_cell_(raw, h, c)   # in-place state update, ONE kernel
            x = h
        logits = ext.decode_gemv(gc["head_t"], x, gc["head_b"])
        return logits.argmax(dim=-1)

    def _gemv_eligible(self, B: int) -> bool:
        from ..ops import extension
        if not extension.extension_available() or self.cfg.bidirectional:
            return False
        ext = extension.get_extension()
        cfg = self.cfg
        K0 = cfg.input_size + cfg.hidden_size
        return bool(ext.decode_gemv_ok(B, K0)
                    and ext.decode_gemv_ok(B, cfg.hidden_size
                                           * cfg.num_directions))

    def _graph_decode(self, cur, state, steps: int,
                      use_gemv: Optional[bool] = None) -> torch.Tensor:
        """Greedy decode via a replayed hipGraph (see generate()).  The
        captured graph + its static buffers are CACHED on the model keyed
        by (batch size, gemv), so steady-state serving is replay-only.
        use_gemv (auto: on when eligible) streams the weights through the
        hand-written serving GEMV instead of library mm."""
        B = cur.shape[0]
        dev = cur.device
        if use_gemv is None:
            use_gemv = self._gemv_eligible(B)
        if use_gemv:
            # MUST run before the cache check: if the weights version
            # moved, this rebuilds the serving-weight tensors AND drops
            # the captured graph that holds the old tensors' addresses --
            # otherwise a cached gemv graph would replay STALE weights
            # after train -> generate -> train -> generate
            self._gemv_cache()
        cache = getattr(self, "_dec_cache", None)
        if cache is None or cache["B"] != B or cache["gemv"] != use_gemv:
            g_cur = cur.clone()
            g_state = [(h.clone(), c.clone()) for h, c in state]
            out_buf = torch.empty(self._DECODE_CAP, B, dtype=torch.long,
                                  device=dev)
            idx = torch.zeros((), dtype=torch.long, device=dev)

            def body():
                out_buf.index_copy_(0, idx.unsqueeze(0), g_cur.unsqueeze(0))
                idx.add_(1)
                if use_gemv:
                    nxt = self._gemv_step(g_cur, g_state)
                else:
                    logits, new_state = self.forward(g_cur.unsqueeze(0), g_state)
                    nxt = logits[-1].argmax(dim=-1)
                    for (h, c), (nh, nc) in zip(g_state, new_state):
                        h.copy_(nh)
                        c.copy_(nc)
                g_cur.copy_(nxt)

            for _ in range(2):        # warmup (workspaces at stable addrs)
                body()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                body()
            cache = {"B": B, "gemv": use_gemv, "graph": graph, "g_cur": g_cur,
                     "g_state": g_state, "out_buf": out_buf, "idx": idx}
            self._dec_cache = cache
        # (re)prime the static buffers from this call's live state
        cache["g_cur"].copy_(cur)
        for (h, c), (oh, oc) in zip(cache["g_state"], state):
            h.copy_(oh)
            c.copy_(oc)
        outs = []
        done = 0
        while done < steps:
            n = min(steps - done, self._DECODE_CAP)
            cache["idx"].zero_()
            for _ in range(n):
                cache["graph"].replay()
            outs.append(cache["out_buf"][:n].clone())
            done += n
        return outs[0] if len(outs) == 1 else torch.cat(outs, dim=0)

    @staticmethod
    def _sample(logits, temperature, generator, top_k=0, top_p=0.0):
        if temperature <= 0:
            return logits.argmax(dim=-1)
        logits = logits.float() / temperature
        if top_k and top_k > 0 and top_k < logits.shape[-1]:
            kth = logits.topk(top_k, dim=-1).values[..., -1:]
            logits = logits.masked_fill(logits < kth, float("-inf"))
        if 0.0 < top_p < 1.0:
            # nucleus: keep the smallest prefix of the sorted distribution
            # whose mass reaches top_p (always at least the top token)
            srt, idx = logits.sort(dim=-1, descending=True)
            cum = torch.softmax(srt, dim=-1).cumsum(dim=-1)
            drop = cum - torch.softmax(srt, dim=-1) >= top_p
            srt = srt.masked_fill(drop, float("-inf"))
            logits = torch.full_like(logits, float("-inf")).scatter_(
                -1, idx, srt)
        probs = torch.softmax(logits, dim=-1)
        return torch.multinomial(probs, 1, generator=generator).squeeze(-1)

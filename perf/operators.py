"""From a model's hidden states to the log probabilities of its answer, as cases to time.

Three operators, each through `CudaBackend` where `own` is true and as elementary torch operations where it is
not:

* "linear": `matmul_epilogue`, act(x . w^T + bias) + residual.  The layers of models whose projections carry a bias, whose
  MLP is not gated, or whose residual stream is added to without a norm between.
* "logits": `logprob_rows`, the log probabilities of given tokens, the entropy and the best alternatives from rows of logits.
  What a serving API reports beside every token it sends.
* "head": `matmul_logprobs`, the log probability of one given token and the entropy of every row, straight from hidden states
  and the head's weight.  Scoring of prompts and of drafts, whose logits nobody else reads.

Sizes are those of `perf/cases.py` (hidden 1024, 2048 and 4096, vocabularies of 32000 and 50257, sixteen
sequences with five rows each in a verification) and ragged ones.
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
MOST = torch.finfo(torch.float32).max


def _linear(name=None, **kw):
    c = dict(op="linear", x="f32", out="f32", bias=True, act="none", residual=False)
    c.update(kw)
    return dict(c, name=name) if name else c


def _logits(name=None, **kw):
    c = dict(op="logits", x="f32", ids=1, top=0, entropy=True, pad=0, mask="none")
    c.update(kw)
    return dict(c, name=name) if name else c


def _head(name=None, **kw):
    c = dict(op="head", x="f32", entropy=True)
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One user's next token on a small model whose MLP is a plain one: all latency.
        _linear("up_gelu_1row", rows=1, n=2816, k=1024, act="gelu"),
        # The serving loop on a large model: sixteen rows through the down projection, onto the residual stream.
        _linear("down_residual_16rows", rows=16, n=4096, k=14336, residual=True),
        # Verification of five rows for each of sixteen sequences: bf16 attention output through the output projection.
        _linear("attn_out_80rows_bf16", rows=80, n=4096, k=4096, x="bf16", residual=True),
        # A prompt chunk of ragged length on a ragged model, all f32.
        _linear("prompt_ragged_f32", rows=300, n=5633, k=2040, act="silu", residual=True),
        # A prompt chunk on a large model that keeps its activations in bf16.
        _linear("up_gelu_2048rows_bf16", rows=2048, n=14336, k=4096, x="bf16", out="bf16", act="gelu_tanh"),
        # One user's token with its five best alternatives.
        _logits("token_top5", rows=1, vocab=50257, top=5),
        # Sixteen users' tokens with twenty alternatives, logits in bf16.
        _logits("batch_top20_bf16", rows=16, vocab=32000, x="bf16", top=20),
        # Constrained decoding: most tokens forbidden, rows with none left, logits in rows padded to a round length; four
        # continuations are weighed.
        _logits("masked_top8_f16", rows=48, vocab=32003, x="f16", ids=4, top=8, pad=125, mask="inf"),
        # A prompt chunk's logits, scored.
        _logits("prompt_logits_f32", rows=2048, vocab=50257, top=5),
        # One row on a small model, from the hidden state: the smallest call of the head.
        _head("score_1row", rows=1, vocab=32000, k=1024),
        # The drafts of a verification.
        _head("score_80rows_bf16", rows=80, vocab=50257, k=4096, x="bf16"),
        # A prompt chunk on a large model: the largest.
        _head("score_2048rows_f32", rows=2048, vocab=50257, k=4096),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op, rows, x = rng.choice(["linear", "logits", "head"]), _log(rng, 1, 2048), rng.choice(["f32", "f16", "bf16"])
    k = 8 * _log(rng, 16, 512)
    if op == "linear":
        return _linear(rows=rows, n=_log(rng, 100, 14336), k=k, x=x, out=rng.choice(["f32", "f32", x]), bias=rng.random() < 0.7,
                       act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), residual=rng.random() < 0.5)
    vocab = _log(rng, 500, 50257)
    if op == "head":
        return _head(rows=rows, vocab=vocab, k=k, x=x, entropy=rng.random() < 0.7)
    return _logits(rows=rows, vocab=vocab, x=x, ids=rng.choice([1, 1, 1, 2, 5]), top=rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                   entropy=rng.random() < 0.7, pad=rng.choice([0, 0, rng.randint(1, 300)]), mask=rng.choice(["none", "none", "inf", "lowest", "nan"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")    # noqa: E731
    rows, x = case["rows"], TORCH[case["x"]]
    s = SimpleNamespace(case=case)
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        s.x = normal(rows, k).to(x)
        s.w = normal(n, k).mul_(k ** -0.5).bfloat16()
        s.bias = normal(n).mul_(0.2) if case["bias"] else None
        # (a residual stream is several times what one layer adds to it)
        s.residual = normal(rows, n).mul_(4.0).to(TORCH[case["out"]]) if case["residual"] else None
        return s
    vocab = case["vocab"]
    if case["op"] == "head":
        k = case["k"]
        s.w = normal(vocab, k).mul_(2.0 * k ** -0.5).bfloat16()
        # Rows a norm has left at unit size, most of them leaning towards the token that follows.
        s.ids = rng.integers(0, vocab, rows).astype(np.uint32)
        lean = torch.from_numpy(np.maximum(0.0, rng.uniform(-0.8, 3.0, rows)).astype(np.float32)).cuda()
        s.x = (normal(rows, k) + lean[:, None] * s.w[torch.from_numpy(s.ids.astype(np.int64)).cuda()].float()).to(x)
        return s
    # Logits of a language model: a broad bell, and per row some tokens that stand out of it.
    store = normal(rows, vocab + case["pad"]).mul_(2.5)
    out = torch.from_numpy(rng.integers(0, vocab, (rows, 24))).cuda()
    store.scatter_add_(1, out, normal(rows, 24).mul_(2.0).add_(torch.linspace(12.0, 2.0, 24, device="cuda")))
    ids = rng.integers(0, vocab, (rows, case["ids"]))
    told = rng.random(ids.shape) < 0.7   # most given tokens are among those that stand out
    ids[told] = np.take_along_axis(out.cpu().numpy(), rng.integers(0, 24, ids.shape), 1)[told]
    s.ids = ids.astype(np.uint32)
    if case["mask"] != "none":
        # All but some tens of tokens forbidden in most rows, everything in every seventh, nothing in the others.
        free = torch.rand(rows, vocab + case["pad"], generator=gen, device="cuda") < min(0.5, 40.0 / vocab)
        which = torch.arange(rows, device="cuda") % 7
        forbidden = (~free | (which == 3)[:, None]) & (which < 5)[:, None]
        value = {"inf": -math.inf, "lowest": torch.finfo(x).min, "nan": math.nan}[case["mask"]]
        store = store.masked_fill_(forbidden, value)
    s.logits = store.to(x)[:, :vocab]
    return s


_BACKEND = []


def _backend():
    """One backend to a process, as a server holds one."""
    if not _BACKEND:
        from yaxus_b200 import CudaBackend
        _BACKEND.append(CudaBackend(0))
    return _BACKEND[0]


def run(state):
    case = state.case
    if own:
        return _run_own(state, case)
    if case["op"] == "linear":
        return {"out": _plain_linear(state, case)}
    if case["op"] == "head":
        return _plain_logprobs(state.x.float() @ state.w.float().T, state.ids[:, None], 0, case["entropy"], squeeze=True)
    return _plain_logprobs(state.logits.float(), state.ids, case["top"], case["entropy"])


def _run_own(s, case):
    b = _backend()
    if case["op"] == "linear":
        return {"out": b.matmul_epilogue(s.x, s.w, bias=s.bias, activation=case["act"], residual=s.residual, out_dtype=TORCH[case["out"]])}
    if case["op"] == "head":
        r = b.matmul_logprobs(s.x, s.w, s.ids, entropy=case["entropy"])
    else:
        r = b.logprob_rows(s.logits, s.ids, top=case["top"], entropy=case["entropy"])
    out = {"logprob": r.logprob}
    if case["entropy"]:
        out["entropy"] = r.entropy
    if case.get("top"):
        out["top_ids"], out["top_logprob"] = r.top_ids, r.top_logprob
    return out


def _plain_linear(s, case):
    y = s.x.float() @ s.w.float().T
    if s.bias is not None:
        y = y + s.bias
    act = case["act"]
    if act == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif act == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif act == "silu":
        y = y / (1.0 + torch.exp(-y))
    if s.residual is not None:
        y = y + s.residual.float()
    return y.to(TORCH[case["out"]])


def _plain_logprobs(logits, ids, top, entropy, squeeze=False):
    # No number counts as forbidden, and +inf as the largest number; a row with nothing left has no probabilities.
    l = torch.where(torch.isnan(logits), -math.inf, logits).clamp(max=MOST)
    m = l.amax(1, keepdim=True)
    empty = m == -math.inf
    d = l - torch.where(empty, torch.zeros_like(m), m)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(torch.where(empty, torch.ones_like(total), total))
    ids = torch.from_numpy(ids.astype(np.int64)).cuda()
    out = {"logprob": d.gather(1, ids) - log_total}
    if squeeze:
        out["logprob"] = out["logprob"][:, 0]
    if entropy:
        weighted = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1, keepdim=True)
        out["entropy"] = torch.where(empty, torch.zeros_like(total), log_total - weighted / total)[:, 0]
    if top:
        # Largest first, equal ones by their index: one whole number that orders both.
        bits = (l + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * 2 ** 32 + (2 ** 31 - torch.arange(l.shape[1], device=l.device))
        best = torch.topk(order, top, dim=1).indices
        out["top_ids"] = best.int()
        out["top_logprob"] = d.gather(1, best) - log_total
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = torch.matmul(s.x.double(), s.w.double().t())
        y = y.add_(s.bias.double()) if case["bias"] else y
        act = {"none": lambda v: v,
               "relu": lambda v: v.clamp(min=0.0),
               "gelu": lambda v: v * torch.special.ndtr(v),
               "gelu_tanh": lambda v: v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)),
               "silu": lambda v: v * torch.sigmoid(v)}[case["act"]]
        y = act(y)
        return {"out": y + s.residual.double() if case["residual"] else y}
    z = torch.matmul(s.x.double(), s.w.double().t()) if case["op"] == "head" else s.logits.double()
    z = z.masked_fill(torch.isnan(z), -math.inf)
    logp = torch.log_softmax(z, 1)
    logp = logp.masked_fill_(torch.isnan(logp), -math.inf)   # (rows with nothing left)
    ids = torch.as_tensor(s.ids.astype(np.int64), device=z.device).reshape(case["rows"], -1)
    out = {"logprob": torch.take_along_dim(logp, ids, 1)}
    if case["op"] == "head":
        out["logprob"] = out["logprob"].reshape(-1)
    if case["entropy"]:
        out["entropy"] = torch.special.entr(logp.exp()).sum(1)
    if case.get("top"):
        value, at = torch.sort(z, dim=1, descending=True, stable=True)
        out["top_ids"] = at[:, :case["top"]].int()
        out["top_logprob"] = torch.take_along_dim(logp, at[:, :case["top"]], 1)
    return out


def work(case):
    rows, x = case["rows"], SIZE[case["x"]]
    if case["op"] == "linear":
        n, k, out = case["n"], case["k"], SIZE[case["out"]]
        return {"bytes": rows * k * x + n * k * 2 + (4 * n if case["bias"] else 0) + rows * n * out * (2 if case["residual"] else 1),
                "flops": 2 * rows * n * k}
    vocab, results = case["vocab"], 4 * (1 if case["entropy"] else 0)
    if case["op"] == "head":
        return {"bytes": rows * case["k"] * x + vocab * case["k"] * 2 + rows * (4 + 4 + results), "flops": 2 * rows * vocab * case["k"]}
    results += 8 * case["ids"] + 8 * case["top"]
    return {"bytes": rows * (vocab * x + results), "flops": 5 * rows * vocab}

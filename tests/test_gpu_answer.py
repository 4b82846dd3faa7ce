"""The operators between hidden states and log probabilities run together, as a server would: the passes of a small model
(prompt, then one token) with its answer's log probabilities, and a model whose layers have biases and a plain MLP."""
import numpy as np
import pytest
import torch

from yaxus_b200._lib import F32, PAGE
from yaxus_b200.backend import LayerMeta, Rope
from yaxus_b200.kvcache import KvCache

from .test_gpu_forward import EPS, HIDDEN, HKV, INNER, VOCAB, D, TinyWeights, forward_cuda, forward_oracle, on_device

pytestmark = pytest.mark.gpu


def log_softmax64(x):
    x = np.asarray(x, np.float64)
    x = x - x.max(1, keepdims=True)
    return x - np.log(np.exp(x).sum(1, keepdims=True))


def test_a_model_s_answer_with_its_log_probabilities(backend, oracle):
    # a prompt's pass gives its last row's logits; every next token is picked, reported with its alternatives and fed back
    w = TinyWeights(oracle, 2, seed=9)
    dw = on_device(backend, w)
    metas = [LayerMeta(index=0, window=None, rope=Rope.default()), LayerMeta(index=1, window=48, rope=Rope.default())]
    pages, max_pos = 8, 4 * PAGE
    kv = backend.new_kv(HKV, metas, pages, max_pos, F32)
    arenas = [(np.zeros((pages * PAGE, HKV * D), np.float32), np.zeros((pages * PAGE, HKV * D), np.float32)) for _ in metas]
    book = KvCache(pages, max_pos)
    seq = book.new_seq()
    tokens = np.random.default_rng(5).integers(0, VOCAB, 70)
    for step in range(3):
        meta = book.append([(seq, tokens)])
        for src, dst in book.take_copies():
            backend.copy_page(kv, src, dst)
        logits = forward_cuda(backend, dw, kv, metas, meta)
        picked = backend.argmax_rows(logits)
        r = backend.logprob_rows(logits, picked, top=5, entropy=True)
        backend.sync()
        ref = log_softmax64(forward_oracle(oracle, w, arenas, metas, meta, F32))
        # logits agree to 3e-4 (as the forward passes' own test has it), a log probability to twice that
        assert abs(r.logprob.item() - ref[0, picked[0]]) <= 6e-4
        assert abs(r.entropy.item() + (np.exp(ref) * ref).sum()) <= 6e-4 * (2 + np.log(VOCAB))
        assert r.top_ids[0, 0].item() == picked[0] and r.top_logprob[0, 0] == r.logprob[0]
        assert (np.abs(r.top_logprob.cpu().numpy()[0] - ref[0, r.top_ids.cpu().numpy()[0]]) <= 6e-4).all()
        tokens = picked.astype(np.int64)
    kv.close()


@pytest.mark.parametrize("rows", [1, 7, 40, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layers_with_biases_then_a_score(backend, rows, dtype):
    # x += down(gelu(up(norm(x)))), twice, with biases and the residual in the product's epilogue; then every row scored
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    mat = lambda n, k: (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).bfloat16()      # noqa: E731
    vec = lambda n: 0.1 * torch.randn(n, generator=gen, device="cuda")                               # noqa: E731
    layers = [dict(norm=vec(HIDDEN), up=mat(INNER, HIDDEN), up_b=vec(INNER), down=mat(HIDDEN, INNER), down_b=vec(HIDDEN)) for _ in range(2)]
    head, last = mat(VOCAB, HIDDEN), vec(HIDDEN)
    x = torch.randn(rows, HIDDEN, generator=gen, device="cuda")
    ids = np.random.default_rng(rows).integers(0, VOCAB, rows)

    want = x.double()
    norm64 = lambda v, g: (1.0 + g.double()) * v / (v.square().mean(1, keepdim=True) + EPS).sqrt()   # noqa: E731
    for l in layers:
        h = norm64(want, l["norm"])
        h = h @ l["up"].double().T + l["up_b"].double()
        want = want + (h * torch.special.ndtr(h)) @ l["down"].double().T + l["down_b"].double()
    want = torch.log_softmax(norm64(want, last) @ head.double().T, 1)

    for l in layers:
        h = backend.rmsnorm(x, l["norm"], 1.0, EPS)
        h = backend.matmul_epilogue(h, l["up"], bias=l["up_b"], activation="gelu", out_dtype=dtype)
        backend.matmul_epilogue(h, l["down"], bias=l["down_b"], residual=x, out=x)
    h = backend.rmsnorm(x, last, 1.0, EPS)
    score = backend.matmul_logprobs(h, head, ids)
    rows_of = backend.logprob_rows(backend.matmul_epilogue(h, head), ids, top=3, entropy=True)
    backend.sync()
    # Activations kept in bf16 round by 2^-9 of themselves twice, each into a sum of INNER terms of both signs (2-norm); kept
    # in f32 what is lost is the sums' last places.  Logits are of unit size, and a log probability moves by two of them.
    tol = 4 * 2.0 ** -9 if dtype == torch.bfloat16 else 2e-5
    at = torch.as_tensor(ids, device="cuda")[:, None]
    assert (score.logprob - want.gather(1, at)[:, 0]).abs().max() <= 2 * tol * 3
    assert (score.entropy - torch.special.entr(want.exp()).sum(1)).abs().max() <= 2 * tol * (2 + np.log(VOCAB))
    assert torch.allclose(rows_of.logprob, score.logprob, rtol=0, atol=1e-5) and torch.allclose(rows_of.entropy, score.entropy, rtol=0, atol=3e-5)
    assert (rows_of.top_logprob.double() - want.gather(1, rows_of.top_ids.long())).abs().max() <= 2 * tol * 3

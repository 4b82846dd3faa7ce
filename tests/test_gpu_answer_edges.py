"""What the operators between hidden states and log probabilities promise at their edges: how 16-bit results are rounded after long
sums, activations far below zero, rows in which one token has nearly all the weight, results over one another,
empty batches, a device with little memory left, more rows than
are taken at a time, the least values of rows, infinite weights, every way a product is dealt out to the SMs."""
import ctypes

import numpy as np
import pytest
import torch

from yaxus_b200 import _lib
from yaxus_b200.backend import BackendError, CudaBackend

from .test_gpu_logprobs import tolerances

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def product(rows, n, k, dtype, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows * 131 + n * 7 + k + seed)
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).bfloat16()
    return x, w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(16, 4096, 14336), (64, 19100, 6016), (100, 12000, 6016), (80, 4096, 14336), (300, 20000, 4104), (1100, 1000, 14336)])
def test_long_sums_of_16_bit_results(backend, dtype, out_dtype, rows, n, k):
    # whole tiles, shares of left-over tiles, shares that end inside a tile, clusters, each over chains as long as 16-bit results have
    x, w = product(rows, n, k, dtype)
    got = backend.matmul_epilogue(x, w, out_dtype=out_dtype)
    for _ in range(5):
        again = backend.matmul_epilogue(x, w, out_dtype=out_dtype)
        backend.sync()
        assert torch.equal(got, again)
    want = x.double() @ w.double().T
    # A product of 16 k adds to its accumulator and may drop up to a last place of it, half of one in the mean; a chain has up to 384 of
    # them (64 k steps of 4 for one part, 48 of 8 for two, 32 of 12 for three), and the accumulator is of the size of a sum of
    # independent terms.  What is off by err before it is rounded is rounded to a neighbour where a border lies that near.
    err = 384 * 2.0 ** -24 * (x.double().square() @ w.double().square().T).sqrt()
    eps = torch.finfo(out_dtype).eps
    step = eps * torch.exp2(torch.floor(torch.log2(want.abs()))).clamp(min=torch.finfo(out_dtype).smallest_normal)
    share = (err / step).clamp(max=1).mean().item()
    off = (got != want.to(out_dtype)).double().mean().item()
    assert off <= share + 5 * (share / got.numel()) ** 0.5, (off, share)
    # ... and nothing is further off than that neighbour: half a step, and what 384 whole last places of the terms' sum are
    most = 384 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T)
    assert ((got.double() - want).abs() <= step / 2 + most).all()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,k", [(4, 200), (50, 200), (300, 200), (50, 201)])
def test_activations_near_and_far_from_zero(backend, act, rows, k):
    # the product is the row's first value itself, so that all that errs is the activation: each result by its own last places
    y = torch.linspace(-12.0, 12.0, rows, device="cuda")
    x = torch.zeros(rows, k, device="cuda")
    x[:, 0] = y
    w = torch.zeros(24, k, device="cuda").bfloat16()
    w[:, 0] = 1.0
    got = backend.matmul_epilogue(x, w, activation=act).double()
    backend.sync()
    v = y.double()[:, None].expand(rows, 24)
    if act == "gelu":
        want = 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5)
        u = v * v           # erfc(z) moves by 2 z^2 + 1 of z's relative error at most, z = -y / sqrt 2
    else:
        u = -v if act == "silu" else -2 * (2 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3)
        want = v / (1 + u.exp())
    # An argument errs by 8 half units of itself at most (gelu_tanh's polynomial has five operations), the function by four last
    # places (erfc), what is made of it by three more roundings.  Where 1 + exp(u) passes 2^126 its reciprocal is no normal f32 and
    # counts as 0: no more than |y| <= 12 times 2^-126 is lost (gelu_tanh is 1.6e-61 at -12).
    tol = want.abs() * ((u.abs() + 1) * 8 * 2.0 ** -24 + 4 * 2.0 ** -23 + 3 * 2.0 ** -24) + 12 * 2.0 ** -126
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(80, 9000), (3, 9000), (3, 300000)])
def test_two_tokens_with_all_the_weight(backend, dtype, rows, cols):
    # the second best is seen first, by the thread that sees the best later; all others weigh exp(-60)
    d = torch.linspace(0.1, 12.0, rows, device="cuda")
    x = torch.full((rows, cols), -55.0, device="cuda")
    x[:, 4099] = 5.0
    x[:, 3] = 5.0 - d
    x = x.to(dtype)
    r = backend.logprob_rows(x, np.tile([4099, 3], (rows, 1)), top=2, entropy=True)
    backend.sync()
    d = (x[:, 4099].double() - x[:, 3].double())
    w = torch.exp(-d)
    log_s = torch.log1p(w)
    h = log_s + w * d / (1 + w)
    # w: its exponent's argument has two roundings (relative, of d) and 2^x is off by two last places at most.  1 + w is rounded
    # three times on its way (a thread's two sums, their sum; the others' add nothing), the logarithm is off by a last place.
    w_err = w * (2.0 ** -22 + 1.5 * d * 2.0 ** -24)
    s_err = w_err + 3 * 2.0 ** -24
    log_err = s_err + log_s * 2.0 ** -23
    assert ((r.logprob[:, 0] + log_s).abs() <= log_err + log_s * 2.0 ** -23).all()
    assert ((r.logprob[:, 1] + d + log_s).abs() <= log_err + (d + log_s) * 2.0 ** -23).all()
    # t = -w d with w's error and three roundings; t / s with those of s and its own
    t_err = w_err * d + 3 * w * d * 2.0 ** -24
    assert ((r.entropy - h).abs() <= log_err + t_err + w * d * s_err + (w * d + h) * 2.0 ** -23).all()
    assert torch.equal(r.top_logprob, r.logprob)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_probability_exceeds_one(backend, dtype):
    # some token of a row stands 4 to 30 above a bell, anywhere in the row
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    for rows, cols in ((3000, 9001), (3, 150001)):
        for shift in range(4 if rows > 3 else 40):
            x = torch.randn(rows, cols, generator=gen, device="cuda")
            at = torch.randint(0, cols, (rows, 1), generator=gen, device="cuda")
            x.scatter_(1, at, 4 + 26 * torch.rand(rows, 1, generator=gen, device="cuda"))
            r = backend.logprob_rows(x.to(dtype), at.cpu().numpy(), top=3, entropy=True)
            backend.sync()
            assert (r.logprob <= 0).all() and (r.top_logprob <= 0).all() and (r.entropy >= 0).all()


def test_results_over_one_another_are_refused(backend):
    x = torch.randn(3, 50, device="cuda")
    h, w = torch.randn(3, 64, device="cuda"), torch.randn(50, 64, device="cuda").bfloat16()
    out = torch.zeros(64, device="cuda")
    ids = np.zeros((3, 2), np.uint32)
    L, c, i, o = backend._L, backend._ctx, ids.ctypes.data, out.data_ptr()
    rows = lambda p, e, t, l: L.yx_logprob_rows(c, x.data_ptr(), 0, 3, 50, 50, i, 2, 4, p, e, t, l)      # noqa: E731
    # in order: 6 log probabilities, 3 entropies, 12 tokens, 12 of theirs
    places = [o, o + 24, o + 36, o + 84]
    for k in range(4):
        for j in range(4):
            if j != k:
                at = list(places)
                at[k] = places[j]
                assert rows(*at) == _lib.YX_ERR_INVALID, (k, j)
                backend.clear_error()
    for at in ([o, o + 20, o + 36, o + 84], [o, o + 24, o + 32, o + 84], [o, o + 24, o + 36, o + 80], [o + 132, o + 24, o + 36, o + 88]):
        assert rows(*at) == _lib.YX_ERR_INVALID
        backend.clear_error()
    head = lambda p, e: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 3, 50, 64, i, p, e)       # noqa: E731
    for p, e in ((o, o), (o, o + 8), (o + 8, o)):
        assert head(p, e) == _lib.YX_ERR_INVALID
        backend.clear_error()
    torch.cuda.synchronize()
    assert (out == 0).all()
    assert rows(*places) == _lib.YX_OK and head(o + 160, o + 172) == _lib.YX_OK       # side by side they are taken
    backend.sync()
    lp = torch.log_softmax(x.double(), 1)
    assert (out[:6] - lp[:, 0].repeat_interleave(2)).abs().max() <= 1e-5


def test_what_is_asked_for_of_no_rows_and_no_tokens_is_empty(backend):
    x = torch.randn(3, 50, device="cuda")
    for shape in ((0,), (0, 2), (0, 0)):
        r = backend.logprob_rows(x[:0], np.zeros(shape, np.uint32), top=4, entropy=True)
        assert r.logprob.shape == shape and r.entropy.shape == (0,) and r.top_ids.shape == r.top_logprob.shape == (0, 4)
    r = backend.logprob_rows(x, np.zeros((3, 0), np.uint32), top=4)
    backend.sync()
    assert r.logprob.shape == (3, 0) and torch.equal(r.top_ids.long(), x.topk(4).indices)
    r = backend.matmul_logprobs(torch.zeros(0, 64, device="cuda"), torch.zeros(50, 64, device="cuda").bfloat16(), [])
    backend.sync()
    assert r.logprob.shape == r.entropy.shape == (0,)


def test_scratch_takes_what_it_needs_where_more_does_not_fit(backend):
    # an inner size that the tensor cores do not take: the scratch are 2000 rows of 8000 logits, 64 MB
    stream = torch.cuda.Stream()
    b = CudaBackend(0, stream)
    hold = []
    with torch.cuda.stream(stream):
        x = torch.randn(2000, 9, device="cuda")
        w = torch.randn(8000, 9, device="cuda").bfloat16()
        ids = np.zeros(2000, np.uint32)
        want = b.matmul_logprobs(x, w, ids)
        b.close()
        b = CudaBackend(0, stream)
        b.matmul_logprobs(x[:40], w, ids[:40])          # the scratch's first size: the next may be half as large again
        b.sync()
        torch.cuda.empty_cache()
        try:
            # fill the device up to 70 to 82 MiB: 61 fit, 92 do not
            for size in (1 << 30, 64 << 20, 12 << 20):
                while torch.cuda.mem_get_info()[0] > (70 << 20) + size:
                    hold.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
            got = b.matmul_logprobs(x, w, ids)
            b.sync()
            assert torch.equal(got.logprob, want.logprob) and torch.equal(got.entropy, want.entropy)
        finally:
            hold.clear()
            torch.cuda.empty_cache()
    b.close()


def test_an_error_is_its_own_call_s_alone(backend):
    # a call that finds no memory: the next one's launch, and its check, know nothing of it
    stream = torch.cuda.Stream()
    b = CudaBackend(0, stream)
    hold = []
    with torch.cuda.stream(stream):
        x = torch.randn(2000, 9, device="cuda")
        w = torch.randn(8000, 9, device="cuda").bfloat16()
        b.matmul_epilogue(x[:40], w[:8])
        b.sync()
        torch.cuda.empty_cache()
        try:
            for size in (1 << 30, 64 << 20, 12 << 20):
                while torch.cuda.mem_get_info()[0] > (34 << 20) + size:
                    hold.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
            b.matmul_logprobs(x, w, np.zeros(2000, np.uint32))     # logits of 64 MB
            assert b.status() == _lib.YX_ERR_OOM
            with pytest.raises(BackendError):
                b.sync()
            b.clear_error()
            small = b.matmul_epilogue(x[:40], w[:8])
            b.sync()
        finally:
            hold.clear()
            torch.cuda.empty_cache()
        assert (small.double() - x[:40].double() @ w[:8].double().T).abs().max() <= 1e-4
    b.close()


def used_by(call):
    """Bytes of device memory a new context has taken for a call."""
    b = CudaBackend(0, torch.cuda.current_stream())
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    out = call(b)
    b.sync()
    used = before - torch.cuda.mem_get_info()[0]
    b.close()
    return out, used


def test_scratch_does_not_grow_with_all_rows(backend):
    # 256 MB for statistics or parts of rows (either would be some 320 and 390 MB here), 40 for shares, and some for small ones
    most = (256 + 40 + 16) << 20
    x, w = product(16000, 64, 4096, torch.float32)
    bias, res, out = torch.randn(64, device="cuda"), torch.randn(16000, 64, device="cuda"), torch.empty(16000, 64, device="cuda")
    backend.matmul_epilogue(x[:4000], w, bias=bias)                   # (the kernels are on the device before memory is counted)
    _, used = used_by(lambda b: b.matmul_epilogue(x, w, bias=bias, residual=res, activation="relu", out=out))
    assert used <= most, used
    want = (x.double() @ w.double().T + bias.double()).clamp(min=0) + res.double()
    assert (out - want).norm() <= 1e-6 * want.norm()
    # rows under the result are all taken before it is written
    square = x[:, :64].contiguous()
    wide = (torch.randn(64, 64, device="cuda") / 8).bfloat16()
    both = backend.matmul_epilogue(square, wide)
    backend.matmul_epilogue(square, wide, out=square)
    backend.sync()
    assert torch.equal(square, both)

    for dtype in (torch.bfloat16, torch.float32):
        x, w = product(50000, 32000, 64, dtype)
        w *= 8
        ids = np.arange(50000) * 7 % 32000
        backend.matmul_logprobs(x[:4000], w, ids[:4000])
        r, used = used_by(lambda b: b.matmul_logprobs(x, w, ids))
        assert used <= most, used
        for at in (0, 24900, 49700):                                  # ends, and where one slice follows another
            lp = torch.log_softmax(x[at:at + 300].double() @ w.double().T, 1)
            want = lp.gather(1, torch.as_tensor(ids[at:at + 300], device="cuda")[:, None])[:, 0]
            h = torch.special.entr(lp.exp()).sum(1)
            # (sums of 64 products; log probabilities of some -10 in f32, and the sums of 32000 terms)
            assert (r.logprob[at:at + 300] - want).norm() <= 2e-6 * want.norm() and (r.entropy[at:at + 300] - h).norm() <= 4e-6 * h.norm()


@pytest.mark.parametrize("rows,k", [(16, 128), (64, 128), (64, 129)])
def test_the_least_values_of_rows(backend, rows, k):
    # one nonzero in each row and column: results are the rows' own values, whole from 2^-110 on, below that to the least bf16, 2^-133
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    at = torch.arange(rows, device="cuda")
    w = torch.zeros(128, k, device="cuda").bfloat16()
    w[torch.arange(128), torch.arange(128)] = 1
    for e in (-60, -100, -110, -112, -120, -126, -132, -140):
        v = ((torch.randint(1 << 23, 1 << 24, (rows,), generator=gen, device="cuda") | 1).double() * 2.0 ** (e - 23)).float()
        x = torch.zeros(rows, k, device="cuda")
        x[at, 2 * at] = v
        got = backend.matmul_epilogue(x, w)
        backend.sync()
        off = (got[at, 2 * at].double() - v.double()).abs().max().item()
        assert off == 0 if e >= -110 else off < 2.0 ** -133
        got[at, 2 * at] = 0
        assert (got == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(4, 128), (64, 128), (64, 129)])
def test_an_infinite_weight_stays_in_its_column(backend, dtype, rows, k):
    x, w = product(rows, 96, k, dtype)
    want = backend.matmul_epilogue(x, w)
    x[0, 9] = 1
    want[0] = backend.matmul_epilogue(x, w)[0]
    w[17, 9] = float("inf")
    got = backend.matmul_epilogue(x, w)
    backend.sync()
    others = torch.arange(96, device="cuda") != 17
    assert torch.equal(got[:, others], want[:, others])
    assert not got[:, 17].isfinite().any()
    number = ~got[:, 17].isnan()
    assert torch.equal(got[number, 17], torch.sign(x[number, 9].float()) * float("inf"))
    if dtype == torch.bfloat16 or k % 8:            # rows that are not cut into parts
        assert number.all()


# (rows, columns, inner size, how it is dealt out on 148 SMs): tiles' sums added up in clusters, whole tiles, shares that meet in scratch;
# of the pair kernel shares of the tiles behind whole rounds, and shares that run over a tile's end where there is no whole round.
DEALT = [
    (1, 4096, 2048, "few, clusters"), (8, 18000, 1024, "few, whole"), (8, 20000, 4096, "few, shares"), (1, 25600, 1024, "few, shares"),
    (32, 40000, 512, "few, shares"), (17, 38001, 768, "few, shares"), (64, 4096, 2048, "pairs, clusters"), (300, 9400, 512, "pairs, whole"),
    (80, 40000, 2048, "pairs, rest shared"), (64, 19200, 4096, "pairs, rest shared"), (300, 20000, 2048, "pairs, rest shared"),
    (600, 13000, 1024, "pairs, rest shared"), (100, 12000, 4096, "pairs, shares"), (250, 11000, 4096, "pairs, shares"), (130, 11500, 4104, "pairs, shares")]


def dealt_out(backend):
    out = np.zeros(6, np.uint32)
    assert backend._L.yx_hook_last_product(backend._ctx, out.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32))) == _lib.YX_OK
    kind, cluster, rounds, rest, shares, _ = out.tolist()
    if cluster > 1:
        return ("few, " if kind == 1 else "pairs, ") + "clusters"
    if kind == 1:
        return "few, whole" if rounds else "few, shares"
    return "pairs, whole" if shares == rest else "pairs, rest shared" if rounds else "pairs, shares"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k,dealt", DEALT)
def test_products_however_they_are_dealt_out(backend, dtype, rows, n, k, dealt):
    x, w = product(rows, n, k, dtype)
    res = torch.randn(rows, n, device="cuda")
    got = backend.matmul_epilogue(x, w, residual=res)
    assert dealt_out(backend) == dealt
    for _ in range(6):
        again = backend.matmul_epilogue(x, w, residual=res)
        backend.sync()
        assert torch.equal(got, again)
    # (sums within a millionth of the result, and the residual's rounding)
    want = x.double() @ w.double().T
    assert (got.double() - res.double() - want).norm() <= 1e-6 * want.norm() + 2.0 ** -24 * (want + res.double()).norm()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k,dealt", DEALT)
def test_heads_however_they_are_dealt_out(backend, dtype, rows, n, k, dealt):
    x, w = product(rows, n, k, dtype)
    w *= 2
    xd, wd = x.double(), w.double().T
    logits = xd @ wd
    lp = torch.log_softmax(logits, 1)
    h = torch.special.entr(lp.exp()).sum(1)
    # A logit's chains and shares are at most 512 f32 additions one after the other, a last place each; a log probability moves by no more
    # than its own logit and the largest move of any, the entropy by that times 1 + its spread.
    move = 512 * 2.0 ** -23 * (xd.abs() @ wd.abs()).amax(1)
    spread = logits.amax(1) - logits.amin(1)
    for turn in range(4):
        # tokens of every column tile, the ends of tiles among them
        ids = ((np.arange(rows) * 127 + 128 * turn * 37 + 127) % n).astype(np.uint32) if turn else np.full(rows, n - 1, np.uint32)
        r = backend.matmul_logprobs(x, w, ids)
        assert dealt_out(backend) == dealt
        for _ in range(6):
            again = backend.matmul_logprobs(x, w, ids)
            backend.sync()
            assert torch.equal(r.logprob, again.logprob) and torch.equal(r.entropy, again.entropy)
        at = torch.as_tensor(ids.astype(np.int64), device="cuda")[:, None]
        lp_tol, h_tol = tolerances(n, lp, h)
        want = lp.gather(1, at)[:, 0]
        assert ((r.logprob - want).abs() <= 2 * move + lp_tol.gather(1, at)[:, 0]).all()
        assert ((r.entropy - h).abs() <= 2 * move * (1 + spread) + h_tol).all()
        assert (r.logprob - want).norm() <= 2e-6 * want.norm() + 1e-7 * rows ** 0.5
        # The entropy's error is that of independent errors of logits, a millionth of their size each, weighted with p (|log p| + h) and
        # added up as squares, and of its sums of n terms: a place or two of log n.
        assert (r.entropy - h).norm() <= 4e-6 * h.norm()


def test_few_long_rows_are_one_launch(backend):
    # (rows that the kernel cuts itself need no scratch, however long they are)
    x, w = product(32, 8, 1500000, torch.float32)
    before = backend.launch_count()
    got = backend.matmul_epilogue(x, w)
    assert backend.launch_count() - before == 1
    backend.sync()
    want = x.double() @ w.double().T
    # 23438 k steps, eight at a time, in shares of some 160: sums of 2930 chains' f32 at most, half a last place each in the mean
    assert (got - want).norm() <= 2930 ** 0.5 * 2.0 ** -23 * want.norm()

"""`logprob_rows` and `matmul_logprobs` against the softmax in 64 bits: types, rows apart, masks that leave little or nothing,
ties, one column, more rows than a grid's y extent, recorded calls, refusals."""
import numpy as np
import pytest
import torch

from yaxus_b200 import _lib
from yaxus_b200.backend import BackendError, CudaBackend

pytestmark = pytest.mark.gpu
INF = float("inf")
MOST = torch.finfo(torch.float32).max
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def softmax64(logits):
    """(log probabilities, entropy) in 64 bits, as the header defines them."""
    l = logits.double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -INF), l).clamp(max=MOST)
    m = l.amax(1, keepdim=True)
    empty = m == -INF
    d = l - torch.where(empty, torch.zeros_like(m), m)
    e = d.exp()
    s = torch.where(empty, torch.ones_like(m), e.sum(1, keepdim=True))
    h = torch.where(empty, torch.zeros_like(m), s.log() - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1, keepdim=True) / s)
    # (in two steps, so that a distance past f32 is one of its infinities as in any f32 result)
    return (d - s.log()).float().double(), h[:, 0]


def best64(logits, top):
    l = logits.double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -INF), l).clamp(max=MOST)
    return torch.sort(l, dim=1, descending=True, stable=True).indices[:, :top]


def tolerances(cols, lp, h):
    # Every exp errs by 2 units of 2^-23 and by its argument's two roundings, which the weight d exp(-d) <= 0.37 keeps below one
    # more; a thread adds up to cols / 256 + 32 terms, half a unit each.  The logarithm turns relative into absolute.
    sum_err = 4 * 2.0 ** -23 + (cols / 256 + 32) * 2.0 ** -24
    # a log probability is the difference of three numbers of its own size at most, and of |log s| <= log(cols)
    lp_tol = sum_err + (lp.abs() * 2 + 2 * np.log(cols + 1.0) + 1) * 2.0 ** -24
    # t errs by the same relative amount, and |t / s| = log s - h <= log(cols)
    h_tol = sum_err * (2 + 2 * np.log(cols + 1.0)) + (h.abs() + np.log(cols + 1.0)) * 2.0 ** -23
    return lp_tol, h_tol


def check(logits, ids, top, r):
    lp, h = softmax64(logits)
    lp_tol, h_tol = tolerances(logits.shape[1], torch.where(lp.isfinite(), lp, torch.zeros_like(lp)), h)
    near = lambda got, want, tol: bool(((got.double() == want) | ((got.double() - want).abs() <= tol)).all())  # noqa: E731
    if ids is not None:
        at = torch.as_tensor(np.asarray(ids).astype(np.int64), device=logits.device).reshape(logits.shape[0], -1)
        got = r.logprob.reshape(at.shape)
        assert near(got, lp.gather(1, at), lp_tol.gather(1, at))
    if r.entropy is not None:
        assert near(r.entropy, h, h_tol)
    if top:
        want = best64(logits, top)
        assert torch.equal(r.top_ids.long(), want)
        assert near(r.top_logprob, lp.gather(1, want), lp_tol.gather(1, want))


def logits_of(rows, cols, dtype, seed=0, pad=0, scale=3.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows * 1000003 + cols + seed)
    return (torch.randn(rows, cols + pad, generator=gen, device="cuda") * scale).to(dtype)[:, :cols]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,n_ids,top,pad", [
    (1, 1, 1, 1, 0), (1, 2, 2, 2, 0), (3, 31, 1, 31, 0), (2, 32, 1, 32, 5), (1, 1000, 1, 5, 0), (5, 1023, 3, 20, 1), (1, 4097, 1, 32, 0),
    (2, 50257, 1, 20, 7), (17, 8191, 1, 1, 3), (150, 2049, 1, 7, 0), (700, 4100, 1, 0, 0), (600, 513, 2, 32, 0), (1, 300001, 1, 20, 0)])
def test_rows(backend, dtype, rows, cols, n_ids, top, pad):
    x = logits_of(rows, cols, dtype, pad=pad)
    ids = np.random.default_rng(cols).integers(0, cols, (rows, n_ids))
    r = backend.logprob_rows(x, ids, top=top, entropy=True)
    backend.sync()
    assert r.logprob.shape == (rows, n_ids)
    check(x, ids, top, r)
    again = backend.logprob_rows(x, ids, top=top, entropy=True)     # the same call gives the same bits
    backend.sync()
    assert all(a is None or torch.equal(a, b) for a, b in zip(r, again))


def test_parts_of_the_result(backend):
    x = logits_of(4, 777, torch.float32)
    ids = [5, 0, 776, 5]
    r = backend.logprob_rows(x, ids)
    assert r.logprob.shape == (4,) and r.entropy is None and r.top_ids is None and r.top_logprob is None
    check(x, ids, 0, r)
    r = backend.logprob_rows(x, top=3)
    assert r.logprob is None and r.entropy is None
    check(x, None, 3, r)
    r = backend.logprob_rows(x, entropy=True)
    assert r.logprob is None and r.top_ids is None
    check(x, None, 0, r)
    r = backend.logprob_rows(x[:0], np.zeros((0, 1), np.uint32), top=3, entropy=True)
    assert r.top_ids.shape == (0, 3) and r.entropy.shape == (0,)
    backend.sync()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 12, 400])
@pytest.mark.parametrize("value", [-INF, float("nan"), "lowest"])
def test_masks(backend, dtype, rows, value):
    # nothing left, one token left, few, all but a few, a whole stretch forbidden
    cols = 9001
    x = logits_of(rows, cols, dtype).clone()
    v = torch.finfo(dtype).min if value == "lowest" else value
    for r in range(rows):
        kind = r % 6
        if kind == 0:
            x[r] = v
        elif kind == 1:
            keep = x[r, 8123].clone()
            x[r] = v
            x[r, 8123] = keep
        elif kind == 2:
            x[r, torch.arange(cols, device=x.device) % 1500 != 7] = v
        elif kind == 3:
            x[r, ::3000] = v
        elif kind == 4:
            x[r, :5000] = v
    ids = np.tile(np.array([8123, 7, 0, 6001]), (rows, 1))
    r = backend.logprob_rows(x, ids, top=8, entropy=True)
    backend.sync()
    check(x, ids, 8, r)
    if value != "lowest":
        assert r.entropy[0] == 0 and (r.logprob[0] == -INF).all() and (r.top_logprob[0] == -INF).all()
        assert r.top_ids[0].tolist() == list(range(8))


@pytest.mark.parametrize("rows", [1, 300])
def test_orders(backend, rows):
    # rising rows (every column is the best so far), falling ones, all equal, few values, both zeros
    cols = 20000
    up = torch.arange(cols, device="cuda", dtype=torch.float32) * 1e-3
    kinds = [up, up.flip(0), torch.full_like(up, 2.5), (torch.arange(cols, device="cuda") % 7).float(),
             torch.where(torch.arange(cols, device="cuda") % 2 == 0, -0.0, 0.0)]
    for k, row in enumerate(kinds):
        x = row.repeat(rows, 1)
        r = backend.logprob_rows(x, np.full((rows, 1), cols - 1), top=32, entropy=True)
        backend.sync()
        check(x, np.full((rows, 1), cols - 1), 32, r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 60000), (300, 60000), (300, 500001), (2, 2000000)])
def test_large_ones_in_a_few_places(backend, dtype, rows, cols):
    # what is largest lies in every 32nd group of 16 bytes, so that one group of threads holds more than the list takes
    c = torch.arange(cols, device="cuda")
    wide = 4 if dtype == torch.float32 else 8
    row = torch.where(c // wide % 32 == 3, 5.0 + (c % 1009) * 0.01, (c % 7) * 0.1).to(dtype)
    x = row[None].expand(rows, cols).contiguous()
    ids = np.full((rows, 1), 12)
    r = backend.logprob_rows(x, ids, top=32, entropy=True)
    backend.sync()
    for i in range(0, rows, 100):     # (rows of an odd length begin at other alignments, and are summed in other orders)
        check(x[i:i + 100], ids[i:i + 100], 32, type(r)(*(t[i:i + 100] for t in r)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 60000), (300, 20011)])
@pytest.mark.parametrize("top", [2, 20, 21, 32])
def test_the_best_in_one_thread_s_share(backend, dtype, rows, cols, top):
    # a thread's logits are 16 bytes in every 4096: the best lie in one thread's, in one of its tiles, in two or in all of them
    wide = 4 if dtype == torch.float32 else 8
    gen = torch.Generator(device="cuda")
    gen.manual_seed(top)
    x = torch.randn(rows, cols, generator=gen, device="cuda").clamp(-3, 3)
    c = torch.arange(cols, device="cuda")
    own = (c // wide) % 256 == 77
    tile = c // (256 * 16)
    for i in range(rows):
        where = own & (tile == 1) if i % 3 == 0 else own & (tile >= 1) & (tile < 3) if i % 3 == 1 else own
        x[i, where] = 5 + torch.rand(int(where.sum()), generator=gen, device="cuda")
    x = x.to(dtype)
    ids = np.full((rows, 1), 77 * wide)
    r = backend.logprob_rows(x, ids, top=top, entropy=True)
    backend.sync()
    check(x, ids, top, r)


def test_large_numbers(backend):
    x = torch.zeros(7, 5000, device="cuda")
    x[0, 17] = INF                      # counts as the largest f32
    x[1, 17], x[1, 4000] = INF, MOST    # ... and is equal to it
    x[2] = MOST
    x[3] = -MOST
    x[4, 9] = 1e30
    x[5, 9], x[5, 10] = MOST, -MOST     # a distance past f32
    x[6, 9], x[6, 10] = MOST, INF       # equal, and one thread's
    ids = np.tile(np.array([17, 4000, 9, 10]), (7, 1))
    r = backend.logprob_rows(x, ids, top=4, entropy=True)
    backend.sync()
    check(x, ids, 4, r)
    check(x, ids, 1, backend.logprob_rows(x, ids, top=1, entropy=True))
    assert r.logprob[0, 0] == 0 and r.top_ids[1].tolist() == [17, 4000, 0, 1]


@pytest.mark.parametrize("rows,cols", [(70001, 3), (66000, 130)])
def test_many_rows(backend, rows, cols):
    x = logits_of(rows, cols, torch.float32)
    ids = np.random.default_rng(1).integers(0, cols, rows)
    r = backend.logprob_rows(x, ids, top=3, entropy=True)
    backend.sync()
    check(x, ids, 3, r)


@pytest.mark.parametrize("rows,n_ids", [(2, 300), (100, 10), (3, 2667), (1, 17001)])
def test_many_given_tokens(backend, rows, n_ids):
    # past what rides in the kernel's parameters, in one launch and in several
    x = logits_of(rows, 5003, torch.float32)
    ids = np.random.default_rng(n_ids).integers(0, 5003, (rows, n_ids))
    r = backend.logprob_rows(x, ids)
    backend.sync()
    check(x, ids, 0, r)


def test_offsets_past_32_bits(backend):
    # the last rows of 8.6 GB of logits, and of a head's hidden states: both begin past 2^32 elements
    rows, cols = 43000, 100003
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-3:] = logits_of(3, cols, torch.bfloat16)
    ids = np.arange(rows) % cols
    r = backend.logprob_rows(x, ids, top=4, entropy=True)
    backend.sync()
    check(x[-3:], ids[-3:], 4, type(r)(*(t[-3:] for t in r)))
    assert torch.allclose(r.logprob[:5], torch.full((5,), -float(np.log(cols)), device="cuda"))
    del x, r
    rows, k = 270000, 16384
    h = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    h[-40:].normal_()
    w = (torch.randn(100, k, device="cuda") * k ** -0.5).bfloat16()
    ids = np.arange(rows) % 100
    p = backend.matmul_logprobs(h, w, ids)
    backend.sync()
    lp = torch.log_softmax(h[-40:].double() @ w.double().T, 1)
    want = lp.gather(1, torch.as_tensor(ids[-40:], device="cuda")[:, None])[:, 0]
    assert (p.logprob[-40:] - want).abs().max() <= 1e-4 and torch.allclose(p.logprob[:9], torch.full((9,), -float(np.log(100)), device="cuda"))


def test_two_contexts_at_once(backend):
    # each has a stream and scratch of its own: what one computes does not show in the other
    streams = [torch.cuda.Stream() for _ in range(2)]
    backends = [CudaBackend(0, s) for s in streams]
    work = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            w = (torch.randn(6000, 512, device="cuda") * 0.1).bfloat16()
            work.append([(torch.randn(rows, 512, device="cuda").to(t), w, np.random.default_rng(rows).integers(0, 6000, rows))
                         for rows in (1, 30, 70, 300) for t in TYPES])
    torch.cuda.synchronize()
    alone = []
    for b, s, jobs in zip(backends, streams, work):
        with torch.cuda.stream(s):
            alone.append([(b.matmul_logprobs(*j), b.logprob_rows(b.matmul_epilogue(*j[:2]), j[2], top=7)) for j in jobs])
            b.sync()
    together = [[], []]
    for turn in range(3):
        for n in range(len(work[0])):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    j = work[i][n]
                    together[i].append((backends[i].matmul_logprobs(*j), backends[i].logprob_rows(backends[i].matmul_epilogue(*j[:2]), j[2], top=7)))
    for b in backends:
        b.sync()
    for i in range(2):
        for n, (p, r) in enumerate(together[i]):
            q, t = alone[i][n % len(work[0])]
            assert torch.equal(p.logprob, q.logprob) and torch.equal(p.entropy, q.entropy)
            assert torch.equal(r.logprob, t.logprob) and torch.equal(r.top_ids, t.top_ids) and torch.equal(r.top_logprob, t.top_logprob)
    for b in backends:
        b.close()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_off_any_alignment(backend, dtype):
    # a first row that starts one element past an aligned address, rows an odd number of elements apart
    store = logits_of(1, 5 * 4101 + 1, dtype)[0]
    x = torch.as_strided(store, (5, 4099), (4101, 1), 1)
    ids = np.arange(5) * 1000
    r = backend.logprob_rows(x, ids, top=9, entropy=True)
    backend.sync()
    check(x, ids, 9, r)


def test_what_lies_between_rows_is_not_read(backend):
    for dtype in TYPES:
        store = logits_of(9, 4000, dtype).contiguous()
        store[:, 3001:] = INF
        x = store[:, :3001]
        ids = np.arange(9)
        r = backend.logprob_rows(x, ids, top=20, entropy=True)
        backend.sync()
        check(x, ids, 20, r)


@pytest.mark.parametrize("rows,n,k", [(1, 300, 128), (1, 32000, 1024), (8, 1000, 256), (9, 129, 64), (16, 50257, 128), (31, 4096, 1024), (32, 257, 512),
                                      (33, 40, 128), (80, 5000, 1024), (130, 1001, 200), (257, 20001, 136), (300, 512, 2048), (2, 1, 8), (3, 77, 41),
                                      (40, 333, 90), (513, 9999, 96)])
@pytest.mark.parametrize("dtype", TYPES)
def test_head(backend, rows, n, k, dtype):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n * 7 + k)
    w = (torch.randn(n, k, generator=gen, device="cuda") * 2 * k ** -0.5).bfloat16()
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype)
    ids = np.random.default_rng(n).integers(0, n, rows)
    r = backend.matmul_logprobs(x, w, ids)
    backend.sync()
    xd, wd = x.double(), w.double().T
    logits = xd @ wd
    lp = torch.log_softmax(logits, 1)
    h = torch.special.entr(lp.exp()).sum(1)
    # A logit is a sum of at most 512 f32 additions one after the other, a last place each; a log probability moves by no more
    # than its own logit and the largest move of any, the entropy by that times 1 + its spread.
    move = 512 * 2.0 ** -23 * (xd.abs() @ wd.abs()).amax(1)
    lp_tol, h_tol = tolerances(n, lp, h)
    at = torch.as_tensor(ids, device="cuda")[:, None]
    spread = (logits.amax(1) - logits.amin(1))
    assert ((r.logprob - lp.gather(1, at)[:, 0]).abs() <= 2 * move + lp_tol.gather(1, at)[:, 0]).all()
    assert ((r.entropy - h).abs() <= 2 * move * (1 + spread) + h_tol).all()
    # ... and all rows together are as near as f32 products would be
    if n > 1:
        assert (r.logprob - lp.gather(1, at)[:, 0]).norm() <= 2e-6 * lp.gather(1, at).norm() + 1e-7 * rows ** 0.5
    only = backend.matmul_logprobs(x, w, ids, entropy=False)
    backend.sync()
    assert only.entropy is None and torch.equal(only.logprob, r.logprob)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 9480), (32, 11264), (7, 9601), (32, 18941), (20, 25600)])
def test_head_of_tiles_of_other_heights(backend, dtype, rows, n):
    # given tokens of every place in a tile, those at its ends among them
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    w = (torch.randn(n, 64, generator=gen, device="cuda") / 4).bfloat16()
    x = torch.randn(rows, 64, generator=gen, device="cuda").to(dtype)
    logits = x.double() @ w.double().T
    lp = torch.log_softmax(logits, 1)
    h = torch.special.entr(lp.exp()).sum(1)
    lp_tol, h_tol = tolerances(n, lp, h)
    # (the move of test_head; 64 products of three parts at most are 192 additions)
    move = 192 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T).amax(1)
    spread = logits.amax(1) - logits.amin(1)
    for first in range(0, 600, rows):
        ids = np.arange(first, first + rows) * (1 if first < 300 else 17) % n
        r = backend.matmul_logprobs(x, w, ids)
        backend.sync()
        at = torch.as_tensor(ids, device="cuda")[:, None]
        assert ((r.logprob - lp.gather(1, at)[:, 0]).abs() <= 2 * move + lp_tol.gather(1, at)[:, 0]).all()
        assert ((r.entropy - h).abs() <= 2 * move * (1 + spread) + h_tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 4096, 14336), (16, 4096, 14336), (32, 4096, 14336), (25, 50257, 2048), (64, 4096, 14336), (200, 900, 14336)])
def test_head_again_and_again(backend, dtype, rows, n, k):
    # many turns of the operands' ring: a slot filled too early or too late shows in one call of several, and in no two alike
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    for _ in range(4):
        w = (torch.randn(n, k, generator=gen, device="cuda") * 2 * k ** -0.5).bfloat16()
        x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype)
        ids = np.arange(rows) * 7 % n
        lp = torch.log_softmax(x.double() @ w.double().T, 1).gather(1, torch.as_tensor(ids, device="cuda")[:, None])[:, 0]
        first = backend.matmul_logprobs(x, w, ids)
        for _ in range(12):
            got = backend.matmul_logprobs(x, w, ids)
            backend.sync()
            assert torch.equal(got.logprob, first.logprob) and torch.equal(got.entropy, first.entropy)
        # (the bound of test_head, on all rows together)
        assert (first.logprob - lp).norm() <= 2e-6 * lp.norm() + 1e-7 * rows ** 0.5


def test_head_of_no_numbers(backend):
    # a row of hidden states that is no number has no logits left; its neighbours are as they were
    for rows in (3, 40):
        x = torch.randn(rows, 256, device="cuda")
        w = torch.randn(500, 256, device="cuda").bfloat16()
        ids = np.arange(rows)
        want = backend.matmul_logprobs(x, w, ids)
        x[1, 7] = float("nan")
        got = backend.matmul_logprobs(x, w, ids)
        backend.sync()
        keep = torch.arange(rows, device="cuda") != 1
        assert got.logprob[1] == -INF and got.entropy[1] == 0
        assert torch.equal(got.logprob[keep], want.logprob[keep]) and torch.equal(got.entropy[keep], want.entropy[keep])


def test_head_equals_the_rows_of_its_logits(backend):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    for rows in (1, 20, 100):
        x = torch.randn(rows, 512, generator=gen, device="cuda")
        w = (torch.randn(3001, 512, generator=gen, device="cuda") * 0.1).bfloat16()
        ids = np.random.default_rng(rows).integers(0, 3001, rows)
        a = backend.matmul_logprobs(x, w, ids)
        b = backend.logprob_rows(backend.matmul_epilogue(x, w), ids, entropy=True)
        backend.sync()
        assert torch.allclose(a.logprob, b.logprob, rtol=2e-6, atol=2e-6) and torch.allclose(a.entropy, b.entropy, rtol=2e-6, atol=4e-6)


@pytest.mark.parametrize("rows", [1, 40, 1500])
def test_recorded_and_replayed(backend, rows):
    # recorded once, replayed over other logits, with larger calls of the same context in between
    stream = torch.cuda.Stream()
    b = CudaBackend(0, stream)
    with torch.cuda.stream(stream):
        x = logits_of(rows, 3000, torch.float32).contiguous()
        h = torch.randn(rows, 256, device="cuda")
        w = torch.randn(2000, 256, device="cuda").mul_(0.1).bfloat16()
        ids = np.random.default_rng(rows).integers(0, 2000, rows)
        b.logprob_rows(x, ids, top=5, entropy=True)
        b.matmul_logprobs(h, w, ids)
        b.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r = b.logprob_rows(x, ids, top=5, entropy=True)
            p = b.matmul_logprobs(h, w, ids)
        assert b.status() == _lib.YX_OK, b.last_error()
        for step in range(2):
            x.copy_(logits_of(rows, 3000, torch.float32, seed=step + 1))
            h.normal_()
            other = np.zeros(4000, np.uint32)
            b.logprob_rows(logits_of(4000, 100, torch.float32), other, top=5)
            b.matmul_logprobs(torch.randn(4000, 256, device="cuda"), w, other)
            graph.replay()
            want = b.matmul_logprobs(h, w, ids)
            b.sync()
            check(x, ids, 5, r)
            assert torch.equal(p.logprob, want.logprob) and torch.equal(p.entropy, want.entropy)
        del graph
    b.close()


def test_refusals(backend):
    x = logits_of(2, 50, torch.float32)
    w = torch.zeros(50, 64, dtype=torch.bfloat16, device="cuda")
    h = torch.zeros(2, 64, device="cuda")
    L, c = backend._L, backend._ctx
    out = torch.empty(200, device="cuda")
    p, o = x.data_ptr(), out.data_ptr()
    two = np.zeros(2, np.uint32)
    i = two.ctypes.data
    bad = np.array([0, 50], np.uint32)
    calls = [
        lambda: L.yx_logprob_rows(c, p, 7, 2, 50, 50, i, 1, 0, o, None, None, None),        # no such type
        lambda: L.yx_logprob_rows(c, None, 0, 2, 50, 50, i, 1, 0, o, None, None, None),     # no logits
        lambda: L.yx_logprob_rows(c, p, 0, 2, 0, 50, i, 1, 0, o, None, None, None),         # no columns
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 49, i, 1, 0, o, None, None, None),        # rows over one another
        lambda: L.yx_logprob_rows(c, p, 0, 1, 2 ** 31, 2 ** 31, i, 1, 0, o, None, None, None),   # too long a row
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 2 ** 31, 64, i, o, None),
        lambda: L.yx_logprob_rows(c, p + 2, 0, 2, 50, 50, i, 1, 0, o, None, None, None),    # off alignment
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, i, 1, 0, o + 1, None, None, None),
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, bad.ctypes.data, 1, 0, o, None, None, None),   # a token past the vocabulary
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, i, 1, 0, None, None, None, None),     # nowhere to put it
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, None, 1, 0, o, None, None, None),     # no tokens
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, i, 0, 0, o, None, None, None),
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, None, 0, 33, None, None, o, o + 400),  # more than YX_TOP_MAX
        lambda: L.yx_logprob_rows(c, p, 0, 2, 20, 50, None, 0, 21, None, None, o, o + 400),  # more than there are
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, None, 0, 5, None, None, o, None),
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, i, 1, 0, p + 396, None, None, None),  # results over the logits
        lambda: L.yx_logprob_rows(c, p, 0, 2, 50, 50, None, 0, 4, None, p + 400, o, p - 16),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 50, 64, i, h.data_ptr() + 8, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 50, 64, i, o, w.data_ptr()),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 9, w.data_ptr(), 2, 50, 64, i, o, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, None, 2, 50, 64, i, o, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 0, 64, i, o, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 50, 0, i, o, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 50, 64, None, o, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 50, 64, i, None, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr(), 0, w.data_ptr(), 2, 50, 64, bad.ctypes.data, o, None),
        lambda: L.yx_matmul_logprobs(c, h.data_ptr() + 1, 0, w.data_ptr(), 2, 50, 64, i, o, None),
    ]
    for k, call in enumerate(calls):
        assert call() == _lib.YX_ERR_INVALID and backend.status() == _lib.YX_ERR_INVALID, k
        with pytest.raises(BackendError):
            backend.sync()
        backend.clear_error()
    # the binding's own: what would reach the device as another address or another token
    for wrong in (lambda: backend.logprob_rows(x.cpu(), [0, 0]), lambda: backend.logprob_rows(x.double(), [0, 0]),
                  lambda: backend.logprob_rows(x.T, [0] * 50), lambda: backend.logprob_rows(x, [0, -1]),
                  lambda: backend.logprob_rows(x, np.array([0, 2 ** 32])), lambda: backend.logprob_rows(x, [0.0, 1.0]),
                  lambda: backend.logprob_rows(x, [0, 0, 0]), lambda: backend.matmul_logprobs(h, w, [0]),
                  lambda: backend.matmul_logprobs(h[:, :32], w[:, :32], [0, 0]), lambda: backend.matmul_logprobs(h, w.float(), [0, 0])):
        with pytest.raises(AssertionError):
            wrong()
    assert backend.status() == _lib.YX_OK


def test_growing_while_recording_is_refused(backend):
    stream = torch.cuda.Stream()
    b = CudaBackend(0, stream)
    with torch.cuda.stream(stream):
        h, w = torch.randn(600, 64, device="cuda"), torch.randn(64, 64, device="cuda").bfloat16()
        x = torch.zeros(8, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x.add_(1.0)
            b.matmul_logprobs(h, w, np.zeros(600, np.uint32))
        assert b.status() == _lib.YX_ERR_STATE and "captured" in b.last_error()
        b.clear_error()
        graph.replay()                   # the rest of the recording is sound
        b.sync()
        assert x[0] == 1
        del graph
    b.close()

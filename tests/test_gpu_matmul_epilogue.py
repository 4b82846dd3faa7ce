"""`matmul_epilogue` against the formula in 64 bits: every type of rows and result, each activation, with and without bias and
residual, the kernels' tile edges, inner sizes that end inside a step, results over residual and rows, recorded calls, refusals."""
import math

import numpy as np
import pytest
import torch

from yaxus_b200 import _lib
from yaxus_b200.backend import BackendError, CudaBackend

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def activate64(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "gelu":
        return y * torch.special.ndtr(y)
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if act == "silu":
        return y * torch.sigmoid(y)
    return y


def inputs(rows, n, k, dtype, out_dtype=torch.float32, bias=True, residual=True, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows * 7919 + n * 31 + k + seed)
    x = torch.randn(rows, k, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).bfloat16()
    b = torch.randn(n, generator=gen, device="cuda") if bias else None
    r = torch.randn(rows, n, generator=gen, device="cuda").to(out_dtype) if residual else None
    return x, w, b, r


def check(got, x, w, b, r, act):
    xd, wd = x.double(), w.double().T
    y = xd @ wd
    terms = xd.abs() @ wd.abs()
    if b is not None:
        y, terms = y + b.double(), terms + b.double().abs()
    want = activate64(y, act)
    # Every product of parts is exact in f32; at most 512 additions one after the other may drop a last place each.  The
    # activations' slope is at most 1.13, and evaluating one in f32 errs by no more than 16 half units of |y| + 1.
    tol = 1.13 * 512 * 2.0 ** -23 * terms + 16 * 2.0 ** -24 * (y.abs() + 1)
    if r is not None:
        want = want + r.double()
        tol = tol + (want.abs() + r.double().abs()) * 2.0 ** -24
    info = torch.finfo(got.dtype)
    tol = tol + want.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2
    assert got.isfinite().all()
    worst = ((got.double() - want).abs() / tol).max().item()
    assert worst <= 1, worst
    return want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 2816, 1024), (3, 40, 128), (8, 129, 64), (9, 100, 200), (16, 1000, 2048), (17, 130, 24), (32, 512, 4096),
                                      (5, 33, 41), (7, 64, 1030),
                                      (33, 257, 128), (64, 300, 136), (80, 4096, 512), (100, 100, 72), (129, 2049, 256), (170, 3000, 1024), (256, 256, 64),
                                      (257, 513, 640), (300, 5633, 264), (513, 1000, 328), (60, 77, 301), (1000, 8, 8)])
def test_shapes(backend, dtype, rows, n, k):
    x, w, b, r = inputs(rows, n, k, dtype)
    got = backend.matmul_epilogue(x, w, bias=b, activation="silu", residual=r)
    backend.sync()
    check(got, x, w, b, r, "silu")
    again = backend.matmul_epilogue(x, w, bias=b, activation="silu", residual=r)
    backend.sync()
    assert torch.equal(got, again)           # the same call gives the same bits


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("rows", [2, 20, 70, 300])
def test_epilogues(backend, act, bias, residual, rows):
    for out_dtype in TYPES:
        x, w, b, r = inputs(rows, 200, 256, torch.bfloat16, out_dtype, bias, residual)
        got = backend.matmul_epilogue(x, w, bias=b, activation=act, residual=r, out_dtype=out_dtype)
        backend.sync()
        assert got.dtype == out_dtype
        check(got, x, w, b, r, act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 11264, 2048), (16, 4096, 14336), (80, 4096, 4096), (275, 34914, 1152), (262, 1460, 6784), (90, 527, 13312),
                                      (512, 9700, 6016)])
def test_rows_are_taken_exactly(backend, dtype, rows, n, k):
    # x reaches the products whole, so that all that is lost is the sums' rounding: one part in a million of the result at most
    x, w, _, _ = inputs(rows, n, k, dtype, bias=False, residual=False)
    got = backend.matmul_epilogue(x, w)
    backend.sync()
    want = x.double() @ w.double().T
    assert (got - want).norm() <= 1e-6 * want.norm()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 4096, 14336), (8, 4096, 14336), (13, 1001, 14336), (16, 20000, 4096), (20, 4096, 14336), (32, 4096, 14336),
                                      (32, 32000, 2048), (40, 4096, 14336), (150, 700, 14336), (300, 2000, 8200)])
def test_long_sums_again_and_again(backend, dtype, rows, n, k):
    # many turns of the operands' ring: a slot filled too early or too late shows in one call of several, and in no two alike
    for seed in range(4):
        x, w, _, _ = inputs(rows, n, k, dtype, bias=False, residual=False, seed=seed)
        want = x.double() @ w.double().T
        first = backend.matmul_epilogue(x, w)
        for _ in range(12):
            got = backend.matmul_epilogue(x, w)
            backend.sync()
            assert torch.equal(got, first)
        assert (first - want).norm() <= 1e-6 * want.norm()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(1, 9480, 64), (8, 11264, 256), (3, 9601, 136), (32, 18944, 128), (17, 18941, 72), (16, 25600, 128), (2, 40, 64)])
def test_tiles_of_other_heights(backend, dtype, out_dtype, rows, n, k):
    x, w, b, r = inputs(rows, n, k, dtype, out_dtype)
    got = backend.matmul_epilogue(x, w, bias=b, activation="silu", residual=r, out_dtype=out_dtype)
    backend.sync()
    check(got, x, w, b, r, "silu")


@pytest.mark.parametrize("rows", [4, 50])
def test_every_bit_of_a_row_counts(backend, rows):
    # one nonzero in each row and column: the results are the rows' own values, bit for bit (normal numbers whose least bit
    # is one too)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    for dtype in TYPES:
        x = torch.zeros(rows, 128, device="cuda", dtype=dtype)
        v = torch.randn(rows, generator=gen, device="cuda").to(dtype)
        x[torch.arange(rows), torch.arange(rows) * 2] = v
        w = torch.eye(128, device="cuda").bfloat16()
        got = backend.matmul_epilogue(x, w)
        backend.sync()
        assert torch.equal(got, x.float())


@pytest.mark.parametrize("rows", [6, 90])
def test_values_of_f16_past_bf16_and_large_sums(backend, rows):
    x = torch.full((rows, 64), 65504.0, device="cuda", dtype=torch.float16)
    x[:, 1] = 6e-8                                        # the least f16
    w = torch.ones(16, 64, device="cuda").bfloat16()
    got = backend.matmul_epilogue(x, w)
    backend.sync()
    assert ((got.double() - x.double().sum(1, keepdim=True)).abs() <= 63 * 65504 * 64 * 2.0 ** -23).all()
    small = backend.matmul_epilogue(x, w, out_dtype=torch.float16)     # past the type's largest: its infinity
    backend.sync()
    assert (small == float("inf")).all()


@pytest.mark.parametrize("rows", [5, 33, 200])
@pytest.mark.parametrize("dtype", TYPES)
def test_result_over_residual_and_over_rows(backend, rows, dtype):
    x, w, b, r = inputs(rows, 256, 256, dtype, dtype)
    want = backend.matmul_epilogue(x, w, bias=b, residual=r, out_dtype=dtype)
    x0 = x.clone()
    over = r.clone()
    assert backend.matmul_epilogue(x, w, bias=b, residual=over, out=over) is over
    backend.sync()
    assert torch.equal(over, want) and torch.equal(x, x0)
    backend.matmul_epilogue(x, w, bias=b, residual=r, out=x)
    backend.sync()
    assert torch.equal(x, want)
    x.copy_(x0)
    backend.matmul_epilogue(x, w, bias=b, residual=x, out=x)      # rows, residual and result in one
    backend.sync()
    assert torch.equal(x, backend.matmul_epilogue(x0, w, bias=b, residual=x0, out_dtype=dtype))


@pytest.mark.parametrize("rows", [3, 70])
@pytest.mark.parametrize("dtype", TYPES)
def test_tensors_off_a_vector_s_alignment(backend, rows, dtype):
    # rows, weight, bias, residual and result one element past an aligned address
    x, w, b, r = inputs(rows, 130, 256, dtype, dtype)

    def off(t):
        store = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        store[1:] = t.reshape(-1)
        return store[1:].view(t.shape)
    want = backend.matmul_epilogue(x, w, bias=b, residual=r, out_dtype=dtype)
    backend.sync()
    for xo, wo, bo, ro in ((off(x), w, b, r), (x, off(w), b, r), (x, w, off(b), off(r)), (off(x), off(w), off(b), off(r))):
        store = torch.full((rows * 130 + 2,), 7.0, dtype=dtype, device="cuda")
        out = store[1:-1].view(rows, 130)
        backend.matmul_epilogue(xo, wo, bias=bo, residual=ro, out=out)
        backend.sync()
        check(out, x, w, b, r, None)
        assert store[0] == 7 and store[-1] == 7           # nothing beside the result is written
        del want
        want = out


def test_rows_past_the_result_are_left(backend):
    for rows in (5, 40, 270):
        x, w, b, _ = inputs(rows, 300, 192, torch.float32)
        store = torch.full((rows + 3, 300), 9.0, device="cuda")
        backend.matmul_epilogue(x, w, bias=b, out=store[:rows])
        backend.sync()
        check(store[:rows], x, w, b, None, None)
        assert (store[rows:] == 9).all()


def test_empty(backend):
    w = torch.zeros(8, 16, device="cuda").bfloat16()
    assert backend.matmul_epilogue(torch.zeros(0, 16, device="cuda"), w).shape == (0, 8)
    assert backend.matmul_epilogue(torch.zeros(2, 16, device="cuda"), w[:0]).shape == (2, 0)
    backend.sync()


def test_more_rows_than_a_grid_s_extent(backend):
    x, w, b, r = inputs(66000, 3, 9, torch.float32)       # (an odd inner size: the kernel of any shape)
    got = backend.matmul_epilogue(x, w, bias=b, activation="relu", residual=r)
    backend.sync()
    check(got, x, w, b, r, "relu")
    x, w, b, r = inputs(70000, 24, 16, torch.bfloat16)
    got = backend.matmul_epilogue(x, w, bias=b, activation="relu", residual=r)
    backend.sync()
    check(got, x, w, b, r, "relu")


def test_results_past_32_bits(backend):
    x = torch.zeros(70000, 64, device="cuda").bfloat16()
    x[-50:].normal_()
    w = (torch.randn(65536, 64, device="cuda") * 0.125).bfloat16()
    got = backend.matmul_epilogue(x, w, activation="relu", out_dtype=torch.bfloat16)     # 4.6e9 results
    backend.sync()
    check(got[-50:], x[-50:], w, None, None, "relu")
    assert (got[:100] == 0).all()


def test_numbers_that_are_none_stay_in_their_rows_and_columns(backend):
    for rows in (6, 64):
        x, w, b, r = inputs(rows, 160, 192, torch.float32)
        want = backend.matmul_epilogue(x, w, bias=b, activation="gelu", residual=r)
        x[2, 100] = float("nan")
        b[17] = float("inf")
        r[4, 30] = float("-inf")
        got = backend.matmul_epilogue(x, w, bias=b, activation="gelu", residual=r)
        backend.sync()
        assert got[2].isnan().all() and got[4, 30] == float("-inf") and (got[:2, 17] == float("inf")).all()
        same = torch.ones_like(got, dtype=torch.bool)
        same[2], same[:, 17], same[4, 30] = False, False, False
        assert torch.equal(got[same], want[same])


@pytest.mark.parametrize("rows", [3, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_the_largest_numbers(backend, rows, dtype):
    # an infinity in a row is one in its results, of the weight's sign; the largest finite value of the type is no infinity
    x, w, _, _ = inputs(rows, 96, 128, dtype)
    x[1, 70] = float("inf")
    x[2] = 0
    x[2, 9] = torch.finfo(dtype).max
    w[:, 9] = 0.25
    got = backend.matmul_epilogue(x, w)
    backend.sync()
    assert torch.equal(got[1], torch.sign(w[:, 70].float()) * float("inf"))
    assert torch.equal(got[2], torch.full_like(got[2], 0.25 * torch.finfo(dtype).max))
    assert got[0].isfinite().all()


@pytest.mark.parametrize("rows", [1, 24, 100])
@pytest.mark.parametrize("dtype", TYPES)
def test_recorded_and_replayed(backend, rows, dtype):
    stream = torch.cuda.Stream()
    b = CudaBackend(0, stream)
    with torch.cuda.stream(stream):
        x, w, bias, r = inputs(rows, 512, 512, dtype)
        up, _, _, _ = inputs(rows, 512, 512, dtype, seed=1)
        first = b.matmul_epilogue(x, w, bias=bias, activation="gelu", out_dtype=dtype)
        b.matmul_epilogue(first, w, residual=r)
        b.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            mid = b.matmul_epilogue(x, w, bias=bias, activation="gelu", out_dtype=dtype)
            out = b.matmul_epilogue(mid, w, residual=r)
        assert b.status() == _lib.YX_OK, b.last_error()
        for step in range(2):
            x.copy_(inputs(rows, 512, 512, dtype, seed=step + 5)[0])
            big = inputs(700, 1000, 1024, dtype)          # (outgrows the scratch that the recording names)
            b.matmul_epilogue(big[0], big[1])
            graph.replay()
            want = b.matmul_epilogue(b.matmul_epilogue(x, w, bias=bias, activation="gelu", out_dtype=dtype), w, residual=r)
            b.sync()
            assert torch.equal(out, want)
        del graph
    b.close()


def test_a_product_feeds_the_next_as_its_weight(backend):
    # what one call writes may be the next one's weight: nothing is read ahead of the call before
    for rows in (4, 40, 300):
        a = torch.randn(192, 256, device="cuda").bfloat16()
        eye = torch.eye(256, device="cuda").bfloat16()
        x = torch.randn(rows, 256, device="cuda").bfloat16()
        for step in range(20):
            wt = torch.zeros(192, 256, device="cuda", dtype=torch.bfloat16)
            src = (a.float() * (step + 1)).bfloat16()
            backend.matmul_epilogue(src, eye, out=wt)
            got = backend.matmul_epilogue(x, wt)
            backend.sync()
            check(got, x, src, None, None, None)


def test_beside_matmul(backend):
    # the plain product and this one differ by the rounding of the rows to 16 bits of mantissa that yx_matmul makes
    x, w, _, _ = inputs(50, 300, 512, torch.float32)
    a, b = backend.matmul(x, w), backend.matmul_epilogue(x, w)
    backend.sync()
    terms = x.double().abs() @ w.double().abs().T
    assert ((a - b).abs() <= (2.0 ** -17 + 512 * 2.0 ** -23) * terms).all()


def test_refusals(backend):
    x, w, b, r = inputs(4, 64, 128, torch.float32)
    L, c = backend._L, backend._ctx
    out = torch.empty(8, 64, device="cuda")
    args = [c, x.data_ptr(), 0, w.data_ptr(), b.data_ptr(), 1, r.data_ptr(), 4, 64, 128, out.data_ptr(), 0]

    def with_(**kw):
        at = dict(x=1, x_dtype=2, w=3, bias=4, act=5, residual=6, rows=7, n=8, k=9, out=10, out_dtype=11)
        a = list(args)
        for name, v in kw.items():
            a[at[name]] = v
        return L.yx_matmul_epilogue(*a)
    for kw in (dict(x_dtype=3), dict(out_dtype=-1), dict(act=5), dict(act=-1), dict(x=None), dict(w=None), dict(out=None), dict(k=0),
               dict(n=2 ** 31), dict(k=2 ** 31), dict(rows=2 ** 31), dict(x=x.data_ptr() + 2), dict(w=w.data_ptr() + 1), dict(bias=b.data_ptr() + 2), dict(residual=r.data_ptr() + 2), dict(out=out.data_ptr() + 2),
               dict(out=w.data_ptr()), dict(out=b.data_ptr()), dict(residual=out.data_ptr() + 256)):
        assert with_(**kw) == _lib.YX_ERR_INVALID and backend.status() == _lib.YX_ERR_INVALID, kw
        with pytest.raises(BackendError):
            backend.sync()
        backend.clear_error()
    for wrong in (lambda: backend.matmul_epilogue(x.cpu(), w), lambda: backend.matmul_epilogue(x, w.float()), lambda: backend.matmul_epilogue(x.double(), w),
                  lambda: backend.matmul_epilogue(x, w, activation="tanh"), lambda: backend.matmul_epilogue(x[:, :64], w),
                  lambda: backend.matmul_epilogue(x, w, bias=b[:5]), lambda: backend.matmul_epilogue(x, w, bias=b.bfloat16()),
                  lambda: backend.matmul_epilogue(x, w, residual=r, out_dtype=torch.bfloat16), lambda: backend.matmul_epilogue(x, w, out=out),
                  lambda: backend.matmul_epilogue(x.T.contiguous().T, w)):
        with pytest.raises(AssertionError):
            wrong()
    assert backend.status() == _lib.YX_OK
    assert with_() == _lib.YX_OK
    backend.sync()

"""What the operators between hidden states and log probabilities promise at their edges: how 16-bit results are rounded after long
sums."""
import numpy as np  # noqa: F401
import pytest
import torch

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

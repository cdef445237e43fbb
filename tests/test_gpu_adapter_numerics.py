"""How many bits adapter_project keeps, one mechanism at a time: inputs whose products and x.A are exact in fp32, so
that what a kernel rounds on the way is all that is left.

Sizes and the kernels that serve them (latent_adapter_project's rule): up to 64 rows with at most 128 stacked rank
columns one launch with x.A inside; up to 96 rows, or narrow results, x.A and then the product with the columns on the
M side; 2048 rows of 2048 columns x.A and then the product on SM pairs.
"""

import pytest
import torch

from latent_b200 import AdapterSet, adapter_project

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def signed(g, lo, hi, *shape):
    """Random signs, magnitudes in [lo, hi)."""
    u = torch.rand(shape, generator=g, device="cuda") * (hi - lo) + lo
    return torch.where(torch.rand(shape, generator=g, device="cuda") < 0.5, -u, u)


def within(got, y, tol):
    bad = ~((got.double() - y).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - y).abs() / tol).max()))


@pytest.mark.parametrize("T,K,N,n", [(9, 512, 256, 2), (40, 512, 256, 12), (128, 512, 384, 12), (2048, 512, 2048, 3)])
@pytest.mark.parametrize("out", [HF, F32])
@pytest.mark.parametrize("e", [-60, -20, -12, -6, -3, 0, 17])
def test_fp16_intermediate_of_any_magnitude(cuda, T, K, N, n, out, e):
    """scale x.A between 2^-68 and 2^19, rows of two magnitudes in every tile, rows that are zero.

    A row of x has one value, so x.A is one product of 11-bit numbers: exact in fp32, and a power of two scales it.  In
    the tensor cores it is two fp16 parts: off by 2^-22 of itself, or by half a step of the subnormals, 2^-25, which of
    the row's largest is at most 2^-16 in the rows of 16-bit results on SM pairs that go there as they are, and 2^-39
    where rows are scaled first (2^-21 allowed for fp32 results).  Sums of 2 rank terms: 2 rank + 8 steps of 2^-24 of
    the sum of their magnitudes."""
    g = torch.Generator("cuda").manual_seed(T + e)
    rank, rows = 16, torch.arange(T, device="cuda")
    at = torch.randint(0, K, (T,), generator=g, device="cuda")
    x = torch.zeros((T, K), dtype=HF, device="cuda")
    x[rows, at] = signed(g, 1, 2, T).to(HF) * torch.where(rows % 2 == 1, 2.0 ** -8, 1.0).to(HF)
    x[3::7] = 0
    ads = [(signed(g, 1, 2, K, rank).to(HF), (signed(g, 0.25, 2, rank, N) * 2.0 ** max(-10, min(13, -e))).to(HF), 2.0 ** e)
           for _ in range(n)]
    ids = torch.randint(-1, n, (T,), generator=g, device="cuda").to(torch.int32)
    y = torch.zeros((T, N), dtype=torch.float64, device="cuda")
    S, most = y.clone(), y.clone()
    for i, (a, b, s) in enumerate(ads):
        r = ids == i
        t = s * (x[r].double() @ a.double())
        y[r], S[r] = t @ b.double(), t.abs() @ b.double().abs()
        most[r] = t.abs().max(1, keepdim=True).values * b.double().abs().sum(0)
    got = adapter_project(x, torch.zeros((K, N), dtype=HF, device="cuda"), AdapterSet(ads), ids, out_dtype=out)
    tol = (2 * rank + 8) * 2.0 ** -24 * S + (2.0 ** -22 + (2.0 ** -21 if out == F32 else 2.0 ** -16)) * most
    within(got, y, tol + torch.finfo(out).eps / 2 * y.abs() + (2.0 ** -25 if out == HF else 0.0))


@pytest.mark.parametrize("T,K,N,n,out", [(9, 512, 256, 2, HF), (40, 512, 256, 12, HF), (128, 512, 384, 12, HF),
                                         (9, 512, 256, 2, F32), (40, 512, 256, 12, F32), (128, 512, 384, 12, F32),
                                         (2048, 512, 2048, 3, F32)])
def test_fp16_intermediates_of_unlike_magnitudes_in_a_row(cuda, T, K, N, n, out):
    """Rank columns 2^-4, 2^-8 and 2^-12 of the largest, their rows of B as much larger: none is less of the result.

    Where the adapters' part has an accumulator of its own (all but 16-bit results on SM pairs) x.A is off by 2^-22 of
    itself or 2^-39 of its row's largest, 2^-27 of the least of these."""
    g = torch.Generator("cuda").manual_seed(T)
    rank, rows = 16, torch.arange(T, device="cuda")
    down = torch.tensor([2.0 ** -(4 * (r % 4)) for r in range(rank)], device="cuda")
    x = torch.zeros((T, K), dtype=HF, device="cuda")
    x[rows, torch.randint(0, K, (T,), generator=g, device="cuda")] = signed(g, 1, 2, T).to(HF)
    ads = [((signed(g, 1, 2, K, rank) * down).to(HF), (signed(g, 0.25, 2, rank, N) / down[:, None]).to(HF), 2.0 ** -6)
           for _ in range(n)]
    ids = torch.randint(0, n, (T,), generator=g, device="cuda").to(torch.int32)
    y = torch.zeros((T, N), dtype=torch.float64, device="cuda")
    S = y.clone()
    for i, (a, b, s) in enumerate(ads):
        t = s * (x[ids == i].double() @ a.double())
        y[ids == i], S[ids == i] = t @ b.double(), t.abs() @ b.double().abs()
    got = adapter_project(x, torch.zeros((K, N), dtype=HF, device="cuda"), AdapterSet(ads), ids, out_dtype=out)
    tol = ((2 * rank + 8) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -27) * S + torch.finfo(out).eps / 2 * y.abs()
    within(got, y, tol + (2.0 ** -25 if out == HF else 0.0))


@pytest.mark.parametrize("T,K,N,n", [(9, 512, 256, 2), (40, 512, 256, 12), (128, 512, 384, 12), (2048, 512, 2048, 3)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_fp32_results_keep_the_intermediates_bits(cuda, T, K, N, n, dtype):
    """fp32 results take x.A in as many 16-bit parts as hold 24 bits (bf16: three) or 22 (fp16: two).

    One rank column, W = 0: y is one product, x.A one (fp16: 22 bits) or two products 2^-8 apart (bf16: 16 bits each, 24
    in all) that fp32 holds.  Three parts of it, their products and sums: 8 steps of 2^-24.  Two bf16 parts would leave
    2^-17, one fp16 part 2^-12."""
    g = torch.Generator("cuda").manual_seed(T)
    rows = torch.arange(T, device="cuda")
    at = torch.randint(0, K // 2, (T,), generator=g, device="cuda")
    x = torch.zeros((T, K), dtype=dtype, device="cuda")
    x[rows, at] = signed(g, 1, 1.4, T).to(dtype)
    if dtype == BF:
        x[rows, K // 2 + at] = signed(g, 1, 1.4, T).to(dtype) * 2.0 ** -8
    ads = [(signed(g, 1, 1.4, K, 1).to(dtype), signed(g, 0.5, 2, 1, N).to(dtype), 2.0 ** (i % 3)) for i in range(n)]
    ids = torch.randint(0, n, (T,), generator=g, device="cuda").to(torch.int32)
    y = torch.zeros((T, N), dtype=torch.float64, device="cuda")
    for i, (a, b, s) in enumerate(ads):
        t = x[ids == i].double() @ a.double()
        assert torch.equal(t, t.float().double())
        y[ids == i] = s * t @ b.double()
    got = adapter_project(x, torch.zeros((K, N), dtype=dtype, device="cuda"), AdapterSet(ads), ids, out_dtype=F32)
    within(got, y, 8 * 2.0 ** -24 * y.abs())


# The tensor cores cut the sum of a step (16 terms) off: up to 2^-23 of the partial sum.  Positive terms, chains of 512
# (32 steps, partial sums that grow evenly): (1 + .. + 32) / 32 = 16.5 steps of 2^-23 at most; then up to 16 such sums
# are added, half a step of 2^-23 of a growing sum each: 8 more of 2^-24.
# The terms of a step are aligned to its largest first, two bits below the last of fp32.  A product of bf16 values of
# [0.5, 1.5) is a multiple of 2^-16 and a partial sum of 512 of them stays below 2^10: its last bit but two is 2^-16 or
# less and nothing more is cut.  Products of fp16 values reach down to 2^-22: each of the 17 terms loses up to 2^-25 of
# the partial sum as well, 17 / 4 + 1 steps of 2^-23 in place of one.
# One chain over 7168 has 14 times as many steps: four (bf16) and 14 / 5.25 times (fp16, as measured) over these bounds.
CHAIN = {BF: 16.5 * 2.0 ** -23 + 8 * 2.0 ** -24, HF: 16.5 * 5.25 * 2.0 ** -23 + 8 * 2.0 ** -24}


@pytest.mark.parametrize("T,N", [(96, 18944), (2048, 2048)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_fp32_results_of_long_sums(cuda, T, N, dtype):
    K = 7168
    g = torch.Generator("cuda").manual_seed(T)
    pos = lambda *s: (torch.rand(s, generator=g, device="cuda") + 0.5).to(dtype)  # noqa: E731
    x, w = pos(T, K), pos(K, N)
    s = AdapterSet([(pos(K, 4), pos(4, N), 1.0)])
    got = adapter_project(x, w, s, torch.full((T,), -1, dtype=torch.int32, device="cuda"), out_dtype=F32)
    y = x.double() @ w.double()
    within(got, y, CHAIN[dtype] * y)


@pytest.mark.parametrize("T,N", [(40, 256), (500, 256), (18944, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_fp32_results_of_a_long_intermediate(cuda, T, N, dtype):
    """x.A over K = 7168, one or a few blocks to a row tile (18944 rows: 148 of them): its sums are cut like x.W's."""
    K, n = 7168, 12
    g = torch.Generator("cuda").manual_seed(T)
    pos = lambda *s: (torch.rand(s, generator=g, device="cuda") + 0.5).to(dtype)  # noqa: E731
    x = pos(T, K)
    ads = [(pos(K, 1) * 2.0 ** -8, pos(1, N), 1.0) for _ in range(n)]
    ids = (torch.arange(T, device="cuda") * n // T).to(torch.int32)
    y = torch.empty((T, N), dtype=torch.float64, device="cuda")
    for i, (a, b, _) in enumerate(ads):
        y[ids == i] = (x[ids == i].double() @ a.double()) @ b.double()
    got = adapter_project(x, torch.zeros((K, N), dtype=dtype, device="cuda"), AdapterSet(ads), ids, out_dtype=F32)
    within(got, y, (CHAIN[dtype] + 2.0 ** -22 + 8 * 2.0 ** -24) * y)


@pytest.mark.parametrize("T,K,N,n", [(12, 256, 256, 2), (40, 256, 256, 12), (300, 256, 256, 3), (2048, 512, 2048, 3)])
@pytest.mark.parametrize("out", [HF, F32])
def test_fp16_row_that_is_not_finite_stays_alone(cuda, T, K, N, n, out):
    """NaN and infinities of a row of x reach no other row, whichever way fp16 rows beyond the parts' range take."""
    g = torch.Generator("cuda").manual_seed(T)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(HF)  # noqa: E731
    x, w = rand(T, K), rand(K, N)
    s = AdapterSet([(rand(K, 16), rand(16, N), 0.5) for _ in range(n)])
    ids = (torch.arange(T, device="cuda") % (n + 1) - 1).to(torch.int32)
    want = adapter_project(x, w, s, ids, out_dtype=out)
    bad = x.clone()
    bad[3, 5], bad[7, 0], bad[8, 1] = float("nan"), float("inf"), -float("inf")   # adapters 2, 3, none where n = 3
    got = adapter_project(bad, w, s, ids, out_dtype=out)
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[[3, 7, 8]] = False
    assert torch.equal(got[rest], want[rest]) and not bool(torch.isfinite(got[~rest]).any())

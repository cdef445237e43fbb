"""Adapters of many requests beside a shared projection (adapter_project)
against a 64-bit evaluation of y[t] = x[t].W + s_a (x[t].A_a).B_a.

Tolerance, per element.  With S = |x|.|W| + |s| (|x|.|A|).|B| every fp32 sum of
n terms is off by at most n 2^-24 S (n roundings of at most half a step of a
partial sum; the tensor cores cut 16 terms a step off instead of rounding, one
step in 16, which is less): K + 2 rank + 64 terms.  The intermediate x.A enters
the tensor cores as two 16-bit parts, off by 2^-16 of itself.  The result is
rounded once: half a step of its type.
"""

import numpy as np
import pytest
import torch

from latent_b200 import AdapterSet, adapter_project
from latent_b200 import _lib

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def make(T, K, N, ranks, dtype=BF, seed=0, layout="kn", ids="mixed"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = rand(T, K).to(dtype)
    w = (rand(K, N) / K ** 0.5).to(dtype)
    w = w if layout == "kn" else w.t().contiguous().t()
    ads = [((rand(K, r) / K ** 0.5).to(dtype), (rand(r, N) * 0.2).to(dtype), 0.5 + 0.25 * i)
           for i, r in enumerate(ranks)]
    n = len(ranks)
    if ids == "mixed":       # single tokens in any order, some without an adapter
        i = torch.randint(-1, n, (T,), generator=g, device="cuda")
    elif ids == "packed":    # runs of one adapter
        i = torch.arange(T, device="cuda") * (n + 1) // max(T, 1) - 1
    else:
        i = torch.full((T,), int(ids), device="cuda")
    return x, w, ads, i.to(torch.int32)


def reference(x, w, ads, ids):
    """(y, S) in 64 bits; w may be None."""
    xd, xa = x.double(), x.double().abs()
    y = xd @ w.double() if w is not None else torch.zeros((x.shape[0], ads[0][1].shape[1]), dtype=torch.float64,
                                                          device=x.device)
    S = xa @ w.double().abs() if w is not None else y.clone()
    for i, (a, b, s) in enumerate(ads):
        rows = ids == i
        y[rows] += s * ((xd[rows] @ a.double()) @ b.double())
        S[rows] += abs(s) * ((xa[rows] @ a.double().abs()) @ b.double().abs())
    return y, S


def assert_close(got, y, S, K, rank):
    tol = torch.finfo(got.dtype).eps / 2 * y.abs() + ((K + 2 * rank + 64) * 2.0 ** -24 + 2.0 ** -16) * S
    if got.dtype == HF:
        tol = tol + 2.0 ** -25          # half a step of the subnormals
    bad = ~((got.double() - y).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - y).abs() / tol).max()))


SHAPES = [
    # T, K, N, ranks
    (1, 2048, 2048, [16, 16]),
    (1, 64, 8, [1]),
    (2, 8, 16, [3, 1, 2]),
    (7, 1024, 704, [16, 5, 16]),
    (16, 256, 136, [64]),
    (20, 1024, 2048, [32] * 9),
    (33, 2048, 1408, [16] * 40),
    (64, 1024, 256, [8, 16, 3]),
    (128, 512, 384, [33, 64]),
    (129, 520, 264, [16, 16, 32]),
    (200, 1032, 648, [128, 100]),
    (257, 256, 512, [16] * 7),
    (640, 1024, 1024, [16, 32]),
    (1000, 712, 1416, [48, 2, 17]),
    (2047, 1024, 2048, [64, 33]),
]


@pytest.mark.parametrize("T,K,N,ranks", SHAPES)
@pytest.mark.parametrize("dtype,layout,ids", [(BF, "kn", "mixed"), (HF, "nk", "packed"), (BF, "nk", "mixed"),
                                              (HF, "kn", "packed")])
def test_matches_64_bits(cuda, T, K, N, ranks, dtype, layout, ids):
    x, w, ads, i = make(T, K, N, ranks, dtype, seed=T + K, layout=layout, ids=ids)
    s = AdapterSet(ads)
    assert s.dtype == dtype
    y, S = reference(x, w, ads, i)
    for out_dtype in (None, F32):
        got = adapter_project(x, w, s, i, out_dtype=out_dtype)
        assert got.dtype == (out_dtype or dtype)
        assert_close(got, y, S, K, s.rank)
    s.check()


@pytest.mark.parametrize("T,K,N", [(5, 100, 37), (70, 33, 130), (130, 101, 64), (300, 64, 131)])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_odd_widths(cuda, T, K, N, layout):
    x, w, ads, i = make(T, K, N, [5, 20], BF, seed=3, layout=layout)
    assert_close(adapter_project(x, w, AdapterSet(ads), i), *reference(x, w, ads, i), K, 32)


@pytest.mark.parametrize("T,K,N,ranks", [(1, 2048, 1001, [16]), (1, 72, 1, [3]), (9, 1024, 5003, [16] * 12),
                                         (40, 512, 37, [64] * 9), (130, 256, 257, [16, 32]), (300, 520, 1999, [16] * 3), (1, 100, 37, [16]),
                                         (2000, 512, 1001, [16] * 4)])
@pytest.mark.parametrize("dtype,out", [(BF, BF), (HF, HF), (BF, F32)])
def test_odd_result_widths(cuda, T, K, N, ranks, dtype, out):
    """Aligned rows of x and W, results of an odd width: dense, and as columns of a wider matrix that keeps the rest."""
    x, w, ads, i = make(T, K, N, ranks, dtype, seed=N, layout="nk")
    s = AdapterSet(ads)
    y, S = reference(x, w, ads, i)
    assert_close(adapter_project(x, w, s, i, out_dtype=out), y, S, K, s.rank)
    for pad in (N + 3, N + 8 - N % 8):
        big = torch.full((T + 1, pad), 7.0, dtype=out, device="cuda")
        adapter_project(x, w, s, i, out=big[:T, :N])
        assert_close(big[:T, :N], y, S, K, s.rank)
        assert bool((big[T] == 7).all()) and bool((big[:, N:] == 7).all())
    s.check()


@pytest.mark.parametrize("T", [1, 20, 300])
@pytest.mark.parametrize("out", [BF, F32])
def test_odd_contraction_in_padded_rows(cuda, T, out):
    """A width of x and W that ends inside a 16-byte run: what pads the rows is not read."""
    K, N = 101, 77
    x, w, ads, i = make(T, K, N, [16, 5], BF, seed=6, layout="nk")
    s = AdapterSet(ads)
    y, S = reference(x, w, ads, i)
    xp = torch.full((T, 104), float("nan"), dtype=BF, device="cuda")
    wp = torch.full((N, 104), float("nan"), dtype=BF, device="cuda")
    xp[:, :K], wp[:, :K] = x, w.t()
    assert_close(adapter_project(xp[:, :K], wp[:, :K].t(), s, i, out_dtype=out), y, S, K, s.rank)
    kn = torch.full((K, 80), float("nan"), dtype=BF, device="cuda")
    kn[:, :N] = w
    assert_close(adapter_project(xp[:, :K], kn[:, :N], s, i, out_dtype=out), y, S, K, s.rank)


@pytest.mark.parametrize("T", [3, 64, 300])
def test_strided_and_unaligned_rows(cuda, T):
    K, N = 256, 192
    x, w, ads, i = make(T, K, N, [16, 8], BF, seed=5)
    s = AdapterSet(ads)
    y, S = reference(x, w, ads, i)
    wide = torch.full((T, K + 24), float("nan"), dtype=BF, device="cuda")
    for off in (8, 3):                                   # 16-byte aligned rows, and rows that are not
        wide[:, off:off + K] = x
        big = torch.full((T + 2, N + 40), 7.0, dtype=BF, device="cuda")
        out = big[1:T + 1, off:off + N]
        assert adapter_project(wide[:, off:off + K], w, s, i, out=out) is out
        assert_close(out, y, S, K, 16)
        big[1:T + 1, off:off + N] = 7.0
        assert bool((big == 7.0).all())                  # nothing written around it
    ww = torch.full((K, N + 16), float("nan"), dtype=BF, device="cuda")
    ww[:, 8:8 + N] = w
    assert_close(adapter_project(x, ww[:, 8:8 + N], s, i), y, S, K, 16)
    assert_close(adapter_project(x.t().contiguous().t(), w, s, i), y, S, K, 16)      # column-major x


@pytest.mark.parametrize("T", [1, 40, 300])
def test_no_adapter_bad_id_and_one_adapter(cuda, T):
    K, N = 512, 256
    for which in ("-1", "1"):
        x, w, ads, i = make(T, K, N, [16, 16, 16], HF, seed=6, ids=which)
        s = AdapterSet(ads)
        assert_close(adapter_project(x, w, s, i), *reference(x, w, ads, i), K, 16)
        s.check()
    bad = i.clone()
    bad[T // 2] = 3
    got = adapter_project(x, w, s, bad)
    ref = i.clone()
    ref[T // 2] = -1
    assert_close(got, *reference(x, w, ads, ref), K, 16)
    with pytest.raises(_lib.LatentError, match="EXPERT_ID"):
        s.check()
    s.check()                                            # cleared
    assert adapter_project(x[:0], w, s, i[:0]).shape == (0, N)


@pytest.mark.parametrize("T", [40, 300])
def test_every_row_its_own_adapter(cuda, T):
    K, N = 256, 384
    x, w, ads, _ = make(T, K, N, [16] * T, BF, seed=7)
    i = torch.randperm(T, device="cuda").to(torch.int32)
    assert_close(adapter_project(x, w, AdapterSet(ads), i), *reference(x, w, ads, i), K, 16)


@pytest.mark.parametrize("T", [12, 300])
def test_a_row_that_is_not_finite_stays_alone(cuda, T):
    K, N = 256, 256
    x, w, ads, i = make(T, K, N, [16, 16], BF, seed=8)
    y, S = reference(x, w, ads, i)
    x = x.clone()
    x[3, 5], x[7, 0] = float("nan"), float("inf")
    got = adapter_project(x, w, AdapterSet(ads), i)
    rest = [t for t in range(T) if t not in (3, 7)]
    assert_close(got[rest], y[rest], S[rest], K, 16)
    assert not bool(torch.isfinite(got[3]).any()) and not bool(torch.isfinite(got[7]).any())


@pytest.mark.parametrize("T,n,out", [(9, 2, HF), (9, 2, F32), (20, 12, HF), (20, 12, F32), (128, 12, HF), (300, 2, HF),
                                     (300, 2, F32)])
def test_fp16_intermediate_beyond_the_fp16_range(cuda, T, n, out):
    """x.A of some rows passes 65504 while the result does not: B is small."""
    K, N = 512, 256
    x, w, ads, i = make(T, K, N, [16] * n, HF, seed=9, ids="packed")
    x[1::3] *= 400.0
    ads = [((a.float() * 200).to(HF), (b.float() * 1e-4).to(HF), 1.0 + 0.5 * (k % 2)) for k, (a, b, _) in enumerate(ads)]
    y, S = reference(x, w, ads, i)
    t = torch.cat([x[i == k].double() @ ads[k][0].double() for k in range(n)])
    assert float(t.abs().max()) > 65504 and float(y.abs().max()) < 60000
    assert_close(adapter_project(x, w, AdapterSet(ads), i, out_dtype=out), y, S, K, 16)


def test_factor_pair_as_the_shared_projection(cuda):
    from latent_b200 import project
    from latent_b200.quant import quantize_factor
    from latent_b200.runtime import FactorPair
    x, w, ads, i = make(50, 256, 320, [16, 8], BF, seed=10)
    g = torch.Generator().manual_seed(1)
    pair = FactorPair(quantize_factor(torch.randn(256, 64, generator=g) / 16, 20.0).to("cuda"),
                      quantize_factor(torch.randn(64, 320, generator=g) / 8, 20.0).to("cuda"))
    s = AdapterSet(ads)
    base = project(x, pair).double()
    y, S = reference(x, None, ads, i)
    for out_dtype in (None, F32):
        assert_close(adapter_project(x, pair, s, i, out_dtype=out_dtype), base + y, base.abs() + S, 256, 16)
    out = torch.empty((50, 320), dtype=BF, device="cuda")
    assert adapter_project(x, pair, s, i, out=out) is out
    assert_close(out, base + y, base.abs() + S, 256, 16)


@pytest.mark.parametrize("T", [20, 700])
def test_streams_graphs_and_repeats(cuda, T):
    """Bit-equal on another stream, in two captured graphs that run side by side, and on replay with new inputs."""
    K, N = 512, 640
    x, w, ads, i = make(T, K, N, [16, 32, 16], BF, seed=11)
    x2, _, _, i2 = make(T, K, N, [16, 32, 16], BF, seed=12)
    s = AdapterSet(ads)
    want, want2 = adapter_project(x, w, s, i), adapter_project(x2, w, s, i2)
    assert torch.equal(want, adapter_project(x, w, s, i))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = adapter_project(x, w, s, i)
    side.synchronize()
    assert torch.equal(got, want)
    xs, idb = x.clone(), i.clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(adapter_project(xs, w, s, idb))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for a, b, ref in ((x, i, want), (x2, i2, want2)):
        xs.copy_(a)
        idb.copy_(b)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    s.check()


def test_calls_of_all_kinds_on_two_streams_at_once(cuda):
    """Blocks of several calls share the GPU: every result is the one of the call alone."""
    calls = []
    for T, K, N, n in ((1, 1024, 2048, 2), (48, 2048, 1408, 40), (200, 1024, 640, 6), (700, 512, 1024, 3), (64, 7168, 256, 16)):
        for out in (None, F32):
            x, w, ads, i = make(T, K, N, [16] * n, BF, seed=T)
            s = AdapterSet(ads)
            calls.append((x, w, s, i, out, adapter_project(x, w, s, i, out_dtype=out)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for rep in range(6):
        got = []
        for k, (x, w, s, i, out, _) in enumerate(calls):
            with torch.cuda.stream(streams[(k + rep) % 3]):
                got.append(adapter_project(x, w, s, i, out_dtype=out))
        torch.cuda.synchronize()
        for g, c in zip(got, calls):
            assert torch.equal(g, c[5])
    for c in calls:
        c[2].check()


def test_calls_from_two_threads(cuda):
    from concurrent.futures import ThreadPoolExecutor
    calls = []
    for T, K, N, n in ((1, 1024, 2048, 2), (40, 2048, 704, 30), (300, 512, 1024, 3), (9, 100, 37, 2)):
        x, w, ads, i = make(T, K, N, [16] * n, BF, seed=T + 1)
        s = AdapterSet(ads)
        calls.append((x, w, s, i, adapter_project(x, w, s, i)))
    torch.cuda.synchronize()

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [[adapter_project(*c[:4]) for c in calls[k:] + calls[:k]] for _ in range(20)]
            torch.cuda.current_stream().synchronize()
        return all(torch.equal(g, c[4]) for r in got for g, c in zip(r, calls[k:] + calls[:k]))

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(run, (0, 2)))


@pytest.mark.parametrize("T,K,N", [(160000, 64, 14336),   # y beyond 2^31 elements, SM pairs
                                   (70000, 32768, 64),    # x
                                   (2, 8192, 270000),     # w
                                   (20000, 24, 131073)])  # y, CUDA cores
def test_offsets_beyond_32_bits(cuda, T, K, N):
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=BF)  # noqa: E731
    x, w = rand(T, K), rand(K, N) / K ** 0.5
    ads = [(rand(K, 16) / K ** 0.5, rand(16, N) * 0.2, 0.5 + 0.25 * i) for i in range(3)]
    ids = (torch.arange(T, device="cuda") * 4 // T - 1).to(torch.int32)
    y = adapter_project(x, w, AdapterSet(ads), ids)
    rows = torch.arange(T, device="cuda")
    rows = rows[(rows < 2) | (rows >= T - 130)]
    for lo, hi in ((0, 100), (max(0, N - 1000), N)):
        want, S = reference(x[rows], w[:, lo:hi], [(a, b[:, lo:hi], s) for a, b, s in ads], ids[rows])
        assert_close(y[rows, lo:hi], want, S, K, 16)
    del x, w, y, ads
    torch.cuda.empty_cache()


@pytest.mark.parametrize("T", [40, 700])
def test_workspace_of_a_captured_call_stays_the_graphs_own(cuda, T):
    from latent_b200 import balance_loss
    x, w, ads, i = make(T, 512, 640, [16] * 12, BF, seed=T)
    s = AdapterSet(ads)
    l = torch.randn((T, 64), device="cuda")
    slots = torch.randint(0, 64, (T, 4), device="cuda").to(torch.int32)
    want, r = adapter_project(x, w, s, i), balance_loss(l, slots, 0.1, 0.1, gradient=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = adapter_project(x, w, s, i)
        rg = balance_loss(l, slots, 0.1, 0.1, gradient=True)
    mine = [torch.full((n,), 7, dtype=torch.uint8, device="cuda")     # would land on it, had it gone back to all
            for n in (s.workspace_bytes(T), 66560, 70000, 1 << 20) for _ in range(40)]
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert all(bool((m == 7).all()) for m in mine)
    assert torch.equal(y, want) and torch.equal(rg.grad, r.grad) and torch.equal(rg.loss, r.loss)


FIRST_IN_CAPTURE = """
import torch
from latent_b200 import AdapterSet, adapter_project, balance_loss, router_topk_grad
g = torch.Generator("cuda").manual_seed(0)
rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)
w, l = rand(256, 512), torch.randn((100, 64), device="cuda")
s = AdapterSet([(rand(256, 16), rand(16, 512), 1.0) for _ in range(12)])
xs = [rand(T, 256) for T in (1, 40, 700)]
ids = [torch.zeros(x.shape[0], dtype=torch.int32, device="cuda") for x in xs]
slots = torch.randint(0, 64, (100, 4), device="cuda").to(torch.int32)
dw = torch.randn((100, 4), device="cuda")

def step():
    r = balance_loss(l, slots, 0.1, 0.1, gradient=True)
    return [adapter_project(x, w, s, i) for x, i in zip(xs, ids)] + [r.loss, router_topk_grad(l, slots, dw, logits=True, out=r.grad)]

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(out, step()):
    assert torch.equal(a, b)
print("captured")
"""


def test_first_calls_of_a_process_inside_a_capture(cuda):
    import subprocess
    import sys
    from conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE], cwd=ROOT, capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_refusals(cuda):
    x, w, ads, i = make(4, 64, 32, [16], BF)
    s = AdapterSet(ads)
    for bad in (lambda: adapter_project(x[:, :32], w, s, i), lambda: adapter_project(x.float(), w, s, i),
                lambda: adapter_project(x, w.half(), s, i), lambda: adapter_project(x, w[:, :16], s, i),
                lambda: adapter_project(x, w, s, i.long()), lambda: adapter_project(x, w, s, i[:3]),
                lambda: adapter_project(x, w.cpu(), s, i), lambda: adapter_project(x, w, s, i, out_dtype=HF),
                lambda: adapter_project(x, w, s, i, out=torch.empty((4, 31), dtype=BF, device="cuda")),
                lambda: adapter_project(x, w[::2].repeat(2, 2)[:, ::2], s, i),
                lambda: adapter_project(x, w.detach().requires_grad_(), s, i),
                lambda: AdapterSet([]), lambda: AdapterSet(ads, dtype=F32),
                lambda: AdapterSet([(torch.zeros(64, 129), torch.zeros(129, 32))]),
                lambda: AdapterSet([ads[0], (ads[0][0][:32], ads[0][1], 1.0)]),
                lambda: AdapterSet([(ads[0][0], ads[0][1] * float("inf"), 1.0)]),
                lambda: AdapterSet([(ads[0][0], ads[0][1], float("nan"))])):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        adapter_project(x, w.detach().requires_grad_(), s, i)
    np_set = AdapterSet([(ads[0][0].float().cpu().numpy(), ads[0][1].float().cpu().numpy())], dtype=BF)
    assert torch.equal(np_set.a, s.a) and float(np_set.scale) == 1.0

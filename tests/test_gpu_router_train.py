"""balance_loss and router_topk_grad against 64-bit evaluations of their
formulas, 64-bit autograd, and differences of the 64-bit loss.

Tolerance of the fp32 arithmetic: a probability is exp(l - m) / sum with
l - m rounded once (|l - m| 2^-24 in the exponent), expf off by two steps
(2^-22), a sum of at most 32 + 5 roundings and a division: a relative error of
(64 + |l - m|) 2^-24.  The dot products add as many terms again with errors of
their factors, and the coefficients four roundings, so every product p (c - d)
is within (192 + 3 max|l - m|) 2^-24 of p (|c| + |d|).  Then half a step of
the gradient's type (fp16: of its subnormals too).
"""

import numpy as np
import pytest
import torch

from latent_b200 import balance_loss, router_topk, router_topk_grad

pytestmark = pytest.mark.gpu
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def steps(l):
    l = torch.where(torch.isfinite(l), l, 0.0).double()
    return (192 + 3 * float(l.max() - l.min() if l.numel() else 0.0)) * 2.0 ** -24


def rounding(got, y):
    return torch.finfo(got.dtype).eps / 2 * y.abs() + (2.0 ** -25 if got.dtype == HF else 0.0)


def close(got, y, tol):
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    bad = ~((got.double() - y).abs() <= tol) & ~torch.isnan(y)
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - y).abs().max()))


def inputs(T, E, k, dtype=F32, seed=0, drop=True, scale=2.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    l = (scale * torch.randn((T, E), generator=g, device="cuda")).to(dtype)
    ids = torch.topk(torch.rand((T, E), generator=g, device="cuda"), k, dim=1).indices.to(torch.int32)
    if drop:
        keep = torch.randint(0, k + 1, (T, 1), generator=g, device="cuda")      # 0: a row with no kept slot
        ids = torch.where(torch.arange(k, device="cuda")[None] < keep, ids, -1).to(torch.int32)
    return l, ids


def loss64(l, ids, b, z, valid, cu):
    """(loss, balance, z, counts, c, rows that enter, n) of 64-bit logits; c: each row's E f / (S' n_s)."""
    T, E = l.shape
    cu = [0, T] if cu is None else cu.tolist()
    valid = torch.ones(T, dtype=torch.bool, device=l.device) if valid is None else valid
    live = ~(l == -float("inf")).all(1)
    counts = torch.zeros((len(cu) - 1, E), dtype=torch.int64, device=l.device)
    segs = []
    for s, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        rows = torch.arange(lo, hi, device=l.device)[valid[lo:hi]]
        e = ids[rows].reshape(-1).long()
        counts[s] = torch.bincount(e[(e >= 0) & (e < E)], minlength=E)
        segs.append(rows)
    used = max(1, sum(len(r) > 0 for r in segs))
    n = max(1, sum(len(r) for r in segs))
    bal = l.new_zeros(())
    zz = l.new_zeros(())
    coef = torch.zeros((T, E), dtype=torch.float64, device=l.device)
    enters = torch.zeros(T, dtype=torch.bool, device=l.device)
    for s, rows in enumerate(segs):
        if not len(rows):
            continue
        f = counts[s].double() / max(1, int(counts[s].sum()))
        c = E * f / (used * len(rows))
        r = rows[live[rows]]
        bal = bal + (torch.softmax(l[r], 1) * c).sum()
        zz = zz + (torch.logsumexp(l[r], 1) ** 2).sum() / n
        coef[r] = c
        enters[r] = True
    return b * bal + z * zz, bal, zz, counts, coef, enters, n


def check_balance(l, ids, b=0.01, z=0.001, valid=None, cu=None):
    r = balance_loss(l, ids, balance_coef=b, z_coef=z, valid=valid, cu_seqlens=cu, gradient=True)
    l64 = l.double().detach().requires_grad_(True)
    loss, bal, zz, counts, coef, enters, n = loss64(l64, ids, b, z, valid, cu)
    assert torch.equal(r.counts.long().reshape(counts.shape), counts)
    eps = steps(l)
    # (a sequence without a kept slot has coef = 0 and a z term all the same: the rows that enter, not those with coef)
    lse = torch.where(enters, torch.logsumexp(torch.where(torch.isfinite(l64), l64, -1e30), 1), 0.0).detach()
    # lse = m + log(sum): half a step of m, two of the logarithm, the sum's relative error
    lerr = (lse.abs() * 2.0 ** -22 + 64 * 2.0 ** -24)
    assert abs(float(r.balance) - float(bal)) <= eps * float(bal) + 1e-30
    assert abs(float(r.z) - float(zz)) <= float((2 * lse.abs() * lerr).sum()) / n + 2.0 ** -23 * float(zz)
    assert abs(float(r.loss) - float(loss)) <= 2.0 ** -23 * float(loss) + b * eps * float(bal) + \
        z * float((2 * lse.abs() * lerr).sum()) / n + 1e-30
    g = torch.autograd.grad(loss, l64)[0] if loss.requires_grad else torch.zeros_like(l64)
    g = torch.nan_to_num(g)            # rows with no finite logit: none of their values enters
    p = torch.nan_to_num(torch.softmax(l64.detach(), 1))
    d = (p * coef).sum(1, keepdim=True)
    tol = p * (b * (coef + d) * eps + 2 * z / n * (lerr + lse.abs() * eps)[:, None]) + rounding(r.grad, g) + 1e-38
    close(r.grad, g, tol)
    again = balance_loss(l, ids, balance_coef=b, z_coef=z, valid=valid, cu_seqlens=cu, gradient=True)
    for a, c in zip(r, again):
        assert torch.equal(a, c)
    return r


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 4, 2), (3, 8, 2), (64, 64, 6), (65, 63, 5), (100, 33, 1),
                                   (257, 160, 6), (300, 256, 8), (77, 1000, 6), (50, 1024, 32), (2000, 129, 8)])
@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_balance_loss(cuda, T, E, k, dtype):
    l, ids = inputs(T, E, k, dtype, seed=T + E)
    check_balance(l, ids, b=0.5 * T, z=0.25 * T)      # coefficients that keep an fp16 gradient in range


@pytest.mark.parametrize("cu", [[0, 0, 1, 1, 40, 200, 200], [0, 300], [5, 17, 300], [0, 128, 256, 290], [7, 7],
                                list(range(0, 301, 3))])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_balance_loss_sequences_and_masks(cuda, cu, masked, dtype):
    """Empty sequences, rows before the first and behind the last, padded rows with NaN and infinities in them."""
    T, E, k = 300, 72, 6
    l, ids = inputs(T, E, k, dtype, seed=len(cu))
    valid = None
    out = torch.ones(T, dtype=torch.bool, device="cuda")
    out[cu[0]:cu[-1]] = False
    if masked:
        valid = torch.rand(T, generator=torch.Generator("cuda").manual_seed(4), device="cuda") < 0.7
        valid[40:200] = len(cu) != 7                  # a sequence of padded rows alone
        out |= ~valid
    clean = check_balance(l, ids, valid=valid, cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    l2, ids2 = l.clone(), ids.clone()
    l2[out] = torch.tensor([float("nan"), float("inf"), -float("inf")] * (E // 3), device="cuda").to(dtype)
    ids2[out] = 5
    r = balance_loss(l2, ids2, 0.01, 0.001, valid, torch.tensor(cu, dtype=torch.int32, device="cuda"), gradient=True)
    for a, b in zip(r, clean):
        assert torch.equal(a, b)
    assert not bool(r.grad[out].any())


@pytest.mark.parametrize("T,S", [(20000, 1), (40000, 2), (3000, 20), (3000, 60), (2000, 200)])
def test_balance_loss_many_rows_and_many_sequences(cuda, T, S):
    """Every split of a sequence's counting over blocks and threads."""
    l, ids = inputs(T, 48, 6, F32, seed=S)
    g = torch.Generator("cuda").manual_seed(S)
    cu = torch.sort(torch.randint(0, T + 1, (S + 1,), generator=g, device="cuda")).values.to(torch.int32)
    if S <= 2:
        cu[0], cu[-1] = 0, T
    valid = torch.rand(T, generator=g, device="cuda") < 0.9
    check_balance(l, ids, valid=valid, cu=cu)


def test_balance_loss_masked_experts(cuda):
    """Masked experts (-inf, the type's lowest value), rows with every expert masked, and rows of NaN."""
    T, E, k = 60, 40, 4
    l, ids = inputs(T, E, k, F32, seed=3)
    l[:, 7] = -float("inf")
    l[:, 9] = torch.finfo(F32).min
    l[11] = -float("inf")
    l[12, :] = -float("inf")
    l[12, 3] = 1.5
    check_balance(l, ids)
    l[20, 4] = float("nan")
    l[21] = float("nan")
    r = balance_loss(l, ids, gradient=True)
    assert torch.isnan(r.loss) and bool(torch.isnan(r.grad[20:22]).all())
    assert bool(torch.isfinite(r.grad[:20]).all()) and bool(torch.isfinite(r.grad[22:]).all())


def test_balance_loss_odd_ids_and_empty(cuda):
    l, ids = inputs(40, 16, 3, F32, seed=5, drop=False)
    ids[3] = 7                                        # one id in every slot
    ids[4, 0], ids[5, 1] = 16, 2 ** 31 - 1            # no such expert: no slot
    check_balance(l, ids)
    none = torch.full_like(ids, -1)
    r = check_balance(l, none)
    assert float(r.balance) == 0 and not bool(r.counts.any())
    r = balance_loss(l[:0], ids[:0], z_coef=1.0, gradient=True)
    assert float(r.loss) == 0 and r.counts.shape == (16,) and not bool(r.counts.any()) and r.grad.shape == (0, 16)
    # sliced and unaligned logits
    wide = torch.randn((40, 19), device="cuda")
    check_balance(wide[:, 1:17], ids)
    flat = torch.randn(40 * 16 + 1, device="cuda")
    check_balance(flat[1:].view(40, 16), ids)


def test_balance_gradient_against_differences(cuda):
    l, ids = inputs(30, 24, 4, F32, seed=6)
    cu = torch.tensor([0, 4, 30], dtype=torch.int32, device="cuda")
    g = balance_loss(l, ids, 0.7, 0.3, None, cu, gradient=True).grad.double()
    gen = torch.Generator("cuda").manual_seed(2)
    for _ in range(4):
        v = torch.randn(l.shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5
        d = [float(loss64(l.double() + s * h * v, ids, 0.7, 0.3, None, cu)[0]) for s in (1, -1)]
        # central difference: h^2 / 6 of the third derivative and 2^-52 / h of the values
        assert abs((d[0] - d[1]) / (2 * h) - float((g * v).sum())) <= 1e-6 * float((g.abs() * v.abs()).sum()) + 1e-8


def slots64(v, ids, E, logits, renorm):
    kept = (ids >= 0) & (ids < E)
    p = torch.softmax(v, 1) if logits else v
    w = torch.where(kept, p.gather(1, torch.where(kept, ids, 0).long()), 0.0)
    if renorm:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(kept.any(1, keepdim=True), total, 1.0)
    return w


def check_route(v, ids, dw, logits, renorm):
    E = v.shape[1]
    got = router_topk_grad(v, ids, dw, renormalize=renorm, logits=logits)
    # renormalised softmax weights are the softmax over the kept logits: the whole softmax's 64-bit form would leave its
    # own roundings in columns whose gradient is zero
    v64 = v.double().detach().requires_grad_(True)
    kept = (ids >= 0) & (ids < E)
    d = torch.where(kept, dw.double(), 0.0)
    if logits and renorm:
        at = torch.where(kept, ids, 0).long()
        x = torch.where(kept, v64.gather(1, at), -float("inf"))
        w = torch.softmax(torch.where(kept.any(1, keepdim=True), x, 0.0), 1) * kept
    else:
        w = slots64(v64, ids, E, logits, renorm)
    g = torch.autograd.grad((w * d).sum(), v64)[0]
    eps = steps(v) if logits else 192 * 2.0 ** -24
    wd = w.detach().abs()
    c = (wd * d.abs()).sum(1, keepdim=True)
    at = torch.where(kept, ids, 0).long()
    if logits and not renorm:
        p = torch.softmax(v64.detach(), 1)
        tol = p * (torch.zeros_like(p).scatter_add_(1, at, d.abs()) + c) * eps
    else:
        if logits:
            s = wd * (d.abs() + c)
        elif renorm:
            total = torch.where(kept, v.double().gather(1, at), 0.0).sum(1, keepdim=True)
            s = (d.abs() + c) / torch.where(total == 0, 1.0, total)
        else:
            s = d.abs()
        tol = torch.zeros_like(v64).scatter_add_(1, at, torch.where(kept, s, 0.0)) * eps
    tol = tol.detach() + rounding(got, g) + 1e-38
    close(got, g, tol)
    assert torch.equal(got, router_topk_grad(v, ids, dw, renormalize=renorm, logits=logits))
    base = torch.randn(v.shape, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(v.dtype)
    acc = base.clone()
    assert router_topk_grad(v, ids, dw, renormalize=renorm, logits=logits, out=acc) is acc
    close(acc, base.double() + g, tol + rounding(acc, base.double() + g) + 2.0 ** -23 * (base.double().abs() + g.abs()))
    return got


MODES = [(True, True), (True, False), (False, True), (False, False)]


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 7, 2), (64, 64, 6), (65, 63, 5), (300, 256, 8), (77, 1000, 6),
                                   (50, 1024, 32), (1001, 160, 6), (20, 40, 32)])
@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("logits,renorm", MODES)
def test_router_grad(cuda, T, E, k, dtype, logits, renorm):
    v, ids = inputs(T, E, k, dtype, seed=T + E)
    if not logits:
        v = torch.softmax(v.float(), 1).to(dtype)
    dw = torch.randn((T, k), generator=torch.Generator("cuda").manual_seed(9), device="cuda")
    check_route(v, ids, dw, logits, renorm)


@pytest.mark.parametrize("logits,renorm", MODES)
def test_router_grad_odd_ids(cuda, logits, renorm):
    v, ids = inputs(50, 30, 5, F32, seed=2, drop=False)
    if not logits:
        v = torch.softmax(v, 1)
    ids[3] = 7                                        # one id in every slot
    ids[4, 1:3] = ids[4, 0]
    ids[5, 0], ids[6, 1] = 30, 2 ** 31 - 1            # no such expert: dropped
    ids[8] = -1
    dw = torch.randn(ids.shape, generator=torch.Generator("cuda").manual_seed(9), device="cuda")
    dw[8], dw[5, 0] = float("nan"), float("inf")      # of dropped slots: never read
    got = check_route(v, ids, dw, logits, renorm)
    assert not bool(got[8].any())
    if logits:
        v[:, 11] = -float("inf")
        ids[ids == 11] = 12
        check_route(v, ids, dw, logits, renorm)
        v[8] = -float("inf")                          # masked row without a kept slot
        assert not bool(router_topk_grad(v, ids, dw, renorm, logits)[8].any())


def test_router_grad_against_differences(cuda):
    for logits, renorm in MODES:
        v, ids = inputs(20, 16, 4, F32, seed=8)
        v = v if logits else torch.softmax(v, 1)
        dw = torch.randn(ids.shape, generator=torch.Generator("cuda").manual_seed(3), device="cuda")
        g = router_topk_grad(v, ids, dw, renorm, logits).double()
        u = torch.randn(v.shape, generator=torch.Generator("cuda").manual_seed(4), device="cuda", dtype=torch.float64)
        u = u if logits else u * v.double()           # stay inside the positive scores
        h = 1e-5
        d = [float((slots64(v.double() + s * h * u, ids, 16, logits, renorm) * dw.double()).sum()) for s in (1, -1)]
        assert abs((d[0] - d[1]) / (2 * h) - float((g * u).sum())) <= 1e-6 * float((g.abs() * u.abs()).sum()) + 1e-8


def test_autograd_matches_the_explicit_gradients(cuda):
    l, _ = inputs(200, 64, 6, F32, seed=4)
    leaf = l.clone().requires_grad_(True)
    ids, w, nk, counts = router_topk(leaf, 6, 0.9, logits=True, expert_counts=True, differentiable=True)
    with torch.no_grad():
        plain = router_topk(l, 6, 0.9, logits=True, expert_counts=True)
    for a, b in zip((ids, w, nk, counts), plain):
        assert torch.equal(a, b) and not b.requires_grad
    assert w.requires_grad and not ids.requires_grad
    assert not any(t.requires_grad for t in router_topk(leaf, 6, 0.9, logits=True))  # only when asked
    dw = torch.randn(w.shape, device="cuda")
    r = balance_loss(leaf, ids, 0.02, 0.001)
    assert r.grad is None and torch.equal(r.counts, counts)
    total = r.loss
    total *= 3.0                                      # a tensor of its own, not a view of the kernel's results
    (total + (w * dw).sum()).backward()
    g = balance_loss(l, ids, 0.06, 0.003, gradient=True).grad
    g = g.double() + router_topk_grad(l, ids, dw, logits=True).double()
    # two fp32 gradients, each within a few steps of the other form's, and their sum
    assert float((leaf.grad.double() - g).abs().max()) <= 8 * 2.0 ** -24 * float(g.abs().max())
    leaf16 = l.to(BF).requires_grad_(True)
    ids, w, _ = router_topk(leaf16, 6, 0.9, logits=True, renormalize=False, differentiable=True)
    w.sum().backward()
    assert leaf16.grad.dtype == BF
    assert torch.equal(leaf16.grad, router_topk_grad(leaf16.detach(), ids, torch.ones_like(w), False, True))


def test_streams_and_graphs(cuda):
    l, ids = inputs(500, 96, 6, F32, seed=1)
    l2, ids2 = inputs(500, 96, 6, F32, seed=2)
    dw = torch.randn((500, 6), device="cuda")
    cu = torch.tensor([0, 100, 450], dtype=torch.int32, device="cuda")

    def step(l, ids):
        r = balance_loss(l, ids, 0.01, 0.001, None, cu, gradient=True)
        router_topk_grad(l, ids, dw, logits=True, out=r.grad)
        return r.loss, r.counts, r.grad

    want, want2 = step(l, ids), step(l2, ids2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(l, ids)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ls, idb = l.clone(), ids.clone()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(ls, idb))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for a, b, ref in ((l, ids, want), (l2, ids2, want2)):
        ls.copy_(a)
        idb.copy_(b)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(u, v) for u, v in zip(o, ref))
    leaf = l.clone().requires_grad_(True)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="capture"):
                balance_loss(leaf, ids)
            with pytest.raises(RuntimeError, match="capture"):
                router_topk(leaf, 4, logits=True, differentiable=True)
        finally:
            g.capture_end()
    torch.cuda.synchronize()


def test_offsets_beyond_32_bits(cuda):
    T, E, k, n = 2200000, 1000, 2, 64
    g = torch.Generator("cuda").manual_seed(3)
    l = torch.randn((T, E), generator=g, device="cuda", dtype=BF)
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda").to(torch.int32)
    dw = torch.randn((T, k), generator=g, device="cuda")
    r = balance_loss(l, ids, 1e4, 1e4, gradient=True)
    assert torch.equal(r.counts.long(), torch.bincount(ids.view(-1).long(), minlength=E))
    tail = l[-n:].double()
    p, lse = torch.softmax(tail, 1), torch.logsumexp(tail, 1)[:, None]
    c = E * r.counts.double() / (k * T) / T
    d = (p * c).sum(1, keepdim=True)
    want = 1e4 * p * (c - d + 2 * lse / T)
    eps, lerr = steps(l[-n:]), lse.abs() * 2.0 ** -22 + 64 * 2.0 ** -24
    close(r.grad[-n:], want, 1e4 * p * ((c + d) * eps + 2 / T * (lerr + lse.abs() * eps)) + rounding(r.grad, want))
    del r
    for renorm in (True, False):
        got = router_topk_grad(l, ids, dw, renormalize=renorm, logits=True)[-n:].clone()
        assert torch.equal(got, check_route(l[-n:].contiguous(), ids[-n:], dw[-n:], True, renorm))
    torch.cuda.empty_cache()


def test_refusals(cuda):
    l, ids = inputs(10, 16, 3)
    dw = torch.ones((10, 3), device="cuda")
    cu = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    for bad in (lambda: balance_loss(l.cpu(), ids), lambda: balance_loss(l[0], ids), lambda: balance_loss(l.double(), ids),
                lambda: balance_loss(l, ids.long()), lambda: balance_loss(l, ids[:9]), lambda: balance_loss(l, ids.cpu()),
                lambda: balance_loss(l, ids, valid=torch.ones(9, dtype=torch.bool, device="cuda")),
                lambda: balance_loss(l, ids, valid=torch.ones(10, device="cuda")),
                lambda: balance_loss(l, ids, cu_seqlens=cu.long()), lambda: balance_loss(l, ids, cu_seqlens=cu[:1]),
                lambda: balance_loss(l, ids, cu_seqlens=cu.cpu()),
                lambda: router_topk_grad(l, ids, dw[:, :2]), lambda: router_topk_grad(l, ids, dw.half()),
                lambda: router_topk_grad(l, ids, dw, out=l), lambda: router_topk_grad(l, ids, dw, out=l.half()),
                lambda: router_topk_grad(l, ids, dw, out=torch.empty((16, 10), device="cuda").t())):
        with pytest.raises(ValueError):
            bad()


def test_recalibration_step_of_a_compressed_layer(cuda):
    """The operators together, as a router's recalibration uses them: adapted router logits, routing, the packed
    experts, the weights' gradient from the per-slot rows, the balance loss; against the same step in 64 bits."""
    from conftest import golden
    from gpu_helpers import golden_moe_experts
    from latent_b200 import AdapterSet, ExpertFFN, ExpertSet, adapter_project
    z = golden("moe")
    facs, _ = golden_moe_experts(z)
    es = ExpertSet(facs, device="cuda")
    E, d = es.n_expert, es.n_embd
    x = torch.from_numpy(np.ascontiguousarray(z["x"])).cuda().to(BF)
    T = x.shape[0]
    gen = torch.Generator("cuda").manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    w = (rand(E, d) / d ** 0.5).to(BF)
    ads = [((rand(d, 4) / d ** 0.5).to(BF), (rand(4, E) * 0.3).to(BF), 1.0) for _ in range(3)]
    req = (torch.arange(T, device="cuda") % 4 - 1).to(torch.int32)
    logits = adapter_project(x, w.t(), AdapterSet(ads), req, out_dtype=F32)
    l64 = x.double() @ w.t().double()
    for i, (a, b, s) in enumerate(ads):
        l64[req == i] += s * (x[req == i].double() @ a.double()) @ b.double()
    assert float((logits.double() - l64).abs().max()) <= 1e-4 * float(l64.abs().max())
    k = min(2, E)
    ids, wts, nk, counts = router_topk(logits, k, 0.9, logits=True, expert_counts=True)
    y = ExpertFFN(es, path="decode")(x, ids, wts, out_per_slot=True)
    out = (y * wts[:, :, None]).sum(1)
    target = rand(T, d)
    d_out = 2.0 * (out - target) / out.numel()
    d_w = (d_out[:, None, :] * y).sum(-1)
    r = balance_loss(logits, ids, 0.01, 0.001, gradient=True)
    assert torch.equal(r.counts, counts)
    g = router_topk_grad(logits, ids, d_w, logits=True, out=r.grad)
    v = logits.double().requires_grad_(True)
    w64 = slots64(v, ids, E, True, True)
    o64 = (y.double() * w64[:, :, None]).sum(1)
    loss = ((o64 - target.double()) ** 2).mean() + loss64(v, ids, 0.01, 0.001, None, None)[0]
    ref = torch.autograd.grad(loss, v)[0]
    # fp32 d_w: d sums of d terms, then the gradients' own steps
    assert float((g.double() - ref).norm()) <= (d + 256) * 2.0 ** -24 * float(ref.norm()) * 4

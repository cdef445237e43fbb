"""Calls of the adapter and router-training operators at the edges of what their documentation allows."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from latent_b200 import AdapterSet, _lib, adapter_project, balance_loss, router_topk, router_topk_grad
from test_gpu_router_train import close, inputs, loss64, rounding, steps

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16


def small_set(K=64, N=32, n=2):
    g = torch.Generator("cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF)  # noqa: E731
    return rand(6, K), rand(K, N), AdapterSet([(rand(K, 4), rand(4, N), 1.0) for _ in range(n)]), \
        torch.zeros(6, dtype=torch.int32, device="cuda")


def test_an_error_is_reported_whatever_stream_it_comes_from(cuda):
    """Work on another stream records a bad id while this one checks: reported now or by the next check, never lost."""
    x, w, s, ids = small_set()
    bad = ids.clone()
    bad[2] = s.n_adapter
    torch.cuda.synchronize()
    side = torch.cuda.Stream()

    def raised():
        try:
            s.check()
            return False
        except _lib.LatentError as e:
            assert "EXPERT_ID" in str(e)
            return True

    for i in range(300):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100000 + 1000 * i)          # lands between two of the checks below, or inside one
            adapter_project(x, w, s, bad)
        seen = 0
        while not side.query():
            seen += raised()
        torch.cuda.current_stream().wait_stream(side)
        seen += raised()
        assert seen
        assert not raised()                               # reported once, then cleared


def test_tangents_are_refused(cuda):
    x, w, s, ids = small_set()
    l, slots = inputs(10, 16, 3)
    dw = torch.ones((10, 3), device="cuda")
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: adapter_project(dual(x), w, s, ids), lambda: adapter_project(x, dual(w), s, ids),
                     lambda: adapter_project(x, dual(w.t().contiguous()).t(), s, ids),
                     lambda: adapter_project(x, w, s, ids, out=dual(torch.empty((6, 32), dtype=BF, device="cuda"))),
                     lambda: balance_loss(dual(l), slots), lambda: balance_loss(dual(l), slots, gradient=True),
                     lambda: router_topk_grad(dual(l), slots, dw), lambda: router_topk_grad(l, slots, dual(dw)),
                     lambda: router_topk_grad(l, slots, dw, out=dual(torch.zeros_like(l))),
                     lambda: router_topk(dual(l), 3, differentiable=True)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        # without tangents the calls stand, inside a level as outside
        router_topk_grad(l, slots, dw)
        adapter_project(x, w, s, ids)
        balance_loss(l, slots)
    router_topk(l, 3, differentiable=True)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("use", [(1.0, 0.0, 0.0), (0.0, 1.0, 0.0), (0.0, 0.0, 1.0), (0.3, 0.7, 0.2)])
def test_every_loss_carries_its_gradient(cuda, dtype, use):
    """loss, balance and z of balance_loss, weighted by the caller, through autograd against 64-bit autograd."""
    T, E, k, b, z = 300, 72, 6, 2.0, 0.5
    l, ids = inputs(T, E, k, dtype, seed=8)
    cu = torch.tensor([0, 100, 101, 290], dtype=torch.int32, device="cuda")
    leaf = l.clone().requires_grad_(True)
    r = balance_loss(leaf, ids, b, z, cu_seqlens=cu)
    parts = [u * v for u, v in zip(use, (r.loss, r.balance, r.z)) if u]
    assert all(p.requires_grad for p in parts) and not r.counts.requires_grad
    sum(parts).backward()
    l64 = l.double().requires_grad_(True)
    loss, bal, zz, _, coef, enters, n = loss64(l64, ids, b, z, None, cu)
    (use[0] * loss + use[1] * bal + use[2] * zz).backward()
    # as balance_loss with the coefficients that the weights amount to, two more roundings of them
    tb, tz = use[0] * b + use[1], use[0] * z + use[2]
    lse = torch.where(enters, torch.logsumexp(l64.detach(), 1), 0.0)
    p, eps = torch.softmax(l64.detach(), 1), steps(l) + 4 * 2.0 ** -24
    d = (p * coef).sum(1, keepdim=True)
    lerr = lse.abs() * 2.0 ** -22 + 64 * 2.0 ** -24
    tol = p * (tb * (coef + d) * eps + 2 * tz / n * (lerr + lse.abs() * eps)[:, None]) + 1e-38
    assert leaf.grad.dtype == dtype
    close(leaf.grad, l64.grad, tol + rounding(leaf.grad, l64.grad))


def test_losses_may_be_changed_in_place(cuda):
    l, ids = inputs(20, 16, 3)
    leaf = l.clone().requires_grad_(True)
    r = balance_loss(leaf, ids, 0.5, 0.1)
    want = torch.autograd.grad(2.0 * r.loss + 3.0 * r.z, leaf)[0]
    r = balance_loss(leaf, ids, 0.5, 0.1)
    loss, z = r.loss, r.z
    loss *= 2.0
    z *= 3.0
    assert torch.equal(torch.autograd.grad(loss + z, leaf)[0], want)

"""Calls of the adapter and router-training operators at the edges of what their documentation allows."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from latent_b200 import AdapterSet, _lib, adapter_project, balance_loss, router_topk, router_topk_grad
from test_gpu_router_train import inputs

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


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

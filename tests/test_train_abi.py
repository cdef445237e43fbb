"""Host-side validation of the adapter and router-training entry points: bad descriptors are rejected
before anything touches the device (this file needs no GPU)."""

import ctypes as C

import pytest
import torch

from latent_b200 import AdapterSet, _lib, adapter_project, balance_loss, router_topk_grad
from latent_b200.build import build


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.lib()


def test_router_grad_validates_on_the_host(lib):
    def f(**kw):
        d = dict(n_tokens=4, n_expert=8, top_k=2, scores=64, ids=64, d_weights=64, d_scores=64)
        return lib.latent_router_grad(C.byref(_lib.RouterGradDesc(**{**d, **kw})), None)

    assert lib.latent_router_grad(None, None) == 1
    assert f(n_expert=0) == 2 and f(n_tokens=-1) == 2 and f(top_k=0) == 2
    assert f(n_tokens=1 << 28, top_k=32) == 2                             # too many slots
    assert f(flags=8) == 1 and f(reserved=1) == 1 and f(type=7) == 3
    assert f(n_expert=2048) == 9 and f(n_expert=64, top_k=33) == 9
    assert f(n_tokens=0, scores=None) == 0                                # empty batch
    for name in ("scores", "ids", "d_weights", "d_scores"):
        assert f(**{name: None}) == 1, name
        assert f(**{name: 66}) == 4, name


def test_balance_loss_validates_on_the_host(lib):
    n = C.c_size_t()

    def size(**kw):
        return lib.latent_balance_workspace_size(C.byref(_lib.BalanceDesc(**kw)), C.byref(n))

    assert size(n_sequences=0, n_expert=8) == 2 and size(n_sequences=1, n_expert=0) == 2
    assert lib.latent_balance_workspace_size(None, C.byref(n)) == 1
    assert lib.latent_balance_workspace_size(C.byref(_lib.BalanceDesc(n_sequences=1, n_expert=8)), None) == 1
    assert size(n_sequences=1, n_expert=8) == 0 and n.value % 256 == 0

    def f(**kw):
        d = dict(n_tokens=4, n_expert=8, top_k=2, n_sequences=1, type=0, balance_coef=0.1, logits=256, ids=256, losses=256,
                 counts=256, workspace=256, workspace_bytes=n.value)
        return lib.latent_balance_loss(C.byref(_lib.BalanceDesc(**{**d, **kw})), None)

    assert lib.latent_balance_loss(None, None) == 1
    assert f(n_expert=0) == 2 and f(n_tokens=-1) == 2 and f(top_k=0) == 2 and f(n_sequences=0) == 2
    assert f(n_sequences=2) == 2                                          # sequences without borders
    assert f(type=5) == 3 and f(n_expert=1025) == 9 and f(flags=1) == 1
    for name in ("logits", "ids", "losses", "counts", "workspace"):
        assert f(**{name: None}) == 1, name
    assert f(logits=258) == 4 and f(ids=258) == 4 and f(grad=257) == 4 and f(d_loss=2) == 4 and f(workspace=128) == 4
    assert f(workspace_bytes=n.value - 1) == 6


def _desc(**kw):
    d = _lib.AdapterDesc(2, 16, 64, 32, 4, _lib.TYPE_BF16, _lib.TYPE_BF16, 0, 256, 64, 256, 32, 256, 64, 256, 32, 256,
                         256, 256, 32, 256, 256, 1 << 20)
    for name, v in kw.items():
        setattr(d, name, v)
    return C.byref(d)


def test_adapter_project_validates_on_the_host(lib):
    f = lib.latent_adapter_project
    assert f(None, None) == 1
    for bad in ({"n_adapter": -1}, {"n_in": 0}, {"n_out": 0}, {"n_tokens": -1}, {"ldx": 63}, {"ldw": 31}, {"lda": 63},
                {"ldb": 31}, {"ldy": 31}, {"flags": 1, "ldw": 63}, {"n_in": (1 << 30) + 1}, {"n_out": 0x7fffffff}):
        assert f(_desc(**bad), None) == 2, bad
    for bad in ({"rank": 8}, {"rank": 48}, {"rank": 256}):
        assert f(_desc(**bad), None) == 9, bad
    for bad in ({"type": 0}, {"type": 9}, {"y_type": 1}):
        assert f(_desc(**bad), None) == 3, bad
    assert f(_desc(flags=2), None) == 1
    for name in ("x", "a", "b", "scale", "ids", "y", "err", "workspace"):
        assert f(_desc(**{name: None}), None) == 1, name
    for bad in ({"x": 257}, {"w": 257}, {"ids": 258}, {"y": 257}, {"y": 258, "y_type": 0}, {"workspace": 272}):
        assert f(_desc(**bad), None) == 4, bad
    assert f(_desc(workspace_bytes=16), None) == 6
    assert f(_desc(n_tokens=0, x=None), None) == 0                        # empty batch
    n = C.c_size_t()
    assert lib.latent_adapter_workspace_size(_desc(), None) == 1
    assert lib.latent_adapter_workspace_size(_desc(), C.byref(n)) == 0 and n.value % 256 == 0
    assert lib.latent_adapter_check(None, None) == 1


def test_python_refusals_without_a_device():
    l, ids = torch.zeros((4, 8)), torch.zeros((4, 2), dtype=torch.int32)
    on_host = AdapterSet([(torch.zeros(8, 2), torch.zeros(2, 8))], device="cpu", dtype=torch.float16)
    for bad in (lambda: balance_loss(l, ids), lambda: router_topk_grad(l, ids, torch.zeros((4, 2))),
                lambda: adapter_project(l.half(), torch.zeros((8, 8), dtype=torch.float16), on_host, ids[:, 0].contiguous()),
                lambda: AdapterSet([], device="cpu"),
                lambda: AdapterSet([(torch.zeros(8, 2), torch.zeros(3, 8))], device="cpu"),
                lambda: AdapterSet([(torch.full((8, 2), float("inf")), torch.zeros(2, 8))], device="cpu")):
        with pytest.raises(ValueError):
            bad()


def test_adapter_set_layout():
    """Padding: ranks to one of 16, 32, 64, 128, rows to 16 bytes, zeros everywhere else."""
    a, b = torch.randn(10, 17), torch.randn(17, 13)
    s = AdapterSet([(a, b, 0.5), (a[:, :3], b[:3])], device="cpu", dtype=torch.float16)
    assert s.rank == 32 and s.a.shape == (2, 32, 16) and s.b.shape == (2, 32, 16) and s.ranks == [17, 3]
    assert torch.equal(s.a[0, :17, :10], a.t().half()) and torch.equal(s.b[1, :3, :13], b[:3].half())
    live = s.a[0, :17, :10].double().abs().sum() + s.a[1, :3, :10].double().abs().sum()
    assert float((s.a.double().abs().sum() - live).abs()) <= 1e-9 * float(live)
    assert s.scale.tolist() == [0.5, 1.0]


@pytest.mark.parametrize("scale", [1e39, -1e39, float("inf"), float("nan")])
def test_scales_are_finite_as_they_are_kept(scale):
    """A scale that is finite in 64 bits and infinite in the 32 that the device keeps."""
    good = (torch.ones(8, 2), torch.ones(2, 8), 3e38)
    assert AdapterSet([good], device="cpu").scale.isfinite().all()
    with pytest.raises(ValueError, match="finite"):
        AdapterSet([good, (torch.ones(8, 2), torch.ones(2, 8), scale)], device="cpu")


def test_balance_loss_gradients_of_all_three_losses_are_given_as_such(lib):
    d = dict(n_tokens=4, n_expert=8, top_k=2, n_sequences=1, type=0, balance_coef=0.1, logits=256, ids=256, losses=256,
             counts=256, workspace=256, flags=_lib.BALANCE_D_LOSSES)
    f = lambda **kw: lib.latent_balance_loss(C.byref(_lib.BalanceDesc(**{**d, **kw})), None)  # noqa: E731
    assert f() == 1                                                       # the flag without the floats
    assert f(d_loss=256) == 6                                             # on to the workspace's check
    assert f(d_loss=256, flags=_lib.BALANCE_D_LOSSES | 4) == 1

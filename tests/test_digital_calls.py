"""Calls of the digital operators' entry points (layer norm, orthogonalisation, Muon step) that lie beside the ordinary
ones: each is answered right or refused, never answered wrong."""

import pytest
import torch

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

gpu = pytest.mark.gpu
both_devices = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])


@pytest.fixture(autouse=True)
def _built(request):
    if request.node.get_closest_marker("gpu") and not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from isa_b200 import build
    build.build_library()


@pytest.fixture
def norms():
    from isa_b200.kernels.transformer_norm import cuda_add_layer_norm, cuda_layer_norm
    return cuda_layer_norm, cuda_add_layer_norm


@pytest.fixture
def muons():
    from isa_b200.kernels.muon import cuda_muon_step, cuda_orthogonalize
    return cuda_orthogonalize, cuda_muon_step


# ------------------------------------------------- what follows a call by its tensors --

@both_devices
def test_norm_refuses_what_it_cannot_follow(norms, device):
    """Forward-mode tangents, traces and subclasses with their own dispatch, with and without gradients recorded."""
    import torch.autograd.forward_ad as fwd
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.testing._internal.two_tensor import TwoTensor
    layer_norm, add_layer_norm = norms
    x, w = torch.randn(3, 16, device=device), torch.ones(16, device=device)
    with fwd.dual_level():
        dual, dual_w = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(w, torch.ones_like(w))
        calls = [lambda: layer_norm(dual), lambda: layer_norm(x, dual_w), lambda: layer_norm(x, None, dual_w),
                 lambda: add_layer_norm(dual, x), lambda: add_layer_norm(x, dual),
                 lambda: layer_norm(dual, w.clone().requires_grad_(True))]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
    for trace in (lambda f: torch.jit.trace(f, (x,)), lambda f: make_fx(f, tracing_mode="real")(x)):
        with pytest.raises(RuntimeError, match="traced"):
            trace(lambda t: layer_norm(t))
        with pytest.raises(RuntimeError, match="traced"):
            trace(lambda t: add_layer_norm(t, t)[0])
    for call in (lambda: layer_norm(TwoTensor(x, x)), lambda: layer_norm(x, TwoTensor(w, w))):
        with pytest.raises(RuntimeError, match="subclass"):
            call()


@both_devices
def test_muon_refuses_what_it_cannot_follow(muons, device):
    import torch.autograd.forward_ad as fwd
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.testing._internal.two_tensor import TwoTensor
    orthogonalize, muon_step = muons
    g, p, m = torch.randn(6, 8, device=device), torch.ones(6, 8, device=device), torch.zeros(6, 8, device=device)
    with fwd.dual_level():
        dual = fwd.make_dual(g, torch.ones_like(g))
        with pytest.raises(RuntimeError, match="forward-mode"):
            orthogonalize(dual)
        for args in (([dual], [g], [m]), ([p], [dual], [m]), ([p], [g], [dual])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                muon_step(*args, lr=0.1)
    for trace in (lambda f: torch.jit.trace(f, (g,)), lambda f: make_fx(f, tracing_mode="real")(g)):
        with pytest.raises(RuntimeError, match="traced"):
            trace(lambda t: orthogonalize(t))
        with pytest.raises(RuntimeError, match="traced"):
            trace(lambda t: muon_step([p], [t], [m], lr=0.1) or t)
    with pytest.raises(RuntimeError, match="subclass"):
        orthogonalize(TwoTensor(g, g))
    with pytest.raises(RuntimeError, match="subclass"):
        muon_step([p], [TwoTensor(g, g)], [m], lr=0.1)
    assert (p == 1).all() and not m.any()


@gpu
def test_dispatch_modes_that_only_look_on(norms):
    """Modes that count or cache operations without standing in for them leave the calls alone."""
    from torch.utils.flop_counter import FlopCounterMode
    layer_norm, _ = norms
    x = torch.randn(5, 48, device="cuda", requires_grad=True)
    want = layer_norm(x)
    with FlopCounterMode(display=False):
        got = layer_norm(x)
        g, = torch.autograd.grad(got.sum(), x)
    assert torch.equal(got, want) and torch.equal(g, torch.autograd.grad(want.sum(), x)[0])
    again = torch.utils.checkpoint.checkpoint(layer_norm, x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again.sum(), x)[0], g)

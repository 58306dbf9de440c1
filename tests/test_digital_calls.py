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


# ------------------------------------------------------------------------ views --

@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_of_negative_views(norms, dtype):
    """Memory that holds the negatives of a tensor's values (the imaginary part of a conjugate is one)."""
    layer_norm, add_layer_norm = norms
    neg = torch._neg_view
    x, d, dy, dh = (torch.randn(9, 40, device="cuda").to(dtype) for _ in range(4))
    w, b = torch.randn(40, device="cuda").to(dtype), torch.randn(40, device="cuda").to(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, d, w, b)]
    want = add_layer_norm(*leaves)
    want += torch.autograd.grad(want, leaves, (dy, dh))
    others = [(-t).requires_grad_(True) for t in (x, d, w, b)]
    got = add_layer_norm(*(neg(t) for t in others))
    got += tuple(-g for g in torch.autograd.grad(got, others, (neg(-dy), neg(-dh))))
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert torch.equal(layer_norm(neg(x), neg(w), neg(b)), layer_norm(-x, -w, -b))
    z = torch.complex(torch.randn(6, 40, device="cuda"), torch.randn(6, 40, device="cuda"))
    assert z.conj().imag.is_neg() and torch.equal(layer_norm(z.conj().imag), layer_norm(-z.imag))


@gpu
def test_muon_of_negative_views(muons):
    orthogonalize, muon_step = muons
    neg = torch._neg_view
    g = torch.randn(3, 30, 20, device="cuda")
    assert torch.equal(orthogonalize(neg(g)), orthogonalize(-g))
    p, m = torch.randn_like(g), torch.randn_like(g)
    want = p.clone(), m.clone()
    muon_step([want[0]], [-g], [want[1]], lr=0.1)
    got = p.clone(), m.clone()
    for bad in (([neg(got[0])], [g], [got[1]]), ([got[0]], [g], [neg(got[1])])):
        with pytest.raises(RuntimeError, match="negative bit"):
            muon_step(*bad, lr=0.1)
    muon_step([got[0]], [neg(g)], [got[1]], lr=0.1)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    # a gradient that is its momentum's negative is written out first, so nothing overlaps
    a, c = (p.clone(), m.clone()), (p.clone(), m.clone())
    muon_step([a[0]], [neg(a[1])], [a[1]], lr=0.1)
    muon_step([c[0]], [-c[1]], [c[1]], lr=0.1)
    assert all(torch.equal(s, t) for s, t in zip(a, c))


# ----------------------------------------------------------------------- numbers --

@gpu
def test_steps_beyond_an_int(muons):
    """2^32 + 5 steps are refused, not taken for 5."""
    orthogonalize, muon_step = muons
    g = torch.randn(8, 8, device="cuda")
    p, m = torch.ones_like(g), torch.zeros_like(g)
    for steps in (2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, 65, 0, -1):
        with pytest.raises(RuntimeError, match="1 to 64 steps"):
            orthogonalize(g, steps=steps)
        with pytest.raises(RuntimeError, match="1 to 64 steps"):
            muon_step([p], [g], [m], lr=0.1, steps=steps)
    assert (p == 1).all() and not m.any()


def _accepted(lib, steps, a, b, c):
    rc = lib.cimekv_orthogonalize(None, 0, 0, 0, 0, 8, 8, steps, a, b, c, 1e-7, None, None, 0, None)  # of no matrices
    assert rc in (0, 1) and (rc == 0 or b"beyond" in lib.cimekv_last_error())
    return rc == 0


def test_coefficients_by_what_they_let_grow():
    """Accepted are those whose singular values stay below 3.9 and whose factors stay below 15, by dense sampling."""
    import numpy as np
    from isa_b200 import _lib
    lib = _lib.load()
    rng = np.random.default_rng(0)
    seen = set()
    for k in range(3000):
        a, b, c = (float(np.float32(v)) for v in rng.normal(size=3) * rng.choice([0.3, 2.0, 6.0], 3))
        if k % 5 == 0:
            c = 0.0
        if k % 7 == 0:
            b = 0.0
        steps = int(rng.integers(1, 7))
        s, shift, size, sure = 1.001, 0.5 * b / c if c else 0.0, 0.0, True
        for _ in range(steps):
            t = np.linspace(0.0, s, 20001)
            q = a + (b + c * t * t) * t * t
            s = np.abs(t * q).max() * 1.001
            size = max(size, s / 3.9, np.abs(q).max() / 15.0, np.abs(t * t + shift).max() / 15.0, abs(shift) / 15.0)
            if size > 1e6:
                break
        if abs(size - 1.0) > 1e-4:  # on either side of the limit by more than the sampling
            assert _accepted(lib, steps, a, b, c) == (size < 1.0), (steps, a, b, c, size)
            seen.add(size < 1.0)
    assert seen == {True, False}
    for known in ((3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5), (1.0, 0.0, 0.0)):
        assert _accepted(lib, 5, *known)


def test_checking_coefficients_takes_no_time():
    """The checks before a launch are a few microseconds of the host's (sampling the polynomial took 50)."""
    import time
    from isa_b200 import _lib
    lib = _lib.load()
    times = []
    for _ in range(7):
        began = time.process_time()
        for _ in range(500):
            _accepted(lib, 5, 3.4445, -4.7750, 2.0315)
        times.append((time.process_time() - began) / 500)
    assert min(times) < 20e-6, min(times)


@gpu
@pytest.mark.parametrize("momentum", [0.0, 0.5, 0.9, 0.95, 0.999, 0.99999, 1.0])
def test_weight_of_the_gradient(muons, momentum):
    """From zeros the momentum is (1 - momentum) g: one rounding of the weight and one of the product, each half of 2^-23
    (a weight formed from the rounded momentum is off by up to 2^-25 / (1 - momentum) of itself)."""
    _, muon_step = muons
    g = torch.randn(70, 90, device="cuda")
    m = torch.zeros_like(g)
    muon_step([torch.zeros_like(g)], [g], [m], lr=0.1, momentum=momentum)
    want = (1.0 - momentum) * g.double()
    assert ((m.double() - want).abs() <= 2.01 * 2.0 ** -24 * want.abs()).all()


# ------------------------------------------------------------------------ memory --

def _peak(call):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    return torch.cuda.max_memory_allocated() - before


@gpu
def test_workspace_does_not_grow_with_the_number_of_matrices(muons):
    """16 bytes an element held at once for 200 matrices of 1,024 x 1,024 would be 3.4 GB: 2 GiB are the limit, and the
    launches that this makes get each matrix right."""
    from tests.test_muon import _assert_near, _exact, _update, _want_step
    orthogonalize, muon_step = muons
    g = torch.cat([_update("cuda", 50, 1024, 1024, seed=i, dtype=BF16) for i in range(4)])
    out = []
    assert _peak(lambda: out.append(orthogonalize(g))) < (2 << 30) + 2 * g.numel() + (1 << 20)
    out = out[0]
    for i in (0, 99, 100, 199):
        _assert_near(out[i], *_exact(g[i]), f"matrix {i}")
    wide = g[::2].transpose(1, 2)[:, :, :900]  # rows and matrices further apart than they are large
    assert torch.equal(orthogonalize(wide), orthogonalize(wide.contiguous()))
    del out
    p, m = torch.zeros(200, 1024, 1024, device="cuda"), torch.zeros(200, 1024, 1024, device="cuda")
    assert _peak(lambda: muon_step([p], [g], [m], lr=1.0, weight_decay=0.0)) < (2 << 30) + (1 << 20)
    zero = torch.zeros(1024, 1024, device="cuda")
    for i in (0, 99, 100, 127, 128, 199):
        want, bound, _, _ = _want_step(zero, g[i], zero, 1.0, weight_decay=0.0)
        _assert_near(p[i], want, bound, f"matrix {i}")


@gpu
@pytest.mark.parametrize("shapes", [[(1500, 1300), (4096, 4096)], [(64, 64), (64, 96), (4096, 4096)]])
def test_muon_step_without_memory_leaves_everything_as_it_was(muons, shapes):
    """Room for the first shape's workspace and not for the last one's: nothing of the call is carried out."""
    _, muon_step = muons
    p, g, m = ([torch.full(s, v, device="cuda", dtype=t) for s in shapes] for v, t in ((1.0, BF16), (2.0, BF16), (0.0, F32)))
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (150 << 20)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            muon_step(p, g, m, lr=0.1)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert all((t == 1.0).all() for t in p) and not any(t.any() for t in m)
    muon_step(p, g, m, lr=0.1)
    assert all(t.any() for t in m)


# ------------------------------------------------------------- waits that run out --

def test_lost_waits_without_a_device():
    from isa_b200 import _lib
    lib = _lib.load()
    assert lib.cimekv_lost_waits(0) == 0 and lib.cimekv_lost_waits(1) == 0
    for kind, ms in ((2, 1.0), (-1, 1.0), (0, 0.0), (0, -1.0), (0, 2000.0), (0, float("nan"))):
        assert lib.cimekv_debug_lose_wait(kind, ms, None) == 1


@gpu
@pytest.mark.parametrize("kind", [0, 1])
def test_a_wait_that_runs_out_is_told(norms, muons, kind):
    """A wait for an arrival that never comes, given up after a millisecond: the next call fails, whichever it is, writes
    nothing, and the one after it runs."""
    from isa_b200 import _lib
    lib = _lib.load()
    (layer_norm, add_layer_norm), (orthogonalize, muon_step) = norms, muons
    x = torch.randn(6, 32, device="cuda")
    leaf, p, m = x.clone().requires_grad_(True), torch.ones_like(x), torch.zeros_like(x)
    y = layer_norm(leaf)
    calls = [lambda: layer_norm(x), lambda: add_layer_norm(x, x), lambda: orthogonalize(x), lambda: muon_step([p], [x], [m], lr=0.1),
             lambda: torch.autograd.grad(y.sum(), leaf, retain_graph=True)]
    for call in calls:
        assert lib.cimekv_debug_lose_wait(kind, 1.0, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert lib.cimekv_lost_waits(0) == 1 << kind
        with pytest.raises(RuntimeError, match="status 5.*ran out"):
            call()
        assert lib.cimekv_lost_waits(0) == 0 and (p == 1).all() and not m.any()
        if call is not calls[3]:
            call()
    assert lib.cimekv_debug_lose_wait(kind, 1.0, None) == 0
    torch.cuda.synchronize()
    assert lib.cimekv_lost_waits(1) == 1 << kind  # read and cleared
    muon_step([p], [x], [m], lr=0.1)
    torch.cuda.synchronize()
    assert lib.cimekv_lost_waits(0) == 0 and torch.isfinite(p).all()


@gpu
def test_first_call_of_a_process_inside_a_capture():
    """What the library sets up at its first call is no part of the capture."""
    import subprocess
    import sys
    from pathlib import Path
    code = f"""
import sys
sys.path.insert(0, {str(Path(__file__).resolve().parent.parent / 'isa-_b200')!r})
import torch
from isa_b200.kernels.muon import cuda_orthogonalize
from isa_b200.kernels.transformer_norm import cuda_layer_norm
x = torch.randn(64, 128, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, o = cuda_layer_norm(x), cuda_orthogonalize(x)
for t in (y, o):
    t.fill_(float("nan"))
graph.replay()
print(torch.equal(y, cuda_layer_norm(x)), torch.equal(o, cuda_orthogonalize(x)))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.split() == ["True", "True"], (r.stdout, r.stderr[-2000:])


# --------------------------------------------------------------------- precision --

@gpu
@pytest.mark.parametrize("shape", [(1, 1100, 1100), (48, 384, 384), (10, 768, 768), (1500, 900)])
def test_fp32_parameters_of_large_matrices_get_the_precision_of_fp32_results(muons, shape):
    """From zeros, with lr s = 1, no decay and no momentum, a step leaves exactly -NS(g): the bits of cuda_orthogonalize
    (the one kernel of small matrices sums more coarsely for a step)."""
    orthogonalize, muon_step = muons
    g = torch.randn(shape, device="cuda")
    p, m = torch.zeros_like(g), torch.zeros_like(g)
    scale = max(1.0, shape[-2] / shape[-1]) ** 0.5
    muon_step([p], [g], [m], lr=1.0 / scale, momentum=0.0, weight_decay=0.0)
    if scale == 1.0:
        assert torch.equal(p, -orthogonalize(g))
    else:  # lr s is 1 but for its roundings
        assert float((p + orthogonalize(g)).abs().max()) <= 4 * 2.0 ** -24 * float(p.abs().max())


def _products_in_fp32(g):
    """Five steps on g[..., rows, cols] in the type of g, by its own products."""
    tall = g.shape[-2] > g.shape[-1]
    x = g.mT if tall else g
    x = x / x.double().norm(dim=(-2, -1), keepdim=True).to(x.dtype)
    for _ in range(5):
        a = x @ x.mT
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    return x.mT if tall else x


@gpu
@pytest.mark.parametrize("rows,cols", [(96, 96), (161, 161), (176, 176), (192, 192), (222, 200), (223, 223)])
def test_fp32_results_below_the_crossing_are_no_further_off_than_fp32_products(muons, rows, cols):
    """Decaying spectra, whose small directions show what rounds: the completed square leaves these sizes 1.13 to 1.33 times
    as far off as products in fp32, the polynomial as it stands 0.70 to 0.87 times."""
    from tests.test_muon import _update
    orthogonalize, _ = muons
    assert not torch.backends.cuda.matmul.allow_tf32
    g = _update("cuda", 6, rows, cols, seed=11)
    want = _products_in_fp32(g.double())
    off = lambda t: float((t.double() - want).norm())  # noqa: E731
    assert off(orthogonalize(g)) <= off(_products_in_fp32(g))


# -------------------------------------------------------------------- in the models --

@gpu
@pytest.mark.parametrize("fused", [False, True])
def test_hooks_and_wrappers_of_blocks_and_norms_run(fused):
    """Hooks on every module, and a block's forward replaced by a checkpointed one, with and without fused norms."""
    import torch.nn as nn
    from torch.utils.checkpoint import checkpoint
    from isa_b200.language import GPT2Model, ModelConfig
    torch.manual_seed(0)
    cfg = ModelConfig.from_preset("tiny", "standard", vocab_size=61, max_seq_len=24, fused_norm=fused)
    cfg.depth = 2
    model = GPT2Model(cfg).cuda()
    ids = torch.randint(0, 61, (2, 24), device="cuda")
    plain = model(ids)
    want = torch.autograd.grad(plain.square().mean(), list(model.parameters()))
    seen = {"pre": set(), "out": set(), "back": set()}
    names = [f"blocks.{i}{k}" for i in range(2) for k in ("", ".ln1", ".ln2")] + ["ln_f"]
    for name in names:
        module = model.get_submodule(name)
        module.register_forward_pre_hook(lambda m, args, name=name: seen["pre"].add(name))
        module.register_forward_hook(lambda m, args, out, name=name: seen["out"].add(name))
        module.register_full_backward_hook(lambda m, gi, go, name=name: seen["back"].add(name))
    entered = []
    for i, blk in enumerate(model.blocks):
        def wrapped(*args, own=blk.forward, i=i):
            entered.append(i)
            return checkpoint(own, *args, use_reentrant=False)
        blk.forward = wrapped
    logits = model(ids)
    assert torch.equal(logits, plain) and entered == [0, 1]
    got = torch.autograd.grad(logits.square().mean(), list(model.parameters()))
    for a, b in zip(got, want):  # the same sums, where torch's own gradients add in any order: 2^-24 of many terms
        assert float((a - b).norm()) <= 1e-5 * float(b.norm())
    assert all(seen[k] == set(names) for k in ("pre", "out"))
    assert seen["back"] >= {f"blocks.{i}" for i in range(2)} | {"ln_f"}


@gpu
def test_hooks_of_the_vit_norms_run():
    from isa_b200.harness.vit import PhysicalViT, ViTConfig
    model = PhysicalViT(ViTConfig(img_size=16, patch_size=8, num_classes=5, embed_dim=48, num_heads=3, depth=1, fused_norm=True)).cuda()
    seen = []
    for name in ("blocks.0.norm1", "blocks.0.norm2", "norm"):
        model.get_submodule(name).register_forward_hook(lambda m, args, out, name=name: seen.append(name))
    model(torch.randn(2, 3, 16, 16, device="cuda"))
    assert seen == ["blocks.0.norm1", "blocks.0.norm2", "norm"]


# --------------------------------------------------------------------------- building --

def test_the_library_needs_nvcc_alone(monkeypatch, tmp_path, capsys):
    """Without torch, without g++ or unasked for the binding is left out and the library built all the same; the binding
    of another torch is not taken for this one's."""
    from isa_b200 import _lib, build
    here = build.binding_path()
    assert here.exists() and torch.__version__ in here.name
    calls = []
    monkeypatch.setattr(build, "build_binding", lambda force=False: calls.append(force))
    build.build_library(binding=False)
    build.build_library(debug=True)
    assert not calls
    build.build_library()
    assert len(calls) == 1
    with monkeypatch.context() as m:
        m.setattr(build.shutil, "which", lambda name: None if name == "g++" else "/usr/bin/" + name)
        assert build.build_library() == build.LIB_PATH
        assert "g++ not found" in capsys.readouterr().err
        m.setattr(build.importlib.util, "find_spec", lambda name: None)
        assert build.build_library() == build.LIB_PATH
        assert "torch and g++ not found" in capsys.readouterr().err
    assert len(calls) == 1
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "1.0.0+none")
        m.setattr(_lib, "_binding", None)
        assert build.binding_path() != here
        with pytest.raises(RuntimeError, match="no tensor binding for this torch"):
            _lib.binding()


# ---------------------------------------------------------------------------- layouts --

@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,cols", [(700, 100), (300, 256), (90, 1000), (41, 4000), (11, 16000), (9, 16384)])
def test_16_bit_rows_that_no_vector_fits(norms, rows, cols, dtype):
    """Rows from any element of a buffer, any distance apart, in input, branch and both gradients; the row before and behind
    them is full of NaN."""
    from tests.test_layer_norm import _assert_near, _plain
    layer_norm, add_layer_norm = norms
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)

    def rows_at(offset, apart):
        buf = torch.full((rows + 2, cols + apart), float("nan"), device="cuda", dtype=dtype).view(-1)
        t = buf[cols + apart + offset:][:rows * (cols + apart)].view(rows, cols + apart)[:, :cols]
        t.copy_(torch.randn(rows, cols, device="cuda", generator=gen))
        return t

    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=gen)).to(dtype).requires_grad_(True)
    b = (0.2 * torch.randn(cols, device="cuda", generator=gen)).to(dtype).requires_grad_(True)
    for places in ([(1, 1)] * 4, [(0, 1), (1, 3), (2, 5), (3, 0)], [(3, 0), (5, 0), (7, 0), (1, 0)], [(4, 4), (0, 8), (4, 12), (0, 4)]):
        x, d, dy, dh = (rows_at(*at) for at in places)
        x, d = x.requires_grad_(True), d.requires_grad_(True)
        want = _plain(x.detach(), d.detach(), w.detach(), b.detach(), 1e-5, dy, dh)
        y, h = add_layer_norm(x, d, w, b)
        assert torch.equal(h.double(), want["h"][0])
        got = torch.autograd.grad((y, h), (x, d, w, b), (dy, dh))
        for t, k in zip((y, *got), ("y", "dx", "dx", "dw", "db")):
            _assert_near(t.detach(), *want[k], f"{k} {places}")
        want = _plain(x.detach(), None, w.detach(), None, 1e-5, dy, None)
        y = layer_norm(x, w)
        for t, k in zip((y, *torch.autograd.grad(y, (x, w), dy)), ("y", "dx", "dw")):
            _assert_near(t.detach(), *want[k], f"{k} alone {places}")


@gpu
def test_matrices_beyond_32_bits(muons):
    """2.7e9 elements in one call: the last matrices equal those of a call of their own."""
    orthogonalize, muon_step = muons
    g = torch.empty(40, 8192, 8192, device="cuda", dtype=BF16).normal_()
    out = orthogonalize(g, steps=1)
    assert torch.equal(out[-2:], orthogonalize(g[-2:], steps=1)) and torch.equal(out[:2], orthogonalize(g[:2], steps=1))
    p = out  # as parameters
    m = torch.zeros(40, 8192, 8192, device="cuda")
    small = p[-2:].clone(), m[-2:].clone()
    muon_step([p], [g], [m], lr=0.1, steps=1)
    muon_step([small[0]], [g[-2:]], [small[1]], lr=0.1, steps=1)
    assert torch.equal(p[-2:], small[0]) and torch.equal(m[-2:], small[1])


@gpu
@pytest.mark.parametrize("x_t,d_t,y_t", [(F32, F32, F32), (F32, BF16, BF16), (BF16, BF16, F32), (F16, F16, F16)])
def test_rows_that_just_fill_48_kb(x_t, d_t, y_t):
    """Widths whose rows take all of the 48 KB of shared memory that a kernel has without asking, but for what its own
    variables need: in a process of its own, where no wider row has asked before."""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    widths = [108, 172, 216, 228, 344, 364, 492, 588, 728, 736, 748, 984, 996, 1204, 1496, 1504, 1516, 2008, 2020, 3032, 3052, 6104]
    code = f"""
import sys
sys.path[:0] = [{str(root / 'isa-_b200')!r}, {str(root)!r}]
import torch
from tests.test_layer_norm import _assert_near, _case, _plain, _run_and_check
from isa_b200.kernels.transformer_norm import cuda_add_layer_norm, cuda_layer_norm
dev = torch.device("cuda")
for cols in {widths}:
    for d_t in (None, {d_t}):
        _run_and_check(*_case(dev, 9, cols, {x_t}, d_t, {x_t}, {y_t}), {y_t})
    buf = torch.randn(9 * cols + 1, device=dev).to({x_t})[1:].view(9, cols)  # rows that no vector fits
    y, h = cuda_add_layer_norm(buf, buf)
    _assert_near(y, *_plain(buf, buf, None, None, 1e-5, None, None)["y"], "y")
    _assert_near(cuda_layer_norm(buf), *_plain(buf, None, None, None, 1e-5, None, None)["y"], "y")
    w = torch.ones(cols, device=dev, requires_grad=True)
    dy = torch.randn(9 * cols + 1, device=dev)[1:].view(9, cols)
    gw, = torch.autograd.grad(cuda_layer_norm(buf, w, None, 1e-5, torch.float32), w, dy)
    _assert_near(gw, *_plain(buf, None, w.detach(), None, 1e-5, dy, None)["dw"], "dw")
print("all")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["all"], (r.stdout, r.stderr[-2000:])


@gpu
def test_calls_from_several_threads_at_once(muons):
    """Kernels whose CTAs wait for one another, from streams of different priority, with others between them: the same bits
    as alone, and no wait runs out."""
    import threading
    from isa_b200 import _lib
    orthogonalize, muon_step = muons
    wrong = []

    def run(seed, shapes, priority):
        stream = torch.cuda.Stream(priority=priority)
        with torch.cuda.stream(stream):
            gen = torch.Generator(device="cuda").manual_seed(seed)
            g = [torch.randn(s, device="cuda", generator=gen) for s in shapes]

            def call():
                if len(g) == 1:
                    return [orthogonalize(g[0])]
                p, m = [torch.zeros_like(t) for t in g], [torch.zeros_like(t) for t in g]
                muon_step(p, g, m, lr=1.0, weight_decay=0.0)
                return p

            want = call()
            stream.synchronize()
            for _ in range(20):
                got = [call() for _ in range(10)]
                stream.synchronize()
                if not all(torch.equal(a, b) for out in got for a, b in zip(out, want)):
                    wrong.append((shapes, priority))

    threads = [threading.Thread(target=run, args=args) for args in
               ((0, [(40, 192, 192)], 0), (1, [(768, 768)], -2), (2, [(30, 192, 192), (8, 192, 768)], -1), (3, [(6, 640, 640)], 0))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong and _lib.load().cimekv_lost_waits(0) == 0

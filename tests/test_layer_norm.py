"""Layer norm and residual layer norm: kernels against the formulas in 64 bits.

Bounds.  u = 2^-24 is the rounding of fp32, eta_t half a step of type t.  A
row's mean is a sum of at most N = 32 terms in a thread, 5 shuffles, 16 warps and
a product: off by n u mean|h| with n = 55.  The centred value adds its own
rounding, and the variance, a sum of squares of the same shape whose first-order
dependence on the mean cancels, is off by n u relative plus the square of the
mean's error over it.  So u_hat = (h - mean) rstd is off by

    du = rstd n u mean|h| + |u_hat| (n/2 + 6) u + |u_hat| (rstd n u mean|h|)^2

(rsqrtf: 2 ulp), y by |w| du + 4 u (|y| + |b|) + eta |y|; the gradients follow by
the product rule, with sums of n terms over columns and of n + rows terms over rows.
"""

import pytest
import torch

U = 2.0 ** -24
N = 55
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _eta(t, dtype):
    """Half a step of ``dtype`` at the values of ``t`` (its smallest step below the normal range)."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.smallest_normal * info.eps


def _plain(x, delta, w, b, eps, dy, dh):
    """y, h, dx, dw, db and their bounds (without the last rounding) in 64 bits."""
    h = x.double() if delta is None else (x.double() + delta.double()).to(x.dtype).double()
    rows, c = h.shape
    one, zero = torch.ones(c, dtype=torch.float64, device=h.device), torch.zeros(c, dtype=torch.float64, device=h.device)
    w = one if w is None else w.double()
    b = zero if b is None else b.double()
    mean = h.mean(1, keepdim=True)
    rstd = ((h - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    u = (h - mean) * rstd
    y = u * w + b
    off = rstd * N * U * h.abs().mean(1, keepdim=True)
    du = off + u.abs() * ((N / 2 + 6) * U + off.square())
    out = {"y": (y, w.abs() * du + 4 * U * (y.abs() + b.abs())), "h": (h, None)}
    if dy is None:
        return out
    g = dy.double()
    gw = g * w
    c1, c2 = gw.mean(1, keepdim=True), (gw * u).mean(1, keepdim=True)
    dx = rstd * (gw - c1 - u * c2)
    d1 = (N + 2) * U * gw.abs().mean(1, keepdim=True)
    d2 = (N + 2) * U * (gw * u).abs().mean(1, keepdim=True) + (gw.abs() * du).mean(1, keepdim=True)
    size = gw.abs() + c1.abs() + (u * c2).abs()
    ddx = rstd * (d1 + u.abs() * d2 + du * c2.abs() + 6 * U * size) + dx.abs() * (N / 2 + 6) * U \
        + rstd * size * off.square()
    if dh is not None:
        dx = dx + dh.double()
        ddx = ddx + U * dx.abs()
    out["dx"] = (dx, ddx)
    k = (N + rows) * U
    out["dw"] = ((g * u).sum(0), (g.abs() * du).sum(0) + k * (g * u).abs().sum(0))
    out["db"] = (g.sum(0), k * g.abs().sum(0))
    return out


def _assert_near(got, want, bound, what):
    assert got.shape == want.shape, what
    tol = _eta(want, got.dtype) * (1 + 2 ** -6) + bound
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max())} of the bound"


def _ops():
    from isa_b200.kernels.transformer_norm import cuda_add_layer_norm, cuda_layer_norm
    return cuda_layer_norm, cuda_add_layer_norm


# ------------------------------------------------------------- CPU: refusals --

def test_refuses_cpu_tensors():
    from isa_b200 import build
    build.build_library()
    layer_norm, add_layer_norm = _ops()
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        add_layer_norm(x, x)


def test_c_entry_refusals_before_any_launch():
    import ctypes
    from isa_b200 import _lib, build
    build.build_library()
    lib = _lib.load()
    p = ctypes.c_void_p(256)
    fwd = lambda rows, cols, x_type=0, x=p, h=None, delta=None, eps=1e-5: lib.cimekv_layer_norm_forward(  # noqa: E731
        x, x_type, cols, delta, 0, cols, None, None, 0, rows, cols, eps, h, p, 0, None, None, None)
    assert fwd(-1, 8) == 1 and b"negative" in lib.cimekv_last_error()
    assert fwd(4, 0) == 1 and b"columns" in lib.cimekv_last_error()
    assert fwd(4, 16385) == 1 and b"columns" in lib.cimekv_last_error()
    assert fwd(4, 8, x_type=7) == 1 and b"type" in lib.cimekv_last_error()
    assert fwd(4, 8, x=None) == 1 and b"null" in lib.cimekv_last_error()
    assert fwd(4, 8, delta=p) == 1  # a branch without a place for the sum
    assert fwd(4, 8, eps=-1.0) == 1 and fwd(4, 8, eps=float("nan")) == 1
    assert fwd(0, 8) == 0  # nothing to do
    bwd = lambda rows, cols, dy=p: lib.cimekv_layer_norm_backward(  # noqa: E731
        dy, 0, cols, None, 0, p, 0, cols, None, 0, p, p, rows, cols, p, None, 0, None, None, None, 0, None)
    assert bwd(-1, 8) == 1 and bwd(4, 0) == 1 and bwd(4, 8, dy=None) == 1
    assert lib.cimekv_layer_norm_workspace_bytes(0, 8) == 0
    assert lib.cimekv_layer_norm_workspace_bytes(8, 16385) == 0


# --------------------------------------------------------------------- GPU ---

gpu = pytest.mark.gpu


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from isa_b200 import build
    build.build_library()
    return torch.device("cuda")


def _case(dev, rows, cols, x_t, d_t, w_t, y_t, seed=0, offset=0.0):
    gen = torch.Generator(device=dev).manual_seed(seed + rows * 7 + cols)
    r = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    x = (r(rows, cols) * 2 + offset + r(cols)).to(x_t).requires_grad_(True)
    d = None if d_t is None else r(rows, cols).to(d_t).requires_grad_(True)
    w = None if w_t is None else (1 + 0.3 * r(cols)).to(w_t).requires_grad_(True)
    b = None if w_t is None else (0.2 * r(cols)).to(w_t).requires_grad_(True)
    return x, d, w, b, r(rows, cols).to(y_t), None if d is None else r(rows, cols).to(x_t)


def _run_and_check(x, d, w, b, dy, dh, y_t, eps=1e-5):
    layer_norm, add_layer_norm = _ops()
    want = _plain(x.detach(), None if d is None else d.detach(), None if w is None else w.detach(),
                  None if b is None else b.detach(), eps, dy, dh)
    if d is None:
        y, h = layer_norm(x, w, b, eps, out_dtype=y_t), None
    else:
        y, h = add_layer_norm(x, d, w, b, eps, out_dtype=y_t)
        assert h.dtype == x.dtype and torch.equal(h.double(), want["h"][0])
    assert y.dtype == y_t
    _assert_near(y.detach(), *want["y"], "y")
    leaves = [t for t in (x, d, w, b) if t is not None]
    outs, grads = ((y,), (dy,)) if d is None else ((y, h), (dy, dh))
    got = dict(zip([k for k, t in (("dx", x), ("dd", d), ("dw", w), ("db", b)) if t is not None],
                   torch.autograd.grad(outs, leaves, grads)))
    for k, t in (("dx", x), ("dd", d), ("dw", w), ("db", b)):
        if t is not None:
            assert got[k].dtype == t.dtype and got[k].shape == t.shape
            _assert_near(got[k], *want["dx" if k == "dd" else k], k)
    return y, h, got


WIDTHS = [1, 2, 3, 16, 31, 33, 128, 132, 192, 257, 384, 500, 512, 516, 768, 1000, 1023, 1024, 1028, 1537, 2048, 2052,
          4095, 4096, 4100, 8192, 8196, 16383, 16384]


@gpu
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("add", [False, True])
def test_widths_fp32(dev, cols, add):
    _run_and_check(*_case(dev, 37, cols, F32, F32 if add else None, F32, F32), F32)


@gpu
@pytest.mark.parametrize("x_t,d_t,w_t,y_t", [
    (F32, None, F32, BF16), (F32, None, F32, F16), (BF16, None, BF16, BF16), (BF16, None, F32, F32),
    (F16, None, F16, F16), (F16, None, F32, F32), (F32, BF16, F32, F32), (F32, BF16, F32, BF16),
    (F32, F16, F32, F16), (F32, F32, BF16, F32), (BF16, BF16, BF16, BF16), (BF16, BF16, F32, F32),
    (F16, F16, F16, F16), (F16, F16, F32, F32), (F32, None, None, F32), (BF16, BF16, None, BF16)])
@pytest.mark.parametrize("rows,cols", [(65, 192), (9, 257), (33, 1028), (5, 5001)])
def test_types(dev, rows, cols, x_t, d_t, w_t, y_t):
    _run_and_check(*_case(dev, rows, cols, x_t, d_t, w_t, y_t, seed=1), y_t)


@gpu
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 1183, 1185, 9000])
@pytest.mark.parametrize("cols", [96, 97, 1536])
def test_row_counts(dev, rows, cols):
    _run_and_check(*_case(dev, rows, cols, F32, BF16, F32, F32, seed=2), F32)


@gpu
def test_rows_far_from_zero(dev):
    """A mean 4096 times the width: the centred squares do not cancel."""
    _run_and_check(*_case(dev, 64, 768, F32, None, F32, F32, offset=8192.0), F32)


@gpu
def test_only_one_of_weight_and_bias(dev):
    layer_norm, _ = _ops()
    x, _, w, b, dy, _ = _case(dev, 20, 200, F32, None, F32, F32)
    for ww, bb in ((w, None), (None, b)):
        want = _plain(x.detach(), None, None if ww is None else ww.detach(), None if bb is None else bb.detach(), 1e-5, dy, None)
        y = layer_norm(x, ww, bb)
        _assert_near(y.detach(), *want["y"], "y")
        gx, gp = torch.autograd.grad(y, (x, w if bb is None else b), dy)
        _assert_near(gx, *want["dx"], "dx")
        _assert_near(gp, *want["dw" if bb is None else "db"], "dw or db")


@gpu
def test_no_rows(dev):
    layer_norm, add_layer_norm = _ops()
    x = torch.empty(0, 5, 24, device=dev, requires_grad=True)
    w = torch.ones(24, device=dev, requires_grad=True)
    b = torch.zeros(24, device=dev, requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape and not w.grad.any() and not b.grad.any()
    y, h = add_layer_norm(x, x.detach(), w, b)
    assert y.shape == h.shape == x.shape


@gpu
def test_layouts(dev):
    """Class-token slices, strided and misaligned rows, a transposed matrix, repeated rows."""
    layer_norm, add_layer_norm = _ops()
    base = torch.randn(6, 17, 132, device=dev)
    odd = torch.randn(20 * 129 + 1, device=dev)
    views = [base[:, 0], base[:, 3:9], base[..., 4:100], base[..., 1:130], odd[1:].view(20, 129)[:, :128],
             base[0].t(), base[0, :1].expand(40, 132), base[0, :, ::2]]
    for v in views:
        x = v.detach()
        cols = x.shape[-1]
        w, b = torch.randn(cols, device=dev), torch.randn(cols, device=dev)
        want = _plain(x.reshape(-1, cols), None, w, b, 1e-5, None, None)["y"]
        _assert_near(layer_norm(x, w, b).reshape(-1, cols), *want, "y")
        y, h = add_layer_norm(x, x, w, b)
        want = _plain(x.reshape(-1, cols), x.reshape(-1, cols), w, b, 1e-5, None, None)
        assert torch.equal(h, x + x)
        _assert_near(y.reshape(-1, cols), *want["y"], "y")
    # gradients that arrive expanded or transposed, an input that is a strided view
    leaf = torch.randn(30, 2, 64, device=dev, requires_grad=True)
    w = torch.randn(64, device=dev, requires_grad=True)
    for dy in (torch.randn(64, device=dev).expand(30, 64), torch.randn(64, 30, device=dev).t(),
               torch.randn(30, 1, device=dev).expand(30, 64)):
        want = _plain(leaf.detach()[:, 1], None, w.detach(), None, 1e-5, dy, None)
        gl, gw = torch.autograd.grad(layer_norm(leaf[:, 1], w), (leaf, w), dy)
        _assert_near(gl[:, 1], *want["dx"], "dx")
        assert not gl[:, 0].any()
        _assert_near(gw, *want["dw"], "dw")


@gpu
def test_special_rows_stay_their_own(dev):
    """Constant, zero, infinite and NaN rows: defined results, and no other row is touched."""
    layer_norm, add_layer_norm = _ops()
    for cols in (64, 65, 2048):
        x = torch.randn(12, cols, device=dev)
        clean = layer_norm(x)
        bad = x.clone()
        bad[1], bad[2] = 0.0, 3.0
        bad[4, 5], bad[7, 3], bad[8, 0] = float("inf"), float("nan"), -float("inf")
        w, b = torch.randn(cols, device=dev), torch.randn(cols, device=dev)
        y = layer_norm(bad)
        keep = [0, 3, 5, 6, 9, 10, 11]
        assert torch.equal(y[keep], clean[keep])
        assert not y[1].any() and not y[2].any()  # a constant row is its own mean
        assert torch.equal(layer_norm(bad, w, b)[1], b)
        for r in (4, 7, 8):
            assert y[r].isnan().all()
        y2, h = add_layer_norm(bad, torch.zeros_like(bad))
        assert torch.equal(y2[keep], clean[keep]) and torch.equal(h[keep], x[keep])
    # a constant row without eps: 0 * inf where its sum rounds to 48 times the value, else +-1 ulp (1e23) with squares
    # that overflow, so rstd = 0 and the row is 0; nothing else is possible
    assert not layer_norm(torch.full((2, 48), 1e30, device=dev), eps=0.0).nan_to_num().any()
    big = torch.randn(3, 48, device=dev, dtype=F16) * 0 + 60000.0
    y, h = add_layer_norm(big, big)  # the fp16 sum overflows as a torch sum does
    assert h.isinf().all() and y.isnan().all()


@gpu
def test_partial_gradients(dev):
    """Each subset of gradients that a caller may want, and only one of the two outputs used."""
    _, add_layer_norm = _ops()
    x, d, w, b, dy, dh = _case(dev, 19, 192, F32, BF16, F32, F32, seed=3)
    full = torch.autograd.grad(add_layer_norm(x, d, w, b), (x, d, w, b), (dy, dh))
    for k, t in enumerate((x, d, w, b)):
        args = [v if i == k else v.detach() for i, v in enumerate((x, d, w, b))]
        got, = torch.autograd.grad(add_layer_norm(*args), t, (dy, dh))
        assert torch.equal(got, full[k])
    only_y = torch.autograd.grad(add_layer_norm(x, d, w, b)[0], (x, d, w, b), dy)
    zero_h = torch.autograd.grad(add_layer_norm(x, d, w, b), (x, d, w, b), (dy, torch.zeros_like(dh)))
    assert all(torch.equal(p, q) for p, q in zip(only_y, zero_h))
    gx, gd, gw, gb = torch.autograd.grad(add_layer_norm(x, d, w, b)[1], (x, d, w, b), dh, allow_unused=True)
    assert torch.equal(gx, dh) and torch.equal(gd, dh.to(BF16)) and not gw.any() and not gb.any()


@gpu
def test_one_tensor_as_stream_and_branch(dev):
    _, add_layer_norm = _ops()
    x = torch.randn(10, 96, device=dev, requires_grad=True)
    dy, dh = torch.randn(10, 96, device=dev), torch.randn(10, 96, device=dev)
    g, = torch.autograd.grad(add_layer_norm(x, x), x, (dy, dh))
    want = _plain(x.detach(), x.detach(), None, None, 1e-5, dy, dh)["dx"]
    _assert_near(g, 2 * want[0], 2 * want[1] + 2 * _eta(want[0], F32), "dx")


@gpu
def test_gradient_against_differences(dev):
    """Directional derivatives of the 64-bit formula: step 1e-4, error O(step^2) of its third derivative and
    2^-53 / step; the kernel's own bound on top."""
    x, _, w, b, dy, _ = _case(dev, 11, 320, F32, None, F32, F32, seed=4)
    layer_norm, _ = _ops()
    grads = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    want = _plain(x.detach(), None, w.detach(), b.detach(), 1e-5, dy, None)
    f = lambda *a: float((torch.nn.functional.layer_norm(a[0], (320,), a[1], a[2], 1e-5) * dy.double()).sum())  # noqa: E731
    args = [t.detach().double() for t in (x, w, b)]
    for k, name in enumerate(("dx", "dw", "db")):
        v = torch.randn_like(args[k])
        step = 1e-4
        plus, minus = ([a + s * step * v if i == k else a for i, a in enumerate(args)] for s in (1, -1))
        slope = (f(*plus) - f(*minus)) / (2 * step)
        got = float((grads[k].double() * v).sum())
        size = float((want[name][0] * v).abs().sum())
        # third derivative: a row's unit vector turns by at most step |v| rstd, so step^2 of the size covers it 10 times over
        tol = float(((want[name][1] + _eta(want[name][0], F32)) * v.abs()).sum()) + 10 * step ** 2 * size + 1e-9 * size
        assert abs(got - slope) <= tol, (name, got, slope, tol)


@gpu
def test_same_bits_every_time(dev):
    _, add_layer_norm = _ops()
    x, d, w, b, dy, dh = _case(dev, 5000, 384, F32, BF16, F32, F32, seed=5)
    first = None
    for _ in range(3):
        y, h = add_layer_norm(x, d, w, b)
        got = [y, h, *torch.autograd.grad((y, h), (x, d, w, b), (dy, dh))]
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(first, got))


@gpu
def test_other_stream_and_graph(dev):
    layer_norm, _ = _ops()
    x, _, w, b, dy, _ = _case(dev, 300, 768, F32, None, F32, F32, seed=6)

    def step():
        y = layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graphs = []
    for _ in range(2):  # two graphs of the same call, replayed alternately
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    with torch.no_grad():
        x.copy_(x.flip(0) * 0.5)
    want = step()
    for g, out in graphs * 2:
        for t in out:
            t.fill_(float("nan"))
        g.replay()
        assert all(torch.equal(p, q) for p, q in zip(want, out))


@gpu
def test_offsets_beyond_32_bits(dev):
    """2.3e9 elements: rows do not depend on one another, so the last ones equal a small call's."""
    layer_norm, add_layer_norm = _ops()
    x = torch.empty(140000, 16384, device=dev, dtype=BF16).normal_()
    w = torch.rand(16384, device=dev, dtype=BF16).requires_grad_(True)
    leaf = x.requires_grad_(True)
    y = layer_norm(leaf, w)
    tail = x.detach()[-5:].clone().requires_grad_(True)
    small = layer_norm(tail, w)
    assert torch.equal(y[-5:], small) and torch.equal(y[:5], layer_norm(x.detach()[:5].clone(), w))
    dy = torch.zeros((), device=dev, dtype=BF16).expand_as(x).clone()
    dy[-5:] = 1.0
    gx, gw = torch.autograd.grad(y, (leaf, w), dy)
    sx, sw = torch.autograd.grad(small, (tail, w), torch.ones_like(small))
    assert torch.equal(gx[-5:], sx) and not gx[:-5].any()
    _assert_near(gw, sw.double(), _eta(sw.double(), BF16) * 2, "dw")  # either sum rounded to bf16 once


@gpu
def test_no_memory_is_kept(dev):
    """Outputs that are dropped without a backward free everything, a saved output among it."""
    _, add_layer_norm = _ops()
    x, d, w, b, dy, dh = _case(dev, 500, 256, F32, BF16, F32, F32, seed=7)
    add_layer_norm(x, d, w, b)
    before = torch.cuda.memory_allocated()
    for _ in range(3):
        add_layer_norm(x, d, w, b)
        y, h = add_layer_norm(x, d, w, b)
        torch.autograd.grad((y, h), (x, d), (dy, dh))
    del y, h
    assert torch.cuda.memory_allocated() == before


@gpu
@pytest.mark.parametrize("how", ["backward", "grad", "other", "released"])
def test_capture_while_an_eager_graph_lives(dev, how):
    """In a process of its own: a capture that would reach the default stream raises, and the process goes on."""
    import subprocess
    import sys
    from pathlib import Path
    code = f"""
import sys
sys.path.insert(0, {str(Path(__file__).resolve().parent.parent / 'isa-_b200')!r})
import torch
from isa_b200.kernels.transformer_norm import cuda_layer_norm
how = {how!r}
x, w = torch.randn(64, 128, device="cuda"), torch.ones(128, device="cuda", requires_grad=True)
v = torch.ones(128, device="cuda", requires_grad=True)
eager = cuda_layer_norm(x, w)
if how == "released":
    eager.sum().backward()
    del eager
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        y = cuda_layer_norm(x, w, v)
        if how == "grad":
            torch.autograd.grad(y.sum(), w)
        elif how == "other":  # only a leaf that no eager graph holds
            out, = torch.autograd.grad(y.sum(), v)
        else:
            y.sum().backward()
    graph.replay()
    print("captured")
except RuntimeError as e:
    print("refused" if "eager graph" in str(e) else e)
torch.cuda.synchronize()
print("alive", float((x * 0 + 1).sum()))
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    want = "captured" if how in ("other", "released") else "refused"
    assert r.returncode == 0 and r.stdout.split() == [want, "alive", "8192.0"], (r.stdout, r.stderr[-2000:])


@gpu
def test_changes_behind_its_back_are_noticed(dev):
    layer_norm, add_layer_norm = _ops()
    x, w = torch.randn(4, 32, device=dev, requires_grad=True), torch.ones(32, device=dev, requires_grad=True)
    for change in ("w", "h"):
        y, h = add_layer_norm(x, x.detach(), w)
        with torch.no_grad():
            (w if change == "w" else h).mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), x)


@gpu
def test_gpu_refusals(dev):
    layer_norm, add_layer_norm = _ops()
    x = torch.zeros(4, 32, device=dev)
    with pytest.raises(RuntimeError, match="weight must be on the device"):
        layer_norm(x, torch.ones(32))
    with pytest.raises(RuntimeError, match="shape"):
        layer_norm(x, torch.ones(16, device=dev))
    with pytest.raises(RuntimeError, match="one type"):
        layer_norm(x, torch.ones(32, device=dev), torch.ones(32, device=dev, dtype=BF16))
    with pytest.raises(RuntimeError, match="float32, bfloat16"):
        layer_norm(x.double())
    with pytest.raises(RuntimeError, match="out_dtype"):
        layer_norm(x.half(), out_dtype=BF16)
    with pytest.raises(RuntimeError, match="columns"):
        layer_norm(torch.zeros(2, 16385, device=dev))
    with pytest.raises(RuntimeError, match="columns"):
        layer_norm(torch.zeros(2, 0, device=dev))
    with pytest.raises(RuntimeError, match="eps"):
        layer_norm(x, eps=-1e-5)
    with pytest.raises(RuntimeError, match="shape of x"):
        add_layer_norm(x, x[:1])
    with pytest.raises(RuntimeError, match="not available"):
        add_layer_norm(x.bfloat16(), x)
    with pytest.raises(RuntimeError, match="device"):
        add_layer_norm(x, x.cpu())


@gpu
def test_double_backward_refused(dev):
    layer_norm, _ = _ops()
    x = torch.randn(4, 32, device=dev, requires_grad=True)
    g, = torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1001, 384), (333, 768), (1, 384), (700, 4096), (40, 16384), (500, 257)])
def test_weight_gradients_alone_of_strided_rows(dev, rows, cols, dtype, add):
    """Rows one to seven elements further apart than they are wide, in the input and in the gradient that arrives, and
    no gradient of the input: nothing of the call begins every row at the same place of a vector."""
    layer_norm, add_layer_norm = _ops()
    gen = torch.Generator(device=dev).manual_seed(rows + cols)
    for apart in (1, 2, 4, 7):
        wide = lambda: torch.randn(rows, cols + apart, device=dev, generator=gen).to(dtype)[:, :cols]  # noqa: E731
        x, d, dy, dh = wide(), wide(), wide(), wide()
        w = (1 + 0.3 * torch.randn(cols, device=dev, generator=gen)).to(dtype).requires_grad_(True)
        b = torch.zeros(cols, device=dev, dtype=dtype, requires_grad=True)
        want = _plain(x, d if add else None, w.detach(), b.detach(), 1e-5, dy, dh if add else None)
        if add:
            gw, gb = torch.autograd.grad(add_layer_norm(x, d, w, b), (w, b), (dy, dh))
        else:
            gw, gb = torch.autograd.grad(layer_norm(x, w, b), (w, b), dy)
        _assert_near(gw, *want["dw"], f"dw, {apart} apart")
        _assert_near(gb, *want["db"], f"db, {apart} apart")
        gw, = torch.autograd.grad(layer_norm(x, w), w, dy)
        _assert_near(gw, *_plain(x, None, w.detach(), None, 1e-5, dy, None)["dw"], f"dw alone, {apart} apart")

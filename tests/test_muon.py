"""Newton-Schulz orthogonalisation and the Muon step against their definitions in 64 bits.

Bound.  u = 2^-24.  An operand held as two fp16 planes is off by 2^-22 of its value (half a step of 11 bits, twice);
a product of two drops lo x lo, another 2^-22 of |L| |R|.  A step of the tensor core (16 products) cuts the products
and the sum so far off below 2^-25 of the largest: 17 / 2 u.  Of such steps with terms at full size an accumulator takes
at most 4 for fp32 results and 16 otherwise, and the accumulators are added in fp32, K / 64 of them at most:
e = 3 * 2^-22 + (34 or 136 + K / 64) u of |L| |R|, whose norm is at most |L|_F |R|_F.  With A = X X^T, P = a I + b A + c A^2
(computed as c B^2 + ..., B = A + b / 2c I, so |B| <= max(|b / 2c|, |A + b / 2c|)) one step X' = P X adds

    dA = e |X|_F^2 + 2^-22 |B|_F,  dP = |c| (2 |B|_2 dA + e |B|_F^2) + 2^-22 |P|_F  (c = 0: dP = |b| dA + 2^-22 |P|_F),
    d  = dP |X|_2 + e |P|_F |X|_F + 2^-22 |X'|_F

fp32 results of at most 160 rows form P as it stands: S = A in place of B where it is stored and multiplied (not in |B|_2, the derivative of P
by A is c (B dA + dA B) either way), and four roundings of its sum, 4 u (|c| |A|_F^2 + |b| |A|_F).  For others S = B:

    dA = e |X|_F^2 + 2^-22 |S|_F,  dP = |c| (2 |B|_2 dA + e |S|_F^2) + 2^-22 |P|_F

and an error before a step is multiplied by at most L = max(|p'(s)|, |p(s) / s|) over the singular values there.
"""

import array
import ctypes
import math

import pytest
import torch

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NS = (3.4445, -4.7750, 2.0315)
CUBIC = (1.5, -0.5, 0.0)


def _ops():
    from isa_b200.kernels.muon import cuda_muon_step, cuda_orthogonalize
    return cuda_orthogonalize, cuda_muon_step


def _exact(g, steps=5, coefficients=NS, eps=1e-7, fine=None):
    """(result, bound on the Frobenius norm of the error) of one matrix, in 64 bits."""
    a, b, c = coefficients
    fine = g.dtype == F32 if fine is None else fine
    cut = 34 if fine else 136
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / max(float(x.norm()), eps)
    m, n = x.shape
    eye = torch.eye(m, dtype=torch.float64, device=x.device)
    err = 2 * 2.0 ** -22 * float(x.norm())
    for _ in range(steps):
        A = x @ x.T
        P = a * eye + b * A + c * (A @ A)
        new = P @ x
        s = torch.linspace(0, 1, 257, dtype=torch.float64) * float(torch.linalg.matrix_norm(x, 2))
        lip = float(torch.maximum((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs(), (a + b * s ** 2 + c * s ** 4).abs()).max())
        e = lambda k: 3 * 2.0 ** -22 + (cut + k / 64) * U  # noqa: E731
        B = A + (0.5 * b / c if c else 0.0) * eye
        fro, two = (lambda t: float(t.norm())), (lambda t: float(torch.linalg.matrix_norm(t, 2)))  # noqa: E731
        S = A if fine and m <= 160 else B
        dA = e(n) * fro(x) ** 2 + 2.0 ** -22 * fro(S)
        dP = (abs(c) * (2 * two(B) * dA + e(m) * fro(S) ** 2) if c else abs(b) * dA) + 2.0 ** -22 * fro(P)
        if fine and m <= 160 and c:
            dP += 4 * U * (abs(c) * fro(A) ** 2 + abs(b) * fro(A))
        err = lip * err + dP * two(x) + e(m) * fro(P) * fro(x) + 2.0 ** -22 * fro(new)
        x = new
    return (x.T if tall else x), err


def _assert_near(got, want, bound, what):
    """Frobenius norm; the result's own rounding is half a step of its type, element by element."""
    info = torch.finfo(got.dtype)
    rounding = float((want.abs() * (info.eps / 2) + info.smallest_normal * info.eps).norm())
    err = float((got.double() - want).norm())
    assert err <= bound + rounding, f"{what}: off by {err}, bound {bound} + {rounding} (norm {float(want.norm())})"


def _update(dev, *shape, seed=0, dtype=F32, scale=1e-3):
    """A decaying spectrum over a floor of noise."""
    gen = torch.Generator(device=dev).manual_seed(seed + sum(shape))
    *batch, m, n = shape
    r = max(1, min(m, n, 16))
    w = 2.0 ** -torch.arange(r, device=dev, dtype=F32).div(3.0)
    low = (torch.randn(*batch, m, r, device=dev, generator=gen) * w) @ torch.randn(*batch, r, n, device=dev, generator=gen)
    return ((low + 0.3 * torch.randn(*shape, device=dev, generator=gen)) * scale).to(dtype)


# ------------------------------------------------------------- CPU: refusals --

def test_refuses_cpu_tensors():
    from isa_b200 import build
    build.build_library()
    orthogonalize, muon_step = _ops()
    g = torch.ones(4, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        orthogonalize(g)
    with pytest.raises(RuntimeError, match="CUDA"):
        muon_step([g], [g], [g], lr=0.1)
    with pytest.raises(ValueError, match="adjust_lr"):
        muon_step([], [], [], lr=0.1, adjust_lr="other")
    with pytest.raises(RuntimeError, match="as many"):
        muon_step([g], [], [g], lr=0.1)
    muon_step([], [], [], lr=0.1)


def test_c_entry_refusals_before_any_launch():
    import ctypes
    from isa_b200 import _lib, build
    build.build_library()
    lib = _lib.load()
    p = ctypes.c_void_p(256)

    def orth(batch=1, rows=8, cols=8, steps=5, c=NS, eps=1e-7, type_=0, g=p, ws=p, ws_bytes=1 << 40):
        return lib.cimekv_orthogonalize(g, type_, 64, 8, batch, rows, cols, steps, *c, eps, p, ws, ws_bytes, None)

    err = lambda: lib.cimekv_last_error()  # noqa: E731
    assert orth(batch=-1) == 1 and b"negative" in err()
    assert orth(rows=32769) == 1 and orth(cols=32769) == 1 and orth(batch=65536) == 1
    assert orth(batch=65535, rows=32768, cols=32768) == 1 and b"too many" in err()
    assert orth(steps=0) == 1 and orth(steps=65) == 1 and b"steps" in err()
    assert orth(eps=0.0) == 1 and orth(eps=float("nan")) == 1
    assert orth(eps=1e-38) == 1 and b"at least 1e-30" in err()
    assert orth(c=(float("nan"), 0.0, 0.0)) == 1 and b"finite" in err()
    assert orth(c=(8.0, 0.0, 0.0)) == 1 and b"beyond 3.9" in err()  # grows without bound
    assert orth(c=(1.5, -0.5, 1e-4)) == 1 and b"beyond 15" in err()  # b / 2c does not fit
    assert orth(type_=3) == 1 and b"type" in err()
    assert orth(g=None) == 1 and b"null" in err()
    assert orth(ws=None) == 4 and orth(ws_bytes=64) == 4
    assert orth(ws=ctypes.c_void_p(264)) == 1 and b"aligned" in err()
    for empty in (dict(batch=0), dict(rows=0), dict(cols=0)):
        assert orth(**empty) == 0
    assert lib.cimekv_orthogonalize_workspace_bytes(0, 8, 8) == 0
    assert lib.cimekv_orthogonalize_workspace_bytes(1, 40000, 8) == 0

    def step(ps, gs, ms, momentum=0.95, rows=4, cols=4, count=None):
        t = lambda v: (ctypes.c_void_p * len(v))(*v)  # noqa: E731
        return lib.cimekv_muon_step(len(ps) if count is None else count, t(ps), t(gs), t(ms), 0, 0, rows, cols, 0.1, None,
                                    momentum, 1, 0.0, 1.0, 5, *NS, 1e-7, p, 1 << 40, None)

    assert step([4096], [8192], [None]) == 1 and b"null" in err()
    assert step([4096], [8192], [4096]) == 1 and b"overlap" in err()
    assert step([4096, 4096], [8192, 8192], [16384, 32768]) == 1 and b"overlap" in err()
    assert step([4096, 4096 + 32], [8192, 8192], [16384, 32768]) == 1 and b"overlap" in err()
    assert step([4096], [8192], [16384], momentum=1.5) == 1 and b"momentum" in err()
    assert step([4096] * 200, [8192] * 200, [16384] * 200) == 1 and b"too many" in err()


# --------------------------------------------------------------------- GPU ---

gpu = pytest.mark.gpu


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from isa_b200 import build
    build.build_library()
    return torch.device("cuda")


SHAPES = [(1, 1), (1, 7), (7, 1), (5, 5), (16, 16), (33, 40), (64, 64), (65, 63), (127, 130), (128, 128), (129, 129),
          (192, 192), (192, 768), (768, 192), (200, 1000), (257, 1001), (256, 256), (300, 257), (384, 384), (513, 520),
          (640, 640), (1000, 40), (1100, 1300)]


@gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_orthogonalize_shapes(dev, shape, dtype):
    orthogonalize, _ = _ops()
    g = _update(dev, *shape, dtype=dtype)
    got = orthogonalize(g)
    assert got.shape == g.shape and got.dtype == dtype
    _assert_near(got, *_exact(g), f"{shape} {dtype}")


@gpu
@pytest.mark.parametrize("shape", [(64, 130, 600), (64, 600, 130), (150, 150, 150), (100, 160, 161), (100, 161, 161), (3, 160, 160)])
@pytest.mark.parametrize("c", [NS, CUBIC])
def test_both_forms_of_the_polynomial(dev, shape, c):
    """fp32 results on both sides of 160 rows, from the kernels of single products and from the one of all steps."""
    orthogonalize, _ = _ops()
    g = _update(dev, *shape, seed=3)
    got = orthogonalize(g, coefficients=c)
    assert torch.equal(orthogonalize(g, coefficients=c), got)
    for k in (0, shape[0] // 2, shape[0] - 1):
        _assert_near(got[k], *_exact(g[k], coefficients=c), f"{shape} {k}")
    assert torch.isfinite(got).all()


@gpu
@pytest.mark.parametrize("shape", [(2, 100, 30), (3, 128, 128), (50, 64, 64), (200, 48, 72), (2, 2, 90, 33), (20, 256, 320),
                                   (9, 384, 384), (40, 192, 192)])
def test_batches(dev, shape):
    orthogonalize, _ = _ops()
    g = _update(dev, *shape, seed=1)
    got = orthogonalize(g).reshape(-1, *shape[-2:])
    flat = g.reshape(-1, *shape[-2:])
    for i in range(0, flat.shape[0], max(1, flat.shape[0] // 7)):
        _assert_near(got[i], *_exact(flat[i]), f"matrix {i}")


@gpu
@pytest.mark.parametrize("shape", [(1500, 1500), (2048, 1024)])
def test_large(dev, shape):
    orthogonalize, _ = _ops()
    g = _update(dev, *shape, seed=2)
    _assert_near(orthogonalize(g), *_exact(g), f"{shape}")


@gpu
@pytest.mark.parametrize("steps,coefficients", [(1, NS), (2, NS), (3, NS), (8, NS), (5, CUBIC), (10, CUBIC), (1, CUBIC),
                                                (5, (1.875, -1.25, 0.375)), (3, (2.0, -1.5, 0.5)), (2, (1.0, 0.0, 0.0))])
@pytest.mark.parametrize("shape", [(96, 160), (300, 300)])
def test_steps_and_coefficients(dev, shape, steps, coefficients):
    orthogonalize, _ = _ops()
    g = _update(dev, *shape, seed=3)
    _assert_near(orthogonalize(g, steps=steps, coefficients=coefficients), *_exact(g, steps, coefficients), "result")


@gpu
def test_singular_values_and_vectors(dev):
    """What it is for: singular values between 0.65 and 1.25, the vectors kept (the product with G is symmetric)."""
    orthogonalize, _ = _ops()
    g = torch.randn(256, 320, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    o = orthogonalize(g).double()
    s = torch.linalg.svdvals(o)
    assert 0.65 < float(s.min()) and float(s.max()) < 1.25
    cross = o @ g.double().T
    assert float((cross - cross.T).norm()) <= 1e-4 * float(cross.norm())


@gpu
@pytest.mark.parametrize("n", [40, 200])
def test_special_matrices(dev, n):
    orthogonalize, _ = _ops()
    g = _update(dev, 6, n, n, seed=5)
    clean = orthogonalize(g)
    g[1] = 0.0
    g[2, 3, 4] = float("nan")
    g[3, 0, 1] = float("inf")
    g[4] *= 1e30   # squares beyond fp32
    g[5] *= 1e-28  # squares below it; the norm is under eps
    got = orthogonalize(g)
    assert torch.equal(got[0], clean[0])
    assert not got[1].any()
    assert got[2].isnan().all() and got[3].isnan().all()
    for i in (4, 5):
        want, bound = _exact(g[i])
        # below eps the values reach 1e-21 of the planes' scale: what 2^-37 (the planes' smallest step) leaves
        _assert_near(got[i], want, bound + 2.0 ** -37 * n * 4.0 ** 5, f"matrix {i}")
    assert float((got[4] - clean[4]).abs().max()) < 1e-3


@gpu
def test_layouts(dev):
    orthogonalize, _ = _ops()
    base = _update(dev, 4, 90, 140, seed=6)
    odd = torch.randn(50 * 70 + 1, device=dev)[1:].view(50, 70)
    views = [base[:, :, 3:131], base[:, 5:60], base.transpose(1, 2), base[::2], base[1], base[0].t(), base[:1].expand(3, 90, 140),
             odd, base[:, :, ::2], base.half()[:, :, 1:66]]
    for v in views:
        got = orthogonalize(v)
        assert got.shape == v.shape and got.is_contiguous()
        assert torch.equal(got, orthogonalize(v.contiguous().clone()))
        flat, o = v.reshape(-1, *v.shape[-2:]), got.reshape(-1, *v.shape[-2:])
        _assert_near(o[-1], *_exact(flat[-1]), "view")


@gpu
def test_empty(dev):
    orthogonalize, muon_step = _ops()
    for shape in [(0, 4, 4), (3, 0, 4), (4, 0), (0, 0)]:
        assert orthogonalize(torch.empty(shape, device=dev)).shape == shape
    e = torch.empty(0, 8, device=dev)
    muon_step([e], [e], [e], lr=0.1)


@gpu
@pytest.mark.parametrize("shape", [(3, 150, 150), (1, 700, 900)])
def test_same_bits_streams_and_graphs(dev, shape):
    orthogonalize, _ = _ops()
    g = _update(dev, *shape, seed=7)
    want = orthogonalize(g)
    for _ in range(3):
        assert torch.equal(orthogonalize(g), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [orthogonalize(g) for _ in range(4)]
    here = [orthogonalize(g) for _ in range(4)]  # at the same time as the other stream's
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got + here)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = orthogonalize(g)
        graphs.append((graph, out))
    g.copy_(g.flip(1) * 3)
    want = orthogonalize(g)
    for graph, out in graphs * 2:
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, want)


@gpu
def test_gpu_refusals(dev):
    orthogonalize, muon_step = _ops()
    g = torch.randn(8, 8, device=dev)
    with pytest.raises(RuntimeError, match="two axes"):
        orthogonalize(g[0])
    with pytest.raises(RuntimeError, match="float32, bfloat16"):
        orthogonalize(g.double())
    with pytest.raises(RuntimeError, match="sides of at most"):
        orthogonalize(torch.empty(1, 32769, device=dev))
    with pytest.raises(RuntimeError, match="beyond 3.9"):
        orthogonalize(g, coefficients=(5.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="steps"):
        orthogonalize(g, steps=0)
    m = torch.zeros_like(g)
    with pytest.raises(RuntimeError, match="shape mismatch"):
        muon_step([g], [g[:4]], [m], lr=0.1)
    with pytest.raises(RuntimeError, match="momentum must be float32"):
        muon_step([g], [g], [m.half()], lr=0.1)
    with pytest.raises(RuntimeError, match="contiguous"):
        muon_step([g.t()], [g], [m], lr=0.1)
    with pytest.raises(RuntimeError, match="one device"):
        muon_step([g], [g.cpu()], [m], lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        muon_step([g, g], [g, g], [m, torch.zeros_like(m)], lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        muon_step([g], [m], [g], lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        muon_step([g], [m], [m], lr=0.1)  # a gradient that is its own momentum
    with pytest.raises(RuntimeError, match="overlap"):
        muon_step([torch.ones(4, 4, device=dev), g], [torch.ones(4, 4, device=dev), g], [torch.zeros(4, 4, device=dev), m], lr=0.1)
    p = torch.ones(4, 4, device=dev)
    with pytest.raises(RuntimeError, match="overlap"):  # nothing of a refused call is carried out
        muon_step([p, g, g], [torch.ones_like(p), torch.ones_like(g), torch.ones_like(g)],
                  [torch.zeros_like(p), m, torch.zeros_like(g)], lr=0.1)
    assert (p == 1).all()
    muon_step([p, g], [torch.ones(4, 4, device=dev).expand(4, 4)] + [torch.ones_like(g)], [torch.zeros_like(p), m], lr=0.1)
    both = torch.ones(4, 4, device=dev)
    muon_step([p, torch.ones_like(p)], [both, both], [torch.zeros_like(p), torch.zeros_like(p)], lr=0.1)  # one gradient twice
    with pytest.raises(RuntimeError, match="one-element"):
        muon_step([g], [m], [m], lr=torch.zeros(2, device=dev))
    with pytest.raises(RuntimeError, match="momentum must be"):
        muon_step([g], [torch.ones_like(g)], [m], lr=0.1, momentum=-0.5)


# ---------------------------------------------------------------------- step --

def _want_step(p, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0.1, match_rms=False):
    """(parameter, its bound, momentum, its bound) of one matrix."""
    g, m0 = g.double(), m.double()
    new = momentum * m0 + (1 - momentum) * g
    # three roundings of the momentum, and its parameters' own in fp32
    dm = 4 * U * (m0.abs() + g.abs())
    u = momentum * new + (1 - momentum) * g if nesterov else new
    o, bound = _exact(u, fine=False)
    rows, cols = p.shape
    s = 0.2 * math.sqrt(max(rows, cols)) if match_rms else math.sqrt(max(1.0, rows / cols))
    # the update's rounding (4 u of |m| + |g|) enters like the planes' rounding, times the steps' growth a^5
    bound += 8 * U * float((m0.abs() + g.abs()).norm()) / max(float(u.norm()), 1e-7) * 3.4445 ** 5
    want = p.double() * (1 - lr * weight_decay) - lr * s * o
    rounding = 4 * U * (p.double().abs() + lr * s * o.abs())
    return want, lr * s * bound + float(rounding.norm()), new, dm


def _matrices(t):
    return t.reshape(-1, *t.shape[-2:])


@gpu
@pytest.mark.parametrize("options", [dict(), dict(nesterov=False), dict(weight_decay=0.0), dict(momentum=0.0),
                                     dict(adjust_lr="match_rms_adamw")])
@pytest.mark.parametrize("p_type,g_type", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32)])
def test_muon_step(dev, options, p_type, g_type):
    """Shapes of several kinds in one call: projections, fused projections as three matrices, tall, wide, odd."""
    _, muon_step = _ops()
    shapes = [(64, 64), (3, 64, 64), (64, 192), (192, 64), (64, 64), (37, 55), (130, 129)]
    gen = torch.Generator(device=dev).manual_seed(8)
    params = [(0.05 * torch.randn(*s, device=dev, generator=gen)).to(p_type) for s in shapes]
    grads = [_update(dev, *s, seed=9 + i).to(g_type) for i, s in enumerate(shapes)]
    momenta = [_update(dev, *s, seed=20 + i) for i, s in enumerate(shapes)]
    plain = {k: v for k, v in options.items() if k != "adjust_lr"}
    want = [[_want_step(*t, 0.02, match_rms="adjust_lr" in options, **plain)
             for t in zip(_matrices(p), _matrices(g), _matrices(m))] for p, g, m in zip(params, grads, momenta)]
    before = [g.clone() for g in grads]
    versions = [t._version for t in params + momenta]
    muon_step(params, grads, momenta, lr=0.02, **options)
    assert all(torch.equal(a, b) for a, b in zip(before, grads))
    assert all(t._version > v for t, v in zip(params + momenta, versions))
    for p, m, ws in zip(params, momenta, want):
        for pi, mi, (wp, bound, wm, dm) in zip(_matrices(p), _matrices(m), ws):
            _assert_near(pi, wp, bound, "parameter")
            assert ((mi.double() - wm).abs() <= dm + 1e-30).all()


@gpu
def test_muon_many_matrices(dev):
    """More matrices than one call of the library takes: the second part reuses the workspace."""
    _, muon_step = _ops()
    params = [torch.zeros(100, 24, 24, device=dev) for _ in range(3)]
    grads = [_update(dev, 100, 24, 24, seed=i) for i in range(3)]
    momenta = [torch.zeros_like(p) for p in params]
    muon_step(params, grads, momenta, lr=1.0, weight_decay=0.0)
    for i, k in ((0, 0), (1, 27), (1, 28), (2, 55), (2, 56), (2, 99)):
        want, bound, _, _ = _want_step(torch.zeros(24, 24, device=dev), grads[i][k], torch.zeros(24, 24, device=dev), 1.0,
                                       weight_decay=0.0)
        _assert_near(params[i][k], want, bound, f"{i} {k}")


def test_muon_shares():
    """How steps of several shapes share the SMs (no GPU: their number is given)."""
    from isa_b200 import _lib
    lib = _lib.load()

    def shares(*groups, sms=148, c=2.0):
        counts, rows, cols = (array.array("i", v) for v in zip(*groups))
        out = array.array("i", [-1] * len(groups))
        at = lambda a: a.buffer_info()[0]  # noqa: E731
        assert lib.cimekv_muon_shares(len(groups), at(counts), at(rows), at(cols), c, sms, at(out)) == 0
        return list(out)

    for c in (0.0, 2.0):
        for groups in ([(40, 192, 192), (10, 192, 768)], [(1, 64, 64), (1, 64, 65), (1, 65, 64)], [(3, 200, 100)] * 4):
            got = shares(*groups, c=c)
            assert all(s >= 2 for s in got) and sum(got) <= 148, got
    big = [(48, 768, 768), (1, 4096, 4096)]
    assert shares(*big) == [0, 0]  # each fills the chip
    got = shares(*big, (1, 64, 64), (1, 64, 256))
    assert got[:2] == [0, 0] and all(s >= 2 for s in got[2:])
    assert shares((5, 64, 64)) == [0]
    assert shares((0, 64, 64), (5, 0, 64), (5, 64, 64)) == [0, 0, 0]
    assert shares((1, 64, 64), (1, 64, 65), sms=3) == [0, 0]
    many = shares(*[(1, 32, 32 + i) for i in range(40)])
    assert sum(many) <= 148 and sum(s > 0 for s in many) == 16
    assert lib.cimekv_muon_shares(1, None, None, None, 2.0, 148, None) == 1
    one, bad = array.array("i", [1]), array.array("i", [40000])
    a, b = one.buffer_info()[0], bad.buffer_info()[0]
    assert lib.cimekv_muon_shares(1, a, b, a, 2.0, 148, a) == 1 and lib.cimekv_muon_shares(1, a, a, a, 2.0, -1, a) == 1
    assert lib.cimekv_muon_shares(0, None, None, None, 2.0, 148, None) == 0
    t = (ctypes.c_void_p * 1)(256)
    for share in (1, -1):
        assert lib.cimekv_muon_step_on(share, 1, t, t, t, 0, 0, 8, 8, 0.1, None, 0.9, 1, 0.0, 1.0, 5, *NS, 1e-7, 256,
                                       1 << 40, None) == 1
        assert b"share" in lib.cimekv_last_error()


SEVERAL = [(6, 192, 192), (3, 192, 768), (2, 100, 37), (1, 300, 300), (2, 33, 500)]


@gpu
@pytest.mark.parametrize("c", [NS, CUBIC])
def test_muon_several_shapes_side_by_side(dev, c):
    """Small matrices of several shapes, a large one among them, in one call: on another stream and from two graphs too."""
    _, muon_step = _ops()
    shapes = SEVERAL + [(1, 1500, 1300)]
    p0 = [torch.randn(s, device=dev) for s in shapes]
    m0 = [_update(dev, *s, seed=i) for i, s in enumerate(shapes)]
    g = [_update(dev, *s, seed=50 + i) for i, s in enumerate(shapes)]
    g[2] = g[2].transpose(1, 2).contiguous().transpose(1, 2)  # copied first

    def call(p, m):
        muon_step(p, g, m, lr=0.02, coefficients=c, weight_decay=0.1)

    def fresh():
        return [t.clone() for t in p0], [t.clone() for t in m0]

    p, m = fresh()
    call(p, m)
    if c == NS:
        for i, s in enumerate(shapes):
            for k in range(s[0]):
                want_p, bound_p, want_m, bound_m = _want_step(p0[i][k], g[i][k], m0[i][k], 0.02)
                _assert_near(p[i][k], want_p, bound_p, f"{s} {k}")
    side = torch.cuda.Stream()
    sets = [fresh() for _ in range(6)]
    torch.cuda.synchronize()
    for k, (q, n) in enumerate(sets):  # on two streams at the same time; workspaces are freed and taken again
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
            call(q, n)
    torch.cuda.synchronize()
    for q, n in sets:
        assert all(map(torch.equal, q, p)) and all(map(torch.equal, n, m))
    graphs = []
    for q, n in sets[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(q, n)
        graphs.append(graph)
    for round_ in range(2):
        for (q, n), graph in zip(sets, graphs):
            for t, u in zip(q + n, p0 + m0):
                t.copy_(u)
            graph.replay()
        for q, n in sets[:2]:
            assert all(map(torch.equal, q, p)) and all(map(torch.equal, n, m))


@gpu
def test_muon_several_shapes_during_another_capture(dev):
    """Calls outside a capture that goes on meanwhile stay out of it, whichever of torch's streams it has taken."""
    _, muon_step = _ops()
    shapes = SEVERAL[:2]
    g = [_update(dev, *s, seed=i) for i, s in enumerate(shapes)]

    def fresh():
        return [torch.ones(s, device=dev) for s in shapes], [torch.zeros(s, device=dev) for s in shapes]

    want = fresh()
    muon_step(want[0], g, want[1], lr=0.02)
    inside, outside = fresh(), [fresh() for _ in range(40)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, capture_error_mode="relaxed"):
        muon_step(inside[0], g, inside[1], lr=0.02)
        for _ in range(8):  # a stream of ours that the capture has not taken
            other = torch.cuda.Stream()
            with torch.cuda.stream(other):
                if not torch.cuda.is_current_stream_capturing():
                    break
        with torch.cuda.stream(other):
            for p, m in outside:
                muon_step(p, g, m, lr=0.02)
    torch.cuda.synchronize()
    for p, m in outside:
        assert all(map(torch.equal, p, want[0])) and all(map(torch.equal, m, want[1]))
    assert not any(m.any() for m in inside[1])
    graph.replay()
    torch.cuda.synchronize()
    assert all(map(torch.equal, inside[0], want[0])) and all(map(torch.equal, inside[1], want[1]))


@gpu
def test_muon_learning_rate_on_the_device_and_graph(dev):
    _, muon_step = _ops()
    p0, g, m0 = torch.randn(96, 80, device=dev), _update(dev, 96, 80), _update(dev, 96, 80, seed=1)
    lr = torch.tensor([0.03], device=dev)
    p, m = p0.clone(), m0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step([p], [g], [m], lr=lr)
    p.copy_(p0)
    m.copy_(m0)
    want_p, want_m = p0.clone(), m0.clone()
    for rate in (0.03, 0.01, 0.0):
        lr.fill_(rate)
        graph.replay()
        muon_step([want_p], [g], [want_m], lr=float(lr))
        assert torch.equal(p, want_p) and torch.equal(m, want_m)


@gpu
def test_muon_leaves_neighbours_alone(dev):
    """Matrices inside larger buffers: what lies around them keeps its values."""
    _, muon_step = _ops()
    for rows, cols in ((50, 70), (70, 50), (64, 64), (129, 131)):
        n = rows * cols
        buf = torch.full((2, 3 * n), 7.0, device=dev)
        p, m = buf[0, n:2 * n].view(rows, cols), buf[1, n:2 * n].view(rows, cols)
        p.copy_(torch.randn(rows, cols, device=dev))
        m.zero_()
        muon_step([p], [_update(dev, rows, cols)], [m], lr=0.1)
        assert (buf[:, :n] == 7.0).all() and (buf[:, 2 * n:] == 7.0).all()
        assert torch.isfinite(p).all() and m.any()

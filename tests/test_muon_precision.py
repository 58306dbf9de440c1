"""Newton-Schulz results and Muon's parameters held against what products in fp32 give.

The bounds of tests/test_muon.py hold for any input and are far above the errors of these.  Here the same iteration in
fp32 products is the measure: an operand of two fp16 planes is off by 2^-22 of its value where an fp32 one is by 2^-24, so
an error may be four times theirs, element by element (of the largest) and in norm.  Where fp32 happens to be exact (a
number, a few rows) the roundings themselves remain: three products a step for five steps and the first planes, 16 of
2^-22.  The result's own rounding, half a step of its type, is added.  On the CPU the same criterion refuses an iteration
with one plane, one without the cross products, and results with a tile missing.
"""

import math

import pytest
import torch

from tests.test_muon import SHAPES, _update

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NS = (3.4445, -4.7750, 2.0315)
gpu = pytest.mark.gpu


def _iterate(g, product=torch.matmul, hold=lambda t: t, steps=5):
    """The iteration on g[..., rows, cols] in the type of g, with its products and what it holds in between given."""
    a, b, c = NS
    tall = g.shape[-2] > g.shape[-1]
    x = g.mT if tall else g
    x = hold(x / x.double().norm(dim=(-2, -1), keepdim=True).clamp_min(1e-7).to(x.dtype))
    eye = torch.eye(x.shape[-2], dtype=x.dtype, device=x.device)
    for _ in range(steps):
        gram = hold(product(x, x.mT))
        x = hold(product(hold(a * eye + b * gram + c * product(gram, gram)), x))
    return x.mT if tall else x


def _excess(got, want, fp32, extra=0.0):
    """Largest of: error over tolerance element by element, and in norm.  extra: further roundings of an element."""
    info = torch.finfo(got.dtype)
    rounding = want.abs() * (info.eps / 2) * (1 + 2.0 ** -6) + info.smallest_normal * info.eps + extra
    floor = 16 * 2.0 ** -22
    err, theirs = (got.double() - want).abs(), (fp32.double() - want).abs()
    one = err / (rounding + max(4 * float(theirs.max()), floor * float(want.abs().max())))
    norm = float(err.norm()) / (float(rounding.norm()) + max(4 * float(theirs.norm()), floor * float(want.norm())))
    worst = max(float(one.max()), norm)
    return worst if math.isfinite(worst) else math.inf


def _check(got, g, what):
    want = _iterate(g.double())
    worst = _excess(got, want, _iterate(g.float()))
    assert worst <= 1.0, f"{what}: {worst} of the tolerance"


# ----------------------------------------------------- CPU: what the criterion sees --

def _planes(t, count):
    """t as `count` fp16 planes of 2^12 t hold it."""
    hi = (t * 4096).half()
    lo = (t * 4096 - hi.double()).half()
    return (hi.double() + (lo.double() if count == 2 else 0.0)) / 4096


def _two_planes(x, y):
    """hi hi + hi lo + lo hi."""
    xh, yh = _planes(x, 1), _planes(y, 1)
    return x @ y - (x - xh) @ (y - yh)


@pytest.mark.parametrize("shape", [(5, 5), (33, 40), (192, 192), (300, 257), (640, 640), (1100, 1300)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_criterion_refuses_what_it_should(shape, dtype):
    g = _update("cpu", *shape, dtype=dtype)
    want, fp32 = _iterate(g.double()), _iterate(g.float())
    good = _iterate(g.double(), _two_planes, lambda t: _planes(t, 2))
    assert _excess(good.to(dtype), want, fp32) <= 1.0
    assert _excess(fp32.to(dtype), want, fp32) <= 1.0
    one_plane = _iterate(g.double(), hold=lambda t: _planes(t, 1))
    assert _excess(one_plane.to(dtype), want, fp32) > 1.0
    no_cross = _iterate(g.double(), lambda x, y: _planes(x, 1) @ _planes(y, 1), lambda t: _planes(t, 2))
    assert _excess(no_cross.to(dtype), want, fp32) > 1.0
    for side in (16, 64, 128):  # a tile that was not written, in the middle and at the ragged end
        for r, c in ((0, 0), (shape[0] // side * side, shape[1] // side * side)):
            if r < shape[0] and c < shape[1]:
                hole = good.clone()
                hole[r:r + side, c:c + side] = 0.0
                assert _excess(hole.to(dtype), want, fp32) > 1.0
    assert _excess(good.to(dtype) * float("nan"), want, fp32) > 1.0


# ---------------------------------------------------------------------------- GPU --

@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from isa_b200 import build
    build.build_library()
    assert not torch.backends.cuda.matmul.allow_tf32
    return torch.device("cuda")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES + [(223, 223), (224, 224), (1500, 1500), (2048, 1024), (4096, 1100)])
def test_orthogonalize(dev, shape, dtype):
    from isa_b200.kernels.muon import cuda_orthogonalize
    for g in (_update(dev, *shape, dtype=dtype), torch.randn(shape, device=dev).to(dtype)):
        _check(cuda_orthogonalize(g), g, f"{shape} {dtype}")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 100, 30), (50, 64, 64), (200, 48, 72), (40, 192, 192), (20, 256, 320), (9, 384, 384),
                                   (48, 768, 768), (64, 130, 600), (100, 161, 161), (100, 230, 230), (6, 1100, 900)])
def test_batches(dev, shape, dtype):
    """Every matrix of a batch."""
    from isa_b200.kernels.muon import cuda_orthogonalize
    g = _update(dev, *shape, seed=1, dtype=dtype)
    got, want, fp32 = cuda_orthogonalize(g), _iterate(g.double()), _iterate(g.float())
    worst = max(_excess(*t) for t in zip(got, want, fp32))
    assert worst <= 1.0, f"{shape}: {worst} of the tolerance"


def _step(p, g, m, dtype, lr, momentum, nesterov, weight_decay):
    """Parameter and orthogonalised update, with arithmetic in `dtype`."""
    p, g, m = p.to(dtype), g.to(dtype), m.to(dtype)
    m = momentum * m + (1 - momentum) * g
    u = momentum * m + (1 - momentum) * g if nesterov else m
    o = math.sqrt(max(1.0, p.shape[-2] / p.shape[-1])) * _iterate(u)
    return p * (1 - lr * weight_decay) - lr * o


@gpu
@pytest.mark.parametrize("options", [dict(momentum=0.95, nesterov=True, weight_decay=0.1),
                                     dict(momentum=0.9, nesterov=False, weight_decay=0.0)])
@pytest.mark.parametrize("p_type,g_type", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32)])
def test_muon_parameters(dev, options, p_type, g_type):
    """Several shapes in one call, from parameters of ordinary size and from zeros (where all that is left is the update),
    each matrix on its own.  Beside the result's rounding an fp32 parameter takes three of its sum, 2^-24 each."""
    from isa_b200.kernels.muon import cuda_muon_step
    for shapes in ([(64, 64), (3, 64, 64), (64, 192), (192, 64), (37, 55), (130, 129)], [(40, 192, 192), (10, 192, 768)],
                   [(12, 768, 768), (300, 1200), (1500, 700)]):
        for size, lr in ((0.05, 0.02), (0.0, 1.0)):
            gen = torch.Generator(device=dev).manual_seed(8)
            params = [(size * torch.randn(*s, device=dev, generator=gen)).to(p_type) for s in shapes]
            grads = [_update(dev, *s, seed=9 + i).to(g_type) for i, s in enumerate(shapes)]
            momenta = [_update(dev, *s, seed=20 + i) for i, s in enumerate(shapes)]
            want, fp32 = ([_step(*t, dtype, lr, **options) for t in zip(params, grads, momenta)] for dtype in (torch.float64, F32))
            start = [p.clone() for p in params]
            cuda_muon_step(params, grads, momenta, lr=lr, **options)
            for s, p0, p, w, f in zip(shapes, start, params, want, fp32):
                flat = lambda t: t.reshape(-1, *s[-2:])  # noqa: E731
                worst = max(_excess(a, b, c, 3 * U * (d.double().abs() + b.abs()))
                            for a, b, c, d in zip(flat(p), flat(w), flat(f), flat(p0)))
                assert worst <= 1.0, f"{s} from {size}: {worst} of the tolerance"

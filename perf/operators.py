"""Cases of the digital operators around the CIM layers: layer normalisation
(alone and joined with the residual sum) with its backward pass, the
Newton-Schulz orthogonalisation of an update matrix, and the optimiser step
that uses it.

``run`` computes a case in its plain form (``own`` false: elementary torch
operations in 32 bits, rounded once at the end) or through the package's entry
points (``own`` true).  ``exact`` computes it in 64 bits from the definitions.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5
# Coefficients and number of the Newton-Schulz steps, and the floor of the norm.
_NS = (3.4445, -4.7750, 2.0315)
_STEPS = 5
_NORM_FLOOR = 1e-7
_LR, _MOMENTUM, _DECAY = 0.02, 0.95, 0.1


def listed():
    return [
        # Final norm of the last tokens of a few sequences in evaluation (tiny GPT preset): launch latency counts.
        dict(name="norm_eval_tail", op="norm", rows=8, cols=192, x="fp32", y="fp32", w="fp32", train=False),
        # ln1 of one block of the mid GPT preset, 32 sequences of 1024 tokens shifted by one, fp32 residual stream.
        dict(name="norm_gpt_mid", op="norm", rows=32736, cols=384, x="fp32", y="fp32", w="fp32", train=True),
        # norm1 of a ViT block (256 images of 197 tokens) whose stream is kept in fp16, normalised to fp32.
        dict(name="norm_vit_fp16", op="norm", rows=50432, cols=384, x="fp16", y="fp32", w="fp32", train=True),
        # ln2 of the tiny GPT preset on one short sequence: fp32 stream plus the bf16 attention output of autocast.
        dict(name="add_norm_tiny", op="add_norm", rows=127, cols=192, x="fp32", d="bf16", y="fp32", w="fp32"),
        # ln2 of the small GPT preset at the benchmark's batch, normalised output handed to a bf16 projection.
        dict(name="add_norm_gpt_small", op="add_norm", rows=32736, cols=768, x="fp32", d="bf16", y="bf16", w="fp32"),
        # Odd row length: rows that no vector load fits.
        dict(name="add_norm_odd", op="add_norm", rows=4099, cols=1537, x="bf16", d="bf16", y="bf16", w="bf16"),
        # A wide bf16 model.
        dict(name="add_norm_wide", op="add_norm", rows=16384, cols=4096, x="bf16", d="bf16", y="bf16", w="bf16"),
        # One attention projection of the tiny GPT preset.
        dict(name="orthogonal_tiny", op="orthogonal", batch=1, rows=192, cols=192, x="fp32"),
        # Odd sides, more columns than rows.
        dict(name="orthogonal_odd", op="orthogonal", batch=2, rows=257, cols=1001, x="fp16"),
        # A large square weight.
        dict(name="orthogonal_large", op="orthogonal", batch=1, rows=4096, cols=4096, x="bf16"),
        # Digital matrices of a tiny hybrid GPT: query, key and value as three matrices, output and down projections.
        dict(name="muon_tiny_hybrid", op="muon", depth=10, dim=192, ffn=768, g="fp32"),
        # Digital matrices of the small physical GPT (attention only, the FFN is thresholds).
        dict(name="muon_small_physical", op="muon", depth=12, dim=768, ffn=0, g="fp32"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most_bytes, most_flops = (max(work(c)[k] for c in listed() if c["op"] in ops)
                              for k, ops in (("bytes", ("norm", "add_norm")), ("flops", ("orthogonal", "muon"))))
    while True:
        op = rng.choice(["norm", "add_norm", "orthogonal", "muon"])
        if op == "norm":
            x = rng.choice(["fp32", "bf16", "fp16"])
            c = dict(op=op, rows=_log_uniform(rng, 1, 65536), cols=_log_uniform(rng, 16, 8192), x=x,
                     y=rng.choice(["fp32", "bf16", "fp16"] if x == "fp32" else ["fp32", x]),
                     w=rng.choice(["fp32", x]), train=rng.random() < 0.75)
        elif op == "add_norm":
            x = rng.choice(["fp32", "bf16", "fp16"])
            c = dict(op=op, rows=_log_uniform(rng, 1, 65536), cols=_log_uniform(rng, 16, 8192), x=x,
                     d=rng.choice(["fp32", "bf16", "fp16"]) if x == "fp32" else x,
                     y=rng.choice(["fp32", "bf16", "fp16"] if x == "fp32" else ["fp32", x]), w=rng.choice(["fp32", x]))
        elif op == "orthogonal":
            c = dict(op=op, batch=_log_uniform(rng, 1, 16), rows=_log_uniform(rng, 32, 4096),
                     cols=_log_uniform(rng, 32, 4096), x=rng.choice(["fp32", "bf16", "fp16"]))
        else:
            dim = _log_uniform(rng, 64, 1024)
            c = dict(op=op, depth=rng.randint(1, 10), dim=dim,
                     ffn=rng.choice([0, _log_uniform(rng, dim, 4 * dim)]), g=rng.choice(["fp32", "bf16"]))
        if op in ("norm", "add_norm"):  # half the even sizes of a model, half anything
            if rng.random() < 0.5:
                c["cols"] = max(16, c["cols"] // 16 * 16)
            if work(c)["bytes"] <= most_bytes:
                return c
        elif work(c)["flops"] <= most_flops:
            return c


def _size(t):
    return _DTYPES[t].itemsize


def _ns_flops(batch, m, n):
    """The steps' products with the symmetry of two of them used: X X^T and its
    square from one triangle each, then the product with X."""
    m, n = min(m, n), max(m, n)
    return batch * _STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    op = case["op"]
    if op in ("norm", "add_norm"):
        n, c = case["rows"] * case["cols"], case["cols"]
        b = n * (_size(case["x"]) + _size(case["y"])) + 2 * c * _size(case["w"])
        f = 8 * n
        if op == "add_norm":
            b += n * (_size(case["d"]) + _size(case["x"]))  # the residual branch in, the sum out
            f += n
        if op == "add_norm" or case["train"]:
            b += n * (_size(case["y"]) + _size(case["x"])) + 2 * c * _size(case["w"])  # dy in; dx, dw, db out
            f += 14 * n
        if op == "add_norm":
            b += n * (_size(case["x"]) + _size(case["d"]))  # gradient of the sum in, of the branch out
        return {"bytes": b, "flops": f}
    if op == "orthogonal":
        k = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * k * _size(case["x"]), "flops": _ns_flops(case["batch"], case["rows"], case["cols"])}
    d, f, layers = case["dim"], case["ffn"], case["depth"]
    k = layers * (4 * d * d + d * f)
    flops = _ns_flops(4 * layers, d, d) + (_ns_flops(layers, d, f) if f else 0)
    return {"bytes": k * (_size(case["g"]) + 16), "flops": flops}  # gradient in; momentum and parameter in and out


def _gradient(gen, dev, *shape):
    """An update with a decaying spectrum (a few strong directions over a noise
    floor), at the magnitude of a mean-reduced loss."""
    *batch, m, n = shape
    r = max(1, min(m, n, 32))
    weight = 2.0 ** -torch.arange(r, device=dev, dtype=torch.float32).div(4.0)
    low = (torch.randn(*batch, m, r, device=dev, generator=gen) * weight) @ torch.randn(*batch, r, n, device=dev,
                                                                                      generator=gen)
    return (low + 0.3 * torch.randn(*shape, device=dev, generator=gen)) * 1e-3


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    op = case["op"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    if op in ("norm", "add_norm"):
        rows, cols = case["rows"], case["cols"]
        train = op == "add_norm" or case["train"]
        x_t, w_t, y_t = _DTYPES[case["x"]], _DTYPES[case["w"]], _DTYPES[case["y"]]
        # a residual stream: a mean and a width of its own for each channel, a few of them far out
        width = 1.0 + 0.5 * torch.rand(cols, device=dev, generator=gen)
        width[:: max(1, cols // 4)] *= 8.0
        s = {"op": op, "train": train, "y_type": y_t}
        s["x"] = (normal(rows, cols) * width + 0.3 * normal(cols)).to(x_t).requires_grad_(train)
        s["weight"] = (1.0 + 0.2 * normal(cols)).to(w_t).requires_grad_(train)
        s["bias"] = (0.1 * normal(cols)).to(w_t).requires_grad_(train)
        if op == "add_norm":
            s["delta"] = (0.5 * normal(rows, cols)).to(_DTYPES[case["d"]]).requires_grad_(True)
            s["grad_sum"] = (0.02 * normal(rows, cols)).to(x_t)
        if train:
            s["grad"] = (0.02 * normal(rows, cols)).to(y_t)
        return s
    if op == "orthogonal":
        return {"op": op, "update": _gradient(gen, dev, case["batch"], case["rows"], case["cols"]).to(_DTYPES[case["x"]])}
    d, f = case["dim"], case["ffn"]
    shapes = ([(3, d, d), (d, d)] + ([(d, f)] if f else [])) * case["depth"]
    return {"op": op,
            "params": [0.02 * normal(*s) for s in shapes],
            "grads": [_gradient(gen, dev, *s).to(_DTYPES[case["g"]]) for s in shapes],
            "momenta": [_gradient(gen, dev, *s) for s in shapes]}


# ---------------------------------------------------------------- plain form --

def _plain_norm(x, weight, bias, y_type, grad, grad_sum, delta=None):
    """(y, [sum], [dx, [d delta], dw, db]) of y = LN(x + delta) in 32 bits. The
    sum is an output in the type of x, and y is that output's norm."""
    h = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    h32 = h.float()
    mean = h32.mean(-1, keepdim=True)
    centred = h32 - mean
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
    unit = centred * rstd
    out = [(unit * weight.float() + bias.float()).to(y_type)] + ([] if delta is None else [h])
    if grad is None:
        return out
    g = grad.float()
    gw = g * weight.float()
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - unit * (gw * unit).mean(-1, keepdim=True))
    if grad_sum is not None:
        dx = dx + grad_sum.float()
    out.append(dx.to(x.dtype))
    if delta is not None:
        out.append(dx.to(delta.dtype))
    return out + [(g * unit).sum(0).to(weight.dtype), g.sum(0).to(bias.dtype)]


def _plain_orthogonal(u):
    """Newton-Schulz steps on a batch of matrices in 32 bits."""
    a, b, c = _NS
    x = u / u.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(_NORM_FLOOR)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(_STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def _plain_muon(params, grads, momenta):
    """One step over matrices of one shape, stacked: parameters and momenta in place."""
    m, n = params[0].shape[-2:]

    def stacked(ts):
        return torch.cat([t.reshape(-1, m, n).float() for t in ts])

    g, mom, p = stacked(grads), stacked(momenta), stacked(params)
    mom = _MOMENTUM * mom + (1.0 - _MOMENTUM) * g
    o = _plain_orthogonal((1.0 - _MOMENTUM) * g + _MOMENTUM * mom)
    p = p * (1.0 - _LR * _DECAY) - (_LR * max(1.0, m / n) ** 0.5) * o
    sizes = [t.numel() // (m * n) for t in params]
    torch._foreach_copy_(params, [t.view_as(q) for t, q in zip(p.split(sizes), params)])
    torch._foreach_copy_(momenta, [t.view_as(q) for t, q in zip(mom.split(sizes), momenta)])


def _by_shape(s):
    groups = {}
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        for to, t in zip(groups.setdefault(tuple(p.shape[-2:]), ([], [], [])), (p, g, m)):
            to.append(t)
    return groups.values()


def _package():
    root = str(Path(__file__).resolve().parent.parent / "isa-_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


def run(state):
    op = state["op"]
    if own:
        return _run_own(state)
    with torch.no_grad():
        if op in ("norm", "add_norm"):
            return _plain_norm(state["x"], state["weight"], state["bias"], state["y_type"], state.get("grad"),
                               state.get("grad_sum"), state.get("delta"))
        if op == "orthogonal":
            return _plain_orthogonal(state["update"].float()).to(state["update"].dtype)
        for group in _by_shape(state):
            _plain_muon(*group)
        return state["params"] + state["momenta"]


def _run_own(s):
    _package()
    if s["op"] == "norm":
        from isa_b200.kernels.transformer_norm import cuda_layer_norm

        if not s["train"]:
            with torch.no_grad():
                return [cuda_layer_norm(s["x"], s["weight"], s["bias"], _EPS, out_dtype=s["y_type"])]
        y = cuda_layer_norm(s["x"], s["weight"], s["bias"], _EPS, out_dtype=s["y_type"])
        return [y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])]
    if s["op"] == "add_norm":
        from isa_b200.kernels.transformer_norm import cuda_add_layer_norm

        y, h = cuda_add_layer_norm(s["x"], s["delta"], s["weight"], s["bias"], _EPS, out_dtype=s["y_type"])
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), (s["x"], s["delta"], s["weight"], s["bias"]),
                                                             (s["grad"], s["grad_sum"]))]
    from isa_b200.kernels.muon import cuda_muon_step, cuda_orthogonalize

    if s["op"] == "orthogonal":
        return cuda_orthogonalize(s["update"], steps=_STEPS, coefficients=_NS, eps=_NORM_FLOOR)
    cuda_muon_step(s["params"], s["grads"], s["momenta"], lr=_LR, momentum=_MOMENTUM, nesterov=True,
                   weight_decay=_DECAY, steps=_STEPS, coefficients=_NS, eps=_NORM_FLOOR)
    return s["params"] + s["momenta"]


# ------------------------------------------------------- definition, 64 bits --

def _exact_norm(s):
    x, w = s["x"].detach(), s["weight"].detach().double()
    h = x.double()
    out = []
    if "delta" in s:
        h = h + s["delta"].detach().double()
        out = [h]
        h = h.to(x.dtype).double()  # the sum is held in the type of x, and y is what is held normalised
    n = h.shape[-1]
    var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
    inv = (var + _EPS) ** -0.5
    out = [torch.addcmul(s["bias"].detach().double(), (h - mean) * inv, w)] + out
    if not s["train"]:
        return out
    # row by row dx = J^T (w g) with J = inv (I - 1 1^T/n - u u^T/n)
    u = (h - mean) * inv
    v = s["grad"].double() * w
    dx = inv * (v - v.sum(-1, keepdim=True) / n - u * torch.einsum("rc,rc->r", u, v).unsqueeze(-1) / n)
    if "delta" in s:
        dx = dx + s["grad_sum"].double()
        out += [dx, dx]
    else:
        out += [dx]
    return out + [torch.einsum("rc,rc->c", s["grad"].double(), u), s["grad"].double().sum(0)]


def _exact_orthogonal(u):
    """The steps as one matrix function: with G = X X^T of the normalised
    matrix, every factor is a polynomial in G, so G and the product Q of the
    factors are carried instead of X, and the answer is Q X."""
    a, b, c = _NS
    tall = u.shape[-2] > u.shape[-1]
    x = u.double().mT if tall else u.double()
    x = x / torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True).clamp_min(_NORM_FLOOR)
    eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    g, q = torch.matmul(x, x.mT), eye
    for k in range(_STEPS):
        f = a * eye + g @ (b * eye + c * g)
        q = f @ q
        if k + 1 < _STEPS:
            g = f @ g @ f
    x = q @ x
    return x.mT if tall else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "add_norm"):
        return _exact_norm(s)
    if case["op"] == "orthogonal":
        return _exact_orthogonal(s["update"])
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g = g.double()
        m = torch.lerp(g, m.double(), _MOMENTUM)
        o = _exact_orthogonal(torch.lerp(g, m, _MOMENTUM))
        scale = _LR * math.sqrt(max(1.0, p.shape[-2] / p.shape[-1]))
        params.append(p.double() - _LR * _DECAY * p.double() - scale * o)
        momenta.append(m)
    return params + momenta

"""The digital operators where the package uses them: LayerNorm as nn.LayerNorm, the GPT and ViT blocks with
``fused_norm``, the Muon optimiser, and a whole training step of all of them."""

import pytest
import torch
import torch.nn as nn

U = 2.0 ** -24


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


# ----------------------------------------------------------------------- CPU --

def test_layer_norm_is_a_drop_in():
    from isa_b200.operators import LayerNorm
    ours, theirs = LayerNorm(24, eps=1e-6), nn.LayerNorm(24, eps=1e-6)
    assert list(ours.state_dict()) == list(theirs.state_dict())
    ours.load_state_dict(theirs.state_dict())
    assert LayerNorm(8, bias=False).bias is None and LayerNorm(8, elementwise_affine=False).weight is None
    with pytest.raises(ValueError, match="last axis"):
        LayerNorm((4, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        ours(torch.zeros(2, 24))
    with pytest.raises(RuntimeError, match="24 features"):
        ours(torch.zeros(2, 1))


def test_fused_norm_keeps_the_checkpoint_layout():
    from isa_b200.language import GPT2Model, ModelConfig
    small = dict(vocab_size=50, max_seq_len=16)
    for kind in ("standard", "hybrid", "physical"):
        plain = GPT2Model(ModelConfig.from_preset("tiny", kind, **small))
        fused = GPT2Model(ModelConfig.from_preset("tiny", kind, fused_norm=True, **small))
        assert list(plain.state_dict()) == list(fused.state_dict())
        fused.load_state_dict(plain.state_dict())


def test_muon_takes_the_digital_matrices():
    from isa_b200.language import GPT2Model, ModelConfig
    for kind, linears in (("standard", 2), ("hybrid", 1), ("physical", 0)):
        cfg = ModelConfig.from_preset(kind and "tiny", kind, vocab_size=50, max_seq_len=16)
        model = GPT2Model(cfg)
        muon, rest = model.configure_muon_groups(0.01, 1e-3, 0.1, 0.02)
        names = {id(p): n for n, p in model.named_parameters()}
        fused, single = muon
        assert fused["matrices"] == 3 and [names[id(p)] for p in fused["params"]] == [
            f"blocks.{i}.attn.in_proj_weight" for i in range(cfg.depth)]
        assert len(single["params"]) == (1 + linears) * cfg.depth
        taken = [id(p) for g in muon + rest for p in g["params"]]
        assert sorted(taken) == sorted(id(p) for p in model.parameters())  # each once, none left out
        assert not any("vth" in names[id(p)] or "embedding" in names[id(p)] for g in muon for p in g["params"])


def test_muon_constructor_refusals():
    from isa_b200.optim import Muon
    w = nn.Parameter(torch.zeros(6, 4))
    with pytest.raises(ValueError, match="stacked"):
        Muon([nn.Parameter(torch.zeros(6))])
    with pytest.raises(ValueError, match="stacked"):
        Muon([w], matrices=4)
    for bad in (dict(lr=-1.0), dict(momentum=1.5), dict(weight_decay=-0.1), dict(adjust_lr="none")):
        with pytest.raises(ValueError):
            Muon([w], **bad)
    opt = Muon([w], lr=0.1)
    opt.step()  # no gradients: nothing to do
    assert not opt.state


# ----------------------------------------------------------------------- GPU --

gpu = pytest.mark.gpu


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from isa_b200 import build
    build.build_library()
    return torch.device("cuda")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_module_against_nn_layer_norm(dev, dtype):
    """Two roundings of the result and of the fp32 arithmetic between the modules: 2 eta + 200 u."""
    from isa_b200.operators import LayerNorm
    ours, theirs = LayerNorm(192).to(dev, dtype), nn.LayerNorm(192).to(dev, dtype)
    with torch.no_grad():
        theirs.weight.uniform_(0.5, 1.5)
        theirs.bias.uniform_(-0.5, 0.5)
    ours.load_state_dict(theirs.state_dict())
    x = torch.randn(3, 41, 192, device=dev, dtype=dtype)
    tol = torch.finfo(dtype).eps + 200 * U
    assert ours(x).dtype == theirs(x).dtype == dtype and _rel(ours(x), theirs(x)) <= tol
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert ours(x).dtype == theirs(x).dtype == torch.float32
        assert ours(x, torch.bfloat16 if dtype != torch.float16 else None).dtype == torch.bfloat16
    y, h = ours.add(x, x)
    assert torch.equal(h, x + x) and _rel(y, theirs(x + x)) <= tol
    y, h = ours.add(x, x.float())  # a wider branch widens the stream, as a torch sum does
    assert h.dtype == torch.float32 and torch.equal(h, x.float() + x.float())


def _models(dev, kind, depth=2):
    from isa_b200.language import GPT2Model, ModelConfig
    out = []
    for fused in (False, True):
        cfg = ModelConfig.from_preset("tiny", kind, vocab_size=211, max_seq_len=48, fused_norm=fused)
        cfg.depth = depth
        torch.manual_seed(0)
        out.append(GPT2Model(cfg).to(dev))
    out[1].load_state_dict(out[0].state_dict())
    return out


@gpu
@pytest.mark.parametrize("kind", ["standard", "hybrid", "physical"])
@pytest.mark.parametrize("autocast", [False, True])
def test_fused_model_against_plain_model(dev, kind, autocast):
    """The same weights with and without fused norms, logits and every gradient, norm-wise.  Without autocast the two
    differ by fp32 roundings of the norms (a few u each, 5 norms deep, and sums over 188 tokens): 1e-4 leaves three
    orders for what the layers between make of them.  Under bf16 autocast the norms' outputs are rounded to bf16 by
    the projection in one case and by the norm in the other, which is the same rounding of values that differ by
    fp32 roundings, so a few flip by a bf16 step: the tolerance of the package's autocast comparisons, 2e-2."""
    plain, fused = _models(dev, kind)
    ids = torch.randint(0, 211, (4, 48), device=dev)
    tol = 2e-2 if autocast else 1e-4
    grads = []
    for model in (plain, fused):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            logits = model(ids[:, :-1])
            loss = nn.functional.cross_entropy(logits.float().reshape(-1, 211), ids[:, 1:].reshape(-1))
        loss.backward()
        grads.append((logits, {n: p.grad for n, p in model.named_parameters()}))
    assert _rel(grads[1][0].float(), grads[0][0].float()) < tol
    for name, g in grads[0][1].items():
        if g is None:
            assert grads[1][1][name] is None
        else:
            assert _rel(grads[1][1][name], g) < tol, name
    # with intermediate results the model takes the unfused path through the same modules
    logits, inter = fused(ids[:, :-1], need_intermediate=True)
    assert len(inter) == 2 and _rel(logits, fused(ids[:, :-1])) < 1e-4


@gpu
def test_fused_vit_against_plain_vit(dev):
    from isa_b200.harness.vit import PhysicalViT, ViTConfig
    small = dict(img_size=32, patch_size=8, num_classes=11, embed_dim=48, num_heads=3, depth=2)
    torch.manual_seed(0)
    plain = PhysicalViT(ViTConfig(**small)).to(dev)
    fused = PhysicalViT(ViTConfig(fused_norm=True, **small)).to(dev)
    fused.load_state_dict(plain.state_dict())
    img = torch.randn(5, 3, 32, 32, device=dev)
    y0, y1 = plain(img), fused(img)
    assert _rel(y1, y0) < 1e-4
    for m, y in ((plain, y0), (fused, y1)):
        y.square().mean().backward()
    for (n, p), q in zip(plain.named_parameters(), fused.parameters()):
        assert _rel(q.grad, p.grad) < 1e-4, n


@gpu
def test_muon_optimizer_against_the_formula(dev):
    """Three steps with new gradients against 64 bits, stacked matrices among them."""
    from isa_b200.optim import Muon
    from tests.test_muon import _exact
    torch.manual_seed(1)
    fused, single = nn.Parameter(torch.randn(96, 32, device=dev) * 0.1), nn.Parameter(torch.randn(32, 80, device=dev) * 0.1)
    idle = nn.Parameter(torch.randn(8, 8, device=dev))
    opt = Muon([{"params": [fused], "matrices": 3, "lr": 0.02}, {"params": [single, idle], "lr": 0.01, "nesterov": False}],
               weight_decay=0.05)
    before = idle.detach().clone()
    want = {p: (p.detach().double().clone(), torch.zeros_like(p, dtype=torch.float64)) for p in (fused, single)}
    bounds = {fused: 0.0, single: 0.0}
    for step in range(3):
        for p in (fused, single):
            p.grad = torch.randn_like(p) * 1e-3
            w, m = want[p]
            m = 0.95 * m + 0.05 * p.grad.double()
            u = 0.95 * m + 0.05 * p.grad.double() if p is fused else m
            lr, parts = (0.02, 3) if p is fused else (0.01, 1)
            o, bound = zip(*(_exact(t, fine=False) for t in u.chunk(parts)))
            # fp32 momenta: a relative rounding of 8 u in the update, at most times the growth of five steps
            bounds[p] += lr * (sum(bound) + parts * 8 * U * 3.4445 ** 5) + 4 * U * float(w.norm())
            want[p] = (w * (1 - lr * 0.05) - lr * torch.cat(o), m)  # none of these matrices is tall: s = 1
        opt.step()
    for p in (fused, single):
        assert float((p.detach().double() - want[p][0]).norm()) <= bounds[p]
        assert _rel(opt.state[p]["momentum_buffer"], want[p][1]) <= 16 * U
    assert torch.equal(idle, before) and idle not in opt.state


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_muon_state_dict_round_trip(dev, dtype):
    from isa_b200.optim import Muon
    torch.manual_seed(2)
    a = nn.Parameter((torch.randn(40, 24, device=dev) * 0.1).to(dtype))
    b = nn.Parameter(a.detach().clone())
    one = Muon([a], lr=0.02)
    a.grad = torch.randn_like(a)
    one.step()
    with torch.no_grad():
        b.copy_(a)
    two = Muon([b], lr=0.5)
    two.load_state_dict(one.state_dict())
    assert two.state[b]["momentum_buffer"].dtype == torch.float32
    assert torch.equal(two.state[b]["momentum_buffer"], one.state[a]["momentum_buffer"])
    assert two.state[b]["momentum_buffer"].data_ptr() != one.state[a]["momentum_buffer"].data_ptr()
    a.grad = torch.randn_like(a)
    b.grad = a.grad.clone()
    one.step()
    two.step()
    assert torch.equal(a, b)


@gpu
def test_muon_captured_step(dev):
    """The first step makes the momenta and is refused in a capture; a later one replays as the plain step."""
    from isa_b200.optim import Muon
    torch.manual_seed(3)
    a = nn.Parameter(torch.randn(40, 72, device=dev))
    a.grad = torch.randn_like(a)
    before = a.detach().clone()
    opt = Muon([a], lr=0.02)
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert torch.equal(a, before)
    opt.step()
    b = nn.Parameter(a.detach().clone())
    b.grad = a.grad.clone()
    plain = Muon([b], lr=0.02)
    plain.load_state_dict(opt.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for seed in range(3):
        a.grad.copy_(torch.randn(40, 72, generator=torch.Generator().manual_seed(seed)))
        b.grad.copy_(a.grad)
        graph.replay()
        plain.step()
        assert torch.equal(a, b)
    assert torch.equal(opt.state[a]["momentum_buffer"], plain.state[b]["momentum_buffer"])


@gpu
def test_muon_zero_matrix_at_the_smallest_eps(dev):
    from isa_b200.kernels.muon import cuda_orthogonalize
    assert not cuda_orthogonalize(torch.zeros(2, 20, 30, device=dev), eps=1e-30).any()


@gpu
def test_training_steps_of_everything(dev):
    """Fused norms, CIM layers and Muon with AdamW in the package's own training step: it runs, and Muon's matrices
    and the norms move.  (A step of Muon does not depend on the gradient's size; AdamW's does below its eps, where the
    threshold voltages of an untrained model are.)"""
    from isa_b200.harness.gpt import GPTConfig, PhysicalGPT, train_step
    torch.manual_seed(3)
    model = PhysicalGPT(GPTConfig(vocab_size=97, max_seq_len=32, size="tiny", fused_norm=True)).to(dev)
    model.blocks = model.blocks[:2]
    opts = model.muon_optimizers(lr=1e-3, muon_lr=0.01)
    ids = torch.randint(0, 97, (3, 32), device=dev)
    start = {n: p.detach().clone() for n, p in model.named_parameters()}
    for _ in range(2):
        loss = train_step(model, opts, ids, model.cim_layers())
    assert torch.isfinite(loss)
    moved = {n for n, p in model.named_parameters() if not torch.equal(p, start[n])}
    assert all(torch.isfinite(p).all() for p in model.parameters())
    for i in range(2):
        for name in ("attn.in_proj_weight", "attn.out_proj.weight", "ln1.weight", "ln2.weight"):
            assert f"blocks.{i}.{name}" in moved, name
    loss = train_step(model, torch.optim.AdamW(model.parameters(), lr=1e-3), ids, model.cim_layers())  # one optimizer alone
    assert torch.isfinite(loss)

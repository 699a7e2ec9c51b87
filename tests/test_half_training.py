"""The mixed-precision operators together, as the denoisers use them: ddpm.Backbone and the direction denoiser with bf16 / fp16
weights against the same networks in 64 bits (outputs and gradients), training steps through DataParallelTrainer and
optim.AdamW, the captured step."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _gelu(z):
    return z * 0.5 * torch.erfc(-z / math.sqrt(2.0))


def _backbone64(bb, x, idx):
    """the formulas of ddpm.py:17-41 in 64 bits on detached copies of the parameters: (output, parameters)"""
    ps = {n: p.detach().double().requires_grad_(True) for n, p in bb.named_parameters()}

    def mlp(pre, h):
        n = len(getattr(bb, pre).layers)
        for k in range(n):
            z = h @ ps[f"{pre}.layers.{k}.weight"].t() + ps[f"{pre}.layers.{k}.bias"]
            h = z if k == n - 1 else (_gelu(z) if k == 0 else h + _gelu(z))
        return h
    h = mlp("linear_model1", x.double()) + ps["embedding_layer.weight"][idx]
    return mlp("linear_model2", h), ps


def _near(got, want, layers, dtype, what):
    """Every layer rounds what it stores and reads (activation, pre-activation, weight gradient's operand) by at most half a
    step each, relative to values whose size the layers keep (|GELU'| <= 1.13, weights of norm about 1, skips): three half
    steps a layer bound the 2-norm error."""
    err = float((got.double() - want).norm() / want.norm().clamp(min=1e-30))
    assert err <= 3 * layers * HALF[dtype], (what, err)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 200, 1500])
def test_backbone_and_gradients(dtype, rows):
    from hypdiff_amd.ddpm import Backbone
    torch.manual_seed(rows)
    bb = Backbone(64, 96, 2, 50).cuda().to(dtype)
    x = torch.randn(rows, 64, device="cuda").to(dtype).float()
    idx = torch.randint(0, 50, (rows,), device="cuda")
    want, ps = _backbone64(bb, x, idx)
    with torch.no_grad():
        out = bb(x, idx)
    assert out.dtype == torch.float32                     # x's type around weights of 16 bits
    layers = 8
    _near(out, want.detach(), layers, dtype, "output")
    g = torch.randn(rows, 64, device="cuda").to(dtype)
    y = bb(x, idx)
    assert torch.equal(y, out)
    y.backward(g.float())
    want.backward(g.double())
    for n, p in bb.named_parameters():
        assert p.grad.dtype == dtype
        _near(p.grad, ps[n].grad, layers, dtype, n)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_direction_denoiser(dtype):
    from hypdiff_amd.models.direction_diffusion import mlp
    torch.manual_seed(3)
    net = mlp(30).cuda().to(dtype)
    x = torch.randn(333, 30, device="cuda").to(dtype).float()
    t = torch.rand(333, device="cuda").to(dtype).float()
    ps = {n: p.detach().double().requires_grad_(True) for n, p in net.named_parameters()}
    h = torch.cat([x, t[:, None]], 1).double()
    for k in range(1, 6):
        h = h @ ps[f"fc{k}.weight"].t() + ps[f"fc{k}.bias"]
        h = _gelu(h) if k < 5 else h
    with torch.no_grad():
        out = net(x, t)
    assert out.dtype == torch.float32
    _near(out, h.detach(), 5, dtype, "output")
    g = torch.randn(333, 30, device="cuda").to(dtype)
    net(x, t).backward(g.float())
    h.backward(g.double())
    for n, p in net.named_parameters():
        _near(p.grad, ps[n].grad, 5, dtype, n)


def _trainer(state_bits, dtype=torch.bfloat16, master=True):
    from hypdiff_amd import dist as hdist, optim
    from hypdiff_amd.ddpm import Model
    torch.manual_seed(11)
    model = Model(64, 96, 2, 50, 1e-4, 0.02).cuda().to(dtype)
    opt = optim.AdamW(model.parameters(), lr=1e-3, state_bits=state_bits, master_weights=master and dtype != torch.float32)
    return model, hdist.DataParallelTrainer(model, optimizer=opt)


@gpu
@pytest.mark.parametrize("state_bits", [32, 8])
def test_training_step_is_the_operators_composed(state_bits):
    """A trainer's step = loss and gradients of the model, then AdamW on them: the weights after two steps are those of a
    plain loop over an identical model, bit for bit."""
    from hypdiff_amd import optim
    model, tr = _trainer(state_bits)
    other, _ = _trainer(state_bits)
    opt = optim.AdamW(other.parameters(), lr=1e-3, state_bits=state_bits, master_weights=True)
    x = torch.randn(200, 64, device="cuda")
    for s in range(2):
        idx = torch.randint(0, 50, (200,), device="cuda")
        eps = torch.randn(200, 64, device="cuda")
        loss = tr.step(lambda: model.loss_fn(x, idx=idx, epsilon=eps))
        for p in other.parameters():
            p.grad = None
        ref = other.loss_fn(x, idx=idx, epsilon=eps)
        ref.backward()
        opt.step()
        assert torch.equal(loss, ref.detach()) and bool(torch.isfinite(loss))
    for p, q in zip(model.parameters(), other.parameters()):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("dtype,state_bits", [(torch.bfloat16, 32), (torch.bfloat16, 8), (torch.float16, 32), (torch.float32, 8)])
def test_captured_training_step(dtype, state_bits):
    """DataParallelTrainer.capture with optim.AdamW: replays, with the program's own eager work between them, against eager
    steps of an identical model on the same inputs.  The step count lives on the device in a replay: the corrections are
    one fp32 step off at most, which may move a stored weight by one of its own steps, and then by the sum of such moves."""
    a, ta = _trainer(state_bits, dtype)
    b, tb = _trainer(state_bits, dtype)
    x, eps = torch.randn(100, 64, device="cuda"), torch.randn(100, 64, device="cuda")
    idx = torch.randint(0, 50, (100,), device="cuda")
    replay = ta.capture(lambda: a.loss_fn(x, idx=idx, epsilon=eps), warmup=2)
    for _ in range(2):
        tb.step(lambda: b.loss_fn(x, idx=idx, epsilon=eps))
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)                          # the warm-up steps are eager
    for k in range(4):
        gen = torch.Generator(device="cuda").manual_seed(k)
        x.copy_(torch.randn(100, 64, device="cuda", generator=gen))
        eps.copy_(torch.randn(100, 64, device="cuda", generator=gen))
        la = replay()
        lb = tb.step(lambda: b.loss_fn(x, idx=idx, epsilon=eps))
        torch.cuda.synchronize()
        assert abs(float(la) - float(lb)) <= 0.02 * abs(float(lb))
        half = HALF.get(dtype, 2.0 ** -24)
        for p, q in zip(a.parameters(), b.parameters()):
            d = (p.double() - q.double()).norm() / q.double().norm()
            assert float(d.detach()) <= 4 * (k + 1) * half + 1e-3 * 0.05 * (k + 1), float(d.detach())


def test_live_graphs_are_found():
    from hypdiff_amd.dist import _in_a_live_graph
    p, q = torch.nn.Parameter(torch.randn(3)), torch.nn.Parameter(torch.randn(2))
    p.register_post_accumulate_grad_hook(lambda t: None)
    assert _in_a_live_graph([p, q]) == []
    loss = (p * 2).sum()
    assert [t is p for t in _in_a_live_graph([p, q])] == [True]
    loss.backward()
    assert len(_in_a_live_graph([p, q])) == 1            # the tensor still holds the node
    kept = loss.detach()
    ring = [loss]
    ring.append(ring)                                    # dropped, but only the collector will see it
    del loss, ring
    assert _in_a_live_graph([p, q]) == [] and bool(torch.isfinite(kept))


@gpu
def test_capture_is_refused_while_an_eager_graph_lives():
    model, tr = _trainer(32)
    x, eps, idx = torch.randn(20, 64, device="cuda"), torch.randn(20, 64, device="cuda"), torch.zeros(20, dtype=torch.int64, device="cuda")
    kept = model.loss_fn(x, idx=idx, epsilon=eps)
    with pytest.raises(RuntimeError, match="autograd graph"):
        tr.capture(lambda: model.loss_fn(x, idx=idx, epsilon=eps), warmup=1)
    del kept
    replay = tr.capture(lambda: model.loss_fn(x, idx=idx, epsilon=eps), warmup=1)
    assert bool(torch.isfinite(replay()))


@gpu
def test_trainer_gives_16_bit_modules_masters():
    from hypdiff_amd import dist as hdist, optim
    from hypdiff_amd.ddpm import Model
    model = Model(64, 64, 1, 20, 1e-4, 0.02).cuda().bfloat16()
    tr = hdist.DataParallelTrainer(model, lr=1e-3)
    assert isinstance(tr.opt, optim.AdamW) and tr.bucket.flat.dtype == torch.bfloat16
    x = torch.randn(40, 64, device="cuda")
    before = [p.detach().clone() for p in model.parameters()]
    loss = tr.step(lambda: model.loss_fn(x))
    assert bool(torch.isfinite(loss)) and "master" in tr.opt.state_buffers()
    assert any(not torch.equal(p, q) for p, q in zip(model.parameters(), before))


@gpu
def test_sampler_runs_on_16_bit_weights():
    from hypdiff_amd.ddpm import Model
    from hypdiff_amd.ddpm_utils import DDPMSampler
    torch.manual_seed(5)
    model = Model(64, 64, 2, 20, 1e-4, 0.02).cuda().eval()
    x = torch.randn(30, 64, device="cuda")
    s = DDPMSampler(1e-4, 0.02, 20, model, "cuda", (64,))
    with torch.no_grad():
        want = s.one_step(x, 7, None)
        model.bfloat16()
        got = s.one_step(x, 7, None)
        final = s.sampling(30, x, only_final=True)
    # one denoiser pass of 9 stages, weights rounded too (one more half step each), scaled into the update of x
    assert float((got - want).norm() / want.norm()) <= 4 * 9 * 2.0 ** -8
    assert final.shape == (30, 64) and bool(torch.isfinite(final).all())


@gpu
def test_capture_of_an_fp32_module_beside_an_eager_graph():
    """BucketAdam: refused while a loss holds the parameters' nodes (the captured backward pass would join their stream), and
    nothing has changed by then; captured once it is dropped, detached losses may stay."""
    from hypdiff_amd import dist as hdist
    from hypdiff_amd.ddpm import Model
    torch.manual_seed(11)
    model = Model(64, 96, 2, 50, 1e-4, 0.02).cuda()
    tr = hdist.DataParallelTrainer(model)
    assert isinstance(tr.opt, hdist.BucketAdam)
    x, eps, idx = torch.randn(20, 64, device="cuda"), torch.randn(20, 64, device="cuda"), torch.zeros(20, dtype=torch.int64, device="cuda")
    loss_fn = lambda: model.loss_fn(x, idx=idx, epsilon=eps)  # noqa: E731
    kept, before = loss_fn(), [p.detach().clone() for p in model.parameters()]
    for _ in range(2):
        with pytest.raises(RuntimeError, match="autograd graph"):
            tr.capture(loss_fn, warmup=1)
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), before)) and tr.opt.t == 0
    kept = kept.detach()
    first = tr.step(loss_fn)
    assert torch.equal(first, kept)
    replay = tr.capture(loss_fn, warmup=1)
    assert bool(torch.isfinite(replay())) and bool(torch.isfinite(first))

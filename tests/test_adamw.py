"""optim.AdamW (csrc/adamw.hip): one step against the formulas in 64 bits, the 8-bit moments bit for bit against a numpy
restatement in fp32, histories, refusals, capture, saving and loading."""
import copy
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
H = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative
SHAPES = [(1,), (7,), (255,), (256,), (257,), (33, 31), (512,), (513, 8), (0,), (3000,)]


def _params(dtype, shapes=SHAPES, seed=0, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ps = []
    for s in shapes:
        n = int(np.prod(s))
        base = (torch.randn(n + offset, device="cuda", generator=gen) * 0.05).to(dtype)
        p = torch.nn.Parameter(base[offset:].view(s))
        p.grad = (torch.randn(n + offset, device="cuda", generator=gen) * 0.01).to(dtype)[offset:].view(s)
        ps.append(p)
    return ps


def _step64(p, g, m, v, t, lr, betas, eps, weight_decay):
    b1, b2 = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = np.sqrt(v1) / math.sqrt(1 - b2 ** t) + eps
    upd = lr / (1 - b1 ** t) * (m1 / den)
    # the largest that the update could be without cancellation between its two terms: what roundings are relative to
    size = lr / (1 - b1 ** t) * ((b1 * np.abs(m) + (1 - b1) * np.abs(g)) / den)
    return p * (1 - lr * weight_decay) - upd, m1, v1, size


def _np64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


@gpu
@pytest.mark.parametrize("dtype,master,offset", [(torch.float32, False, 0), (torch.float32, False, 1), (torch.bfloat16, False, 0),
                                                 (torch.bfloat16, True, 0), (torch.bfloat16, True, 3), (torch.float16, True, 0),
                                                 (torch.float16, False, 1)])
def test_step_32(dtype, master, offset):
    """Three steps; every step is compared with the formulas in 64 bits from the state that it started from.  Bounds in
    units u = 2^-24: m is three roundings and two constants: 5 u of |b1 m| + |(1-b1) g|; v likewise 6 u; the update adds
    sqrt, two products, a sum, a quotient and two constants: 16 u of its size; p itself 4 u; 16-bit storage half a step."""
    from hypdiff_amd.optim import AdamW
    ps = _params(dtype, offset=offset)
    opt = AdamW(ps, master_weights=master, **H)
    u = 2.0 ** -24
    first = opt.state_buffers()          # the state exists, at step 0
    assert all(b.dtype == torch.float32 for b in first.values())
    for t in (1, 2, 3):
        st = [opt.state[p] for p in ps]
        w0 = [_np64(s["master"]) if master else _np64(p) for p, s in zip(ps, st)]
        m0, v0 = [_np64(s["exp_avg"]) for s in st], [_np64(s["exp_avg_sq"]) for s in st]
        opt.step()
        for i, p in enumerate(ps):
            g = _np64(p.grad)
            w, m, v, size = _step64(w0[i], g, m0[i], v0[i], t, **H)
            assert np.all(np.abs(_np64(st[i]["exp_avg"]) - m) <= 5 * u * (0.9 * np.abs(m0[i]) + 0.1 * np.abs(g)))
            assert np.all(np.abs(_np64(st[i]["exp_avg_sq"]) - v) <= 6 * u * v + 1e-44)
            bound = 4 * u * np.abs(w0[i]) + 16 * u * size
            if master:
                assert np.all(np.abs(_np64(st[i]["master"]) - w) <= bound)
                assert torch.equal(p.detach(), st[i]["master"].to(dtype))
            else:
                half = 0.0 if dtype == torch.float32 else EPS[dtype]
                assert np.all(np.abs(_np64(p) - w) <= bound * (1 + half) + half * np.abs(w) + (2.0 ** -25 if dtype == torch.float16 else 0))
            assert st[i]["step"] == t
        for p in ps:
            p.grad.mul_(-1.5)


def _f32(x):
    return np.float32(x)


def _step8(w, g, m, s, t, lr, betas, eps, weight_decay):
    """numpy restatement in fp32, one rounding per operation: (w, m, s) before rounding to codes"""
    b1, b2 = betas
    m = m * _f32(b1) + g * _f32(1 - b1)
    v = (s * s) * _f32(b2) + (g * g) * _f32(1 - b2)
    s = np.sqrt(v)
    den = s * _f32(1 / math.sqrt(1 - b2 ** t)) + _f32(eps)
    return w * _f32(1 - lr * weight_decay) - (m / den) * _f32(lr / (1 - b1 ** t)), m, s


def _blocks(x):
    return np.concatenate([x, np.zeros(-len(x) % 256, np.float32)]).reshape(-1, 256)


def _scales(x):
    amax = np.abs(_blocks(x)).max(1)
    scale = np.maximum(amax, _f32(2.0 ** -100)) * _f32(1 / 448)
    inv = _f32(1) / scale
    return np.where(amax == 0, _f32(0), scale), np.where(amax == 0, _f32(0), inv)


def _root_codes(s, inv, t):
    y = _blocks(s) * inv[:, None]
    i = np.arange(y.size, dtype=np.uint64).reshape(y.shape)
    d = ((i * 2654435761 + t * 1779033703) & 0xFFFFFFFF) >> 12
    normal = ((np.ascontiguousarray(y).view(np.uint32).astype(np.uint64) + d) >> 20).astype(np.int64) - 960
    small = np.floor(y * _f32(512) + d.astype(np.float32) * _f32(2.0 ** -20)).astype(np.int64)
    code = np.minimum(np.where(y < 2.0 ** -6, small, normal), 126)
    return np.where(_blocks(s) > 0, np.maximum(code, 1), 0).reshape(-1)[:len(s)].astype(np.uint8)


@gpu
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True), (torch.bfloat16, False),
                                          (torch.float16, True)])
def test_step_8_bit_for_bit(dtype, master):
    from hypdiff_amd.optim import AdamW
    ps = _params(dtype, seed=3)
    opt = AdamW(ps, state_bits=8, master_weights=master, **H)
    opt.state_buffers()
    for t in (1, 2, 3, 4):
        before = []
        for p in ps:
            st = opt.state[p]
            dec = lambda k: np.float32(1) * st[k].float().cpu().numpy().reshape(-1) * \
                np.repeat(st[k + "_scale"].cpu().numpy(), 256)[:p.numel()]  # noqa: E731
            w = (st["master"] if master else p.detach().float()).cpu().numpy().reshape(-1).copy()
            before.append((w, p.grad.float().cpu().numpy().reshape(-1), dec("exp_avg"), dec("exp_avg_sq_root")))
        opt.step()
        for p, (w, g, m, s) in zip(ps, before):
            st = opt.state[p]
            w, m, s = _step8(w, g, m, s, t, **H)
            got_w = (st["master"] if master else p.detach()).cpu().reshape(-1)
            want_w = torch.from_numpy(w)
            assert torch.equal(got_w, want_w if master else want_w.to(dtype))
            if master:
                assert torch.equal(p.detach().cpu().reshape(-1), want_w.to(dtype))
            sm, im = _scales(m)
            ss, iss = _scales(s)
            assert np.array_equal(st["exp_avg_scale"].cpu().numpy(), sm)
            assert np.array_equal(st["exp_avg_sq_root_scale"].cpu().numpy(), ss)
            want_m = torch.from_numpy((_blocks(m) * im[:, None]).reshape(-1)[:len(m)]).to(torch.float8_e4m3fn)
            assert torch.equal(st["exp_avg"].cpu().reshape(-1).view(torch.uint8) & 0x7F, want_m.view(torch.uint8) & 0x7F)
            assert torch.equal(st["exp_avg"].float().cpu().reshape(-1), want_m.float())
            assert np.array_equal(st["exp_avg_sq_root"].cpu().view(torch.uint8).numpy().reshape(-1), _root_codes(s, iss, t))
        for p in ps:
            p.grad.mul_(-0.7)


@gpu
def test_roots_decay_without_gradient():
    """With g = 0, sqrt(v) falls by 0.05 % a step, a hundredth of a code: rounding has to let it through.  Per element the
    codes wander (about 6 moves of 6-12 % in 1000 steps, a spread near 0.2), the mean of 4096 elements by 0.2 / 64 = 0.3 %:
    half a code, 2^-4, is far outside that."""
    from hypdiff_amd.optim import AdamW
    p = torch.nn.Parameter(torch.randn(4096, device="cuda"))
    p.grad = torch.randn(4096, device="cuda").abs() + 0.5
    opt = AdamW([p], state_bits=8, lr=0.0)
    opt.step()
    st = opt.state[p]

    def root():
        return st["exp_avg_sq_root"].double() * st["exp_avg_sq_root_scale"].double().repeat_interleave(256)
    r0 = root()
    p.grad.zero_()
    for _ in range(1000):
        opt.step()
    ratio = float((root() / r0).mean()) / 0.999 ** 500
    assert abs(ratio - 1) < 2.0 ** -4, ratio


@gpu
def test_small_root_never_becomes_zero_and_nonfinite_spreads_to_its_block_only():
    from hypdiff_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(768, device="cuda"))
    g = torch.full((768,), 1e-12, device="cuda")
    g[0] = 1e3
    g[600] = float("nan")
    p.grad = g
    opt = AdamW([p], state_bits=8)
    opt.step()
    st = opt.state[p]
    assert bool((st["exp_avg_sq_root"].view(torch.uint8)[:512] > 0).all())
    assert torch.isnan(st["exp_avg_scale"]).tolist() == [False, False, True]
    assert torch.isnan(p).nonzero().flatten().tolist() == [600]
    p.grad = torch.full((768,), 1e-3, device="cuda")
    opt.step()
    assert torch.isnan(p).tolist() == [False] * 512 + [True] * 256


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradient_and_zero_state(bits):
    from hypdiff_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.zeros(300, device="cuda")
    AdamW([p], lr=0.5, weight_decay=0.5, state_bits=bits).step()
    assert torch.equal(p.detach(), torch.full_like(p, 0.75))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_skipped_gradients_groups_and_padding(bits):
    """More tensors than one launch takes, two groups with their own options, parameters that miss steps: each tensor must
    come out as if it were alone in an optimizer (its own step count), and the state's padding stays zero."""
    from hypdiff_amd.optim import AdamW
    shapes = [(5 + 3 * i,) for i in range(200)]
    a, b = _params(torch.float32, shapes, seed=1), _params(torch.float32, shapes, seed=1)
    groups = [{"params": a[:150]}, {"params": a[150:], "lr": 3e-3, "weight_decay": 0.0}]
    many = AdamW(groups, state_bits=bits, **H)
    one = [AdamW([p], state_bits=bits, **(H if i < 150 else {**H, "lr": 3e-3, "weight_decay": 0.0})) for i, p in enumerate(b)]
    for t in range(3):
        for i, (p, q) in enumerate(zip(a, b)):
            if i % 7 == t:
                p.grad = q.grad = None
            else:
                p.grad = torch.sin(torch.arange(p.numel(), device="cuda") * (1.0 + i + t))
                q.grad = p.grad.clone()
        many.step()
        for o in one:
            o.step()
    for i, (p, q) in enumerate(zip(a, b)):
        assert torch.equal(p, q), i
        assert many.state[p]["step"] == one[i].state[q]["step"]
    for gi in (0, 1):
        fl = many._flats[gi]
        live = torch.zeros(fl.total, dtype=torch.bool, device="cuda")
        for f, n in zip(fl.first, fl.numels):
            live[f:f + n] = True
        for k, buf in fl.buffers.items():
            if not k.endswith("_scale"):
                assert int(buf.view(torch.uint8 if bits == 8 else torch.int32)[~live].ne(0).sum()) == 0, k


@gpu
@pytest.mark.parametrize("bits,dtype,master", [(32, torch.float32, False), (8, torch.bfloat16, True)])
def test_state_dict_round_trip_and_types(bits, dtype, master):
    from hypdiff_amd.optim import AdamW
    a = _params(dtype, seed=5)
    opt = AdamW(a, state_bits=bits, master_weights=master, **H)
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    other = AdamW(b, lr=1.0, state_bits=bits, master_weights=master)
    other.load_state_dict(sd)
    opt.step()
    other.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q) and other.state[q]["step"] == 2
    for k, buf in opt.state_buffers().items():
        assert torch.equal(buf.view(torch.uint8), other.state_buffers()[k].view(torch.uint8)), k


@gpu
def test_loads_a_state_of_torchs_adamw():
    from hypdiff_amd.optim import AdamW
    a = _params(torch.float32, seed=6)
    ref = torch.optim.AdamW(a, **H)
    ref.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    opt = AdamW(b)
    opt.load_state_dict(ref.state_dict())
    ref.step()
    opt.step()
    for p, q in zip(a, b):     # both a handful of fp32 roundings from the formula: 2 * 20 u of the larger of |p| and lr
        assert torch.all((p - q).abs() <= 40 * 2.0 ** -24 * torch.clamp(p.abs(), min=H["lr"] * 1.5)), (p - q).abs().max()


@gpu
def test_offsets_beyond_32_bits():
    """a tensor of 2^32 + 300 elements, alike everywhere: every element takes the step that a small tensor's take"""
    from hypdiff_amd.optim import AdamW
    out = []
    for n in ((1 << 32) + 300, 300):
        p = torch.nn.Parameter(torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16))
        p.grad = torch.full((n,), -0.25, device="cuda", dtype=torch.bfloat16)
        opt = AdamW([p], state_bits=8, **H)
        opt.step()
        opt.step()
        out.append((p.detach(), opt.state_buffers()["exp_avg"].view(torch.uint8)[:n]))
    for big, small in zip(*out):
        assert bool((small == small[0]).all()) and float(small[0]) != 0.5
        for k in range(0, big.numel(), 1 << 30):
            assert bool((big[k:k + (1 << 30)] == small[0]).all())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_on_the_device(bits):
    from hypdiff_amd.optim import AdamW
    a, b = _params(torch.float32, seed=7), _params(torch.float32, seed=7)
    o1, o2 = AdamW(a, state_bits=bits, **H), AdamW(b, state_bits=bits, **H)
    for _ in range(2):
        o1.step()
        o2.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o1.step()
    for k in range(3):
        graph.replay()
        o1.replayed()
        o2.step()
        for p, q in zip(a, b):
            # eager: corrections rounded from the host's pow, replay: from the device's, at most one fp32 step apart each
            # (the moments and their codes do not depend on them: equal bits)
            tol = 8 * 2.0 ** -24 * torch.clamp(p.abs(), min=H["lr"] * 8)
            assert torch.all((p - q).abs() <= tol * (k + 1)), (k, (p - q).abs().max())
            for name in (x for x in o1.state[p] if x != "step"):
                assert torch.equal(o1.state[p][name].view(torch.uint8), o2.state[q][name].view(torch.uint8)), name
    o1.step()                                             # eager again: the device's count goes on
    assert o1.state_dict()["state"][0]["step"] == 6


@gpu
@pytest.mark.parametrize("bits,dtype,master", [(32, torch.float32, False), (8, torch.bfloat16, True)])
def test_a_state_loaded_after_a_capture_is_the_one_that_replays_continue(bits, dtype, master):
    from hypdiff_amd.optim import AdamW
    a, b = _params(dtype, seed=8), _params(dtype, seed=8)
    make = lambda ps: AdamW(ps, state_bits=bits, master_weights=master, **H)  # noqa: E731
    o1, o2 = make(a), make(b)
    o1.step()
    o2.step()
    sd, weights = copy.deepcopy(o2.state_dict()), [p.detach().clone() for p in b]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o1.step()
    for _ in range(3):
        graph.replay()
        o1.replayed()
    with torch.no_grad():
        for p, w in zip(a, weights):
            p.copy_(w)
    o1.load_state_dict(sd)
    junk = torch.full((1 << 22,), 7.0, device="cuda")     # would land in memory that the load had let go of
    assert o1.state_dict()["state"][0]["step"] == 1
    for k in range(2):
        graph.replay()
        o1.replayed()
        o2.step()
        for p, q in zip(a, b):                            # as test_captured_step_counts_on_the_device; 16-bit: half a step more
            u = torch.finfo(p.dtype).eps if p.dtype != torch.float32 else 0.0
            tol = (8 * 2.0 ** -24 * (k + 1) + u) * torch.clamp(p.abs(), min=H["lr"] * 8).double()
            assert torch.all((p.double() - q.double()).abs() <= tol)
            for name in (x for x in o1.state[p] if x not in ("step", "master")):
                assert torch.equal(o1.state[p][name].view(torch.uint8), o2.state[q][name].view(torch.uint8)), name
    assert torch.all(junk == 7.0)
    with pytest.raises(RuntimeError, match="captured"):
        o1.load_state_dict(AdamW(b, state_bits=40 - bits, **H).state_dict())


@gpu
def test_loading_its_own_state_changes_nothing_and_a_refused_state_neither():
    from hypdiff_amd.optim import AdamW
    a = _params(torch.bfloat16, seed=9)
    opt = AdamW(a, state_bits=8, master_weights=True, **H)
    opt.step()
    opt.step()
    before = {k: v.view(torch.uint8).clone() for k, v in opt.state_buffers().items()}
    opt.load_state_dict(opt.state_dict())
    broken = copy.deepcopy(opt.state_dict())
    del broken["state"][len(a) - 1]["exp_avg_scale"]
    with pytest.raises(ValueError, match="exp_avg_scale"):
        opt.load_state_dict(broken)
    for k, v in opt.state_buffers().items():
        assert torch.equal(v.view(torch.uint8), before[k]), k
    assert all(opt.state[p]["step"] == 2 for p in a)


def test_refusals_on_the_host():
    from hypdiff_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                dict(state_bits=16), dict(betas=(0.9,))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    with pytest.raises(TypeError):
        AdamW([p], lr=torch.tensor(1e-3))
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(4, 6).t())])
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        AdamW([p]).step()
    with pytest.raises(TypeError, match="state_dict"):
        copy.deepcopy(AdamW([p]))
    sd = torch.optim.AdamW([p], amsgrad=True).state_dict()
    with pytest.raises(ValueError, match="amsgrad"):
        AdamW([p]).load_state_dict(sd)


def test_refusals_of_the_entry_point():
    """Bad arguments come back as a status before anything is launched (no GPU needed)."""
    from hypdiff_amd import _lib
    from hypdiff_amd.optim import _JOB

    def call(job=(256, 256, 0, 100, 0), n=1, dt=0, bits=32, m=256, v=256, ms=None, vs=None, master=None, total=256, lr=1e-3,
             b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1, table=None, rows=0):
        a = np.array([job] * max(n, 1), dtype=_JOB)
        _lib.call("hd_adamw_step", a.ctypes.data, n, dt, bits, m, v, ms, vs, master, total, lr, b1, b2, eps, wd, step, table,
                  rows, None)
    for bad, what in ((dict(n=-1), "jobs"), (dict(n=1000), "jobs"), (dict(dt=7), "element type"), (dict(bits=16), "bits"),
                      (dict(master=256), "own master"), (dict(b1=1.0), "hyper"), (dict(step=0), "step"), (dict(total=100), "whole blocks"),
                      (dict(job=(0, 256, 0, 100, 0)), "null"), (dict(job=(256, 256, 0, -1, 0)), "null"),
                      (dict(job=(258, 256, 0, 100, 0)), "aligned"), (dict(job=(256, 256, 100, 100, 0)), "segment"),
                      (dict(job=(256, 256, 0, 257, 0)), "segment"), (dict(job=(256, 256, 256, 1, 0)), "segment"),
                      (dict(table=256, rows=1, job=(256, 256, 0, 100, 1)), "row"), (dict(bits=8), "null state"),
                      (dict(m=None), "null state"), (dict(m=260), "16-byte")):
        with pytest.raises(RuntimeError, match=what):
            call(**bad)


BAD_STEPS = [None, -1, 1.5, float("nan"), float("inf"), "3", True, torch.tensor([1.0, 2.0]), torch.tensor(-2.0), torch.tensor(float("nan"))]


def _saved_step(sd, k, step):
    sd = {"state": {i: dict(st) for i, st in sd["state"].items()}, "param_groups": [dict(g, lr=0.5) for g in sd["param_groups"]]}
    if step is None:
        del sd["state"][k]["step"]
    else:
        sd["state"][k]["step"] = step
    return sd


def test_a_state_without_a_step_is_refused_before_anything_changes():
    from hypdiff_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    opt = AdamW([p], lr=1e-3)
    whole = {"state": {0: {"step": 1, "exp_avg": torch.zeros(4), "exp_avg_sq": torch.zeros(4)}}, "param_groups": opt.state_dict()["param_groups"]}
    for bad in BAD_STEPS:
        with pytest.raises(ValueError, match="step"):
            opt.load_state_dict(_saved_step(whole, 0, bad))
    for entry in (None, 3.0, torch.zeros(4, dtype=torch.complex64)):
        sd = _saved_step(whole, 0, 1)
        sd["state"][0]["exp_avg_sq"] = entry
        with pytest.raises(TypeError, match="exp_avg_sq"):
            opt.load_state_dict(sd)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.load_state_dict(_saved_step(whole, 0, torch.tensor(2.0)))
    assert opt.param_groups[0]["lr"] == 1e-3 and not opt.state


@gpu
@pytest.mark.parametrize("captured", [False, True])
def test_a_refused_step_changes_nothing_on_the_device(captured):
    from hypdiff_amd.optim import AdamW
    a = _params(torch.bfloat16, seed=9)
    opt = AdamW(a, state_bits=8, master_weights=True, **H)
    opt.step()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    if captured:
        with torch.cuda.graph(graph):
            opt.step()
        graph.replay()
    sd = copy.deepcopy(opt.state_dict())
    before = {k: v.view(torch.uint8).clone() for k, v in opt.state_buffers().items()}
    table = opt._flats[0].table.clone()
    for bad in BAD_STEPS:
        with pytest.raises(ValueError, match="step"):
            opt.load_state_dict(_saved_step(sd, len(a) - 2, bad))
    for k, v in opt.state_buffers().items():
        assert torch.equal(v.view(torch.uint8), before[k]), k
    assert torch.equal(opt._flats[0].table, table) and opt.param_groups[0]["lr"] == H["lr"]
    assert opt.state_dict()["state"][0]["step"] == 2 + captured
    opt.load_state_dict(sd)
    if captured:
        graph.replay()
        assert opt.state_dict()["state"][0]["step"] == 4


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate")
def test_a_parameter_twice_is_refused():
    """one launch would read and write it from two places at once"""
    from hypdiff_amd.optim import AdamW
    p, q = (torch.nn.Parameter(torch.zeros(n)) for n in (600, 4))
    with pytest.raises(ValueError, match="twice"):
        AdamW([p, q, p])
    opt = AdamW([p])
    with pytest.raises(ValueError, match="twice"):
        opt.add_param_group({"params": [q, q]})
    assert len(opt.param_groups) == 1
    base = torch.zeros(600)
    apart = [torch.nn.Parameter(base[:300]), torch.nn.Parameter(base[300:]), torch.nn.Parameter(torch.zeros(0)), q]
    AdamW._check_apart(apart)
    with pytest.raises(ValueError, match="share memory"):
        AdamW._check_apart(apart + [torch.nn.Parameter(base[299:301])])


@gpu
def test_parameters_that_share_memory_are_refused():
    from hypdiff_amd.optim import AdamW
    base = torch.zeros(600, device="cuda")
    ps = [torch.nn.Parameter(base[:301]), torch.nn.Parameter(base[300:])]
    for p in ps:
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="share memory"):
        AdamW(ps).step()
    assert not base.any()
    ps = [torch.nn.Parameter(base[:300]), torch.nn.Parameter(base[300:])]
    for p in ps:
        p.grad = torch.ones_like(p)
    AdamW(ps, lr=0.5, weight_decay=0.0).step()          # neighbours in one buffer: m / sqrt(v) = 1
    assert float((base + 0.5).abs().max()) <= 0.5 * 16 * 2.0 ** -24 + 0.5e-8

"""ops.linear_act (csrc/gemm_half.hip): forward and gradients of resid + act(x W^T + b) on 16-bit operands against 64 bits,
over sizes, layouts and types; NaN and infinities; the same bits on every call; refusals; captured and replayed."""
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step, relative
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}             # half of fp16's smallest step


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _act64(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def _reference(x, w, b, r, g, act, dtype):
    """Results in 64 bits and what each may be off by, from arithmetic:

    z     K products of 16-bit numbers are exact in fp32; their sum in any order is off by K u sum|x w|, the bias by one
          more rounding: ez.
    y     act is 1.13-Lipschitz (GELU) and evaluated to 2e-6 |z| (the kernel's fit of erfc) + 4 u |z|, the residual one
          rounding, storage half a step.
    dz    z was stored in fp16 (its relative half step and smallest step), g times a slope that moves by at most 0.8 per
          unit of z, except at ReLU's border, where an element within the error of 0 may count or not; the product and the
          slope's evaluation (2e-6 for erfc, 8 u for the rest): 2.5e-6 |g|; storage of dz another h.
    dx dw db   sums of those errors against |W|, |x|, 1, and the sum's own roundings."""
    h, tiny = HALF[dtype], TINY[dtype]
    K = x.shape[1]
    z = x @ w.t()
    ez = (K + 1) * U * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b
        ez = ez + U * b.abs()
    a, slope = _act64(z, act)
    y = a if r is None else a + r
    ey = 1.13 * ez + 2.3e-6 * z.abs() + U * y.abs()
    out = {"y": (y, ey * (1 + h) + h * y.abs() + tiny)}
    if g is None:
        return out
    moved = ez * (1 + h) + (0.0 if act == "identity" else HALF[torch.float16]) * z.abs() + TINY[torch.float16]
    if act == "relu":
        ds = (z.abs() <= moved).double()
    else:
        ds = (0.8 * moved) if act == "gelu" else torch.zeros_like(z)
    dz = g * slope
    ed = g.abs() * (ds + (2.5e-6 if act == "gelu" else 0.0))
    ed16 = ed + h * (dz.abs() + ed) + tiny
    n = lambda k: (k + 1) * U  # noqa: E731
    for key, val, err, size, k in (("dx", dz @ w, ed16 @ w.abs(), (dz.abs() + ed16) @ w.abs(), w.shape[0]),
                                   ("dw", dz.t() @ x, ed16.t() @ x.abs(), (dz.abs() + ed16).t() @ x.abs(), x.shape[0]),
                                   ("db", dz.sum(0), ed.sum(0), (dz.abs() + ed).sum(0), x.shape[0])):
        e = err + n(k) * size
        out[key] = (val, e * (1 + h) + h * val.abs() + tiny)
    return out


def _check(got, want, bound, what):
    got = got.detach().double()
    assert got.shape == want.shape, what
    over = (got - want).abs() - bound
    assert not bool((over > 0).any()) and not bool(torch.isnan(got).any()), \
        (what, float(over.max()), float(((got - want).abs() / bound.clamp(min=1e-300)).max()))


def _run(M, N, K, dtype, act, bias, resid, seed, pitch=0, lead=None, w_pitch=0, g_kind="dense"):
    from hypdiff_amd import ops
    gen = _gen(seed)
    x = torch.randn(M, K + pitch, device="cuda", generator=gen).to(dtype)[:, pitch // 2:pitch // 2 + K]
    w = (torch.randn(N, K + w_pitch, device="cuda", generator=gen) / math.sqrt(K)).to(dtype)[:, :K]
    b = torch.randn(N, device="cuda", generator=gen).to(dtype) if bias else None
    r = torch.randn(M, N, device="cuda", generator=gen).to(dtype) if resid else None
    g = torch.randn(M, N, device="cuda", generator=gen).to(dtype)
    if g_kind == "slice":
        g = torch.randn(M, N + 3, device="cuda", generator=gen).to(dtype)[:, 2:N + 2]
    elif g_kind == "row":
        g = g[:1].expand(M, N)
    if lead is not None:
        x, g = x.reshape(lead + (K,)), g.reshape(lead + (N,))
        r = None if r is None else r.reshape(lead + (N,))
    leaves = {"dx": x, "dw": w}
    if bias:
        leaves["db"] = b
    if resid:
        leaves["dr"] = r
    leaves = {k: t.detach().requires_grad_(True) for k, t in leaves.items()}
    y0 = ops.linear_act(x, w, b, act=act, resid=r)
    y = ops.linear_act(leaves["dx"], leaves["dw"], leaves.get("db"), act=act, resid=leaves.get("dr"))
    assert torch.equal(y0, y) and y.dtype == dtype
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), g)))
    d = lambda t, c: None if t is None else t.reshape(-1, c).double()  # noqa: E731
    want = _reference(d(x, K), w.double(), None if b is None else b.double(), d(r, N), d(g, N), act, dtype)
    _check(y.reshape(-1, N), *want["y"], "y")
    for k in ("dx", "dw") + (("db",) if bias else ()):
        assert grads[k].dtype == dtype and grads[k].shape == leaves[k].shape
        _check(grads[k].reshape(want[k][0].shape), *want[k], k)
    if resid:
        assert torch.equal(grads["dr"], g)
    y2 = ops.linear_act(leaves["dx"], leaves["dw"], leaves.get("db"), act=act, resid=leaves.get("dr"))
    for k, t in zip(leaves, torch.autograd.grad(y2, list(leaves.values()), g)):
        assert torch.equal(t, grads[k]), k               # no order of sums to differ in


SIZES = [(1, 1, 1), (700, 90, 3), (5000, 5, 7), (3, 9, 8), (1, 512, 512), (2, 7, 5), (15, 16, 17), (16, 8, 8), (33, 40, 24), (64, 64, 64), (127, 129, 72), (128, 128, 128),
         (130, 136, 264), (200, 512, 512), (200, 64, 512), (200, 512, 64), (257, 300, 513), (1000, 14, 15), (300, 900, 800),
         (2049, 72, 88), (4100, 260, 136)]


@gpu
@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sizes(M, N, K, dtype):
    k = SIZES.index((M, N, K))
    _run(M, N, K, dtype, ("gelu", "relu", "identity")[k % 3], k % 4 != 3, k % 2 == 0, k)


# outputs narrower than a chunk beside inputs that have to be staged through registers; few and many rows
@gpu
@pytest.mark.parametrize("M,N,K", [(50, 5, 13), (3000, 1, 41), (9000, 7, 129), (700, 3, 515), (1, 6, 9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_narrow_outputs_of_odd_inputs(M, N, K, dtype):
    _run(M, N, K, dtype, "relu", True, False, 21)
    _run(M, N, K, dtype, "identity", True, True, 22)


@gpu
@pytest.mark.parametrize("act", ["gelu", "relu", "identity"])
@pytest.mark.parametrize("bias,resid", [(False, False), (True, True)])
def test_activations_and_epilogues(act, bias, resid):
    _run(300, 200, 160, torch.bfloat16, act, bias, resid, 5)
    _run(70, 99, 161, torch.float16, act, bias, resid, 6)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layouts(dtype):
    """pitched rows (aligned, odd, starting off a 16-byte border), pitched weights, leading axes, gradients that are slices
    or one row for all"""
    _run(140, 136, 128, dtype, "gelu", True, True, 1, pitch=8)
    _run(140, 136, 128, dtype, "gelu", True, False, 2, pitch=16)
    _run(140, 136, 128, dtype, "relu", True, True, 3, pitch=37, w_pitch=1)
    _run(140, 136, 128, dtype, "gelu", True, True, 4, w_pitch=24, g_kind="slice")
    _run(140, 136, 128, dtype, "identity", True, True, 5, g_kind="row")
    _run(140, 133, 120, dtype, "gelu", True, True, 6, lead=(4, 5, 7))
    _run(140, 136, 128, dtype, "identity", True, False, 7, pitch=3, g_kind="slice")


@gpu
def test_transposed_and_strided_operands():
    from hypdiff_amd import ops
    gen = _gen(9)
    x = torch.randn(96, 50, device="cuda", generator=gen).bfloat16()
    w = torch.randn(96, 80, device="cuda", generator=gen).bfloat16()
    for xs, wsx in ((x.t(), w.t()), (x.t()[::2], w.t()[::3])):
        got = ops.linear_act(xs, wsx)
        assert torch.equal(got, ops.linear_act(xs.contiguous(), wsx.contiguous()))
    row = torch.randn(96, device="cuda", generator=gen).bfloat16()
    assert torch.equal(ops.linear_act(row, w.t()), ops.linear_act(row[None], w.t())[0])
    one = ops.linear_act(row.expand(40, 96), w.t(), resid=row[:80].expand(40, 80))
    assert torch.equal(one, one[:1].expand_as(one))


@gpu
@pytest.mark.parametrize("M,N", [(40, 72), (300, 136), (5000, 264), (20000, 520), (130, 33)])
def test_skip_connection(M, N):
    """resid is x: the skip's gradient is added to dx in fp32, before its one rounding"""
    from hypdiff_amd import ops
    gen = _gen(M)
    x = torch.randn(M, N, device="cuda", generator=gen).bfloat16().requires_grad_(True)
    w = (torch.randn(N, N, device="cuda", generator=gen) / math.sqrt(N)).bfloat16().requires_grad_(True)
    g = torch.randn(M, N, device="cuda", generator=gen).bfloat16()
    y = ops.linear_act(x, w, act="gelu", resid=x)
    dx, dw = torch.autograd.grad(y, [x, w], g)
    xd, wd, gd = x.detach().double(), w.detach().double(), g.double()
    want = _reference(xd, wd, None, xd, gd, "gelu", torch.bfloat16)
    _check(y, *want["y"], "y")
    _check(dw, *want["dw"], "dw")
    v, e = want["dx"]
    h = HALF[torch.bfloat16]
    _check(dx, v + gd, e - h * v.abs() + (h + 2 * U) * (v + gd).abs(), "dx")
    only = torch.autograd.grad(ops.linear_act(x, w.detach(), act="relu", resid=x), [x], g)[0]
    apart = x.detach().requires_grad_(True)
    other = torch.autograd.grad(ops.linear_act(apart, w.detach(), act="relu", resid=x.detach()), [apart], g)[0]
    assert float((only.double() - other.double() - gd).abs().max()) <= 2 * h * float((other.double().abs() + gd.abs()).max())


@gpu
def test_no_rows():
    from hypdiff_amd import ops
    x = torch.zeros(0, 24, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(16, 24, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = torch.randn(16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = ops.linear_act(x, w, b, act="gelu", resid=torch.zeros(0, 16, device="cuda", dtype=torch.bfloat16))
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.zeros(0, 16, device="cuda", dtype=torch.bfloat16))
    assert dx.shape == (0, 24) and not dw.any() and not db.any()


@gpu
@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_large_and_tiny_preactivations_keep_their_slope(act):
    """z far outside fp16 (it is kept clamped) has slope 0 or 1; a tiny positive z counts for ReLU; an infinite y is passed on"""
    from hypdiff_amd import ops
    x = torch.tensor([[3e38], [1e30], [7e4], [1e-30], [-1e-30], [-7e4], [-1e30]], device="cuda").bfloat16().requires_grad_(True)
    w = torch.ones(8, 1, device="cuda", dtype=torch.bfloat16)
    y = ops.linear_act(x, w, act=act)
    dx = torch.autograd.grad(y, [x], torch.ones(7, 8, device="cuda", dtype=torch.bfloat16))[0].flatten().tolist()
    small = (0.5, 0.5) if act == "gelu" else (1.0, 0.0)
    assert dx == [8.0, 8.0, 8.0, 8 * small[0], 8 * small[1], 0.0, 0.0]
    assert torch.equal(y[:3, 0], x.detach()[:3, 0]) and float(y.detach()[5:].abs().max()) == 0.0


@gpu
@pytest.mark.parametrize("K", [64, 65, 200])
def test_nonfinite_values_stay_in_their_row_and_column(K):
    from hypdiff_amd import ops
    gen = _gen(11)
    x = torch.randn(150, K, device="cuda", generator=gen).bfloat16()
    w = torch.randn(140, K, device="cuda", generator=gen).bfloat16()
    clean = ops.linear_act(x, w, act="relu")
    x[149, K - 1], x[3, 0] = float("nan"), float("inf")
    w[139, 1] = float("nan")
    got = ops.linear_act(x, w, act="relu")
    hit = torch.zeros(150, 140, dtype=torch.bool, device="cuda")
    hit[149] = True
    hit[3] = True
    hit[:, 139] = True
    assert bool(torch.isnan(got[149]).all()) and bool(torch.isnan(got[:, 139]).all())
    assert torch.equal(got[~hit], clean[~hit])


@gpu
@pytest.mark.parametrize("act", ["relu", "identity"])
def test_nonfinite_gradients(act):
    """an infinite gradient stays in its row; behind a closed ReLU it is gone; a NaN pre-activation passes the gradient on"""
    from hypdiff_amd import ops
    x = torch.tensor([[-1.0], [1.0], [1.0], [float("nan")]], device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(9, 1, device="cuda", dtype=torch.bfloat16)
    g = torch.ones(4, 9, device="cuda", dtype=torch.bfloat16)
    g[0, 2] = g[1, 3] = float("inf")
    dx = torch.autograd.grad(ops.linear_act(x, w, act=act), [x], g)[0].flatten().tolist()
    assert dx == [0.0 if act == "relu" else float("inf"), float("inf"), 9.0, 9.0]


@gpu
def test_offsets_beyond_32_bits():
    """x and dx of 4.4 GB: the last rows come out like the formula's, and dW sees them (all others are zeros)"""
    from hypdiff_amd import ops
    gen = _gen(15)
    M, N, K, last = (1 << 22) + 3, 8, 520, 5
    x = torch.zeros(M, K, device="cuda", dtype=torch.bfloat16)
    x[-last:] = torch.randn(last, K, device="cuda", generator=gen).bfloat16()
    w = (torch.randn(N, K, device="cuda", generator=gen) / math.sqrt(K)).bfloat16().requires_grad_(True)
    g = torch.randn(M, N, device="cuda", generator=gen).bfloat16()
    x.requires_grad_(True)
    y = ops.linear_act(x, w, act="gelu")
    dx, dw = torch.autograd.grad(y, [x, w], g)
    d = lambda t: t.detach()[-last:].double()  # noqa: E731
    want = _reference(d(x), w.detach().double(), None, None, d(g), "gelu", torch.bfloat16)
    _check(y[-last:], *want["y"], "y")
    _check(dx[-last:], *want["dx"], "dx")
    _check(dw, *want["dw"], "dw")


@gpu
def test_gradient_against_differences():
    """L = sum(g * y) along a random direction in x, W, b: central differences in 64 bits of the formula against the
    kernel's gradients: what the gradients may be off by (see _reference) summed along the direction."""
    from hypdiff_amd import ops
    gen = _gen(12)
    x = torch.randn(40, 24, device="cuda", generator=gen).half()
    w = (torch.randn(32, 24, device="cuda", generator=gen) / 5).half()
    b = torch.randn(32, device="cuda", generator=gen).half()
    g = torch.randn(40, 32, device="cuda", generator=gen).half()
    ls = [t.detach().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.linear_act(*ls, act="gelu"), ls, g)
    want = _reference(x.double(), w.double(), b.double(), None, g.double(), "gelu", torch.float16)
    for k, (t, gr) in enumerate(zip((x, w, b), grads)):
        d = torch.randn(t.shape, device="cuda", generator=gen, dtype=torch.float64)
        h = 1e-4

        def loss(s):
            ops64 = [v.double() for v in (x, w, b)]
            ops64[k] = ops64[k] + s * d
            return float((_act64(ops64[0] @ ops64[1].t() + ops64[2], "gelu")[0] * g.double()).sum())
        diff = (loss(h) - loss(-h)) / (2 * h)
        bound = float((want[("dx", "dw", "db")[k]][1] * d.abs()).sum())
        assert abs(diff - float((gr.double() * d).sum())) <= bound + 1e-5 * abs(diff) + 1e-5


@gpu
@pytest.mark.parametrize("M,N,K", [(200, 136, 128), (70, 33, 41)])
def test_captured_and_replayed(M, N, K):
    from hypdiff_amd import ops
    gen = _gen(13)
    new = lambda *s: torch.randn(*s, device="cuda", generator=gen).bfloat16()  # noqa: E731
    x, w, b, g = new(M, K), new(N, K), new(N), new(M, N)

    def both():
        ls = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.linear_act(*ls, act="gelu")
        return (y.detach(),) + torch.autograd.grad(y, ls, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(3):
        for t in (x, w, b, g):
            t.copy_(new(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, both()):
            assert torch.equal(a, c)


@gpu
def test_two_streams_at_once():
    from hypdiff_amd import ops
    gen = _gen(14)
    new = lambda *s: torch.randn(*s, device="cuda", generator=gen).bfloat16()  # noqa: E731
    sets = [(new(3000, 512), new(512, 512), new(512), new(3000, 512)) for _ in range(2)]

    def step(x, w, b, g):
        ls = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.linear_act(*ls, act="gelu")
        return (y.detach(),) + torch.autograd.grad(y, ls, g)
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([step(*s) for _ in range(5)])
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        for o in outs:
            assert all(torch.equal(a, c) for a, c in zip(o, w))


@gpu
def test_second_derivatives_are_refused():
    from hypdiff_amd import ops
    x, w = (torch.randn(8, 8, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    with pytest.raises(NotImplementedError, match="create_graph"):
        torch.autograd.grad(ops.linear_act(x, w, act="gelu").sum(), [x], create_graph=True)
    with pytest.raises(NotImplementedError, match="create_graph"):
        torch.autograd.grad(ops.embedding(torch.zeros(1, dtype=torch.int64, device="cuda"), w).sum(), [w], create_graph=True)


def test_refusals_on_the_host():
    from hypdiff_amd import ops
    x, w = torch.zeros(3, 4).bfloat16(), torch.zeros(5, 4).bfloat16()
    for args, kw, err in (((x.float(), w.float()), {}, TypeError), ((x, w.half()), {}, TypeError), ((x, w[0]), {}, ValueError),
                          ((x, w[:, :3]), {}, ValueError), ((x, w[:0]), {}, ValueError), ((x, w), dict(act="silu"), ValueError),
                          ((x, w, torch.zeros(4).bfloat16()), {}, ValueError), ((x, w, torch.zeros(5)), {}, TypeError),
                          ((x, w), dict(resid=torch.zeros(5).bfloat16()), ValueError),
                          ((x, w), dict(resid=torch.zeros(3, 5)), TypeError)):
        with pytest.raises(err, match="linear_act"):
            ops.linear_act(*args, **kw)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_act(x, w)


def test_refusals_of_the_entry_points():
    from hypdiff_amd import _lib

    def fwd(x=256, ldx=16, w=256, ldw=16, bias=None, resid=None, ldr=0, dt=1, M=4, N=8, K=16, act=0, y=256, z=None):
        _lib.call("hd_linear_act_fwd", x, ldx, w, ldw, bias, resid, ldr, dt, M, N, K, act, y, z, None)

    def bwd(g=256, ldg=8, z=256, x=256, ldx=16, w=256, ldw=16, dt=1, M=4, N=8, K=16, act=6, add=None, dx=256, dw=256, db=256,
            ws=256, nbytes=1 << 30):
        _lib.call("hd_linear_act_bwd", g, ldg, z, x, ldx, w, ldw, dt, M, N, K, act, add, 16, dx, dw, db, ws, nbytes, None)
    for fn in (fwd, bwd):
        for bad, what in ((dict(dt=0), "element type"), (dict(act=2), "activation"), (dict(M=-1), "shape"), (dict(N=0), "shape"),
                          (dict(K=0), "shape"), (dict(M=1 << 30), "shape"), (dict(ldx=15), "pitch"), (dict(ldw=15), "pitch"),
                          (dict(x=257), "aligned"), (dict(x=None), "null|needs")):
            with pytest.raises(RuntimeError, match=what):
                fn(**bad)
    for bad, what in ((dict(ws=None), "workspace"), (dict(nbytes=16), "workspace of"), (dict(M=0), "no rows"), (dict(z=None), "null"),
                      (dict(ldg=7), "pitch"), (dict(w=None), "needs"), (dict(add=256, dx=None), "dx_add"), (dict(add=257), "aligned")):
        with pytest.raises(RuntimeError, match=what):
            bwd(**bad)
    assert _lib.load().hd_linear_act_bwd_workspace_bytes(1 << 30, 8, 8, 6) == 0


@gpu
@pytest.mark.filterwarnings("ignore:.*torch.jit:DeprecationWarning")
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(grad):
    """a tangent may not get lost, whether or not an operand requires a gradient; operands without one pass"""
    import torch.autograd.forward_ad as fwd
    from hypdiff_amd import ops
    x, w = (torch.randn(8, 8, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    idx = torch.arange(8, device="cuda")
    y, e = ops.linear_act(x, w, act="gelu"), ops.embedding(idx, w, add=x)
    w.requires_grad_(grad)
    with fwd.dual_level():
        assert torch.equal(ops.linear_act(x, w, act="gelu"), y) and torch.equal(ops.embedding(idx, w, add=x), e)
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.linear_act(dual, w), lambda: ops.linear_act(x, w, resid=dual), lambda: ops.linear_act(x, dual),
                     lambda: ops.linear_act(x, w, dual[0]), lambda: ops.linear_act(dual, w, resid=dual),
                     lambda: ops.embedding(idx, dual), lambda: ops.embedding(idx, w, add=dual)):
            with pytest.raises(NotImplementedError, match="forward mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                call()


@gpu
@pytest.mark.parametrize("M,N,K,pitch,w_pitch", [(300, 136, 128, 37, 5), (300, 136, 128, 0, 8), (40, 33, 41, 7, 0), (3000, 264, 200, 24, 16)])
def test_saved_tensors_that_change_their_layout(M, N, K, pitch, w_pitch):
    """hooks on saved tensors bring back contiguous copies of pitched operands (save_on_cpu), or pitched ones of contiguous: the
    same gradients; a hook that changes the type is refused"""
    from hypdiff_amd import ops
    gen = _gen(16)
    x = torch.randn(M, K + pitch, device="cuda", generator=gen).bfloat16()[:, :K].detach().requires_grad_(True)
    w = torch.randn(N, K + w_pitch, device="cuda", generator=gen).bfloat16()[:, :K].detach().requires_grad_(True)
    g = torch.randn(M, N, device="cuda", generator=gen).bfloat16()
    run = lambda act: torch.autograd.grad(ops.linear_act(x, w, act=act), [x, w], g)  # noqa: E731

    def widen(t):
        big = torch.full((t.shape[0], t.shape[1] + 9), float("nan"), device="cuda", dtype=t.dtype)
        big[:, 3:3 + t.shape[1]] = t
        return big[:, 3:3 + t.shape[1]]
    for act in ("gelu", "identity"):
        want = run(act)
        for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, widen),
                      torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t)):
            with hooks:
                got = run(act)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()), pytest.raises(RuntimeError, match="came back"):
        run("gelu")


def test_grids_beyond_the_limit_are_refused():
    """an input narrower than a chunk takes 32 x 32 tiles whatever their number: 2^24 of them are 2^32 threads, which no grid
    holds (no GPU needed: refused before anything is launched)"""
    from hypdiff_amd import _lib

    def fwd(M, N, K):
        _lib.call("hd_linear_act_fwd", 256, K, 256, K, None, None, 0, 1, M, N, K, 0, 256, None, None)
    for M, N, K in ((1 << 24, 1024, 3), (1 << 19, 1 << 15, 7), ((1 << 29) - 1, 33, 1), (1 << 26, 4096, 8), (1 << 26, 4096, 9)):
        with pytest.raises(RuntimeError, match="too many tiles"):
            fwd(M, N, K)


def _tiles(M, N, bm, bn):
    return -(-M // bm) * -(-N // bn)


def _kind(M, N, K, direct):
    """the kernel that hd_linear_act_fwd takes (csrc/gemm_half.hip, choose_tiles): 0 the 32 x 32 one, then by tile size"""
    if (K < 8 and not direct) or _tiles(M, N, 32, 32) <= (512 if direct else 64):
        return 0
    cost = [max(least, start + (per if direct else odd) / 256 * _tiles(M, N, bm, bn)) for bm, bn, start, per, odd, least in (
        (64, 64, 6, 2.85, 3.6, 11), (64, 128, 6, 4.6, 5.4, 13), (128, 128, 8, 8, 8, 18), (128, 192, 8, 12, 12, 20))]
    return 1 + cost.index(min(cost))


# every tile size with rows staged straight to LDS (K a multiple of 8) and through registers, none of the sizes a multiple of a tile
@gpu
@pytest.mark.parametrize("M,N,K,kind", [(4101, 260, 136, 1), (8055, 264, 72, 2), (5003, 776, 200, 2), (7750, 776, 136, 3),
                                        (6225, 904, 104, 4), (9003, 906, 64, 4),
                                        (674, 72, 101, 1), (7994, 201, 67, 2), (5001, 777, 129, 2), (7262, 521, 131, 3), (6164, 905, 77, 4),
                                        (9001, 907, 70, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_tile_size(M, N, K, kind, dtype):
    assert _kind(M, N, K, K % 8 == 0) == kind
    _run(M, N, K, dtype, ("gelu", "relu", "identity")[M % 3], True, M % 2 == 0, M)


# the weight gradient in 192 x 192 tiles (from 8e9 products and 6 tiles on), rows straight to LDS and through registers; also
# the input gradient of a wide layer in the larger tiles
@gpu
@pytest.mark.parametrize("M,N,K", [(20011, 600, 680), (20011, 601, 681), (12007, 1000, 904), (12007, 905, 1001), (41003, 385, 577)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_weight_gradients(M, N, K, dtype):
    assert M * N * K >= 8e9 and _tiles(N, K, 192, 192) >= 6 and M % 64 and N % 192 and K % 192
    _run(M, N, K, dtype, "gelu" if M % 2 else "relu", True, False, N)

"""ops.embedding (csrc/embedding.hip): lookup and table gradient against 64 bits, over types, sizes, layouts, empty and hot
tokens; the same bits on every call; refusals; captured and replayed; next to the fp32 form of ddpm.Backbone."""
import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # storage: half a step, relative
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}            # half of fp16's smallest step


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _idx(rows, T, kind, dtype, seed):
    g = _gen(seed)
    if kind == "one":
        return torch.full((rows,), T - 1, dtype=dtype, device="cuda")
    if kind == "hot":                                    # three quarters on one token, the rest anywhere
        i = torch.randint(0, T, (rows,), device="cuda", generator=g)
        return torch.where(torch.rand(rows, device="cuda", generator=g) < 0.75, T // 3, i).to(dtype)
    return torch.randint(0, T, (rows,), device="cuda", generator=g).to(dtype)


def _check(got, want, size, dtype):
    """|got - want| <= size (the fp32 roundings, in absolute numbers) + the rounding to the storage type"""
    got, want = got.detach().double().cpu(), want.double().cpu()
    bound = size.double().cpu() * (1 + HALF[dtype]) + HALF[dtype] * want.abs() + TINY[dtype] + 1e-300
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), ((got - want).abs() / bound).max()


def _lookup64(idx, table, scale, add):
    y = table.detach().double()[idx.long()] * scale
    size = 3 * U * y.abs()                               # scale to fp32, the product, the sum's share
    if add is not None:
        y = y + add.detach().double()
        size = size + U * y.abs()
    return y, size


def _grad64(idx, g, T, scale, padding):
    idx, g = idx.reshape(-1).cpu().numpy().astype(np.int64), g.reshape(-1, g.shape[-1]).double().cpu().numpy()
    gt, ab, n = np.zeros((T, g.shape[1])), np.zeros((T, g.shape[1])), np.zeros(T)
    ok = (idx >= 0) & (idx < T) & (idx != (-1 if padding is None else padding))
    np.add.at(gt, idx[ok], g[ok])
    np.add.at(ab, idx[ok], np.abs(g[ok]))
    np.add.at(n, idx[ok], 1)
    size = (n[:, None] + 2) * U * ab * abs(scale)        # a sum of n terms in any order: n - 1 roundings; the scale: 2
    return torch.from_numpy(gt * scale), torch.from_numpy(size)


CASES = [  # rows, T, D, index kind
    (1, 1, 1, "any"), (1, 1000, 512, "any"), (3, 2, 7, "any"), (200, 1000, 512, "any"), (257, 17, 700, "hot"), (63, 5000, 33, "any"),
    (4096, 100, 64, "any"), (4097, 100, 65, "any"), (5000, 1, 16, "one"), (20000, 300, 12, "hot"), (30011, 70000, 24, "any"),
    (9000, 255, 1000, "hot"), (9000, 256, 130, "one"), (300000, 40, 8, "hot"), (6000, 1 << 17, 5, "any"),
]


@gpu
@pytest.mark.parametrize("rows,T,D,kind", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lookup_and_gradient(rows, T, D, kind, dtype):
    from hypdiff_amd import ops
    k = CASES.index((rows, T, D, kind))
    idx = _idx(rows, T, kind, torch.int32 if k % 2 else torch.int64, k)
    table = torch.randn(T, D, device="cuda", generator=_gen(k + 1)).to(dtype).requires_grad_(True)
    add = torch.randn(rows, D, device="cuda", generator=_gen(k + 2)).to(dtype).requires_grad_(True) if k % 3 else None
    scale, padding = (1.0, None) if k % 2 else (-1.7, T // 3)
    g = torch.randn(rows, D, device="cuda", generator=_gen(k + 3)).to(dtype)
    y = ops.embedding(idx, table, scale=scale, add=add, padding_idx=padding)
    assert y.dtype == dtype and y.shape == (rows, D)
    _check(y, *_lookup64(idx, table, scale, add), dtype)
    leaves = [table] + ([add] if add is not None else [])
    grads = torch.autograd.grad(y, leaves, g)
    _check(grads[0], *_grad64(idx, g, T, scale, padding), dtype)
    if add is not None:
        assert torch.equal(grads[1], g)
    again = torch.autograd.grad(ops.embedding(idx, table, scale=scale, add=add, padding_idx=padding), [table], g)[0]
    assert torch.equal(again, grads[0])                  # the order of the sums is fixed


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """pitched tables, transposed tables, scalar and 2-D indices, strided indices, gradients that are slices, transposes or
    expanded, and the autograd of a broadcast add"""
    from hypdiff_amd import ops
    wide = torch.randn(50, 41, device="cuda", generator=_gen(0)).to(dtype)
    for table in (wide[:, 3:36], wide.t()[3:36], wide[::2, 1:]):
        table = table.detach().requires_grad_(True)
        T, D = table.shape
        base = torch.randint(0, T, (6, 22), device="cuda", generator=_gen(1))
        for idx in (base[0, 0], base, base[:, ::2], base.t(), base[:0]):
            bias = torch.randn(D, device="cuda", generator=_gen(2)).to(dtype).requires_grad_(True)
            y = ops.embedding(idx, table, scale=2.0, add=bias.expand(tuple(idx.shape) + (D,)))
            _check(y, *_lookup64(idx, table, 2.0, bias.expand(tuple(idx.shape) + (D,))), dtype)
            big = torch.randn(tuple(idx.shape) + (D + 5,), device="cuda", generator=_gen(3)).to(dtype)
            gs = [big[..., 2:2 + D], torch.ones(D, device="cuda", dtype=dtype).expand(tuple(idx.shape) + (D,))]
            for g in gs:
                gt, gb = torch.autograd.grad(y, [table, bias], g, retain_graph=True)
                _check(gt, *_grad64(idx, g, T, 2.0, None), dtype)
                assert gb.shape == bias.shape and torch.allclose(
                    gb.double(), g.reshape(-1, D).double().sum(0), rtol=HALF[dtype] + 1e-5, atol=1e-2 if dtype == torch.bfloat16 else 1e-4)


@gpu
def test_indices_outside_the_table():
    from hypdiff_amd import ops
    table = torch.randn(10, 8, device="cuda").requires_grad_(True)
    idx = torch.tensor([3, -1, 10, 1 << 40, -(1 << 40), 9], device="cuda")
    y = ops.embedding(idx, table, add=torch.zeros(6, 8, device="cuda"))
    assert torch.isnan(y).all(1).tolist() == [False, True, True, True, True, False]
    assert torch.equal(y[[0, 5]], table[[3, 9]])
    gt = torch.autograd.grad(y, [table], torch.ones(6, 8, device="cuda"))[0]
    assert gt.sum(1).tolist() == [0, 0, 0, 8, 0, 0, 0, 0, 0, 8]


@gpu
def test_gradient_against_differences():
    """The table's gradient of L = sum(w * y) is linear in the table: L(table + d) - L(table - d) = 2 <dL/dtable, d>.
    In fp32 with |terms| summed in fp64: 4 roundings of u per term of L."""
    from hypdiff_amd import ops
    g = _gen(4)
    idx = torch.randint(0, 30, (500,), device="cuda", generator=g)
    table = torch.randn(30, 20, device="cuda", generator=g)
    d = torch.randn(30, 20, device="cuda", generator=g)
    w = torch.randn(500, 20, device="cuda", generator=g)
    gt = ops._embedding_sum(w, idx, 30, 0.5, None)

    def loss(t):
        y = ops.embedding(idx, t, scale=0.5).double() * w.double()
        return float(y.sum()), float(y.abs().sum())
    (a, sa), (b, sb) = loss(table + d), loss(table - d)
    want = 2 * float((gt.double() * d.double()).sum())
    bound = 4 * U * (sa + sb) + 2 * 502 * U * float((gt.double().abs() * d.double().abs()).sum()) + 40 * U * float(
        (torch.zeros(30, 20, device="cuda", dtype=torch.float64).index_add_(0, idx, w.double().abs()) * d.double().abs()).sum())
    assert abs((a - b) - want) <= bound


@gpu
def test_captured_and_replayed_with_new_indices():
    from hypdiff_amd import ops
    table = torch.randn(100, 40, device="cuda", generator=_gen(5)).bfloat16().requires_grad_(True)
    for rows in (300, 6000):                             # both sorts
        idx = torch.randint(0, 100, (rows,), device="cuda", generator=_gen(6))
        g = torch.randn(rows, 40, device="cuda", generator=_gen(7)).bfloat16()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops._embedding_sum(g, idx, 100, 1.0, None)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops._embedding_lookup(table, idx, 1.0, None)
            gt = ops._embedding_sum(g, idx, 100, 1.0, None)
        for k in range(3):
            idx.copy_(torch.randint(0, 100, (rows,), device="cuda", generator=_gen(20 + k)))
            g.copy_(torch.randn(rows, 40, device="cuda", generator=_gen(30 + k)).bfloat16())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, ops._embedding_lookup(table, idx, 1.0, None))
            assert torch.equal(gt, ops._embedding_sum(g, idx, 100, 1.0, None))


@gpu
@pytest.mark.parametrize("rows", [511, 512, 513, 1024, 1025, 2049])
def test_gradient_around_the_borders_of_the_sorts(rows):
    from hypdiff_amd import ops
    for T, kind in ((3, "any"), (70000, "hot"), (256, "one")):
        idx = _idx(rows, T, kind, torch.int64, rows)
        g = torch.randn(rows, 9, device="cuda", generator=_gen(rows + 1))
        want, size = _grad64(idx, g, T, 0.5, None)
        _check(ops._embedding_sum(g, idx, T, 0.5, None), want, size, torch.float32)


@gpu
def test_two_streams_at_once():
    from hypdiff_amd import ops
    sets = [(torch.randint(0, 300, (20000,), device="cuda", generator=_gen(k)), torch.randn(300, 96, device="cuda", generator=_gen(k + 2)),
             torch.randn(20000, 96, device="cuda", generator=_gen(k + 4))) for k in range(2)]

    def step(idx, table, g):
        t = table.detach().requires_grad_(True)
        y = ops.embedding(idx, t)
        return y.detach(), torch.autograd.grad(y, [t], g)[0]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([step(*s) for _ in range(5)])
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        for o in outs:
            assert all(torch.equal(a, c) for a, c in zip(o, w))


@gpu
def test_offsets_beyond_32_bits():
    """a result and a gradient of 4.4 GB (many rows), then a table of that size (many tokens)"""
    from hypdiff_amd import ops
    rows, T, D = (1 << 22) + 7, 5, 520
    table = torch.randn(T, D, device="cuda", generator=_gen(40)).bfloat16().requires_grad_(True)
    idx = torch.arange(rows, device="cuda") % T
    g = torch.zeros(rows, D, device="cuda", dtype=torch.bfloat16)
    g[-3:] = torch.randn(3, D, device="cuda", generator=_gen(41)).bfloat16()
    y = ops.embedding(idx, table)
    assert torch.equal(y[-300:], table.detach()[idx[-300:]])
    gt = torch.autograd.grad(y, [table], g)[0]
    want = torch.zeros(T, D, device="cuda", dtype=torch.bfloat16)
    want[idx[-3:]] = g[-3:]                              # one row a token, zeros besides: no rounding
    assert torch.equal(gt, want)
    del y, g
    table = torch.randn(rows, D, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    idx = torch.arange(rows - 300, rows, device="cuda", dtype=torch.int32)
    g = torch.randn(300, D, device="cuda", generator=_gen(42)).bfloat16()
    y = ops.embedding(idx, table)
    assert torch.equal(y, table.detach()[-300:])
    gt = torch.autograd.grad(y, [table], g)[0]
    assert torch.equal(gt[-300:], g) and not bool(gt[:-300].any())


@gpu
def test_agrees_with_the_fp32_embedding_of_the_backbone():
    from hypdiff_amd import autograd as hag, ops
    g = _gen(8)
    idx = torch.randperm(1000, device="cuda", generator=g)[:200]      # no token twice: no order of sums to differ in
    table = torch.randn(1000, 512, device="cuda", generator=g).requires_grad_(True)
    h = torch.randn(200, 512, device="cuda", generator=g)
    gy = torch.randn(200, 512, device="cuda", generator=g)
    new = ops.embedding(idx, table, add=h)
    old = hag.EmbeddingAdd.apply(h.clone(), table, idx)
    assert torch.equal(new, old)
    assert torch.equal(torch.autograd.grad(new, [table], gy)[0], torch.autograd.grad(old, [table], gy)[0])


def test_refusals_on_the_host():
    from hypdiff_amd import ops
    t, i = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="table"):
        ops.embedding(i, t.double())
    with pytest.raises(TypeError, match="indices"):
        ops.embedding(i.to(torch.int16), t)
    with pytest.raises(ValueError, match="table"):
        ops.embedding(i, t[0])
    with pytest.raises(ValueError, match="table"):
        ops.embedding(i, t[:0])
    with pytest.raises(TypeError, match="add"):
        ops.embedding(i, t, add=torch.zeros(2, 3).bfloat16())
    with pytest.raises(ValueError, match="add"):
        ops.embedding(i, t, add=torch.zeros(3))
    with pytest.raises(ValueError, match="padding_idx"):
        ops.embedding(i, t, padding_idx=4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.embedding(i, t)


def test_refusals_of_the_entry_points():
    from hypdiff_amd import _lib

    def look(table=256, ldt=8, idx=256, bits=64, add=None, lda=0, dt=0, T=4, rows=2, dim=8, out=256):
        _lib.call("hd_embedding_lookup", table, ldt, idx, bits, add, lda, 1.0, dt, T, rows, dim, out, None)

    def summed(g=256, ldg=8, idx=256, bits=64, dt=0, T=4, rows=2, dim=8, out=256, ws=256, nbytes=1 << 20):
        _lib.call("hd_embedding_sum", g, ldg, idx, bits, -1, 1.0, dt, T, rows, dim, out, ws, nbytes, None)
    for fn in (look, summed):
        for bad, what in ((dict(dt=3), "element type"), (dict(bits=16), "bits"), (dict(T=0), "shape"), (dict(rows=-1), "shape"),
                          (dict(rows=1 << 31), "shape"), (dict(dim=0), "shape"), (dict(T=1 << 31), "shape"), (dict(out=None), "null"),
                          (dict(idx=None), "null"), (dict(out=257, dt=1), "aligned"), (dict(idx=260), "aligned")):
            with pytest.raises(RuntimeError, match=what):
                fn(**bad)
    with pytest.raises(RuntimeError, match="workspace of"):
        summed(nbytes=16)
    with pytest.raises(RuntimeError, match="null"):
        summed(ws=None)
    assert _lib.load().hd_embedding_sum_workspace_bytes(1 << 31, 8, 4, 0) == 0


@gpu
@pytest.mark.parametrize("T", [(1 << 24) + 5, 1 << 24, (1 << 16) - 1, 1 << 16])
def test_gradient_at_every_number_of_radix_passes(T):
    """tokens of 17, 16 and 25 bits (3, 2, 4 passes): the named rows against 64 bits, all others zero"""
    from hypdiff_amd import ops
    rows, D = 3000, 2
    idx = _idx(rows, T, "hot", torch.int64, 50)
    idx[-1] = T - 1
    g = torch.randn(rows, D, device="cuda", generator=_gen(51))
    got = ops._embedding_sum(g, idx, T, 1.0, None)
    names, at = torch.unique(idx, return_inverse=True)
    want, size = _grad64(at, g, names.numel(), 1.0, None)
    _check(got[names], want, size, torch.float32)
    got[names] = 0
    assert not bool(got.any())

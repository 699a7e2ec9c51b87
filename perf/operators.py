"""What is measured of the mixed-precision training operators: the fused Linear, the embedding and the AdamW step.

Three operators of one training step of a denoiser in 16 bits, each in a plain form (elementary torch operations in
32 bits, rounded once at the end) and through the framework's entry points:

  linear     y = resid + act(x W^T + b), 16-bit operands.  mode "infer": y; mode "train": y and the gradients of x, W, b.
  embedding  y = add + scale * table[idx].  mode "infer": y; mode "train": y and the table's gradient (the rows of dL/dy
             summed by token).
  adamw      one step of AdamW over a list of tensors, with the moments in 32 bits or in 8.

The 8-bit moments: every tensor is cut into blocks of 256 elements (the last one of a tensor may be shorter), and a block
holds m and s = sqrt(v) as e4m3 codes with one fp32 scale each, max|.| / 448.  m is rounded to the nearest code.  s is
rounded up or down by comparing the dropped bits with the Weyl sequence frac(i * 2654435761 / 2^32 + t * 1779033703 / 2^32)
of the element's index i in its tensor and the step t (an average over steps is not biased: round-to-nearest would never let
v decay, its relative change per step, 1 - beta2, is far below half a code), and a positive s never becomes code 0.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 256                     # elements of one scale of the 8-bit moments
LR, B1, B2, EPS, WD = 1e-3, 0.9, 0.999, 1e-8, 1e-2
STEP0 = 1000                    # steps behind the state that an optimizer case starts from

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

# parameter lists: (shape, how many)
LISTS = {
    # graph-level DDPM backbone: 2 MLPs of 12 Linear each at width 512 on 64-wide latents, and the time embedding
    "backbone": [((512, 64), 1), ((512, 512), 22), ((64, 512), 1), ((1000, 512), 1), ((512,), 23), ((64,), 1)],
    # direction denoiser at latent width 512: D+1 -> 800 -> 900 -> 800 -> 700 -> D
    "denoiser": [((800, 513), 1), ((900, 800), 1), ((800, 900), 1), ((700, 800), 1), ((512, 700), 1),
                 ((800,), 2), ((900,), 1), ((700,), 1), ((512,), 1)],
    # a large model's share of one GPU: matrices of ragged widths, their biases, one big table
    "wide": [((2048, 1365), 16), ((1365, 2048), 16), ((2048,), 16), ((32000, 400), 1)],
}


def listed():
    return [
        # one latent row through one hidden layer of the graph-level denoiser (sampling one graph): latency
        {"name": "linear_row", "op": "linear", "mode": "infer", "M": 1, "N": 512, "K": 512, "type": "bf16", "act": "gelu",
         "bias": True, "resid": True, "pitch": 0},
        # first layer of the direction denoiser over every node of the ego graph set: cat(x, t) makes an odd width
        {"name": "linear_odd", "op": "linear", "mode": "infer", "M": 15777, "N": 800, "K": 513, "type": "fp16", "act": "gelu",
         "bias": True, "resid": False, "pitch": 0},
        # widest layer of the direction denoiser over every node of the BA graph set
        {"name": "linear_nodes", "op": "linear", "mode": "infer", "M": 74750, "N": 900, "K": 800, "type": "bf16", "act": "gelu",
         "bias": True, "resid": False, "pitch": 0},
        # training: a hidden residual layer on the graph-level batch of 200
        {"name": "linear_train_batch", "op": "linear", "mode": "train", "M": 200, "N": 512, "K": 512, "type": "bf16",
         "act": "gelu", "bias": True, "resid": True, "pitch": 0},
        # training: the odd first layer over the community graph set
        {"name": "linear_train_odd", "op": "linear", "mode": "train", "M": 7850, "N": 800, "K": 513, "type": "fp16",
         "act": "gelu", "bias": True, "resid": False, "pitch": 0},
        # training: the widest layer over the BA graph set
        {"name": "linear_train_nodes", "op": "linear", "mode": "train", "M": 74750, "N": 900, "K": 800, "type": "bf16",
         "act": "gelu", "bias": True, "resid": False, "pitch": 0},
        # the time embedding added to the activations of a batch of 200
        {"name": "embed_batch", "op": "embedding", "mode": "infer", "rows": 200, "T": 1000, "D": 512, "type": "bf16",
         "add": True, "scaled": False, "padding": False, "hot": 0.0, "wide_idx": True},
        # training: the time embedding with every node of the BA set, drawn unevenly (few steps own most rows)
        {"name": "embed_train_hot", "op": "embedding", "mode": "train", "rows": 74750, "T": 1000, "D": 512, "type": "fp32",
         "add": True, "scaled": True, "padding": False, "hot": 1.2, "wide_idx": True},
        # training: a token table at a long batch, frequencies as in text, with a padding token
        {"name": "embed_train_tokens", "op": "embedding", "mode": "train", "rows": 131072, "T": 50000, "D": 700, "type": "bf16",
         "add": False, "scaled": True, "padding": True, "hot": 1.0, "wide_idx": False},
        # the direction denoiser's parameters in fp32, moments in 8 bits
        {"name": "adamw_denoiser_8", "op": "adamw", "list": "denoiser", "type": "fp32", "bits": 8, "master": False},
        # the graph-level backbone in bf16 with fp32 masters, moments in 32 bits
        {"name": "adamw_backbone_32", "op": "adamw", "list": "backbone", "type": "bf16", "bits": 32, "master": True},
        # a large model's share: moments in 8 bits, bf16 parameters, fp32 masters
        {"name": "adamw_wide_8", "op": "adamw", "list": "wide", "type": "bf16", "bits": 8, "master": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "embedding", "adamw"])
    if op == "linear":
        return {"op": op, "mode": rng.choice(["infer", "train"]), "M": _log_int(rng, 1, 74750), "N": _log_int(rng, 8, 900),
                "K": _log_int(rng, 8, 800), "type": rng.choice(["bf16", "fp16"]), "act": rng.choice(["identity", "relu", "gelu"]),
                "bias": rng.random() < 0.8, "resid": rng.random() < 0.4, "pitch": rng.choice([0, 0, 1, 8, 37])}
    if op == "embedding":
        return {"op": op, "mode": rng.choice(["infer", "train"]), "rows": _log_int(rng, 1, 131072), "T": _log_int(rng, 2, 50000),
                "D": _log_int(rng, 8, 700), "type": rng.choice(["bf16", "fp16", "fp32"]), "add": rng.random() < 0.5,
                "scaled": rng.random() < 0.5, "padding": rng.random() < 0.3, "hot": rng.choice([0.0, 0.7, 1.2]),
                "wide_idx": rng.random() < 0.5}
    kind = rng.choice(["bf16", "fp16", "fp32"])
    return {"op": op, "list": "drawn", "tensors": rng.randint(1, 40), "largest": _log_int(rng, 16, 2_000_000),
            "shapes": rng.randint(0, 1 << 30), "type": kind, "bits": rng.choice([8, 32]),
            "master": kind != "fp32" and rng.random() < 0.6}


def _shapes(case):
    if case["list"] != "drawn":
        return [s for s, n in LISTS[case["list"]] for _ in range(n)]
    rs = np.random.RandomState(case["shapes"] % (1 << 31))
    n = [max(1, int(round(math.exp(rs.uniform(0.0, math.log(case["largest"])))))) for _ in range(case["tensors"])]
    return [(v,) if v % 2 else (2, v // 2) for v in n]


def _segments(numels):
    """(first element, number) of every tensor in the flat state: a tensor starts a block of its own"""
    at, out = 0, []
    for n in numels:
        out.append((at, n))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return out, at


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)

    def randn(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    dt = TYPES[case["type"]]
    if case["op"] == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        lim = 1.0 / math.sqrt(k)                       # nn.Linear's initialisation
        st = {"case": case, "x": randn(m, k + case["pitch"]).to(dt)[:, :k]}
        st["w"] = ((torch.rand(n, k, device="cuda", generator=gen) * 2 - 1) * lim).to(dt)
        st["b"] = ((torch.rand(n, device="cuda", generator=gen) * 2 - 1) * lim).to(dt) if case["bias"] else None
        st["r"] = randn(m, n).to(dt) if case["resid"] else None
        st["g"] = randn(m, n).to(dt) if case["mode"] == "train" else None
        if case["mode"] == "train":
            for key in ("x", "w", "b"):
                if st[key] is not None:
                    st[key].requires_grad_(True)
        return st
    if case["op"] == "embedding":
        rows, t, d = case["rows"], case["T"], case["D"]
        if case["hot"]:                                # token ranks by a power law, ranks dealt out over the table
            p = torch.arange(1, t + 1, device="cuda", dtype=torch.float64).pow(-case["hot"])
            edges = torch.cumsum(p / p.sum(), 0)
            rank = torch.searchsorted(edges, torch.rand(rows, device="cuda", generator=gen, dtype=torch.float64)).clamp_(max=t - 1)
            idx = torch.randperm(t, device="cuda", generator=gen)[rank]
        else:
            idx = torch.randint(0, t, (rows,), device="cuda", generator=gen)
        st = {"case": case, "idx": idx.to(torch.int64 if case["wide_idx"] else torch.int32), "table": randn(t, d).to(dt),
              "add": randn(rows, d).to(dt) if case["add"] else None, "scale": math.sqrt(d) if case["scaled"] else 1.0,
              "padding": t // 2 if case["padding"] else None, "g": randn(rows, d).to(dt) if case["mode"] == "train" else None}
        if case["mode"] == "train":
            st["table"].requires_grad_(True)
        return st
    shapes = _shapes(case)
    numels = [int(np.prod(s)) for s in shapes]
    segs, total = _segments(numels)
    real = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, n in segs:
        real[a:a + n] = True
    master = randn(total, std=0.05) * real
    st = {"case": case, "step": STEP0, "segs": segs}
    st["params"] = [torch.nn.Parameter(master[a:a + n].to(dt).view(s)) for (a, n), s in zip(segs, shapes)]
    for p in st["params"]:
        p.grad = randn(*p.shape, std=1e-2).to(dt)
    if case["master"]:
        st["master"] = master
    m = randn(total, std=3e-3) * real
    s = torch.exp(randn(total, std=0.7)) * 1e-2 * real
    if case["bits"] == 32:
        st["exp_avg"], st["exp_avg_sq"] = m, s * s
    else:
        st["exp_avg_scale"] = m.view(-1, BLOCK).abs().amax(1) * (1.0 / 448.0)
        st["exp_avg_sq_root_scale"] = s.view(-1, BLOCK).amax(1) * (1.0 / 448.0)
        st["exp_avg"] = (m.view(-1, BLOCK) / st["exp_avg_scale"][:, None]).reshape(-1).to(torch.float8_e4m3fn)
        codes = (s.view(-1, BLOCK) / st["exp_avg_sq_root_scale"][:, None]).reshape(-1).to(torch.float8_e4m3fn).view(torch.uint8)
        st["exp_avg_sq_root"] = torch.where(real, codes.clamp(min=1), torch.zeros_like(codes)).view(torch.float8_e4m3fn)
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "embedding": _own_embedding, "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        return {"linear": _plain_linear, "embedding": _plain_embedding, "adamw": _plain_adamw}[op](state)


def _own_linear(st):
    from hypdiff_amd import ops
    y = ops.linear_act(st["x"], st["w"], st["b"], act=st["case"]["act"], resid=st["r"])
    if st["g"] is None:
        return {"y": y}
    leaves = [("dx", st["x"]), ("dw", st["w"])] + ([("db", st["b"])] if st["b"] is not None else [])
    grads = torch.autograd.grad(y, [t for _, t in leaves], st["g"])
    return {"y": y, **{name: g for (name, _), g in zip(leaves, grads)}}


def _own_embedding(st):
    from hypdiff_amd import ops
    y = ops.embedding(st["idx"], st["table"], scale=st["scale"], add=st["add"], padding_idx=st["padding"])
    if st["g"] is None:
        return {"y": y}
    return {"y": y, "dtable": torch.autograd.grad(y, [st["table"]], st["g"])[0]}


def _own_adamw(st):
    from hypdiff_amd import optim
    case, opt = st["case"], st.get("opt")
    if opt is None:                                    # the optimizer that a program keeps, resumed from its saved state
        opt = st["opt"] = optim.AdamW(st["params"], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=case["bits"],
                                      master_weights=case["master"])
        sd = opt.state_dict()
        per = ["exp_avg", "exp_avg_sq"] if case["bits"] == 32 else ["exp_avg", "exp_avg_sq_root"]
        per_block = [] if case["bits"] == 32 else ["exp_avg_scale", "exp_avg_sq_root_scale"]
        sd["state"] = {}
        for i, ((a, n), p) in enumerate(zip(st["segs"], st["params"])):
            s = {"step": st["step"], **{k: st[k][a:a + n].view(p.shape) for k in per + (["master"] if case["master"] else [])}}
            s.update({k: st[k][a // BLOCK:(a + n + BLOCK - 1) // BLOCK] for k in per_block})
            sd["state"][i] = s
        opt.load_state_dict(sd)
    opt.step()
    return {"params": [p.detach() for p in st["params"]], **opt.state_buffers()}


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    return z * (0.5 * torch.erfc(z * -math.sqrt(0.5))) if act == "gelu" else z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * (torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))


def _plain_linear(st):
    case = st["case"]
    dt = TYPES[case["type"]]
    x, w = st["x"].float(), st["w"].float()
    z = x @ w.t()
    if st["b"] is not None:
        z = z + st["b"].float()
    y = _act(z, case["act"])
    if st["r"] is not None:
        y = y + st["r"].float()
    out = {"y": y.to(dt)}
    if st["g"] is None:
        return out
    dz = st["g"].float()
    if case["act"] != "identity":
        dz = dz * _act_slope(z, case["act"])
    out["dx"] = (dz @ w).to(dt)
    out["dw"] = (dz.t() @ x).to(dt)
    if st["b"] is not None:
        out["db"] = dz.sum(0).to(dt)
    return out


def _plain_embedding(st):
    dt = TYPES[st["case"]["type"]]
    idx = st["idx"].long()
    y = st["table"][idx].float() * st["scale"]
    if st["add"] is not None:
        y = y + st["add"].float()
    out = {"y": y.to(dt)}
    if st["g"] is not None:
        gt = torch.zeros(st["table"].shape, device="cuda", dtype=torch.float32).index_add_(0, idx, st["g"].float())
        gt = gt * st["scale"]
        if st["padding"] is not None:
            gt[st["padding"]] = 0
        out["dtable"] = gt.to(dt)
    return out


def _flat(tensors):
    pad = torch.nn.functional.pad
    return torch.cat([pad(t.detach().reshape(-1).float(), (0, -t.numel() % BLOCK)) for t in tensors])


def _block_scale(amax):
    """max|.| / 448 of a block, 0 for a block of zeros, NaN where the block holds an infinity or a NaN; and its reciprocal"""
    scale = torch.clamp(amax, min=2.0 ** -100) * (1.0 / 448.0)
    inv = 1.0 / scale
    zero = amax == 0
    scale = torch.where(zero, torch.zeros_like(scale), torch.where(torch.isfinite(amax), scale, torch.full_like(scale, math.nan)))
    return scale, torch.where(zero, torch.zeros_like(inv), inv)


def _root_codes(s, inv, index, step):
    """e4m3 codes of s * inv >= 0, rounded by the Weyl sequence of (index, step)"""
    y = s.view(-1, BLOCK) * inv[:, None]
    u = (index * 2654435761 + step * 1779033703) & 0xFFFFFFFF
    d = (u >> 12).view(-1, BLOCK)                                          # 20 bits
    normal = ((y.contiguous().view(torch.int32).long() + d) >> 20) - 960   # exponent bias 127 -> 7, 23 -> 3 mantissa bits
    small = torch.floor(y * 512.0 + d.float() * 2.0 ** -20).long()
    code = torch.clamp(torch.where(y < 2.0 ** -6, small, normal), max=126)
    code = torch.where(s.view(-1, BLOCK) > 0, torch.clamp(code, min=1), torch.zeros_like(code))
    return code.to(torch.uint8).view(-1).view(torch.float8_e4m3fn)


def _plain_adamw(st):
    case, segs = st["case"], st["segs"]
    st["step"] += 1
    t = st["step"]
    step_size, r2 = LR / (1.0 - B1 ** t), 1.0 / math.sqrt(1.0 - B2 ** t)
    g = _flat([p.grad for p in st["params"]])
    p = st["master"] if case["master"] else _flat(st["params"])
    if case["bits"] == 32:
        m, v = st["exp_avg"], st["exp_avg_sq"]
    else:
        m = (st["exp_avg"].float().view(-1, BLOCK) * st["exp_avg_scale"][:, None]).view(-1)
        v = (st["exp_avg_sq_root"].float().view(-1, BLOCK) * st["exp_avg_sq_root_scale"][:, None]).view(-1)
        v = v * v
    m = m * B1 + g * (1.0 - B1)
    v = v * B2 + (g * g) * (1.0 - B2)
    s = torch.sqrt(v)
    p = p * (1.0 - LR * WD) - (m / (s * r2 + EPS)) * step_size
    if case["bits"] == 32:
        st["exp_avg"], st["exp_avg_sq"] = m, v
    else:
        if "index" not in st:
            st["index"] = torch.cat([torch.arange(n + -n % BLOCK, device="cuda") for _, n in segs])
        scale, inv = _block_scale(m.view(-1, BLOCK).abs().amax(1))
        st["exp_avg_scale"], st["exp_avg"] = scale, (m.view(-1, BLOCK) * inv[:, None]).view(-1).to(torch.float8_e4m3fn)
        scale, inv = _block_scale(s.view(-1, BLOCK).amax(1))
        st["exp_avg_sq_root_scale"], st["exp_avg_sq_root"] = scale, _root_codes(s, inv, st["index"], t)
    if case["master"]:
        st["master"] = p
    torch._foreach_copy_([q.data for q in st["params"]], [p[a:a + n].view(q.shape) for (a, n), q in zip(segs, st["params"])])
    keys = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale", "master")
    return {"params": [q.detach() for q in st["params"]], **{k: st[k] for k in keys if k in st}}


# ---- the bytes and operations that a pass cannot do without ---------------------------------------------------------
def work(case):
    e = SIZE[case["type"]]
    if case["op"] == "linear":
        m, n, k = case["M"], case["N"], case["K"]
        nb = (m * k + n * k + m * n * (2 if case["resid"] else 1) + (n if case["bias"] else 0)) * e
        fl = 2.0 * m * n * k
        if case["mode"] == "train":
            nb += (m * n + m * k + n * k + (n if case["bias"] else 0)) * e     # dL/dy in; dx, dW, db out
            fl *= 3
        return {"bytes": nb, "flops": fl}
    if case["op"] == "embedding":
        rows, t, d = case["rows"], case["T"], case["D"]
        nb = rows * (8 if case["wide_idx"] else 4) + (min(rows, t) + rows * (2 if case["add"] else 1)) * d * e
        fl = rows * d * 2.0
        if case["mode"] == "train":
            nb += (rows + t) * d * e
            fl += rows * d
        return {"bytes": nb, "flops": fl}
    n = sum(int(np.prod(s)) for s in _shapes(case))
    per = 3 * e + (8 if case["master"] else 0) - (e if case["master"] else 0)      # p, g in; p out (a master replaces p in)
    per += 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK
    return {"bytes": float(n * per), "flops": 14.0 * n}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "linear":
            x, w = st["x"].double(), st["w"].double()
            z = torch.mm(x, w.t().contiguous())
            if st["b"] is not None:
                z += st["b"].double()
            phi = 0.5 + 0.5 * torch.erf(z / math.sqrt(2.0))
            act = {"identity": lambda: (z, torch.ones_like(z)), "relu": lambda: (z * (z > 0), (z > 0).double()),
                   "gelu": lambda: (z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))}
            y, slope = act[case["act"]]()
            if st["r"] is not None:
                y = y + st["r"].double()
            out = {"y": y}
            if st["g"] is not None:
                dz = st["g"].double() * slope
                out["dx"] = torch.mm(dz, w)
                out["dw"] = torch.mm(dz.t().contiguous(), x)
                if st["b"] is not None:
                    out["db"] = dz.sum(0)
            return out
        if case["op"] == "embedding":
            idx = st["idx"].long().cpu().numpy()
            y = st["table"].double()[st["idx"].long()] * st["scale"]
            out = {"y": y + st["add"].double() if st["add"] is not None else y}
            if st["g"] is not None:
                # sorted by token: differences of the running sums at the tokens' borders, in column slabs
                order = np.argsort(idx, kind="stable")
                ends = torch.from_numpy(np.searchsorted(idx[order], np.arange(case["T"]), side="right")).cuda()
                by = st["g"][torch.from_numpy(order).cuda()].double()
                run_sum = torch.cat([torch.zeros(1, case["D"], device="cuda", dtype=torch.float64), torch.cumsum(by, 0)])
                at = run_sum[ends]
                gt = torch.diff(at, dim=0, prepend=torch.zeros(1, case["D"], device="cuda", dtype=torch.float64)) * st["scale"]
                if st["padding"] is not None:
                    gt[st["padding"]] = 0.0
                out["dtable"] = gt
            return out
        t = st["step"] + 1
        res = {"params": []}
        parts = {}
        for (a, n), p in zip(st["segs"], st["params"]):
            nb, lo = (n + BLOCK - 1) // BLOCK, a // BLOCK
            g = p.grad.double().reshape(-1)
            th = (st["master"][a:a + n] if case["master"] else p.detach().reshape(-1)).double()
            if case["bits"] == 32:
                m0, v0 = st["exp_avg"][a:a + n].double(), st["exp_avg_sq"][a:a + n].double()
            else:
                rep = lambda k: st[k][lo:lo + nb].double().repeat_interleave(BLOCK)[:n]  # noqa: E731
                m0 = st["exp_avg"][a:a + n].double() * rep("exp_avg_scale")
                v0 = (st["exp_avg_sq_root"][a:a + n].double() * rep("exp_avg_sq_root_scale")) ** 2
            m1 = B1 * m0 + (1 - B1) * g
            v1 = B2 * v0 + (1 - B2) * g ** 2
            th = th - LR * WD * th
            th = th - LR * (m1 / (1 - B1 ** t)) / (torch.sqrt(v1 / (1 - B2 ** t)) + EPS)
            res["params"].append(th.view(p.shape))
            fill = lambda v: torch.nn.functional.pad(v, (0, nb * BLOCK - n))  # noqa: E731
            if case["master"]:
                parts.setdefault("master", []).append(fill(th))
            if case["bits"] == 32:
                parts.setdefault("exp_avg", []).append(fill(m1))
                parts.setdefault("exp_avg_sq", []).append(fill(v1))
            else:                                      # the codes' values before they are rounded, in units of the block's scale
                for key, val in (("exp_avg", m1), ("exp_avg_sq_root", torch.sqrt(v1))):
                    blocks = fill(val).view(nb, BLOCK)
                    sc = blocks.abs().amax(1) / 448.0
                    parts.setdefault(key, []).append((blocks / sc[:, None]).reshape(-1))
                    parts.setdefault(key + "_scale", []).append(sc)
        return {**res, **{k: torch.cat(v) for k, v in parts.items()}}

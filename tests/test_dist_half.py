"""CPU, several ranks over gloo: the mean of 16-bit gradients (dist.GradBucket, dist.DataParallelTrainer) against the mean of
the ranks' own gradients in 64 bits."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}     # half of the smallest step


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _gradients(world, dtype):
    """(world, 5 parameters of 40): sizes from fp16's smallest step to half its largest value, alike and apart over the ranks"""
    rs = np.random.RandomState(3)
    size = np.exp2(rs.uniform(-24, 15, (1, 5, 40)) + rs.uniform(-8, 0, (world, 5, 40)))
    size[:, 0] = 2.0 ** -24                              # every rank holds the smallest step
    return torch.from_numpy(np.sign(rs.standard_normal((1, 5, 40))) * size).to(dtype)


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from hypdiff_amd import dist as hdist
    res = {}
    for dtype in (torch.bfloat16, torch.float16):
        c = _gradients(world, dtype)
        want = c.double().mean(0)
        # dividing and adding in fp32: two roundings of 2^-24 a rank, relative to the terms; one rounding to the type
        bound = HALF[dtype] * want.abs() + TINY[dtype] + 2 * world * 2.0 ** -24 * c.double().abs().mean(0) * (1 + HALF[dtype])
        for overlap, chunk in ((True, 64), (True, 4 << 20), (False, 4 << 20)):
            net = torch.nn.ParameterList([torch.nn.Parameter(torch.zeros(40, dtype=dtype)) for _ in range(5)])
            tr = hdist.DataParallelTrainer(net, optimizer=torch.optim.SGD(net.parameters(), lr=0.0), overlap=overlap)
            if chunk == 64:
                tr.bucket = hdist.GradBucket(net.parameters(), chunk_bytes=chunk)
                res[f"{dtype} chunks"] = len(tr.bucket.chunks) >= 3
            for _ in range(2):                           # the second step starts from a used bucket
                tr.step(lambda: sum((p * c[rank, k]).float().sum() for k, p in enumerate(net)))
                for k, p in enumerate(net):
                    ok = p.grad.dtype == dtype and bool(((p.grad.double() - want[k]).abs() <= bound[k]).all())
                    res[f"{dtype} {overlap} {chunk} {k}"] = ok
            res[f"{dtype} {overlap} {chunk} bucket"] = tr.bucket.flat.dtype == dtype and all(
                p.grad.data_ptr() == tr.bucket.flat[lo:].data_ptr() for p in net for lo in (tr.bucket.offsets[id(p)][0],))
        bucket = hdist.GradBucket([torch.nn.Parameter(torch.zeros(40, dtype=dtype)) for _ in range(5)])
        bucket.flat.copy_(c[rank].reshape(-1))
        work = bucket.allreduce_mean_(async_op=True)
        work.wait()
        res[f"{dtype} async"] = bool(((bucket.flat.double() - want.reshape(-1)).abs() <= bound.reshape(-1)).all())
    q.put((rank, res))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_mean_of_16_bit_gradients(world):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = [q.get(timeout=180) for _ in range(world)]
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    for rank, res in got:
        assert all(res.values()), (rank, [k for k, v in res.items() if not v])


def _nccl_worker(port, q):
    res = {}
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY="0")
        torch.cuda.set_device(0)
        dist.init_process_group("nccl", rank=0, world_size=1, device_id=torch.device("cuda", 0))
        from hypdiff_amd import dist as hdist
        from hypdiff_amd.ddpm import Model
        new = lambda: torch.randn(100, 64, device="cuda")  # noqa: E731
        x, eps, idx = new(), new(), torch.randint(0, 50, (100,), device="cuda")

        def trainer(overlap=True):
            torch.manual_seed(11)
            model = Model(64, 96, 2, 50, 1e-4, 0.02).cuda().bfloat16()
            tr = hdist.DataParallelTrainer(model, lr=1e-3, overlap=overlap)
            if overlap:
                tr.bucket = hdist.GradBucket(model.parameters(), chunk_bytes=1 << 14)
            return model, tr, lambda: model.loss_fn(x, idx=idx, epsilon=eps)
        plain, tp, lp = trainer()
        for _ in range(3):
            tp.step(lp)
        hdist.FORCE_COLLECTIVES = True
        weights = lambda m: [p.detach().clone() for p in m.parameters()]  # noqa: E731
        for overlap in (True, False):
            m, t, loss = trainer(overlap)
            for _ in range(3):
                t.step(loss)
            res[f"eager {overlap}"] = all(torch.equal(a, b) for a, b in zip(weights(m), weights(plain)))
        m, t, loss = trainer()
        replay = t.capture(loss, warmup=1)
        hdist.FORCE_COLLECTIVES = False
        plain, tp, lp = trainer()
        tp.step(lp)
        for k in range(3):
            # a replay's corrections come from the device's pow, one fp32 step off at most: it may move a stored weight by one
            # of its own steps (2^-8), and then by the sum of such moves
            eps.copy_(new())
            replay()
            tp.step(lp)
            torch.cuda.synchronize()
            res[f"replay {k}"] = all(float((a.double() - b.double()).norm()) <= (4 * (k + 1) * 2.0 ** -8 + 5e-5 * (k + 1))
                                     * float(b.double().norm()) for a, b in zip(weights(m), weights(plain)))
        dist.destroy_process_group()
    except Exception:                                    # report instead of leaving the parent waiting
        import traceback
        res["error"] = traceback.format_exc()
    q.put(res)


@pytest.mark.gpu
def test_16_bit_bucket_over_rccl_eager_and_captured():
    """A world of one rank whose collectives are really issued: widened chunks from the backward pass, in eager steps (the
    same bits as without) and recorded into the captured step."""
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_nccl_worker, args=(_free_port(), q), daemon=True)
    p.start()
    res = q.get(timeout=100)
    p.join(30)
    assert "error" not in res, res["error"]
    assert p.exitcode == 0 and all(res.values()), res

"""AdamW over many parameter tensors in one launch, moments in 32 bits or in 8 (csrc/adamw.hip).

Stands beside dist.BucketAdam (Adam over the fp32 bucket of the data-parallel trainer): the same kind of one-launch step for
parameters in fp32, bf16 or fp16 with gradients of their own type, with decoupled weight decay and parameter groups.  The
reference trains with optim.Adam(params, lr) (diff.py:107, diff_graphset.py:66, lp_train.py:41-46).
"""
import numbers

import numpy as np
import torch

from . import _lib, ops

BLOCK = 256                 # elements of one scale of the 8-bit moments; every tensor's state starts on a multiple of it
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# struct hd_adamw_job of include/hypdiff.h
_JOB = np.dtype([("param", np.uint64), ("grad", np.uint64), ("first", np.int64), ("count", np.int64), ("row", np.int64)])
_OPTIONS = ("lr", "betas", "eps", "weight_decay", "state_bits", "master_weights")


class _Flat:
    """The state of one parameter group: flat arrays with a segment of whole 256-element blocks for every parameter."""

    def __init__(self, group):
        self.params = list(group["params"])
        self.bits, self.with_master = int(group["state_bits"]), bool(group["master_weights"])
        dev = self.params[0].device
        self.numels = [p.numel() for p in self.params]
        self.first, at = [], 0
        for n in self.numels:
            self.first.append(at)
            at += (n + BLOCK - 1) // BLOCK * BLOCK
        self.total = at
        self.steps = [0] * len(self.params)              # steps taken by each parameter, as the host counts them
        self.table = torch.zeros(len(self.params), 3, dtype=torch.float64, device=dev)     # the device's count
        self.device_count = False                        # True once a step was captured: the device's count is the true one
        self.jobs = np.zeros(len(self.params), dtype=_JOB)     # the launch arguments; a step fills in the pointers
        self.jobs["first"], self.jobs["count"], self.jobs["row"] = self.first, self.numels, range(len(self.params))
        self.checked, self.states = None, []
        self.buffers = {}
        if self.bits == 32:
            self.buffers["exp_avg"] = torch.zeros(at, dtype=torch.float32, device=dev)
            self.buffers["exp_avg_sq"] = torch.zeros(at, dtype=torch.float32, device=dev)
        else:
            for k in ("exp_avg", "exp_avg_sq_root"):
                self.buffers[k] = torch.zeros(at, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
                self.buffers[k + "_scale"] = torch.zeros(at // BLOCK, dtype=torch.float32, device=dev)
        if self.with_master:
            self.buffers["master"] = torch.zeros(at, dtype=torch.float32, device=dev)
            self.take_masters()

    def take_masters(self):
        m = self.buffers["master"]
        torch._foreach_copy_([m[a:a + n] for a, n in zip(self.first, self.numels)], [p.detach().reshape(-1) for p in self.params])

    def clear(self):
        """as before the first step, in the same memory"""
        for k, b in self.buffers.items():
            (b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b).zero_()
        if self.with_master:
            self.take_masters()
        self.set_steps([0] * len(self.params))

    def view(self, key, i):
        """parameter i's part of a buffer: its shape, or one value per block for the scales"""
        a, n, buf = self.first[i], self.numels[i], self.buffers[key]
        if key.endswith("_scale"):
            return buf[a // BLOCK:(a + n + BLOCK - 1) // BLOCK]
        return buf[a:a + n].view(self.params[i].shape)

    def refresh_steps(self):
        if self.device_count:                            # replays of a captured step counted on the device alone
            self.set_steps([int(t) for t in self.table[:, 0].tolist()], False)

    def set_steps(self, steps, device=True):
        self.steps = steps
        for st, t in zip(self.states, steps):
            st["step"] = t
        if device:
            self.table[:, 0] = torch.tensor(steps, dtype=torch.float64)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    in fp32 arithmetic over parameters in fp32, bf16 or fp16 (contiguous, on the current GPU), one launch per 88 tensors of
    a group.

    state_bits=32: moments in fp32, also for 16-bit parameters.
    state_bits=8: m and sqrt(v) as e4m3 codes with one fp32 scale per 256 elements (2.03 bytes per parameter instead of 8).
        sqrt(v) is rounded up or down so that it is right on average over steps (round-to-nearest would never let it decay);
        the rounding depends on the element and the step alone, so a run repeats bit for bit.
    master_weights=True: 16-bit parameters keep fp32 weights in the state and receive their rounding (an update below half a
        step of the type is lost otherwise).  fp32 parameters are their own.  The masters are taken from the parameters at
        the first step (or from a loaded state): parameters changed by hand afterwards are overwritten.

    The parameters of a group are distinct and share no memory.  Sparse, complex and fp64 parameters, lr as a tensor, amsgrad
    and maximize are not offered.  A parameter whose gradient is None is skipped and does not count the step.  Inside a
    captured HIP graph the step count lives on the device, so a replay has the right bias corrections (state_dict reads it
    back); lr and the other options are the captured ones.  Run one step (or load a state) before the capture; a state loaded
    later goes into the same arrays, and replays continue from it.  state_dict / load_state_dict keep the state's own types;
    with state_bits=32 a state saved by torch.optim.AdamW loads; a state that is refused has changed nothing."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, master_weights=False):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                        master_weights=bool(master_weights))
        self._flats = {}
        super().__init__(params, defaults)

    @staticmethod
    def _check_options(g):
        for k in ("lr", "eps", "weight_decay"):
            if torch.is_tensor(g[k]):
                raise TypeError(f"AdamW: {k} is a number here, not a tensor (it is a launch argument)")
            if not 0.0 <= float(g[k]) < float("inf"):
                raise ValueError(f"AdamW: {k} = {g[k]} is not a finite number >= 0")
        if len(g["betas"]) != 2 or not all(0.0 <= float(b) < 1.0 for b in g["betas"]):
            raise ValueError(f"AdamW: betas = {g['betas']} are not two numbers in [0, 1)")
        if g["state_bits"] not in (32, 8):
            raise ValueError(f"AdamW: state_bits is 32 or 8, not {g['state_bits']}")

    def add_param_group(self, group):
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            self._check_options(g)
            if len({id(p) for p in g["params"]}) != len(g["params"]):
                raise ValueError("AdamW: a parameter stands twice in a group (both updates would run at once)")
            for p in g["params"]:
                if p.dtype not in _DT:
                    raise TypeError(f"AdamW: parameters in float32, bfloat16 or float16, not {p.dtype}")
                if p.layout != torch.strided or not p.is_contiguous():
                    raise ValueError("AdamW: a parameter is not contiguous")
        except Exception:
            self.param_groups.pop()
            raise

    def _flat(self, gi):
        fl = self._flats.get(gi)
        if fl is None:
            group = self.param_groups[gi]
            if not group["params"]:
                return None
            ops._dev(*group["params"])
            self._check_apart(group["params"])
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: the state does not exist yet: run one step or load a state before capturing a graph")
            fl = self._flats[gi] = _Flat(group)
            self._link(fl)
        return fl

    @staticmethod
    def _check_apart(params):
        """one launch updates all of them: no two may share memory"""
        end = 0
        for start, stop in sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel()):
            if start < end:
                raise ValueError("AdamW: two parameters of a group share memory (both updates would run at once)")
            end = stop

    def _link(self, fl):
        fl.states = [self.state[p] for p in fl.params]
        for i, (p, st) in enumerate(zip(fl.params, fl.states)):
            # an fp32 parameter is its own master
            st.update({"step": fl.steps[i], **{k: fl.view(k, i) for k in fl.buffers if k != "master" or p.dtype != torch.float32}})

    def state_buffers(self, group=0):
        """The flat state arrays of a parameter group, the ones that the step updates: exp_avg, exp_avg_sq (fp32), or exp_avg,
        exp_avg_sq_root (float8_e4m3fn) with their _scale arrays (fp32, one per 256 elements); master (fp32) where kept.  The
        parameters follow each other in the group's order, each from a multiple of 256 on, with zeros behind it."""
        fl = self._flat(group)
        return {} if fl is None else dict(fl.buffers)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            fl = self._flat(gi)
            if fl is not None:
                self._step_group(group, fl)
        return loss

    def _step_group(self, group, fl):
        # the host's part is most of a small model's step
        options = (group["lr"], group["betas"], group["eps"], group["weight_decay"], group["state_bits"], group["master_weights"])
        if fl.checked != options:
            self._check_options(group)
            if int(group["state_bits"]) != fl.bits or bool(group["master_weights"]) != fl.with_master:
                raise RuntimeError("AdamW: state_bits and master_weights cannot change after a group's first step")
            fl.checked = options
        params = group["params"]
        if len(params) != len(fl.params):
            raise RuntimeError("AdamW: the parameters of a group changed after its first step")
        if torch.cuda.is_current_stream_capturing():
            fl.device_count = True
        cur = torch.cuda.current_device()
        keep = []
        batches, touched = self._all_present(params, fl, cur) or self._one_by_one(params, fl, cur, keep)
        b = fl.buffers
        second = b["exp_avg_sq"] if fl.bits == 32 else b["exp_avg_sq_root"]
        most = _lib.load().hd_adamw_max_jobs()
        (b1, b2), lr, eps, wd = group["betas"], float(group["lr"]), float(group["eps"]), float(group["weight_decay"])
        for (dt, t), (rows, ptrs, grads) in batches.items():
            master = b["master"] if fl.with_master and dt != torch.float32 else None
            jobs = fl.jobs if len(rows) == len(params) else fl.jobs[rows]
            jobs["param"], jobs["grad"] = ptrs, grads
            for k in range(0, len(rows), most):
                _lib.call("hd_adamw_step", jobs.ctypes.data + k * _JOB.itemsize, min(most, len(rows) - k), _DT[dt], fl.bits,
                          ops._p(b["exp_avg"]), ops._p(second), ops._p(b.get("exp_avg_scale")),
                          ops._p(b.get("exp_avg_sq_root_scale")), ops._p(master), fl.total, lr, float(b1), float(b2), eps, wd, t,
                          ops._p(fl.table), len(params), ops._stream())
        steps, states = fl.steps, fl.states
        for i in touched:                                 # counted once the launches are under way
            steps[i] = states[i]["step"] = steps[i] + 1
        # the kernel wrote behind autograd's back: the versions key the caches of weight copies, and a saved tensor must notice
        torch.autograd.graph.increment_version(params if len(touched) == len(params) else [params[i] for i in touched])

    @staticmethod
    def _all_present(params, fl, cur):
        """the usual step: every gradient there, of its parameter's type and size, contiguous, one type and one count in the
        group: the launch's lists and the indices, or None (then _one_by_one looks at every tensor and says what is wrong)"""
        t = fl.steps[0]
        dt = params[0].dtype
        if fl.steps.count(t) != len(params) or 0 in fl.numels:
            return None
        grads = [p.grad for p in params]
        T = torch.Tensor
        try:
            if not (list(map(T.numel, grads)) == fl.numels == list(map(T.numel, params))
                    and {g.dtype for g in grads} == {p.dtype for p in params} == {dt}
                    and set(map(T.get_device, grads)) == set(map(T.get_device, params)) == {cur}
                    and all(map(T.is_contiguous, grads)) and all(map(T.is_contiguous, params))):
                return None
            pointers = list(map(T.data_ptr, params)), list(map(T.data_ptr, grads))
        except (TypeError, RuntimeError):                 # no gradient, or one without strides
            return None
        rows = range(len(params))
        return {(dt, 0 if fl.device_count else t + 1): (rows,) + pointers}, rows

    def _one_by_one(self, params, fl, cur, keep):
        batches, touched = {}, []
        for i, p in enumerate(params):
            g = p.grad
            if g is None:
                continue
            dt, n = p.dtype, fl.numels[i]
            if g.dtype is not dt or g.get_device() != cur or p.get_device() != cur or g.layout is not torch.strided \
                    or p.numel() != n or g.numel() != n or not p.is_contiguous():
                self._refuse(i, p, g, fl, cur)
            if not g.is_contiguous():
                g = g.contiguous()
                keep.append(g)                            # lives until the launch is enqueued; its memory is stream-ordered
            touched.append(i)
            if n:
                # one launch has one element type and one step count
                rows, ptrs, grads = batches.setdefault((dt, 0 if fl.device_count else fl.steps[i] + 1), ([], [], []))
                rows.append(i)
                ptrs.append(p.data_ptr())
                grads.append(g.data_ptr())
        return batches, touched

    @staticmethod
    def _refuse(i, p, g, fl, cur):
        if p.get_device() != cur or g.get_device() != cur:
            raise RuntimeError("AdamW: parameter %d is on %s, its gradient on %s, but the current device is cuda:%d"
                               % (i, p.device, g.device, cur))
        if g.layout is not torch.strided:
            raise RuntimeError("AdamW: sparse gradients are not offered")
        if g.dtype is not p.dtype:
            raise TypeError("AdamW: parameter %d is %s, its gradient %s" % (i, p.dtype, g.dtype))
        if g.numel() != p.numel() or p.numel() != fl.numels[i]:
            raise ValueError("AdamW: parameter %d changed its size" % i)
        raise ValueError("AdamW: parameter %d is not contiguous" % i)

    # ---- replays of a captured step (dist.DataParallelTrainer.capture) ----
    def replayed(self):
        """To be called after a replay of a graph that holds step(): the parameters changed without the host's doing."""
        torch.autograd.graph.increment_version([p for g in self.param_groups for p in g["params"] if p.grad is not None])

    # ---- saving and loading: the state's own types, not the parameters' ----
    def __getstate__(self):
        raise TypeError("AdamW: save or copy state_dict(), not the optimizer (its state lives in shared flat arrays)")

    def state_dict(self):
        for fl in self._flats.values():
            fl.refresh_steps()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        saved, groups = state_dict["state"], state_dict["param_groups"]
        if len(groups) != len(self.param_groups) or any(len(a["params"]) != len(b["params"])
                                                        for a, b in zip(groups, self.param_groups)):
            raise ValueError("AdamW: the saved state has other parameter groups")
        # a state saved by torch.optim.AdamW has no state_bits.  Everything is looked at before anything changes
        options = [{k: g.get(k, mine[k]) for k in _OPTIONS} for g, mine in zip(groups, self.param_groups)]
        for gi, (g, mine, opt) in enumerate(zip(groups, self.param_groups, options)):
            self._check_options(opt)
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("AdamW: the saved options ask for amsgrad or maximize, which are not offered")
            if self._captured(gi) and not self._keeps(gi, opt):
                raise RuntimeError("AdamW: a captured step updates this state; state_bits and master_weights cannot change "
                                   "under it")
            for pid, p in zip(g["params"], mine["params"]):
                if saved.get(pid):
                    self._check_saved(saved[pid], p, opt)
            if any(saved.get(pid) for pid in g["params"]):
                ops._dev(*mine["params"])
        # and the saved state may be this optimizer's own: that is copied before it is overwritten
        own = {b.untyped_storage().data_ptr() for fl in self._flats.values() for b in fl.buffers.values()}
        kept = lambda v: v.detach().clone() if v.untyped_storage().data_ptr() in own else v.detach()  # noqa: E731
        parts = [[saved.get(pid) and {k: int(v) if k == "step" else kept(v) if torch.is_tensor(v) else v
                                      for k, v in saved[pid].items()} for pid in g["params"]] for g in groups]
        super().load_state_dict({**state_dict, "state": {}})
        for gi, (mine, opt, part) in enumerate(zip(self.param_groups, options, parts)):
            mine.update(opt)
            if not self._keeps(gi, opt) or not (any(part) or self._captured(gi)):
                self._flats.pop(gi, None)
                if not any(part):
                    continue                              # made anew at the next step
            if gi in self._flats:
                fl = self._flats[gi]                      # the arrays stay where they are: a captured step names them
                fl.clear()
                self._link(fl)
            else:
                fl = self._flat(gi)
            steps, to, frm = list(fl.steps), [], []
            for i, (st, p) in enumerate(zip(part, fl.params)):
                if not st:
                    continue
                for k in fl.buffers:
                    if k == "master" and (k not in st or p.dtype == torch.float32):
                        continue                          # taken from the parameter
                    dst, src = fl.view(k, i), st[k]
                    if dst.dtype == torch.float8_e4m3fn:
                        dst, src = dst.view(torch.uint8), src.view(torch.uint8)
                    to.append(dst)
                    frm.append(src.detach().to(dst.device).reshape(dst.shape))
                steps[i] = st["step"]
            if to:
                with torch.no_grad():
                    torch._foreach_copy_(to, frm)
            fl.set_steps(steps)

    def _captured(self, gi):
        return gi in self._flats and self._flats[gi].device_count

    def _keeps(self, gi, opt):
        fl = self._flats.get(gi)
        return fl is not None and (fl.bits, fl.with_master) == (int(opt["state_bits"]), bool(opt["master_weights"]))

    @staticmethod
    def _check_saved(st, p, opt):
        n, bits = p.numel(), int(opt["state_bits"])
        blocks = (n + BLOCK - 1) // BLOCK
        want = {"exp_avg": n, "exp_avg_sq": n} if bits == 32 else \
            {"exp_avg": n, "exp_avg_sq_root": n, "exp_avg_scale": blocks, "exp_avg_sq_root_scale": blocks}
        if opt["master_weights"] and p.dtype != torch.float32 and "master" in st:
            want["master"] = n
        step = st.get("step")
        if torch.is_tensor(step):
            step = step.item() if step.numel() == 1 else None
        if isinstance(step, bool) or not isinstance(step, numbers.Real) or not 0 <= step < 1 << 53 or step != int(step):
            raise ValueError(f"AdamW: the saved step is {st.get('step')!r}, not a whole number >= 0")
        for k, count in want.items():
            if k not in st:
                raise ValueError(f"AdamW: the saved state has no {k} (state_bits={bits})")
            if not torch.is_tensor(st[k]) or st[k].is_complex():
                raise TypeError(f"AdamW: the saved {k} is not a tensor of real numbers")
            if st[k].numel() != count:
                raise ValueError(f"AdamW: the saved {k} has {st[k].numel()} elements, not {count}")
            codes = bits == 8 and k in ("exp_avg", "exp_avg_sq_root")
            if (st[k].dtype == torch.float8_e4m3fn) != codes:
                raise ValueError(f"AdamW: the saved {k} is {st[k].dtype}, not {torch.float8_e4m3fn if codes else torch.float32}")

"""Graph-level latent DDPM on HIP kernels -- drop-in for the reference's ddpm.py
(`MLP`, `Backbone`, `Model`), the denoiser of diff_graphset.py (config 3).

Same constructors and state_dict keys (`backbone.linear_model1.layers.N.*`,
`backbone.embedding_layer.weight`, `backbone.linear_model2.layers.N.*`).  Every Linear
is one MFMA GEMM launch with its bias, exact-erf GELU and residual add fused into the
accumulator write-out (ddpm.py:17-27); the time embedding is added in place.  With weights in
bf16 or fp16 (`model.bfloat16()`) the denoiser runs and trains on the 16-bit operators
(ops.linear_act, ops.embedding; optim.AdamW keeps fp32 masters).
"""
import numpy as np
import torch
import torch.nn as nn

from . import autograd as hag
from . import ops


class MLP(nn.Module):
    """ddpm.py:9-27"""

    def __init__(self, dim_in, dim_hidden, dim_out, num_layer):
        super().__init__()
        self.layers = nn.ModuleList(
            [nn.Linear(dim_in, dim_hidden)] + [nn.Linear(dim_hidden, dim_hidden) for _ in range(num_layer)] + [
                nn.Linear(dim_hidden, dim_out)])
        self.gelu = nn.GELU()

    def forward(self, x):
        ops._dev(x)
        if self.layers[0].weight.dtype in ops.HALF_TYPES:
            return self._forward_half(x)
        x = x.to(torch.float32).contiguous()
        last = len(self.layers) - 1
        if hag.chain_wants_grad(self.chain(), x):
            # training (diff_graphset.py:64-75): HIP forward + backward, see hypdiff_amd/autograd.py
            if x.shape[1] % 4:
                x = ops._pad_k(x, (x.shape[1] + 3) // 4 * 4)
            kinds = (hag.GELU,) + (hag.RES,) * (last - 1) + (hag.LIN,)
            return hag.linear_stack(x, list(self.layers), kinds)
        chain = self.chain()
        if ops.chain_small_ok(x, chain):                 # small batch: the whole stack in one launch
            return ops.linear_chain_small(x, chain)
        return ops.linear_chain(x, chain)

    def _forward_half(self, x):
        """the stack on bf16 / fp16 weights (module.bfloat16() / module.half()), inference and training: one fused launch a
        layer, activations in the weights' type"""
        first, last = self.layers[0], self.layers[-1]
        h = ops.linear_act(x.to(first.weight.dtype), first.weight, first.bias, act="gelu")
        for layer in self.layers[1:-1]:
            h = ops.linear_act(h, layer.weight, layer.bias, act="gelu", resid=h)
        return ops.linear_act(h, last.weight, last.bias)

    def chain(self):
        """gelu(layer(x)) first, x0 + gelu(layer(x0)) in between, plain layer last (ddpm.py:17-27)"""
        last = len(self.layers) - 1
        return [(layer.weight, layer.bias, 1 if idx == 0 else (0 if idx == last else 2))
                for idx, layer in enumerate(self.layers)]


class Backbone(nn.Module):
    """ddpm.py:30-41"""

    def __init__(self, dim_in, dim_hidden, num_layer, n_steps):
        super().__init__()
        self.linear_model1 = MLP(dim_in, dim_hidden, dim_hidden, num_layer)
        self.embedding_layer = nn.Embedding(n_steps, dim_hidden)
        self.linear_model2 = MLP(dim_hidden, dim_hidden, dim_in, num_layer)

    def forward(self, x, idx):
        kind = self.embedding_layer.weight.dtype
        if not (self.linear_model1.layers[0].weight.dtype is kind is self.linear_model2.layers[0].weight.dtype):
            # activations of one type would reach an embedding that reads and writes another
            raise TypeError("Backbone: linear_model1, embedding_layer and linear_model2 have weights of one type, not "
                            f"{self.linear_model1.layers[0].weight.dtype}, {kind}, {self.linear_model2.layers[0].weight.dtype}")
        ops._dev(x)
        if kind in ops.HALF_TYPES:
            # bf16 / fp16 weights: the result comes back in x's type (the noising and the sampler around it stay in fp32)
            h = self.linear_model1(x)
            h = ops.embedding(idx.to(device=x.device, dtype=torch.int64), self.embedding_layer.weight, add=h)
            return self.linear_model2(h).to(x.dtype)
        c1, c2 = self.linear_model1.chain(), self.linear_model2.chain()
        if not hag.chain_wants_grad(c1 + c2, x, self.embedding_layer.weight):
            xf = x.to(torch.float32)
            if ops.chain_small_ok(xf, c1 + c2) and c1[-1][0].shape[0] == self.embedding_layer.weight.shape[1]:
                # inference on a small batch (config 3, B = 200): both MLPs and the time embedding in ONE launch
                idx = idx.to(device=x.device, dtype=torch.int64).contiguous()
                return ops.linear_chain_small(xf, c1 + c2, emb_after=len(c1) - 1, emb=self.embedding_layer.weight,
                                              emb_idx=idx)
        h = self.linear_model1(x)
        idx = idx.to(device=h.device, dtype=torch.int64).contiguous()
        if hag.wants_grad(h, self.embedding_layer.weight):
            return self.linear_model2(hag.EmbeddingAdd.apply(h, self.embedding_layer.weight, idx))
        tab = self.embedding_layer.weight.detach()
        ops._lib.call("hd_embedding_add", ops._p(h), ops._p(tab), ops._p(idx), tab.shape[0], h.shape[0], h.shape[1],
                      ops._stream())
        return self.linear_model2(h)


class Model(nn.Module):
    """ddpm.py:44-111"""

    def __init__(self, dim_in, dim_hidden, num_layer, T, beta_1, beta_T):
        super().__init__()
        self.beta = torch.linspace(start=beta_1, end=beta_T, steps=T)
        self.alpha_bars = torch.cumprod(1 - self.beta, dim=0)
        self.snr = (1 - self.alpha_bars) / self.alpha_bars
        self.deta = 0.01
        self.c = 1.0
        self.backbone = Backbone(dim_in, dim_hidden, num_layer, T)
        self._ab_dev = None

    def getpri(self, t):
        """ddpm.py:63-69"""
        out = self.deta * torch.tanh(np.sqrt(self.c) * t / 2000)
        return out.reshape(t.shape[0], 1)

    def _alpha_bars_dev(self, device):
        if self._ab_dev is None or self._ab_dev.device != torch.device(device):
            self._ab_dev = self.alpha_bars.to(device).contiguous()
        return self._ab_dev

    def loss_fn(self, x, idx=None, target='pred_noise', epsilon=None):
        """ddpm.py:71-85 (forward value; `idx` / `epsilon` optionally inject the draws)"""
        output, epsilon, alpha_bar = self.forward(x, idx=idx, get_target=True, epsilon=epsilon, _train=True)
        if target == 'pred_noise':
            return hag.mse_loss(output, epsilon)
        return hag.mse_loss(output, x)

    def forward(self, x, idx=None, get_target=False, restrict=False, epsilon=None, _train=False):
        """ddpm.py:87-111.  idx None (or `_train`): training-time noising at random / given
        per-row steps; idx int: inference at that step on the already perturbed x."""
        ops._dev(x)
        if idx is None or _train:
            if idx is None:
                if x.is_cuda and torch.cuda.is_current_stream_capturing():
                    # under HIP graph capture the draw has to happen on the device (the reference draws on the host
                    # and copies, ddpm.py:93: same distribution, another generator)
                    idx = torch.randint(0, len(self.alpha_bars), (x.size(0),), device=x.device)
                else:
                    idx = torch.randint(0, len(self.alpha_bars), (x.size(0),)).to(x.device)
            idx = idx.to(device=x.device, dtype=torch.int64).contiguous()
            ab = self._alpha_bars_dev(x.device)
            used_alpha_bars = ab[idx][:, None]
            # fp32 whatever x and the weights are: the kernel reads fp32 rows, the loss is taken on them
            epsilon = torch.randn_like(x, dtype=torch.float32) if epsilon is None else epsilon.to(torch.float32)
            x = x.to(torch.float32).contiguous()
            if epsilon.shape != x.shape:
                raise ValueError(f"Model: epsilon has shape {tuple(epsilon.shape)}, x {tuple(x.shape)}")
            x_tilde = torch.empty_like(x)
            ops._lib.call("hd_ddpm_noise", ops._p(x), ops._p(epsilon.contiguous()), ops._p(idx), ops._p(ab), ab.shape[0],
                          ops._p(x_tilde), x.shape[0], x.shape[1], 1 if restrict else 0, self.deta,
                          float(np.sqrt(self.c)), 2000.0, ops._stream())
        else:
            idx = torch.full((x.size(0),), int(idx), dtype=torch.int64, device=x.device)
            x_tilde = x
            used_alpha_bars = None
        output = self.backbone(x_tilde, idx)
        return (output, epsilon, used_alpha_bars) if get_target else output

"""Alignments drawn from a trained generator in evaluation (BatchNorm with its running statistics, so that an alignment does
not depend on what it is drawn beside), the 2-D tower's products in 8 bits (src/layers.py:91-147, 223-288).

A transposed convolution with kernel 4 and stride 2 is a product -- every pixel's channels times a [channels, 16 x channels]
weight, one column for each tap -- and a fold that sums each output pixel's four taps.  The products run on 8-bit rows
(HipOps.linear_q8 / gemm_q8: a scale for each pixel and each column); the BatchNorm's factor is part of the column scales, its
shift and the LeakyReLU of the fold (HipOps.up_fold_q8), which hands the next product its codes.  Between product and fold
the taps are held in bfloat16: their rounding (2^-9) is below that of the codes they come from (1/254 of a row's largest).
The position tower, a thousandth of the work, stays in fp32.
"""
from __future__ import annotations

from typing import Dict, Tuple

import torch

from pgan_engine import net_dims
from pgan_hip import PganError, rows8

BN_EPS = 1e-5


class Sampler8:
    """sites, positions = Sampler8(...).draw(z), z [n <= batch, latent], of the weights and running statistics that the last
    refresh() took over, also where a captured draw is replayed."""

    def __init__(self, ops, params: Dict[str, torch.Tensor], buffers: Dict[str, torch.Tensor], batch: int, act: str = "sigmoid",
                 latent: int = 128, data: int = 64):
        """params / buffers: the generator's state_dict entries on the GPU (FlatStore.p of an Engine or of a module)."""
        if batch < 1:
            raise ValueError(f"batch must be at least 1, got {batch}")
        if act not in ("sigmoid", "tanh"):
            raise ValueError(f"act must be 'sigmoid' or 'tanh', got {act!r}")
        self.ops, self.P, self.Bf, self.batch, self.latent, self.data = ops, params, buffers, int(batch), int(latent), int(data)
        self.act_id = 1 if act == "sigmoid" else 2
        dm = net_dims(self.data, self.latent)
        self.g2c, self.g2h, self.g1c, self.g1l = dm["g2c"], dm["g2h"], dm["g1c"], dm["g1l"]
        self.n = len(self.g2c) - 2                       # BatchNorm stages of each tower
        dev, B = params["twod_conv_layers.0.weight"].device, self.batch
        f = dict(dtype=torch.float32, device=dev)
        c, h = self.g2c, self.g2h
        # stage i: rows of c[i] channels, one for each pixel of an h[i] x h[i] image (stage 0: the latent vector)
        self.q = [rows8(B * h[i] ** 2, c[i], dev) for i in range(self.n + 1)]
        self.qs = [torch.zeros(B * h[i] ** 2, **f) for i in range(self.n + 1)]
        self.y = [torch.zeros(B * h[i] ** 2, 16 * c[i + 1], dtype=torch.bfloat16, device=dev) for i in range(self.n + 1)]
        self.w = [rows8(16 * c[i + 1], c[i], dev) for i in range(self.n + 1)]
        self.ws = [torch.zeros(16 * c[i + 1], **f) for i in range(self.n + 1)]
        self.shift = [torch.zeros(c[i + 1], **f) for i in range(self.n)]
        self.bias0 = torch.zeros(16 * c[1], **f)
        self.sites, self.pos = torch.zeros(B, self.data, self.data, 1, **f), torch.zeros(B, 1, self.data, **f)
        self.hA = [None] + [torch.zeros(B, self.g1c[i], self.g1l[i], **f) for i in range(1, self.n + 1)]
        self.hH = [None] + [torch.zeros(B, self.g1c[i], self.g1l[i], **f) for i in range(1, self.n + 1)]
        self.stats = [None] + [torch.zeros(2, self.g1c[i], **f) for i in range(1, self.n + 1)]
        self.w1 = [torch.empty_like(params[f"oned_conv_layers.{3 * i}.weight"]) for i in range(self.n + 1)]
        self.norm1 = [None] + [tuple(torch.zeros(self.g1c[i], **f) for _ in range(4)) for i in range(1, self.n + 1)]
        self._parts = {}            # batch size -> running statistics in the form the BatchNorm kernels take sums
        self.refresh()

    def _norm(self, tower: str, i: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Factor and shift of a tower's i-th BatchNorm with its running statistics."""
        k = f"{tower}.{3 * i + 1}"
        gain = self.P[k + ".weight"].double() / torch.sqrt(self.Bf[k + ".running_var"].double() + BN_EPS)
        return gain.float(), (self.P[k + ".bias"].double() - self.Bf[k + ".running_mean"].double() * gain).float()

    @torch.no_grad()
    def refresh(self) -> None:
        """Take over the generator's present weights and running statistics."""
        for i in range(self.n + 1):
            w = self.P[f"twod_conv_layers.{3 * i}.weight"]
            rows = w.detach().permute(2, 3, 1, 0).reshape(-1, w.shape[0]).contiguous()        # (kh, kw, out) x in
            self.ops.quant_rows(rows, self.w[i], self.ws[i])
            if i < self.n:
                gain, shift = self._norm("twod_conv_layers", i)
                self.ws[i].mul_(gain.repeat(16))
                self.shift[i].copy_(shift)
        self.bias0.copy_(self.shift[0].repeat(16))
        for i in range(self.n + 1):
            self.w1[i].copy_(self.P[f"oned_conv_layers.{3 * i}.weight"])
            if i > 0:
                k = f"oned_conv_layers.{3 * (i - 1) + 1}"
                for to, of in zip(self.norm1[i], (self.P[k + ".weight"], self.P[k + ".bias"], self.Bf[k + ".running_mean"],
                                                  self.Bf[k + ".running_var"])):
                    to.copy_(of)
        for n in self._parts:
            self._fill_sums(n)

    def _running_sums(self, n: int):
        """The running statistics as the batch sums that give them: per channel sum and sum of squares of n x length
        values, in the first slice."""
        if n not in self._parts:
            if torch.cuda.is_current_stream_capturing():
                raise PganError(f"draw: make one draw of {n} alignments before capturing one")
            self._parts[n] = [None] + [torch.zeros(self.ops.bn_fwd_partials(n, self.g1c[i], self.g1l[i]), dtype=torch.float64,
                                                   device=self.bias0.device) for i in range(1, self.n + 1)]
            self._fill_sums(n)
        return self._parts[n]

    def _fill_sums(self, n: int) -> None:
        for i in range(1, self.n + 1):
            mean, var = (t.double() for t in self.norm1[i][2:])
            count, slices = n * self.g1l[i], self._parts[n][i].view(self.g1c[i], -1, 2)
            slices[:, 0, 0], slices[:, 0, 1] = mean * count, (var + mean * mean) * count

    @torch.no_grad()
    def draw(self, z: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """sites [n, 1, data, data] and positions [n, 1, data] of z [n, latent] or [n, latent, 1, 1], n <= batch; buffers of
        the sampler, overwritten by the next draw."""
        n = z.shape[0]
        if n > self.batch or z.numel() != n * self.latent:
            raise PganError(f"draw: z {tuple(z.shape)} is not at most {self.batch} rows of {self.latent}")
        o, c, h = self.ops, self.g2c, self.g2h
        if n == 0:
            return self.sites[:0].view(0, 1, self.data, self.data), self.pos[:0]
        z = z.detach().reshape(n, self.latent).to(torch.float32).contiguous()
        # sites
        o.linear_q8(z, self.w[0], self.ws[0], self.y[0][:n], self.q[0], self.qs[0], bias=self.bias0)
        o.quant_rows(self.y[0][:n].view(n * 16, c[1]), self.q[1][:n * 16], self.qs[1], lrelu=True)
        for i in range(1, self.n + 1):
            px = n * h[i] ** 2
            y = self.y[i][:px]
            o.gemm_q8(self.q[i][:px], self.qs[i], self.w[i], self.ws[i], y)
            y = y.view(n, h[i], h[i], -1)
            if i < self.n:
                o.up_fold_q8(y, self.shift[i], self.q[i + 1][:4 * px], self.qs[i + 1])
            else:
                o.up_fold(y, None, self.sites[:n], self.act_id)
        # positions
        parts = self._running_sums(n)
        o.gemm_nn(z, self.w1[0].view(self.latent, -1), self.hA[1][:n].view(n, -1))
        for i in range(1, self.n + 1):
            gain, bias, mean, var = self.norm1[i]        # (momentum 0: the statistics stay)
            o.bn_fwd_apply(self.hA[i][:n], gain, bias, mean, var, self.hH[i][:n], self.stats[i], parts[i], 1, momentum=0.0)
            if i < self.n:
                o.convt1d_up(self.hH[i][:n], self.w1[i], self.hA[i + 1][:n])
            else:
                o.convt1d_up(self.hH[i][:n], self.w1[i], self.pos[:n], self.act_id)
        return self.sites[:n].view(n, 1, self.data, self.data), self.pos[:n]

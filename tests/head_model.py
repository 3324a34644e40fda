"""The softmax head's loss and gradient in float64, and how far a result of
the kernels may be from them, from the roundings that they make.

Roundings counted, with u the half step of the inputs' dtype and
e = 2^-24 that of float32:
  scores    sums of `width` exact products in float32: at most
            (width + 2) e sum_k |h_k W_vk|; tanh under a cap: 4 e cap more
  exp, sum  expf and logf to 4 e; at most 512 additions follow each other
            within a tile and between tiles
  d score   rounded to the dtype twice (the exponential, then the normalised
            value), the label's own once; factors to 16 e; float16 operands
            end at 2^-35 of the largest row weight
  products  sums of vocab (rows) terms in float32: at most that many e of
            the sum of magnitudes; the result rounded once
"""
import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Head:
    def __init__(self, hidden, weight, labels, row_weight=None, reduction="mean", softcap=0.0,
                 z_loss=0.0, grad_scale=1.0):
        self.dtype = hidden.dtype
        width = weight.shape[1]
        vocab = weight.shape[0]
        self.shape = hidden.shape
        h = hidden.detach().reshape(-1, width).double()
        w = weight.detach().double()
        y = labels.reshape(-1).long()
        counts = (y >= 0) & (y < vocab)
        self.counts = counts
        h = torch.where(counts[:, None], h, torch.zeros_like(h))
        y = torch.where(counts, y, torch.zeros_like(y))
        self.h, self.w = h, w
        s = h @ w.T
        err = (width + 2) * E * (h.abs() @ w.abs().T).amax(1, keepdim=True)
        slope = torch.ones_like(s)
        if softcap:
            t = torch.tanh(s / softcap)
            z, slope = softcap * t, 1 - t * t
            err = err + 4 * E * softcap
        else:
            z = s
        lse = torch.logsumexp(z, 1, keepdim=True)
        p = torch.exp(z - lse)
        zy = z.gather(1, y[:, None])
        rl = lse - zy + z_loss * lse ** 2
        u = torch.ones_like(lse) if row_weight is None else row_weight.reshape(-1, 1).double()
        u = torch.where(counts[:, None], u, torch.zeros_like(u))
        if reduction == "mean":
            total = u.sum()
            u = u / total if total != 0 else torch.zeros_like(u)
        keep = counts[:, None].double()
        self.lse, self.row_loss = (lse * keep)[:, 0], (rl * keep)[:, 0]
        self.loss = (u * rl * keep).sum()
        e_lse = err + 600 * E + 4 * E * lse.abs()
        e_rl = e_lse + err + 4 * E * (rl.abs() + lse.abs() + zy.abs()) \
            + z_loss * (2 * lse.abs() * e_lse + 4 * E * lse ** 2)
        self.tol_lse, self.tol_row_loss = (e_lse * keep)[:, 0], (e_rl * keep)[:, 0]
        self.tol_loss = (u.abs() * keep * (e_rl + 4 * E * rl.abs())).sum()

        one = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
        g = u * grad_scale
        f = 1 + 2 * z_loss * lse
        ds = g * (f * p - one) * slope
        half = half_step(self.dtype)
        e_exp = 2 * err + e_lse + 64 * E  # relative error of p
        e_slope = 2 * err / softcap + 16 * E if softcap else torch.zeros_like(err)
        d = ds.abs() * (2 * half + half ** 2) + g.abs() * f * p * (e_exp * slope + e_slope) \
            + one * g.abs() * (f * (e_exp + e_slope) + 32 * E) + 4 * E * ds.abs()
        if self.dtype == torch.float16:
            d = d + g.abs().max() * 2.0 ** -35
        d = d * keep
        self.d_hidden, self.d_weight = ds @ w, ds.T @ h
        n_v, n_r = vocab + 8, h.shape[0] + 8
        tiny = torch.finfo(self.dtype).smallest_normal * torch.finfo(self.dtype).eps
        self.tol_d_hidden = d @ w.abs() + n_v * E * (ds.abs() @ w.abs()) \
            + half * self.d_hidden.abs() + tiny
        self.tol_d_weight = d.T @ h.abs() + n_r * E * (ds.abs().T @ h.abs()) \
            + half * self.d_weight.abs() + tiny

    def check(self, got):
        """Every output of a call within its tolerance, and zeros in rows left out."""
        for name in got._fields:
            x = getattr(got, name).detach()
            want, tol = getattr(self, name), getattr(self, "tol_" + name)
            x = x.double().reshape(want.shape)
            off = (x - want).abs()
            assert bool(torch.isfinite(x).all()), name
            assert bool((off <= tol).all()), \
                f"{name}: {float((off - tol).max()):.3g} beyond its tolerance"
        out = ~self.counts
        assert bool((got.lse.reshape(-1)[out] == 0).all())
        assert bool((got.row_loss.reshape(-1)[out] == 0).all())
        if hasattr(got, "d_hidden"):
            assert bool((got.d_hidden.reshape(len(out), -1)[out] == 0).all())

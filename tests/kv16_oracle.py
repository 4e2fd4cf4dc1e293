"""Attention over the 16-bit paged cache in 64 bits, from its definition, with a bound for what fp32
work and 16-bit roundings may be off by.  Nothing here uses the package."""
import math

import torch


def attention(q, data, tables, lens, starts, *, scale=None, softcap=None, slopes=None, window=None, prefix=None, first=None):
    """(y, bound) in 64 bits ``[T, nh, hd]`` for host lists ``lens``, ``starts`` and tensors on the device.

    The bound of an element, u the half step of the type (eps / 2), p the probabilities:
      u |y|                             the result's own rounding;
      u (sum p |v| + |y|)               the probabilities' rounding before the product with V and before their sum;
      sum p E (|v| + |y|)               an error E of a score moves its probability by E.  E: the products' sum,
                                        (hd + 8) 2^-24 of sum |q k| scale; the cap's tanh 2^-20 of the score, and where
                                        it is c - 2 c / (1 + e) of c up to 512, 2^-22 c (half the exponential's and the
                                        reciprocal's last bits); the distance's product and sum 2^-23 of it; three roundings of
                                        the exponent, 2^-22 of its size;
      (n + 64) 2^-23 (sum p |v| + |y|)  fp32 sums of n terms, the exponential's last bit, the quotient;
      2^-24                             fp16's smallest step.
    """
    T, hd = q.shape[0], data.shape[-1]
    kvh, page = data.shape[1], data.shape[3]
    nh = q.shape[1] // hd
    group = nh // kvh
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    y = torch.zeros((T, nh, hd), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(y)
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        m = hi - lo
        if m <= 0 or n <= 0:
            continue
        pages = data[tables[b, :-(-n // page)].long()]
        rows = q[lo:hi].double().view(m, nh, hd)
        i, j = torch.arange(n - m, n, device=q.device)[:, None], torch.arange(n, device=q.device)[None]
        seen = j <= i
        if prefix is not None:
            seen = seen | ((j < int(prefix[b])) & (i >= 0))
        if window is not None:
            seen = seen & (i - j < window)
        if first is not None:
            seen = seen & (j >= first[lo:hi, None])
        some = seen.any(1)
        for h in range(nh):
            k, v = (pages[:, h // group, c].reshape(-1, hd)[:n].double() for c in (0, 1))
            x = rows[:, h] @ k.t().contiguous() * scale
            err = (rows[:, h].abs() @ k.abs().t().contiguous()) * scale * (hd + 8) * 2.0**-24
            if softcap is not None:
                err = err + x.abs() * 2.0**-20 + (softcap * 2.0**-22 if softcap <= 512 else 0.0)
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                bias = slopes[h].double() * (i - j).abs()
                err = err + (bias.abs() + x.abs()) * 2.0**-23
                x = x - bias
            x = torch.where(seen, x, -math.inf)
            top = x.max(1, keepdim=True).values
            err = err + torch.where(seen, (top - x).abs() + 2, 0.0) * 2.0**-22
            p = torch.where(some[:, None], torch.softmax(x, 1), 0.0)
            v0 = torch.where(seen.any(0)[:, None], v, 0.0)
            o = p @ v0
            a = p @ v0.abs()
            pe = torch.where(p > 0, p * err, 0.0)
            y[lo:hi, h] = o
            bound[lo:hi, h] = (u * (2 * o.abs() + a) * 1.01 + pe @ v0.abs() + pe.sum(1, keepdim=True) * o.abs()
                               + (n + 64) * 2.0**-23 * (a + o.abs()) + 2.0**-24)
    return y, bound


def check(out, y, bound, what=""):
    """Every element within its bound."""
    off = (out.double().view(y.shape) - y).abs()
    assert torch.isfinite(off).all(), f"{what}: {int((~torch.isfinite(off)).sum())} values are not finite"
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst} of the bound"

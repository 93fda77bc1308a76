"""Norm and rotation of heads in 64 bits, one pair at a time, with bounds on what fp32 arithmetic and one rounding may leave."""
import math

import torch


def forward(x, w, pos, freq, R, interleaved, norm, eps, m=1.0):
    """x [..., H, D] with pos [...]: (y, the sum of the magnitudes that each value of y is made of)."""
    x = x.detach().double().cpu()
    r, n, z = _normed(x, w, norm, eps)
    y, size = z.clone(), z.abs()
    for i, (a, b) in enumerate(_pairs(R, interleaved)):
        c, s = _turn(pos, freq[i])
        za, zb = z[..., a], z[..., b]
        y[..., a], y[..., b] = m * (za * c - zb * s), m * (zb * c + za * s)
        size[..., a], size[..., b] = (abs(m) * (za.abs() + zb.abs()),) * 2
    none = (pos.cpu() < 0)[..., None, None]
    return torch.where(none, 0.0, y), torch.where(none, 0.0, size)


def backward(x, w, pos, freq, R, interleaved, norm, eps, g, m=1.0):
    """(dx, its magnitudes, dw, its magnitudes); dw None without norm."""
    x, g = x.detach().double().cpu(), g.detach().double().cpu()
    r, n, _ = _normed(x, w, norm, eps)
    there = (pos.cpu() >= 0)[..., None, None]
    dz, size = g.clone(), g.abs()
    for i, (a, b) in enumerate(_pairs(R, interleaved)):
        c, s = _turn(pos, freq[i])
        ga, gb = g[..., a], g[..., b]
        dz[..., a], dz[..., b] = m * (ga * c + gb * s), m * (gb * c - ga * s)
        size[..., a], size[..., b] = (abs(m) * (ga.abs() + gb.abs()),) * 2
    dz, size = torch.where(there, dz, 0.0), torch.where(there, size, 0.0)
    if not norm:
        return dz, size, None, None
    dw, dw_size = torch.where(there, dz * n, 0.0).flatten(0, -2).sum(0), torch.where(there, size * n.abs(), 0.0).flatten(0, -2).sum(0)
    wd = 1.0 if w is None else w.detach().double().cpu()
    dn, dn_size = dz * wd, size * (wd if w is None else wd.abs())
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    dx_size = r * (dn_size + n.abs() * (dn_size * n.abs()).mean(-1, keepdim=True))
    return torch.where(there, dx, 0.0), torch.where(there, dx_size, 0.0), dw, dw_size


def _normed(x, w, norm, eps):
    if not norm:
        return 1.0, x, x
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * r
    return r, n, n if w is None else n * w.detach().double().cpu()


def _pairs(R, interleaved):
    return [(2 * i, 2 * i + 1) if interleaved else (i, i + R // 2) for i in range(R // 2)]


def _turn(pos, f):
    """Of every position and each head: Python's math.fmod is exact, so the angle is off by the product's rounding alone."""
    a = pos.detach().cpu().double() * f
    return a.cos()[..., None], a.sin()[..., None]


def close(got, want, size, slack):
    """One rounding to got's type (half a step relative to the value, half a step of the subnormals), and `slack` of the magnitudes for fp32."""
    info = torch.finfo(got.dtype)
    got = got.detach().double().cpu()
    tol = info.eps / 2 * want.abs() + slack * size + info.tiny * info.eps / 2
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst by {((got - want).abs() / tol).nan_to_num(math.inf).max():.3g} of what is allowed"

"""Block-scaled FP8 in 64 bits: quantizers, linear and routed experts, with
bounds on how far an f32 implementation may be.

Test infrastructure only. Torch float64 tensors on any device.

Bounds. e4m3 products are exact in f32; a tensor-core sum of K of them in f32
is taken to lose at most ``K / 8`` units of 2^-23 of the sum of magnitudes
(four K = 32 steps per 128 values, each keeping at least f32's 24 bits, and
one scaled addition per 128 values). A bf16 rounding loses 2^-8 of the value.
A value that the implementation knows only to within ``d`` may round to
another e4m3 code: the bound then holds the distance of the codes at both
ends of the interval.
"""
import math

import torch

B = 128
U = 2.0 ** -23
BF16 = 2.0 ** -8


def e4m3(p):
    """p (float64) rounded to the nearest e4m3 value, ties to even, saturated at 448."""
    mag = p.abs()
    _, e = torch.frexp(mag)                        # mag = m 2^e, 1/2 <= m < 1
    step = torch.exp2((e - 1).clamp(-6, 8).double() - 3)
    return torch.sign(p) * torch.minimum(torch.round(mag / step) * step, torch.full_like(mag, 448.0))


def scales(amax):
    """(inverse, scale) of blocks with these maxima, as f32 values in float64."""
    a = torch.where(amax.isfinite(), amax.clamp_min(float(torch.tensor(1e-30))), math.nan)
    return (448.0 / a).float().double(), (a / 448.0).float().double()


def _cut(x, dim):
    n = -(-x.shape[dim] // B)
    return [x.narrow(dim, i * B, min(B, x.shape[dim] - i * B)) for i in range(n)]


def quantize_rows(x):
    """(codes, scale (M, blocks)) of x (M, K), an exact float64 image of the input."""
    qs, ss = [], []
    for v in _cut(x, 1):
        inv, s = scales(v.abs().amax(1, keepdim=True))
        qs.append(e4m3((v * inv).float().double()) if v.numel() else v)
        ss.append(s)
    return torch.cat(qs, 1), torch.cat(ss, 1)


def quantize_blocks(w):
    """(codes, scale) of w (E, N, K)."""
    rows, ss = [], []
    for r in _cut(w, 1):
        cols, sr = [], []
        for v in _cut(r, 2):
            inv, s = scales(v.abs().amax((1, 2), keepdim=True))
            cols.append(e4m3((v * inv).float().double()))
            sr.append(s)
        rows.append(torch.cat(cols, 2))
        ss.append(torch.cat(sr, 2))
    return torch.cat(rows, 1), torch.cat(ss, 1)


def value_rows(q, s):
    return q * s.repeat_interleave(B, -1)[..., : q.shape[-1]]


def value_blocks(q, s):
    return q * s.repeat_interleave(B, -2)[..., : q.shape[-2], :].repeat_interleave(B, -1)[..., : q.shape[-1]]


def product(a, w):
    """(a w^T, bound) of float64 values."""
    return a @ w.mT, (a.shape[-1] / 8 + 4) * U * (a.abs() @ w.abs().mT)


def linear(x, wq, ws, bias=None, out_bf16=True):
    y, tol = product(value_rows(*quantize_rows(x)), value_blocks(wq, ws))
    if bias is not None:
        y = y + bias
    return y, tol + U * y.abs() + (BF16 * y.abs() if out_bf16 else 0.0)


def activation(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    return torch.nn.functional.gelu(g, approximate="tanh")


def experts(x, ids, weights, guq, gus, dwq, dws, act):
    """(out (T, H), bound) of the routed forward; x float64 image of the hidden states."""
    T, H = x.shape
    E, two_i, _ = guq.shape
    xd = value_rows(*quantize_rows(x))
    out, tol = torch.zeros_like(x), torch.zeros_like(x)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        y, dy = product(xd[t], value_blocks(guq[e], gus[e]))
        g, u = y.chunk(2, 1)
        dg, du = dy.chunk(2, 1)
        a = activation(act, g)
        h = a * u
        # |act'| < 1.13; the activation itself to 1e-5 (its exponential's argument)
        dh = 1.13 * dg * u.abs() + (a.abs() + 1.13 * dg) * du + 1e-5 * h.abs()
        hd, dhd = torch.empty_like(h), torch.empty_like(h)
        for lo in range(0, h.shape[1], B):
            v, d = h[:, lo:lo + B], dh[:, lo:lo + B]
            amax = v.abs().amax(1, keepdim=True)
            inv, s = scales(amax)
            r = (d.amax(1, keepdim=True) / amax.clamp_min(1e-30)) + 4 * U      # error of the scale
            p = v * inv
            dp = d * inv + p.abs() * r
            q = e4m3(p)
            hd[:, lo:lo + B] = q * s
            dhd[:, lo:lo + B] = (torch.maximum((e4m3(p + dp) - q).abs(), (e4m3(p - dp) - q).abs()) + q.abs() * r) * s
        dw = value_blocks(dwq[e], dws[e])
        y, dy = product(hd, dw)
        dy = dy + dhd @ dw.abs().T
        w = weights[t, j][:, None]
        out.index_add_(0, t, w * y)
        tol.index_add_(0, t, w.abs() * (dy + (ids.shape[1] + 1) * U * y.abs()))
    return out, tol + BF16 * out.abs()

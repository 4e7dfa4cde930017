"""Plain 64-bit forms of the paged cache's operators, and how far an exact kernel's roundings may take a result from them.

Tolerances count roundings (half a step of type t is torch.finfo(t).eps / 2, relative):
- a rotated element a c - b s: cos and sin, the products and the sum in f32, each within 2^-22 of |a| + |b| times the
  amplitude (five roundings of 2^-24 and the angle's 2^-23), then one rounding of the result;
- attention: scores are sums of head_dim f32 products (head_dim x 2^-24 of the sum of their absolute values, and of the
  largest over the row's keys: `ds`), so a weight is within a factor 1 +- 2 ds; the exponential and its argument add
  2^-20; weights are rounded once to the cache's type (eps / 2) for the product with V and summed in f32 (n x 2^-24); f16
  weights below 2^-24 of the largest lose bits (2^-34 of it at most); the result is rounded once (and below the smallest
  normal number by the subnormal step).
"""
import math

import torch


def rope_freqs(dim, base, scaling="none", factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0):
    th, amp = [], 1.0
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        if scaling == "linear":
            f /= factor
        if scaling == "ntk":
            f = (base * factor ** (dim / (dim - 2))) ** (-2 * i / dim)
        if scaling == "yarn":
            lo = max(math.floor(dim * math.log(original / (beta_fast * 2 * math.pi)) / (2 * math.log(base))), 0)
            hi = min(math.ceil(dim * math.log(original / (beta_slow * 2 * math.pi)) / (2 * math.log(base))), dim - 1)
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = r * f / factor + (1 - r) * f
            amp = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
        if scaling == "bands":
            s = min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low)))
            f = (1 - s) * f / factor + s * f
        th.append(f)
    return th, amp


def rotated(x, pos, dim, layout, th, amp):
    """x [rows, heads, d] at pos [rows] in 64 bits, and the tolerance of each element."""
    y, step = x.double(), torch.finfo(x.dtype).eps / 2
    a = pos.double().view(-1, 1, 1) * torch.tensor(th, dtype=torch.float64, device=x.device)
    c, s = amp * torch.cos(a), amp * torch.sin(a)
    i = torch.arange(dim // 2, device=x.device)
    lo, hi = (i, i + dim // 2) if layout == "half" else (2 * i, 2 * i + 1)
    p, q = y[..., lo], y[..., hi]
    out = y.clone()
    out[..., lo], out[..., hi] = p * c - q * s, q * c + p * s
    tol = torch.zeros_like(y)
    tol[..., lo] = tol[..., hi] = (p.abs() + q.abs()) * amp * 2 ** -22
    tol[..., :dim] += out[..., :dim].abs() * step + torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    return out, tol


def attention(q, k, v, pos0, scale, window=0, sinks=None, gate=None):
    """Tokens q [t, q_heads, d] at positions pos0 .. over k, v [n, kv_heads, d]: result and tolerance, 64 bits. Rows see
    (p - window, p]; what a row does not see is left out, whatever it holds."""
    t, heads, d = q.shape
    n, kv_heads = k.shape[:2]
    eps = torch.finfo(q.dtype).eps
    group = heads // kv_heads
    p = torch.arange(pos0, pos0 + t, device=q.device)[:, None]
    j = torch.arange(n, device=q.device)[None]
    seen = (j <= p) & ((j > p - window) if window else (j >= 0))
    out = torch.empty(t, heads, d, dtype=torch.float64, device=q.device)
    tol = torch.empty_like(out)
    for h in range(heads):
        kk, vv = k[:, h // group].double(), v[:, h // group].double()
        x = scale * (q[:, h].double() @ torch.nan_to_num(kk, 0.0, 0.0, 0.0).T.contiguous())
        # a row that sees NaN or infinities is none of these tests' but test_odd_values', which checks it apart
        ds = scale * (q[:, h].double().abs() @ torch.nan_to_num(kk, 0.0, 0.0, 0.0).abs().T.contiguous())
        x = x.masked_fill(~seen, -math.inf)
        ds = ds.masked_fill(~seen, 0.0).amax(1, keepdim=True) * d * 2.0 ** -24
        top = x.amax(1, keepdim=True)
        if sinks is not None:
            top = torch.maximum(top, sinks[h].double())
        w = torch.exp(x - top)
        total = w.sum(1, keepdim=True)
        if sinks is not None:
            total = total + torch.exp(sinks[h].double() - top)
        w = w / total
        fine = torch.nan_to_num(vv, 0.0, 0.0, 0.0)
        out[:, h] = w @ fine
        size = w @ fine.abs()
        tol[:, h] = size * (eps / 2 + 4 * ds + n * 2.0 ** -24 + 2.0 ** -19) + n * 2.0 ** -34 * fine.abs().max() / total
    if gate is not None:
        s = torch.sigmoid(gate.double())
        out, tol = out * s, tol * s + (out * s).abs() * 2.0 ** -20
    tol = tol + (out.abs() + tol) * eps / 2 + torch.finfo(q.dtype).smallest_normal * eps
    return out, tol


def close(got, want, tol, what=""):
    bad = (got.double() - want).abs() - tol
    assert not (bad > 0).any() and torch.isfinite(got).all(), \
        f"{what}: {int((bad > 0).sum())} of {bad.numel()} values off, the worst by {float((got.double() - want).abs().max()):.3g}, " \
        f"{float(((got.double() - want).abs() / tol).max()):.3g} of its tolerance"

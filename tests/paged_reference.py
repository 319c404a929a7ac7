"""Plain 64-bit statements of the paged cache's operators (cactus_amd/paged.py), on the CPU, one sequence at a time, and the
error bounds that the tests hold the kernels to.  Halves round by at most 2^-11 of the value, floats by 2^-24."""
import math

import torch

U16, U32 = 2.0 ** -11, 2.0 ** -24


def offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32)


def make_tables(gen, used, width, total):
    """Disjoint page lists in random order, -1 behind a sequence's last page."""
    order = torch.randperm(total, generator=gen).int()
    t = torch.full((len(used), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def norm_rope(x, weight, eps, theta, positions):
    """(value, sum of the absolute terms it is made of) of rope(rms_norm(x)); x [n, H, D], positions [n]."""
    x = x.double()
    D = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if not theta:
        return x, x.abs()
    freq = theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = positions.double()[:, None, None] * freq
    a, b = x[..., :D // 2], x[..., D // 2:]
    y = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    s = a.abs() + b.abs()
    return y, torch.cat([s, s], -1)


def row_bound(D):
    """fp32 error of a normed and rotated element, relative to |a| + |b| of its pair: the norm's sum (D terms) and its
    root, the weight, cosine and sine (an angle known to 2^-24 turns is 2 pi 2^-24 off), two products and a sum."""
    return (D + 32) * U32


def finite(x):
    """What the cache stores of infinities and NaN."""
    x = x.double().clone()
    x[torch.isnan(x)] = 0
    return x.clamp(-65504, 65504)


def seen(position, keys, window, sink):
    j = torch.arange(keys)
    ok = j <= position
    if window:
        ok &= (position - j <= window) | (j < sink)
    return ok


def attend(q, k, v, positions, window, sink, scale=0.0, extra=None, ratio=1.0):
    """q [n, Hq, D], k / v [L, Hkv, D] -> (out, bound) [n, Hq, D].  extra [L]: keys that can be seen at all.
    The bound: the output's rounding; every weight rounded to binary16; scores in fp32 (D products, the scale, the base-2
    argument: D + 8 roundings of the sum of |q k|), which enter numerator and denominator; fp32 sums over L keys.
    Binary16 is subnormal below 2^-14: a weight that small beside the largest is rounded by 2^-25 of the largest, however
    small it is.  ratio: how far the page scales of the values lie apart; a weight is rounded together with its page's scale,
    so beside the largest it may be that much smaller, and its value that much larger."""
    n, Hq, D = q.shape
    L, Hkv, _ = k.shape
    scale = scale or 1 / math.sqrt(D)
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros((n, Hq, D), dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(n):
        ok = seen(int(positions[i]), L, window, sink)
        if extra is not None:
            ok &= extra
        if not bool(ok.any()):
            continue
        kk, vv = k[ok], v[ok]
        for h in range(Hq):
            hk = h * Hkv // Hq
            s = kk[:, hk] @ q[i, h] * scale
            mag = (kk[:, hk].abs() @ q[i, h].abs() * abs(scale)).max().item()
            w = torch.softmax(s, 0)
            out[i, h] = w @ vv[:, hk]
            weighted = w @ vv[:, hk].abs()
            delta = (D + 8) * U32 * mag
            tol[i, h] = U16 * out[i, h].abs() + weighted * (U16 + 2 * delta + (int(ok.sum()) + 16) * U32) + 2.0 ** -24
            small = w < w.max() * ratio * 2.0 ** -14
            tol[i, h] += 2.0 ** -25 * w.max() * ratio * vv[small][:, hk].abs().sum(0)
    return out, tol


def gather(pages, scales, table, page, start, count):
    """Tokens start .. start + count - 1 of a sequence as float64 [count, H, D], and which of them have a page."""
    P = pages.shape[2]
    at = torch.arange(start, start + count)
    idx = at // P
    ids = torch.where(idx < table.shape[0], table[idx.clamp(max=table.shape[0] - 1)], torch.tensor(-1, dtype=torch.int32)).long()
    ok = (ids >= 0) & (ids < pages.shape[0])
    ids = torch.where(ok, ids, 0)
    x = pages[ids, :, at % P].double() * scales[ids].double()[:, :, None]
    return x * ok[:, None, None], ok

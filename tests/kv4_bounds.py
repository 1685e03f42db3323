"""Attention over the 4-bit KV cache in 64 bits, with the distance that the kernels' roundings allow per row, head and group of 64 channels.

The roundings are independent of one another, so their squares add up (an error of at most e, uniform, has the variance e^2 / 3); a row is
within six times the root of the sum, plus what is a bound on all of them.  With o the row's output, p its weights, v the values and lo the
low ends of their groups:
  both      o is rounded to bf16: 2^-8 of it at most, and so is its norm.  Scores are sums in 32 bits: 2^-21 of the sum of |q k|, which moves the row by twice that of
            sum p |v - o|.  The final normalisation and an approximate exponential: 2^-19.
  decode    p s is rounded to fp16 (2^-11), the share p n s = p (v - lo) of each value with it, and not below 2^-25 of the largest p s.  Tensor-core
            sums round towards zero, by up to 2^-24 of sum p n s at each of the (at most 256) blocks of a warp.
  prefill   p and v are rounded to fp16, and p not below 2^-25 of the largest; keys too, which moves a score by 2^-11 of q k in each channel.
"""
import math

import torch


def attention(q, k, v, pos, window=0, limit=None, gate=None, prefill=False, keys=None):
    """(rows [T, Hq, D], allowed distance [T, Hq, D / 64] in the 2-norm) of bf16 queries over the values [n, Hkv, D] that the cache stands for.
    ``keys``: [T, n] truth values of what each row sees, in place of positions and window."""
    T, Hq, D = q.shape
    n, Hkv = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    if keys is None:
        kp = torch.arange(n)[None]
        keys = kp <= (pos if limit is None else torch.maximum(pos, limit))[:, None]
        if window:
            keys = keys & (kp > pos[:, None] - window)
    some = keys.any(1)
    want, tol = torch.empty(T, Hq, D, dtype=torch.float64), torch.empty(T, Hq, D // 64, dtype=torch.float64)
    norms = lambda x: x.unflatten(-1, (-1, 64)).square().sum(-1)  # noqa: E731   squared, per group
    for h in range(Hkv):
        kh, vh = (torch.where(keys.any(0)[:, None], x[:, h], 0.0) for x in (k, v))
        lo = vh.unflatten(-1, (-1, 64)).amin(-1).repeat_interleave(64, -1)
        share, step = vh - lo, (vh - lo).unflatten(-1, (-1, 64)).amax(-1) / 15
        for i in range(h * Hq // Hkv, (h + 1) * Hq // Hkv):
            s = (q[:, i] @ kh.T / math.sqrt(D)).masked_fill(~keys, -math.inf)
            p = torch.where(some[:, None], s.softmax(-1), 0.0)
            o = p @ vh
            size = norms(vh) if prefill else norms(share)
            var = (2 if prefill else 1) * 2.0 ** -22 / 3 * (p.square() @ size)
            if prefill:
                var += 2.0 ** -50 / 3 * p.amax(-1, keepdim=True).square() * (keys.double() @ size)
                w = p.square() * (q[:, i].square() @ kh.square().T) / D * 2.0 ** -22 / 3
                var += (w @ norms(vh) + w.sum(-1, keepdim=True) * norms(o) - 2 * ((w @ vh) * o).unflatten(-1, (-1, 64)).sum(-1)).clamp(min=0)
                bound = torch.zeros_like(var)
            else:
                most = torch.stack([(p * step[:, g]).amax(-1) for g in range(D // 64)], -1)
                var += 2.0 ** -50 / 3 * most.square() * 225 * 64 * keys.sum(-1, keepdim=True)
                bound = 2.0 ** -16 * norms(p @ share).sqrt()
            off = 2.0 ** -21 * ((q[:, i].abs() @ kh.abs().T) / math.sqrt(D)).masked_fill(~keys, 0.0).amax(-1, keepdim=True)
            bound += (2 * off + 2.0 ** -19) * (p @ norms(vh).sqrt() + norms(o).sqrt()) + 2.0 ** -8 * norms(o).sqrt()
            g = torch.sigmoid(gate[:, i].double()) if gate is not None else torch.ones_like(o)
            want[:, i] = o * g
            tol[:, i] = (6 * var.sqrt() + bound) * g.unflatten(-1, (-1, 64)).amax(-1) + 1e-37
    return want, tol


def worst(out, want, tol):
    """Largest distance in units of what is allowed: above 1, some row is wrong.  (Infinite where an output is no finite number.)"""
    out = out.double().cpu()
    if not torch.isfinite(out).all():
        return math.inf
    return float(((out - want).unflatten(-1, (-1, 64)).norm(dim=-1) / tol).amax())


def edge_queries(g, k, pos, Hq, window=0):
    """bf16 queries [T, Hq, D] that put weight on the keys at the borders of what each row sees: its own and the next one, the window's first and the
    one before it.  (Against these a row that misses one of them, or sees one too many, is far off; random queries notice it in short contexts only.)"""
    n, Hkv, D = k.shape
    q = torch.randn(len(pos), Hq, D, generator=g, dtype=torch.float64)
    at = [pos, pos + 1] + ([pos - window] if window else [torch.zeros_like(pos)]) + ([pos - window + 1] if window > 1 else [])
    for a in at:
        key = k[a.clamp(0, n - 1)].repeat_interleave(Hq // Hkv, 1) * ((a >= 0) & (a < n))[:, None, None]
        q = q + key * (math.log(n) + 1) * math.sqrt(D) / k.square().sum(-1).mean()
    return q.to(torch.bfloat16)

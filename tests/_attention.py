"""Single-token attention from its definition in 64 bits, with the error that
two-part products leave, element by element.

The kernel carries the rotated query and the softmax weights as hi + lo, two
bf16 numbers each (a rounding to bf16 is off by at most 2^-8 of the value, so the
pair by 2^-16), sums in fp32 and rounds the output to bf16 once (2^-8).  Hence

* a score is off by at most 2^-16 sum |q' k| / sqrt(128) for the split of the
  rotated q', as much again for its fp32 sum (128 terms, each off by at most
  2^-23 of the running magnitude), and 2^-20 sum (|x1| + |x2|) |k| / sqrt(128)
  for the rotation of the pair (x1, x2): an angle off by 2e-7, sine, cosine and
  three operations of 32 bits each;
* a weight is off by its score's error, 2^-16 of itself for its own split and
  at most 2^-16 for exponential, rescaling and the sums of products and weights;
  another 2^-15 covers chains of up to 128 steps of 16 keys (2^-23 of the running
  magnitude each, in the products and in the sum);
* the output is sum p v / sum p, so an error e_j of weight j moves it by at most
  p_j e_j (|v_j| + |o|).
"""
import math

import torch

D = 128


def turned(x, pos, theta):
    """(rotation of x [heads, 128] to `pos` in 64 bits, |x1| + |x2| of each column's pair)."""
    inv = theta ** (-torch.arange(64, dtype=torch.float64, device=x.device) / 64)
    c, s = (pos * inv).cos(), (pos * inv).sin()
    x1, x2 = x.double()[..., :64], x.double()[..., 64:]
    size = x1.abs() + x2.abs()
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1), torch.cat([size, size], -1)


def definition(q, k, v, pos, theta=0.0):
    """(output, bound of its error) of queries q [Hq, 128] at `pos` over keys and values [n, Hkv, 128]."""
    group = q.shape[0] // k.shape[1]
    qq, size = turned(q, pos, theta) if theta else (q.double(), torch.zeros_like(q, dtype=torch.float64))
    kk, vv = k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    p = (torch.einsum("hd,jhd->hj", qq, kk) / math.sqrt(D)).softmax(-1)
    o = torch.einsum("hj,jhd->hd", p, vv)
    error = torch.einsum("hd,jhd->hj", 2.0 ** -15 * qq.abs() + 2.0 ** -20 * size, kk.abs()) / math.sqrt(D) + 2.0 ** -14
    moved = torch.einsum("hj,jhd->hd", p * error, vv.abs()) + (p * error).sum(1, keepdim=True) * o.abs()
    return o, 1.01 * 2.0 ** -8 * o.abs() + moved


def excess(got, q, kc, vc, lengths, theta=0.0):
    """The largest error of got [batch, Hq, 128] beyond its bound over the caches
    [batch, room, Hkv, 128] as they are now; at most 0 where all is well."""
    worst = -math.inf
    for b, n in enumerate(lengths):
        if n == 0:
            worst = max(worst, float(got[b].abs().max()))
            continue
        worst = max(worst, beyond(got[b], *definition(q[b], kc[b, :n], vc[b, :n], n - 1, theta)))
    return worst


def beyond(got, ref, bound):
    over = (got.double() - ref).abs() - bound
    return math.inf if over.isnan().any() else float(over.max())


def heavy_keys(n):
    """Keys to lift: the first, the last and some 30 between, in every part that n keys may be split into."""
    return sorted({*range(0, n, max(1, n // 30)), n - 1})


def lift(q, k, heavy, pos, theta=0.0):
    """Sets the keys `heavy` of k [n, Hkv, 128] so that they share most of the
    weight of the first query head on each (all heads' after rotation to `pos`)."""
    group = q.shape[0] // k.shape[1]
    qq = turned(q, pos, theta)[0] if theta else q.double()
    for h in range(k.shape[1]):
        x = qq[h * group]
        # a score of log n + 2 beside random ones of size about 1
        k[heavy, h] = (x * ((math.log(k.shape[0]) + 2) * math.sqrt(D) / float(x @ x))).to(k.dtype)

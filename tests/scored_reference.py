"""Scored attention in 64 bits, and how far a 16- or 32-bit result may be from it.

``attend`` is the definition: capped, biased and masked scores over a sequence's keys, softmax, weighted sum.
``bound`` adds up the roundings a kernel that sums in fp32 makes, each at most half a step of its type
(``torch.finfo(t).eps / 2``):

* the weights, rounded to the launch's type before the product with V, and the partial outputs of a split range:
  2 half steps of A = sum_k p_k |v_k| (weights are positive and sum to 1);
* the output: a half step of |out|;
* fp32: a score is off by ds = (D + 8) half steps of S, the largest sum_d |q_d k_d| |scale| of the row, plus 4 half
  steps of the largest score in log2 units for the scale and the exponent, plus 2e-7 of the cap (the tanh is
  1 - 2 / (e + 1): a difference of numbers up to 1, three roundings); a weight moves by 2 ds relative (numerator and
  denominator), so the output by 2 ds A; the running sums of n keys add n / 16 + 16 half steps of A (a tile of 16 keys is
  one product, summed as a whole).
"""

from __future__ import annotations

import numpy as np
import torch


def attend(q, k, v, positions, scale, softcap=0.0, slopes=None, first=0, prefix=0, kv_len=None):
    """q (R, Hq, D), k / v (T, Hkv, D) (any float type, on any device), positions (R,). Returns float64
    (out, A, S): (R, Hq, D), (R, Hq, D) and (R, Hq, 2) with the row's S and largest |score|."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    rows, hq, d = q.shape
    t, hkv, _ = k.shape
    kv_len = t if kv_len is None else kv_len
    pos = torch.as_tensor(list(positions), dtype=torch.int64)
    key = torch.arange(t)
    seen = (key[None] >= first) & (key[None] < kv_len) & ((key[None] <= pos[:, None]) | (key[None] < prefix))
    out = torch.zeros((rows, hq, d), dtype=torch.float64)
    weight = torch.zeros_like(out)
    size = torch.zeros((rows, hq, 2), dtype=torch.float64)
    dist = (pos[:, None] - key[None]).abs().double()
    for r in range(rows):
        keep = seen[r].nonzero()[:, 0]
        if keep.numel() == 0:
            continue
        for h in range(hq):
            kk, vv = k[keep, h // (hq // hkv)], v[keep, h // (hq // hkv)]
            s = (kk @ q[r, h]) * scale
            size[r, h, 0] = (kk.abs() @ q[r, h].abs()).max() * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * dist[r, keep]
            size[r, h, 1] = s.abs().max()
            p = torch.softmax(s, 0)
            out[r, h] = p @ vv
            weight[r, h] = p @ vv.abs()
    return out, weight, size


def bound(out, weight, size, dtype, d, keys, softcap=0.0):
    u32, u = torch.finfo(torch.float32).eps / 2, torch.finfo(dtype).eps / 2
    ds = (d + 8) * u32 * size[..., :1] + 4 * u32 * 1.4427 * size[..., 1:] + 2e-7 * softcap
    fp32 = 2 * ds + (keys / 16 + 16) * u32
    p = 0.0 if dtype == torch.float32 else 2 * u
    return u * out.abs() + (p + fp32) * weight * (1 + u)


def check(got, out, weight, size, dtype, d, keys, softcap=0.0, what=""):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    over = (got - out).abs() / bound(out, weight, size, dtype, d, keys, softcap).clamp_min(1e-30)
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound at {np.unravel_index(int(over.argmax()), over.shape)}"


LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def round4(x, dtype):
    """The values rows stand for in a 4-bit pool whose attention runs in ``dtype``: per 32 elements the smallest permitted
    power of two whose sevenfold reaches the largest magnitude, then the nearest level (the even one on a tie); a
    group with a NaN or an infinity is NaN. Float64."""
    g = x.detach().cpu().double().unflatten(-1, (-1, 32)).numpy()
    lo, hi = (-23, 13) if dtype == torch.float16 else (-125, 125)
    top = np.abs(g).max(-1, keepdims=True)
    bad = ~np.isfinite(g).all(-1, keepdims=True)
    top = np.where(bad | (top == 0), 1.0, top)
    e = np.frexp(top)[1] - 3  # top < 2^(e + 3), so 7 * 2^(e - 1) < top
    e = np.where(7.0 * np.exp2(e.astype(np.float64)) < top, e + 1, e)
    e = np.where((np.abs(g).max(-1, keepdims=True) == 0) & ~bad, lo, e)
    step = np.exp2(np.clip(e, lo, hi).astype(np.float64))
    # past 8 the nearest level is 6 in any case (and past 2^53 a difference to a level is rounded away)
    r = np.minimum(np.abs(np.where(bad, 0.0, g)) / step, 8.0)
    gap = np.abs(r[..., None] - np.array(LEVELS))
    near = gap == gap.min(-1, keepdims=True)
    even = np.array([i % 2 == 0 for i in range(8)])
    code = np.where((near & even).any(-1), (near & even).argmax(-1), near.argmax(-1))
    out = np.where(bad, np.nan, np.sign(np.where(bad, 0.0, g)) * np.array(LEVELS)[code] * step)
    return torch.from_numpy(out).flatten(-2)

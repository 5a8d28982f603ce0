"""The paged K/V cache's definitions in 64 bits (numpy / torch double, CPU).

Tolerance of attention against them, per output element, from the kernels' roundings (a rounding is off by at
most half a step: bf16 2^-8, half 2^-11, fp32 2^-24, relative):
  * the bf16 output: 2^-8 |out|;
  * P in half (int4 rows): 2^-11 sum_j p_j |v_j|, and 2^-25 sum_j |v_j| for subnormal P (p <= 1 before the
    division by l >= 1); in two bf16 terms (bf16 rows, at most 16 query rows): 2^-16 sum_j p_j |v_j|, below the
    former; in bf16 (bf16 rows, more query rows): 2^-8 sum_j p_j |v_j|;
  * a score s = scale sum_d q_d k_d in fp32: at most D / 16 additions of 16-term products, each step off by at
    most 2^-22 of B = scale sum_d |q_d k_d|: 2^-19 B for D <= 128, on p through exp twice (numerator and l).
    int4 rows, few query rows: a code c enters as 64 + n, n = c + 8 < 16, and 72 q is taken off again, so the
    sums of a group reach scale sum_d |q_d| 80 s, s = max|k| / 7 of the group; two products and one fused
    multiply-add a group, each off by 2^-23 of that: with B' = scale sum_d |q_d| 80 s_d, 2^-21 B' in all;
    exp2 itself 2^-22, corrections of the running maximum and l: n / 16 steps of 2^-23 each, P V the same."""
import math

import numpy as np
import torch


def bf16_round(x):
    return torch.as_tensor(x, dtype=torch.float32).to(torch.bfloat16)


def codes(x):
    """int4 rows of x (bf16 [..., D]): (integers, scales), in 64 bits."""
    y = x.double()
    y = y.reshape(*y.shape[:-1], -1, 32)
    top = y.abs().amax(-1, keepdim=True)
    s = (top / 7).to(torch.bfloat16).double().clamp(2.0 ** -14, 9344.0)
    c = torch.round(y / s).clamp(-7, 7)
    bad = ~torch.isfinite(y).all(-1, keepdim=True)
    c = torch.where(bad, torch.zeros_like(c), c)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    return c, s


def held(x, int4):
    """The values the cache holds for rows x (bf16), as double."""
    if not int4:
        return x.double()
    c, s = codes(x)
    return (c * s).reshape(x.shape)


def visible(n, i, window, sinks):
    j = torch.arange(n)
    ok = j <= i
    if window:
        ok &= (j > i - window) | (j < sinks)
    return ok


def attend(q, k, v, i0, window=0, sinks=0, scale=None, int4=True):
    """q [t][Hq][D], held k, v [n][H][D] (double): rows i0 .. i0 + t - 1.  Returns (out, tolerance)."""
    t, hq, D = q.shape
    n, H = k.shape[:2]
    G = hq // H
    scale = D ** -0.5 if scale is None else scale
    p_step = 2.0 ** -8 if not int4 and t * G > 16 else 2.0 ** -11
    q = q.double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for x in range(t):
        j = visible(n, i0 + x, window, sinks).nonzero()[:, 0]
        for h in range(hq):
            kk, vv = k[j, h // G], v[j, h // G]
            s = kk @ q[x, h] * scale
            p = torch.softmax(s, 0)
            o = p @ vv
            a = p @ vv.abs()
            B = float((kk.abs() @ q[x, h].abs()).max() * scale) * 2.0 ** -19
            if int4:
                top = kk.abs().reshape(len(j), -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(len(j), D)
                B += float((top @ q[x, h].abs()).max() * scale) * 80 / 7 * 2.0 ** -21
            out[x, h] = o
            tol[x, h] = 2.0 ** -8 * o.abs() + a * (p_step + B + (len(j) / 16 + 64) * 2.0 ** -22) + \
                2.0 ** -25 * vv.abs().sum(0)
    return out, tol


def assert_close(got, want, tol, what=""):
    err = (got.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.2f} of the tolerance"

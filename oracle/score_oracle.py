"""CPU oracle of attention by a score rule, of normed and rotated heads, in float64.  TEST INFRASTRUCTURE ONLY.

Nothing in the product package may import this module.

``score_attention`` restates, key by key and without any tiling, what ``aicomp_paged_score_attn`` computes: for the row at
position p of its sequence and head h,

    s_j = scale q.k_j;  s_j = cap tanh(s_j / cap);  s_j -= slope_h |p - j|
    visible: first <= j, p - j < window, j <= p or j < prefix
    out = sum_j e^{s_j} v_j / sum_j e^{s_j};  0 where nothing is visible

``norm_rope`` restates the norm and the rotation of a head (pairs as complex numbers).  The reference has neither (its decoder
knows the causal mask and the half rotation alone): parity unpinned, the formulas are the definition.
"""
from __future__ import annotations

from typing import Optional

import torch


def score_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first_pos: int, scale: float, cap: float = 0.0,
                    slopes: Optional[torch.Tensor] = None, window: int = 0, first_keys: Optional[torch.Tensor] = None,
                    prefix: int = 0):
    """One sequence: ``q [n, Hq, D]`` at positions ``first_pos ..``, ``k`` / ``v [ctx, Hkv, D]``.  Returns ``out``, the weighted
    mean of ``|v|`` (what a relative error of the weights moves) and, per row and head, the largest
    ``scale * sum_d |q_d k_d|`` of a visible key (what a relative error of the products moves), all float64."""
    n, hq, d = q.shape
    ctx, hkv, _ = k.shape
    q, k, v = q.double(), k.double(), v.double()
    j = torch.arange(ctx)
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    mean_abs = torch.zeros_like(out)
    size = torch.zeros(n, hq, dtype=torch.float64)
    for i in range(n):
        p = first_pos + i
        seen = (j <= p) | (j < prefix)
        if window:
            seen &= p - j < window
        if first_keys is not None:
            seen &= j >= int(first_keys[i])
        if not bool(seen.any()):
            continue
        for h in range(hq):
            kk, vv = k[seen, h // (hq // hkv)], v[seen, h // (hq // hkv)]
            s = kk @ q[i, h] * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            if slopes is not None:
                s = s - float(slopes[h]) * (p - j[seen]).abs().double()
            w = torch.softmax(s, 0)
            out[i, h] = w @ vv
            mean_abs[i, h] = w @ vv.abs()
            size[i, h] = (kk.abs() @ q[i, h].abs()).max() * abs(scale)
    return out, mean_abs, size


def score_attention_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first_pos: int, scale: float, cap: float = 0.0,
                         slopes: Optional[torch.Tensor] = None, window: int = 0, first_keys: Optional[torch.Tensor] = None,
                         prefix: int = 0):
    """``score_attention`` of all rows of a head at once, for thousands of rows: the same values but for the order of sums."""
    n, hq, d = q.shape
    ctx, hkv, _ = k.shape
    q, k, v = q.double(), k.double(), v.double()
    j, p = torch.arange(ctx), torch.arange(first_pos, first_pos + n)[:, None]
    seen = (j <= p) | (j < prefix)
    if window:
        seen &= p - j < window
    if first_keys is not None:
        seen &= j >= first_keys[:, None]
    some = seen.any(1)
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    mean_abs = torch.zeros_like(out)
    size = torch.zeros(n, hq, dtype=torch.float64)
    for h in range(hq):
        kk, vv = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = q[:, h] @ kk.T * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - float(slopes[h]) * (p - j).abs().double()
        w = torch.softmax(torch.where(seen, s, -torch.inf)[some], -1)
        out[some, h] = w @ vv
        mean_abs[some, h] = w @ vv.abs()
        size[some, h] = torch.where(seen, q[:, h].abs() @ kk.abs().T, 0.0).amax(1)[some] * abs(scale)
    return out, mean_abs, size


def norm_rope(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float, angles: Optional[torch.Tensor], interleaved: bool):
    """``x [T, H, D]``, ``angles [T, R/2]`` (or None) -> float64."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if angles is None:
        return x
    T, H, _ = x.shape
    half = angles.shape[1]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    pairs = head.reshape(T, H, half, 2) if interleaved else torch.stack((head[..., :half], head[..., half:]), -1)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angles, dtype=torch.float64),
                                                                                        angles.double())[:, None])
    head = turned.reshape(T, H, 2 * half) if interleaved else torch.cat((turned[..., 0], turned[..., 1]), -1)
    return torch.cat((head, rest), -1)

"""Attention over part of a sequence's keys in 64 bits (oracle; test infrastructure only).

No counterpart in the reference; the definition, token by token: query i sees
the keys of row i of ``seen`` and its output is the softmax-weighted mean of
their values, 0 when it sees none.
"""

from __future__ import annotations

import torch


def window_seen(ctx: int, n: int, window: int, sinks: int) -> torch.Tensor:
    """(n, ctx + n) truth values of queries at positions ctx .. ctx + n - 1."""
    seen = torch.zeros(n, ctx + n, dtype=torch.bool)
    for i in range(n):
        p = ctx + i
        seen[i, max(0, p - window + 1):p + 1] = True
        seen[i, :min(sinks, p + 1)] = True
    return seen


def tree_seen(ctx: int, draft: torch.Tensor) -> torch.Tensor:
    """(n, ctx + n): the whole context and the drafted tokens of ``draft`` (n, n)."""
    return torch.cat([torch.ones(draft.shape[0], ctx, dtype=torch.bool), draft], dim=1)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor, scale: float):
    """q (n, Hq, D), k/v (K, Hkv, D), seen (n, K): outputs (n, Hq, D), sum_k w_k |v_k| and the largest
    sum_e |q_e k_e| * scale of a seen pair (what error bounds need), in float64."""
    n, hq, D = q.shape
    g = hq // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    seen = seen.to(q.device)
    out, wabs = torch.zeros(n, hq, D, dtype=torch.float64, device=q.device), torch.zeros(n, hq, D, dtype=torch.float64,
                                                                                         device=q.device)
    most = 0.0
    for i in range(n):
        at = seen[i].nonzero().squeeze(1)
        if not len(at):
            continue
        for h in range(hq):
            kk, vv = k[at, h // g], v[at, h // g]
            w = torch.softmax(kk @ q[i, h] * scale, 0)
            out[i, h] = w @ vv
            wabs[i, h] = w @ vv.abs()
        if i in (0, n - 1):
            most = max(most, float((k[at].abs().repeat_interleave(g, 1) * q[i].abs()).sum(-1).max()) * abs(scale))
    return out, wabs, most


def tolerance(out, wabs, most: float, keys: int, head_dim: int, dtype: torch.dtype) -> torch.Tensor:
    """Elementwise bound of a kernel that keeps scores, sums and outputs in float32, rounds the weights of 16-bit
    pools to the pool type for the value product, and rounds the output once.

    * a score sums head_dim products in float32: off by at most (head_dim + 4) 2^-24 times the sum of their
      absolute values (scale and base-2 factor included), at most ``2 * most`` (a pair other than the measured ones
      may be larger); the weights are off by twice that (numerator and denominator), so the output by that times
      sum w |v|;
    * exp2 and the divisions: within 2^-20 of sum w |v|; float32 sums over ``keys`` terms: keys * 2^-24 of it;
    * 16-bit weights: half a step each, eps / 2 of sum w |v| (below float16's normal range 2^-25 a key instead);
    * the output's own rounding: eps / 2 of |out|, and half of the type's smallest step.
    """
    eps = torch.finfo(dtype).eps
    rel = 2 * 2 * most * (head_dim + 4) * 2.0 ** -24 * 1.4427 + 2.0 ** -20 + 2 * keys * 2.0 ** -24
    tol = rel * wabs + eps / 2 * out.abs() + torch.finfo(dtype).tiny
    if dtype != torch.float32:
        tol = tol + eps / 2 * wabs * (1 + rel)
        if dtype == torch.float16:
            tol = tol + keys * 2.0 ** -25 * wabs.amax(-1, keepdim=True)
    return tol

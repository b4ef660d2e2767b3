"""Plain restatements of the 4-bit KV cache's operators for the tests: the
number format from its definition (fp32 operations, as the format says), the
attention in 64 bits, and the eviction row by row."""

import numpy as np
import torch

GROUP = 32


def quantise(x):
    """(codes uint8 [..., D], scales bf16 [..., D/32, 2]) of bf16 x, by the format's definition."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)  # NaN where the group holds one
    r = hi - lo
    s = torch.where(r < 2.0**-100, torch.zeros_like(r), r * np.float32(16.0 / 15.0)).bfloat16().float()
    z = (lo - s).bfloat16().float()
    bad = ~(torch.isfinite(s) & torch.isfinite(z))
    s, z = s.masked_fill(bad, float("nan")), z.masked_fill(bad, 0.0)
    live = (s > 0)[..., None]
    inv = torch.where(s > 0, 16.0 / s, torch.zeros_like(s))[..., None]
    t = torch.where(live, (g - z[..., None]) * inv - 16.0, torch.zeros_like(g))
    codes = t.round().clamp(0, 15).to(torch.uint8)
    return codes.flatten(-2), torch.stack([s, z], -1).bfloat16()


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def values(packed, scales):
    """The bf16 values (as float64) that packed codes and scales stand for."""
    n = unpack(packed).double().unflatten(-1, (-1, GROUP))
    s, z = scales[..., 0].double()[..., None], scales[..., 1].double()[..., None]
    return (s * (1 + n / 16) + z).bfloat16().double().flatten(-2)


def limits(offset, s, prefix, cache_len):
    """Visible rows of each query: int64 [B, S] from offsets [B]."""
    off = torch.as_tensor(offset).long().cpu()[:, None]
    lim = torch.maximum(off + 1 + torch.arange(s), torch.full_like(off, prefix))
    return torch.minimum(lim, off + s).clamp(0, cache_len)


def attention(q, k, v, lim, scale, gate=None):
    """64-bit attention and what bounds its fp32 error.

    q [B, H, S, D], k, v [B, Hk, L, D] float64, lim [B, S].  Returns (out [B, S, H, D],
    weights [B, Hk, L], spread [B, S, H, D] = sum p |v| (gated), score [B, H, S] =
    the largest sum |q k| scale of a row).  Rows that a query does not see take no part.
    """
    B, H, S, D = q.shape
    Hk, L = k.shape[1], k.shape[2]
    out = torch.zeros((B, S, H, D), dtype=torch.float64, device=q.device)
    spread, score = torch.zeros_like(out), torch.zeros((B, H, S), dtype=torch.float64, device=q.device)
    w = torch.zeros((B, Hk, L), dtype=torch.float64, device=q.device)
    for b in range(B):
        for h in range(H):
            kv = h * Hk // H
            for s in range(S):
                n = int(lim[b, s])
                if n == 0:
                    continue
                x = k[b, kv, :n] @ q[b, h, s].double() * scale
                p = torch.softmax(x, 0)
                out[b, s, h] = p @ v[b, kv, :n]
                spread[b, s, h] = p @ v[b, kv, :n].abs()
                score[b, h, s] = (k[b, kv, :n].abs() @ q[b, h, s].double().abs()).max() * abs(scale)
                w[b, kv, :n] += p
    if gate is not None:
        sig = torch.sigmoid(gate.double())
        out, spread = out * sig, spread * sig
    return out, w, spread, score


def evict(weights, positions, n, budget, protect):
    """Sources of the kept places [min(n, budget)] of one head (numpy, row by row)."""
    n = max(0, min(n, len(weights)))
    if n <= budget:
        return list(range(n))
    key = []
    for j in range(n):
        w = float(weights[j])
        key.append(float("inf") if positions[j] >= protect else w)
    # NaN ranks below -inf; of equal keys the lower row wins
    order = sorted(range(n), key=lambda j: (np.isnan(key[j]), -key[j] if not np.isnan(key[j]) else 0.0, j))
    kept = set(order[:budget])
    movers = iter(j for j in range(budget, n) if j in kept)
    return [j if j in kept else next(movers) for j in range(budget)]

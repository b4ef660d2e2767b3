"""GPU: the attention over values of 0 and 1, so that each output element is the
probability mass of its own share of the cache rows: a row, a tile or a part that is
lost, counted twice or scaled wrongly shows in its element, whatever the others hold.

Element e is 1 in the rows [n e / D, n (e + 1) / D) and 0 elsewhere; both are exact in
the 4-bit format (S = 1.0664, Z = -S: codes 0 and 15).  An output is a sum of
non-negative terms, so every bound is relative to the element itself (u = 2^-8):
the output's rounding u; a probability's 2^-16 up to 32 query rows of a kv head and u
above; its own 2 e + (n + 64) 2^-23 + 2^-20 with e = (D + 8) 2^-23 sum|q k| scale, as in
tests/test_kv4_gpu.py.  What is below 2^-126 may be 0.

And NaN values in tokens that some of many queries see, with two query tiles per CTA
and caches that are split over CTAs.
"""

import pytest
import torch

import hrm_layer_ops as ops
import kv4_reference as ref
from test_kv4_gpu import U, filled, rand, same

pytestmark = pytest.mark.gpu


def mass_cache(b, h, n, d, seed, drift):
    """Keys with a common direction that grows along the rows; v as above."""
    c = ops.kv4_cache(b, h, n, d, track=True)
    k = rand((b, h, n, d), seed).float()
    k += drift * (torch.arange(n, device="cuda") / n)[:, None] * torch.ones(d, device="cuda")
    v = (torch.arange(n, device="cuda")[:, None] * d // n == torch.arange(d, device="cuda")).float().expand(b, h, n, d)
    for t, x in (("k", k), ("v", v)):
        codes, scales = ref.quantise(x.bfloat16())
        getattr(c, t + "_codes").copy_(ref.pack(codes))
        getattr(c, t + "_scales").copy_(scales)
    stored = ref.values(c.v_codes, c.v_scales)
    assert torch.equal(stored, v.double())
    return c, stored


@pytest.mark.parametrize("b,hk,group,s,n,d", [
    (1, 2, 1, 1, 3000, 128), (2, 1, 4, 1, 9000, 64), (1, 1, 1, 12, 13000, 128), (2, 2, 1, 30, 1500, 256),
    (1, 2, 1, 40, 2048, 128), (1, 1, 2, 50, 6000, 64), (40, 2, 1, 100, 700, 128), (1, 1, 1, 128, 1000, 192),
    (1, 2, 1, 300, 2048, 128), (1, 1, 1, 300, 9000, 64), (40, 4, 1, 150, 600, 64), (1, 1, 3, 170, 3001, 128),
    (1, 1, 1, 300, 2500, 256), (2, 1, 1, 520, 1999, 128)])
@pytest.mark.parametrize("drift", [0.0, 4.0, 16.0])
def test_every_share_of_the_rows_has_its_mass(cuda, b, hk, group, s, n, d, drift):
    c, v = mass_cache(b, hk, n, d, 3 * n + d, drift)
    q = rand((b, hk * group, s, d), 7).float()
    # of every three queries one meets its largest scores last, one first
    q += 0.2 * torch.tensor([1.0, -1.0, 0.0], device="cuda").repeat(s)[:s, None]
    q = q.bfloat16()
    off = n - s
    w0 = c.weights.double()
    got = ops.kv4_attention(q, c, off, accumulate=True).double()
    k = ref.values(c.k_codes, c.k_scales).repeat_interleave(group, 1)
    x = torch.einsum("bhsd,bhld->bhsl", q.double(), k) * d**-0.5
    seen = torch.arange(n, device="cuda") <= off + torch.arange(s, device="cuda")[:, None]
    p = torch.softmax(x.masked_fill(~seen, -float("inf")), -1)
    want = torch.einsum("bhsl,bhld->bshd", p, v.repeat_interleave(group, 1))
    if drift > 10:  # the running maximum grows by far more than the kernels' slack, tile after tile
        grow = x[..., n * 3 // 4:].max() - x[..., : n // 4].max()
        assert float(grow) > 20.0
    score = float(torch.einsum("bhsd,bhld->bhsl", q.double().abs(), k.abs()).amax()) * d**-0.5
    rel = 2 * (d + 8) * 2.0**-23 * score + (n + 64) * 2.0**-23 + 2.0**-20
    bits = 2.0**-16 if group * s <= 32 else U
    err = (got - want).abs()
    tol = (U + bits + rel) * want + 2.0**-126
    assert bool((err <= tol).all()), (float((err - tol).max()), float((err / want.clamp(min=1e-30)).max()))
    w = p.unflatten(1, (hk, group)).sum((2, 3))
    err, tol = (c.weights.double() - w0 - w).abs(), rel * w + (group * s + 2) * 2.0**-23 * (w0 + w) + 2.0**-126 * s
    assert bool((err <= tol).all()), float((err - tol).max())
    assert ops.wait_timeouts() == 0


@pytest.mark.parametrize("b,hk,group,s,off,d", [(1, 1, 1, 300, 5000, 128), (1, 2, 1, 300, 70, 64), (1, 1, 2, 150, 3000, 64),
                                                (30, 5, 1, 140, 33, 128), (1, 1, 1, 300, 4000, 256),
                                                (1, 1, 1, 300, 5000, 192), (2, 1, 1, 600, 1000, 128)])
@pytest.mark.parametrize("place", ["last", "middle", "first"])
def test_nan_values_among_many_queries(cuda, b, hk, group, s, off, d, place):
    """A token whose v is NaN in a group: queries before it as without, later ones NaN there only."""
    c = filled(b, hk, off + s + 9, d, 19)
    q = rand((b, hk * group, s, d), 20)
    w0 = c.weights.clone()
    clean = ops.kv4_attention(q, c, off, accumulate=True)
    w1 = c.weights.clone()
    c.weights.copy_(w0)
    t = {"last": s - 1, "middle": s // 2, "first": 0}[place]
    c.v_scales[:, :, off + t, 1, 0] = float("nan")
    c.v_scales[:, :, off + s:] = float("nan")  # rows behind the sequence
    got = ops.kv4_attention(q, c, off, accumulate=True)
    same(got[:, :t], clean[:, :t], "earlier queries")
    nan = torch.isnan(got[:, t:])
    want = torch.zeros_like(nan)
    want[..., 32:64] = True
    assert torch.equal(nan, want)
    same(got[:, t:][~want], clean[:, t:][~want], "other groups")
    same(c.weights, w1, "weights")


@pytest.mark.parametrize("s", [1, 3, 40, 300])
def test_gate_over_its_whole_range(cuda, s):
    """Every bf16 gate in (-87, 100): values of 1 make the output sigmoid(gate), whose factor
    is within 2^-16 of itself."""
    bits = torch.arange(0x0000, 0x42c9, 1, dtype=torch.int32)
    g = torch.cat([bits.to(torch.int16).view(torch.bfloat16), -bits[bits < 0x42ae].to(torch.int16).view(torch.bfloat16)])
    d, h = 128, -(-g.numel() // (128 * s))
    gate = torch.zeros(h * s * d).bfloat16()
    gate[: g.numel()] = g
    gate = gate.view(1, s, h, d).cuda()
    c = ops.kv4_cache(1, h, 50 + s, d)
    codes, scales = ref.quantise(rand((1, h, 50 + s, d), 1))
    c.k_codes.copy_(ref.pack(codes))
    c.k_scales.copy_(scales)
    c.v_scales[..., 1] = 1.0  # S = 0, Z = 1
    got = ops.kv4_attention(rand((1, h, s, d), 2), c, 50, gate=gate).double()
    want = torch.sigmoid(gate.double())
    bits = 2.0**-16 if s <= 32 else U  # the probabilities', whose sum is 1 unrounded
    assert bool(((got - want).abs() <= (U + bits + 2.0**-16 + 2.0**-18) * want).all())

"""GPU: groups of the 4-bit cache whose largest value S * 31/16 + Z overflows bf16.

S = bf16_rn(range * 16/15) may be rounded up, so that a group that ends near bf16's
largest number would read back as an infinity.  The writes mark such a group as NaN,
as one whose S or Z overflows; and a row that holds one (the caller may have filled
the cache) has no influence on queries that do not see it.
"""

import pytest
import torch

import hrm_layer_ops as ops
import kv4_reference as ref
from test_kv4_gpu import filled, rand, same

pytestmark = pytest.mark.gpu

MOST = torch.finfo(torch.bfloat16).max


def near_the_top():
    """Rows of 64, two groups each: hi = bf16's largest number, the next lower one and one
    16 below, over every bf16 lo from 2^97 up to 2^127, some negative ones and 0."""
    bits = torch.arange(0x7000, 0x7f00, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    lows = torch.cat([bits, -bits[bits < 1e37], torch.zeros(1)])
    rows = []
    for hi in (0x7f7f, 0x7f7e, 0x7f70):
        hi = torch.tensor([hi], dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
        x = lows[:, None] + (hi - lows)[:, None] * torch.linspace(0, 1, 32)
        x[:, 0], x[:, -1] = lows, hi
        rows.append(x.bfloat16())
    x = torch.cat(rows)
    return x[: len(x) // 2 * 2].reshape(1, 1, -1, 64).cuda()


def expected(x):
    """Packed codes and scales by the format's definition.  The codes are worked out here:
    ref.quantise has 16.0 / S, which torch takes as 16 times the reciprocal of S, and that is
    a denormal number of fewer bits where S > 2^126."""
    _, scales = ref.quantise(x)
    s, z = scales[..., 0].double(), scales[..., 1].double()
    over = ~(torch.isfinite((s * 31 / 16 + z).bfloat16()) & torch.isfinite((s + z).bfloat16()))
    s, z = scales[..., 0].float()[..., None], scales[..., 1].float()[..., None]
    t = (x.float().unflatten(-1, (-1, 32)) - z) * torch.div(torch.full_like(s, 16.0), s) - 16.0
    codes = t.round().clamp(0, 15).masked_fill((over | torch.isnan(s[..., 0]) | (s[..., 0] == 0))[..., None], 0)
    codes = codes.to(torch.uint8).flatten(-2)
    scales = torch.where(over[..., None], torch.tensor([float("nan"), 0.0], device=x.device), scales.float())
    return ref.pack(codes), scales.bfloat16(), over


def check(c, x):
    codes, scales, over = expected(x)
    same(c.k_codes, codes, "codes")
    assert torch.equal(torch.isnan(c.k_scales), torch.isnan(scales))
    same(c.k_scales.nan_to_num(7.0), scales.nan_to_num(7.0), "scales")
    # no infinity is left: a group is finite, or NaN as a whole
    v = ref.values(c.k_codes, c.k_scales).unflatten(-1, (-1, 32))
    nan = torch.isnan(v)
    assert not bool(torch.isinf(v).any()) and torch.equal(nan.all(-1), nan.any(-1))
    assert torch.equal(nan.any(-1), over | torch.isnan(scales[..., 0].double()))


def test_a_group_that_would_read_back_as_an_infinity_is_nan(cuda):
    x = near_the_top()
    codes, scales = ref.quantise(x)
    inf = torch.isinf(ref.values(ref.pack(codes), scales)).any(-1)
    assert bool(inf.any())  # there are such groups (by the restatement alone: 25 elements)
    c = ops.kv4_cache(1, 1, x.shape[2], 64)
    ops.kv4_update(c, x, x)
    check(c, x)
    same(c.v_codes, c.k_codes)
    # the prologue, at position 0 (the rotation is by 0): gate, q, k, v of one token per row
    n = x.shape[2]
    c = ops.kv4_cache(1, 1, n, 64)
    gqkv = x.view(1, n, 1, 64).expand(1, n, 4, 64).reshape(n, 1, 256)
    each = ops.kv4_cache(n, 1, 1, 64)
    _, _, k, v = ops.split_gqkv_rope_kv4(gqkv, 1, each, 0)
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        getattr(c, name).copy_(getattr(each, name).view_as(getattr(c, name)))
    check(c, x)
    assert not bool(torch.isinf(k).any()) and not bool(torch.isinf(v).any())


@pytest.mark.parametrize("s", [2, 4, 12, 40, 80, 300])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("s_z", [(3.2965e38, -2.9908e38), (-3.0e38, -1.5e38), (float("inf"), 0.0)])
def test_such_rows_have_no_influence_where_they_are_not_seen(cuda, s, d, s_z):
    off = 37
    c = filled(1, 2, off + s + 3, d, 170)
    q = rand((1, 2, s, d), 171)
    clean = ops.kv4_attention(q, c, off)
    at = off + s - 1  # the last query's own row
    c.v_codes[:, :, at] = 0xff
    c.v_scales[:, :, at, 1] = torch.tensor(s_z).bfloat16().cuda()
    c.k_codes[:, :, at] = 0xff
    c.k_scales[:, :, at, 0] = torch.tensor(s_z).bfloat16().cuda()
    assert not bool(torch.isfinite(ref.values(c.v_codes, c.v_scales)[:, :, at, 32:64]).any())
    got = ops.kv4_attention(q, c, off)
    same(got[:, :-1], clean[:, :-1], "earlier queries")
    assert not bool(torch.isfinite(got[:, -1, :, 32:64]).any())

"""GPU: the 4-bit KV cache's write, attention and eviction against plain
restatements (tests/kv4_reference.py).

Tolerances, fixed before the first run (u = 2^-8 is bf16's rounding, half a step):
* codes, scales, moved rows, lengths, positions: equal bit for bit (the format's
  fp32 operations are IEEE, the eviction moves bytes).
* a stored value against the original x, in 64 bits: half a step S/32; plus the
  grid's shift by the roundings of S and Z, u * (hi - lo) + u * |lo - S|; plus the
  value's own rounding u * |value|; plus 2^-20 of the range for fp32.
* attention: one rounding u |out|; products of bf16 are exact in fp32, and sums on
  the tensor cores lose at most 2^-23 per addition, so a score is off by
  e = (D + 8) 2^-23 sum|q k| scale and a probability by 2 e + (L + 64) 2^-23 + 2^-20
  (exp2, the sum, the quotient) of itself; a probability enters the product with 16
  bits (2^-16) up to 32 rows per kv head and with 8 (u) above.  All of it times
  sum p |v|.  The gate adds 2^-18.
* weights: the same relative error of each probability, plus fp32 additions.
"""

import ctypes

import numpy as np
import pytest
import torch

import hrm_layer_ops as ops
import kv4_reference as ref
from hrm_layer_ops._lib import HrmError

pytestmark = pytest.mark.gpu

U = 2.0**-8
P = ctypes.c_void_p


def rand(shape, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).bfloat16().cuda()


def filled(b, h, n, d, seed, track=True, spread=True):
    """A tracked cache of random keys and values, packed by the restatement."""
    c = ops.kv4_cache(b, h, n, d, track=track)
    for i, t in enumerate("kv"):
        x = rand((b, h, n, d), seed + i).float()
        if spread:
            x[..., :: d // 4] *= 5.0
        codes, scales = ref.quantise(x.bfloat16())
        getattr(c, t + "_codes").copy_(ref.pack(codes))
        getattr(c, t + "_scales").copy_(scales)
    if track:
        c.weights.copy_(torch.rand((b, h, n), generator=torch.Generator().manual_seed(seed + 2)).cuda() * 3)
        c.positions.copy_(torch.arange(n, dtype=torch.int32, device="cuda").expand(b, h, n))
    return c


def buffers(c):
    return {n: getattr(c, n) for n in ("k_codes", "k_scales", "v_codes", "v_scales", "weights", "positions")
            if getattr(c, n) is not None}


def snapshot(c):
    return {n: t.clone() for n, t in buffers(c).items()}


def same(a, b, what=""):
    if a.dtype.is_floating_point:  # bits, so that NaN equals itself
        i = {2: torch.int16, 4: torch.int32}[a.element_size()]
        a, b = a.contiguous().view(i), b.contiguous().view(i)
    assert torch.equal(a, b), f"{what}: {(a != b).sum().item()} of {a.numel()} differ"


# ------------------------------------------------------------------------ write
def check_values(x, packed, scales):
    got = ref.values(packed, scales)
    g = x.double().unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = scales[..., 0].double()[..., None]
    v = got.unflatten(-1, (-1, 32))
    tol = s / 32 + U * (hi - lo) + U * (lo - s).abs() + U * v.abs() + (hi - lo) * 2.0**-20
    err = (v - g).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("b,h,s,d,n,off", [(1, 1, 1, 64, 1, 0), (2, 3, 5, 128, 9, 4), (3, 2, 17, 192, 40, 0),
                                           (1, 4, 33, 256, 64, 31), (5, 1, 1, 128, 7, 6)])
def test_update_matches_the_format(cuda, b, h, s, d, n, off):
    c = filled(b, h, n, d, 1)
    before = snapshot(c)
    k, v = rand((b, h, s, d), 2), rand((b, h, s, d), 3, 0.01)
    k[..., 3] *= 30
    ops.kv4_update(c, k, v, position_offset=1000, cache_offset=off)
    for t, x in (("k", k), ("v", v)):
        codes, scales = ref.quantise(x)
        want = before[t + "_codes"].clone(); want[:, :, off:off + s] = ref.pack(codes)
        same(getattr(c, t + "_codes"), want, t + " codes")
        want = before[t + "_scales"].clone(); want[:, :, off:off + s] = scales
        same(getattr(c, t + "_scales"), want, t + " scales")
        check_values(x, ref.pack(codes), scales)
    want = before["weights"].clone(); want[:, :, off:off + s] = 0
    same(c.weights, want, "weights")
    want = before["positions"].clone()
    want[:, :, off:off + s] = torch.arange(1000, 1000 + s, dtype=torch.int32, device="cuda")
    same(c.positions, want, "positions")


def special_groups():
    """Rows of 64: constants, signed zeros, one outlier, denormals, a huge offset, tiny and huge ranges."""
    z = torch.zeros(64)
    rows = [z.clone(), z - 1.5, torch.where(torch.arange(64) % 2 == 0, 0.0, -0.0), z.clone(), z + 100.0, z.clone(),
            z.clone(), z.clone(), torch.linspace(-1, 1, 64), z.clone()]
    rows[3][5] = 1e30
    rows[4][7] = 100.5
    rows[5] += torch.arange(64) * 2.0**-133           # denormal steps: a range under 2^-100
    rows[6] += torch.arange(64) * 2.0**-99            # just above it
    rows[7][::2], rows[7][1::2] = 3e38, -3e38         # the range overflows binary32: NaN
    rows[9][0] = -3.38e38                             # Z overflows bf16: NaN
    return torch.stack(rows).bfloat16().cuda().view(1, 1, -1, 64)


def test_update_special_values(cuda):
    x = special_groups()
    c = ops.kv4_cache(1, 1, x.shape[2], 64)
    ops.kv4_update(c, x, x)
    codes, scales = ref.quantise(x)
    same(c.k_codes, ref.pack(codes), "codes")
    got, want = c.k_scales.float(), scales.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    assert bool(torch.isnan(ref.values(c.k_codes, c.k_scales)[0, 0, 7]).all())
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = rand((1, 1, 4, 128), 5)
        y[0, 0, 2, 40] = bad
        c = ops.kv4_cache(1, 1, 4, 128)
        ops.kv4_update(c, y, y)
        nan = torch.isnan(ref.values(c.v_codes, c.v_scales))[0, 0]
        want = torch.zeros_like(nan); want[2, 32:64] = True
        assert torch.equal(nan, want)


def test_update_per_sequence_places(cuda):
    """Device offsets: each sequence at its own row; rows outside the cache are dropped."""
    c = filled(4, 2, 10, 128, 7)
    before = snapshot(c)
    k = rand((4, 2, 3, 128), 8)
    off = torch.tensor([0, 7, 9, -2], dtype=torch.int32, device="cuda")
    pos = torch.tensor([50, 0, 3, 2**31 - 10], dtype=torch.int32, device="cuda")
    ops.kv4_update(c, k, k, pos, off)
    codes, scales = ref.quantise(k)
    want, want_pos = before["k_codes"].clone(), before["positions"].clone()
    for b in range(4):
        for s in range(3):
            r = int(off[b]) + s
            if 0 <= r < 10:
                want[b, :, r] = ref.pack(codes)[b, :, s]
                want_pos[b, :, r] = int(pos[b]) + s
    same(c.k_codes, want)
    same(c.positions, want_pos)


@pytest.mark.parametrize("b,s,h,d,table", [(1, 1, 1, 64, True), (3, 7, 4, 128, True), (2, 33, 12, 128, False),
                                           (2, 5, 3, 192, True), (1, 40, 5, 256, True), (700, 1, 2, 128, True),
                                           (2, 400, 16, 64, True)])
@pytest.mark.parametrize("keep", [True, False])
def test_split_rope_kv4_matches_the_bf16_prologue(cuda, b, s, h, d, table, keep):
    """gate and q: the bits of split_gqkv_rope; the cache: its rotated k and v quantised."""
    n, off, pos = s + 6, 3, 11
    gqkv = rand((b, s, 4 * h * d), 21)
    tab = ops.rope_table(pos + s, d, 10000.0) if table else None
    c = filled(b, h, n, d, 22)
    before = snapshot(c)
    gate, q, k, v = ops.split_gqkv_rope_kv4(gqkv, h, c, pos, 10000.0, tab, cache_offset=off, keep_kv=keep)
    g0, q0, k0, v0 = ops.split_gqkv_rope(gqkv, h, pos, 10000.0, tab)
    same(gate, g0, "gate"); same(q, q0, "q")
    for t, x, stored in (("k", k0, k), ("v", v0, v)):
        codes, scales = ref.quantise(x)
        want = before[t + "_codes"].clone(); want[:, :, off:off + s] = ref.pack(codes)
        same(getattr(c, t + "_codes"), want, t + " codes")
        want = before[t + "_scales"].clone(); want[:, :, off:off + s] = scales
        same(getattr(c, t + "_scales"), want, t + " scales")
        if keep:
            same(stored, ref.values(ref.pack(codes), scales).bfloat16(), t + " values")
        else:
            assert stored is None
    assert bool((c.weights[:, :, off:off + s] == 0).all())
    assert torch.equal(c.positions[0, 0, off:off + s].cpu(), torch.arange(pos, pos + s, dtype=torch.int32))


def test_split_rope_kv4_device_offsets_and_table_end(cuda):
    """Per-sequence positions; those past the table (or before 0) take the in-kernel angles, same bits."""
    b, s, h, d = 4, 2, 3, 128
    gqkv = rand((b, s, 4 * h * d), 31)
    pos = torch.tensor([0, 5, 6, 40], dtype=torch.int32, device="cuda")
    off = torch.tensor([0, 1, 6, -5], dtype=torch.int32, device="cuda")
    c, w = ops.kv4_cache(b, h, 8, d, track=True), ops.kv4_cache(b, h, 8, d, track=True)
    gate, q, k, v = ops.split_gqkv_rope_kv4(gqkv, h, c, pos, 10000.0, ops.rope_table(7, d), cache_offset=off)
    for i in range(b):
        one = ops.kv4_cache(1, h, 8, d, track=True)
        fits = 0 <= int(off[i]) and int(off[i]) + s <= 8
        g1, q1, k1, v1 = ops.split_gqkv_rope_kv4(gqkv[i:i + 1].contiguous(), h, one, int(pos[i]),
                                                 cache_offset=int(off[i]) if fits else 0)
        for a, e in ((gate, g1), (q, q1), (k, k1), (v, v1)):
            same(a[i:i + 1], e)
        if fits:
            for name, t in buffers(one).items():
                buffers(w)[name][i] = t[0]
    for name, t in buffers(c).items():
        same(t, buffers(w)[name], name)


# -------------------------------------------------------------------- attention
def run_attention(c, q, off, gate=None, prefix=0, scale=None, accumulate=False):
    b, h, s, d = q.shape
    k, v = ref.values(c.k_codes, c.k_scales), ref.values(c.v_codes, c.v_scales)
    offs = off if isinstance(off, torch.Tensor) else torch.full((b,), off)
    lim = ref.limits(offs, s, prefix, c.shape[2])
    sc = d**-0.5 if scale is None else scale
    want, w, spread, score = ref.attention(q, k, v, lim, sc, gate)
    w0 = c.weights.double() if accumulate else None
    others = {n: t.clone() for n, t in buffers(c).items() if not (accumulate and n == "weights")}
    got = ops.kv4_attention(q, c, off, gate=gate, prefix_len=prefix, scale=scale, accumulate=accumulate)
    e = (d + 8) * 2.0**-23 * score.max() + 0.0
    rel = 2 * e + (c.shape[2] + 64) * 2.0**-23 + 2.0**-20 + 2.0**-18
    p_bits = 2.0**-16 if (h // c.shape[1]) * s <= 32 else U
    tol = U * want.abs() + (rel + p_bits) * spread + 1e-37
    err = (got.double() - want).abs()
    assert not bool(torch.isnan(got).any()) or bool(torch.isnan(want).any())
    assert bool((err <= tol).all()), (float((err - tol).max()), float((err / tol).max()))
    if accumulate:
        rows = (h // c.shape[1]) * s
        err, tol = (c.weights.double() - w0 - w).abs(), rel * w + (rows + 2) * 2.0**-23 * (w0 + w)
        assert bool((err <= tol).all()), float((err - tol).max())
    for n, t in others.items():
        same(buffers(c)[n], t, n)  # the cache is only read
    return got


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 127, 128, 129, 1000, 2049])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_attention_single_token_lengths(cuda, n, d):
    c = filled(2, 3, n, d, n + d)
    run_attention(c, rand((2, 3, 1, d), 5), n - 1, accumulate=True)


@pytest.mark.parametrize("b,hk,group,s,n,d,prefix", [
    (2, 2, 1, 3, 40, 64, 0), (1, 1, 8, 1, 300, 128, 0), (2, 2, 4, 2, 129, 128, 0), (1, 2, 3, 3, 77, 128, 0),
    (1, 1, 5, 6, 200, 192, 50), (1, 2, 1, 17, 150, 256, 0), (2, 1, 1, 32, 64, 128, 40), (1, 2, 1, 33, 33, 128, 0),
    (1, 1, 2, 40, 190, 64, 0), (2, 1, 1, 65, 200, 128, 130), (1, 1, 3, 50, 64, 192, 0), (1, 2, 1, 70, 71, 256, 5),
    (1, 1, 1, 128, 128, 128, 128), (1, 1, 1, 200, 500, 64, 20)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_attention_shapes(cuda, b, hk, group, s, n, d, prefix, accumulate):
    c = filled(b, hk, n + 5, d, 3 * n)
    q, gate = rand((b, hk * group, s, d), 7), rand((b, s, hk * group, d), 8)
    run_attention(c, q, n - s, gate=gate, prefix=prefix, accumulate=accumulate)


@pytest.mark.parametrize("s", [1, 5, 20, 70])
def test_attention_ragged_and_empty_sequences(cuda, s):
    """Per-sequence offsets: full, short, partly visible (negative) and idle sequences."""
    n, d = 300, 128
    c = filled(5, 2, n, d, 50)
    off = torch.tensor([n - s, 0, 37, -(s // 2), -s - 3], dtype=torch.int32, device="cuda")
    got = run_attention(c, rand((5, 2, s, d), 51), off, accumulate=True)
    assert bool((got[4] == 0).all())


def test_attention_offsets_past_the_cache_are_cut(cuda):
    c = filled(2, 1, 50, 64, 60)
    off = torch.tensor([48, 2**31 - 5], dtype=torch.int32, device="cuda")
    run_attention(c, rand((2, 1, 4, 64), 61), off)


@pytest.mark.parametrize("s", [1, 4, 12, 80])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_rows_that_are_not_seen_have_no_influence(cuda, s, d):
    """NaN rows behind the sequence, and NaN values in tokens later than the query."""
    n, off = 150, 40
    c = filled(1, 2, n, d, 70)
    q = rand((1, 2, s, d), 71)
    clean = ops.kv4_attention(q, c, off)
    for t in (c.k_scales, c.v_scales):
        t[:, :, off + s:] = float("nan")
    same(ops.kv4_attention(q, c, off), clean, "rows behind the sequence")
    if s == 1:
        return
    # the last token's v is NaN in its second group, its k in the first
    at = off + s - 1
    c.v_scales[:, :, at, 1, 0] = float("nan")
    got = ops.kv4_attention(q, c, off)
    same(got[:, :-1], clean[:, :-1], "earlier queries")
    nan = torch.isnan(got[0, -1])
    want = torch.zeros_like(nan); want[:, 32:64] = True
    assert torch.equal(nan, want)
    same(got[0, -1][~want], clean[0, -1][~want])
    c.k_scales[:, :, at, 0, 0] = float("nan")
    got = ops.kv4_attention(q, c, off)
    same(got[:, :-1], clean[:, :-1], "earlier queries")
    assert bool(torch.isnan(got[0, -1]).all())


def test_nan_and_infinite_queries_stay_in_their_row(cuda):
    c = filled(1, 1, 90, 128, 75)
    for s in (3, 70):
        q = rand((1, 1, s, 128), 76)
        clean = ops.kv4_attention(q, c, 10)
        q[0, 0, 1, 5] = float("nan")
        got = ops.kv4_attention(q, c, 10)
        assert bool(torch.isnan(got[0, 1]).all())
        same(got[0, [0, 2]], clean[0, [0, 2]])


@pytest.mark.parametrize("s", [1, 40])
def test_large_and_peaked_scores(cuda, s):
    """Scores in the hundreds (one row takes all the probability) and a negative scale."""
    c = filled(1, 2, 400, 128, 80)
    run_attention(c, rand((1, 2, s, 128), 81, 20.0), 400 - s)
    run_attention(c, rand((1, 2, s, 128), 82), 400 - s, scale=-0.3)
    run_attention(c, rand((1, 2, s, 128), 83), 400 - s, scale=0.0)


def test_attention_is_the_same_from_call_to_call(cuda):
    for s in (1, 3, 20, 100):
        c = filled(2, 3, 700, 128, 90)
        q = rand((2, 3, s, 128), 91)
        w0 = c.weights.clone()
        a = ops.kv4_attention(q, c, 600, accumulate=True)
        wa = c.weights.clone()
        for _ in range(5):
            c.weights.copy_(w0)
            same(ops.kv4_attention(q, c, 600, accumulate=True), a)
            same(c.weights, wa)


def test_attention_row_past_four_gigabytes(cuda):
    """Code offsets past 2^32 bytes: the last head of a large cache."""
    b, h, n, d = 3, 12, 1 << 20, 256
    c = ops.kv4_cache(b, h, n, d, track=True)
    assert c.k_codes.numel() > 1 << 32
    small = filled(1, 1, 64, d, 95)
    for name, t in buffers(c).items():
        t[-1, -1, -64:] = buffers(small)[name][0, 0]
        t[-1, -1, :-64] = 0
    k = rand((b, h, 1, d), 96)
    ops.kv4_update(c, k, k, cache_offset=torch.tensor([-1, -1, n - 1], dtype=torch.int32, device="cuda"))
    codes, scales = ref.quantise(k)
    same(c.k_codes[-1, -1, -1], ref.pack(codes)[-1, -1, 0])
    # the query's scores: 0 on the zero rows, so every row counts
    off = torch.tensor([-1, -1, n - 1], dtype=torch.int32, device="cuda")
    q = rand((b, h, 1, d), 97)
    got = ops.kv4_attention(q, c, off)
    kk, vv = ref.values(c.k_codes[-1, -1], c.k_scales[-1, -1]), ref.values(c.v_codes[-1, -1], c.v_scales[-1, -1])
    p = torch.softmax(kk @ q[-1, -1, 0].double() / 16, 0)
    want, spread = p @ vv, p @ vv.abs()
    # fp32 sums of 2^20 rows, in at least 16 partial sums: 2^-23 for each of 2^16 terms, in p and in its sum
    assert bool(((got[-1, 0, -1].double() - want).abs() <= U * want.abs() + spread * (2.0**-15 + 2.0**-6)).all())
    assert bool((got[:2] == 0).all())
    del c
    torch.cuda.empty_cache()


# --------------------------------------------------------------------- eviction
def check_evict(c, lengths, budget, protect, out=None, host=False):
    b, h, n, d = c.shape
    lens = [lengths] * b if isinstance(lengths, int) else lengths
    prot = [protect] * b if isinstance(protect, int) else protect
    before = snapshot(c)
    to_before = snapshot(out) if out is not None else before
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.kv4_evict(c, lengths if host else dev(lens), budget, protect if host else dev(prot), out=out)
    want = {k: v.clone() for k, v in to_before.items()}
    w, p = before["weights"].cpu().numpy(), before["positions"].cpu().numpy()
    for i in range(b):
        for j in range(h):
            src = ref.evict(w[i, j], p[i, j], lens[i], budget, prot[i])
            if src:
                for name in want:
                    want[name][i, j, :len(src)] = before[name][i, j, torch.tensor(src, device="cuda")]
    assert got.tolist() == [min(max(0, min(x, n)), budget) for x in lens]
    for name, t in buffers(out if out is not None else c).items():
        same(t, want[name], name)
    if out is not None:
        for name, t in buffers(c).items():
            same(t, before[name], "source " + name)


@pytest.mark.parametrize("n,budget", [(1, 1), (2, 1), (33, 32), (100, 7), (1025, 1024), (2048, 1000), (2049, 64),
                                      (5000, 4998), (8193, 5000), (33000, 4000), (40000, 39999)])
@pytest.mark.parametrize("place", ["in place", "out"])
def test_evict_sizes(cuda, n, budget, place):
    c = filled(1, 2, n, 64, n)
    out = filled(1, 2, budget + 3, 64, 5) if place == "out" else None
    check_evict(c, n, budget, n - max(1, budget // 4), out, host=True)


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("place", ["in place", "out"])
def test_evict_ragged_batches(cuda, d, place):
    n, budget = 600, 200
    c = filled(6, 3, n, d, 11)
    out = filled(6, 3, 250, d, 12) if place == "out" else None
    check_evict(c, [600, 201, 200, 0, 333, -4], budget, [550, 100, 0, 0, 10**6, 0], out)


def test_evict_ties_nan_infinities_and_zeros(cuda):
    n = 300
    c = filled(1, 6, n, 64, 13)
    c.weights[0, 0] = 1.0                                             # all equal
    c.weights[0, 1] = torch.arange(n, device="cuda").remainder(3).float()  # many ties at the border
    c.weights[0, 2, ::2] = float("nan")
    c.weights[0, 3, :50] = float("inf"); c.weights[0, 3, 60:200] = -float("inf")
    c.weights[0, 4] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 0.0, -0.0)
    c.weights[0, 5] = -torch.rand(n, generator=torch.Generator().manual_seed(1)).cuda()
    c.positions[0, :, 100:140] = 10**6                                # protected rows in the middle
    for budget in (1, 20, 39, 40, 41, 150, 299):
        x = ops.Kv4Cache(**{k: v.clone() for k, v in buffers(c).items()})
        check_evict(x, n, budget, 10**6)
        out = ops.kv4_cache(1, 6, budget, 64, track=True)
        check_evict(c, n, budget, 10**6, out)


def test_evict_all_rows_protected_or_none(cuda):
    c = filled(2, 2, 700, 128, 14)
    out = ops.kv4_cache(2, 2, 128, 128, track=True)
    check_evict(c, 700, 128, 0, out)
    check_evict(c, 700, 128, 10**7, out)
    check_evict(c, 100, 128, 0, out)


# ----------------------------------------------- long caches: shares of all items
@pytest.mark.parametrize("b,hk,group,s,n,d,ragged", [(1, 1, 1, 1, 4097, 64, False), (1, 3, 1, 1, 20000, 128, False),
                                                     (5, 2, 1, 1, 9000, 128, True), (70, 1, 1, 1, 4200, 64, True),
                                                     (3, 1, 4, 2, 6000, 256, True), (2, 1, 2, 9, 5000, 128, True),
                                                     (40, 16, 1, 1, 4500, 64, True), (2, 1, 1, 3, 4300, 192, False)])
def test_attention_long_caches(cuda, b, hk, group, s, n, d, ragged):
    """The rows of all items laid end to end and cut: against the 64-bit form, with weights."""
    c = filled(b, hk, n, d, 7 * n)
    q, gate = rand((b, hk * group, s, d), 1), rand((b, s, hk * group, d), 2)
    if ragged:  # full, empty and short sequences among them
        off = torch.tensor([(n - s) if i % 4 == 0 else (-s - 1 if i % 4 == 1 else (n - s) * i // (4 * b))
                            for i in range(b)], dtype=torch.int32, device="cuda")
    else:
        off = n - s
    if b * hk * group * s <= 40:
        run_attention(c, q, off, gate=gate, accumulate=True)
        return
    # many rows: vectorised over heads
    k, v = ref.values(c.k_codes, c.k_scales), ref.values(c.v_codes, c.v_scales)
    w0 = c.weights.double()
    got = ops.kv4_attention(q, c, off, gate=gate, accumulate=True)
    lim = ref.limits(off, s, 0, n).cuda()
    x = torch.einsum("bhsd,bhld->bhsl", q.double(), k) * d**-0.5
    seen = torch.arange(n, device="cuda") < lim[:, None, :, None]
    p = torch.softmax(x.masked_fill(~seen, -float("inf")), -1).nan_to_num(0.0)
    sig = torch.sigmoid(gate.double())
    want = torch.einsum("bhsl,bhld->bshd", p, v) * sig
    spread = torch.einsum("bhsl,bhld->bshd", p, v.abs()) * sig
    e = (d + 8) * 2.0**-23 * float((q.double().abs().amax() * k.abs().sum(-1).amax())) * d**-0.5
    rel = 2 * e + (n + 64) * 2.0**-23 + 2.0**-20 + 2.0**-18 + 2.0**-16
    assert bool(((got.double() - want).abs() <= U * want.abs() + rel * spread + 1e-37).all())
    err, w = (c.weights.double() - w0 - p.sum(2)).abs(), p.sum(2)
    assert bool((err <= rel * w + 2.0**-21 * (w0 + w)).all())


def test_long_caches_nan_rows_and_lse_order(cuda):
    """Not-seen NaN tokens at the end of a cut item; the same result from call to call."""
    n, d, s = 9000, 128, 4
    c = filled(1, 2, n, d, 33)
    q = rand((1, 2, s, d), 34)
    clean = ops.kv4_attention(q, c, n - s)
    c.v_scales[:, :, n - 1, 1, 0] = float("nan")
    for _ in range(3):
        got = ops.kv4_attention(q, c, n - s)
        same(got[:, :-1], clean[:, :-1])
        nan = torch.isnan(got[0, -1])
        want = torch.zeros_like(nan); want[:, 32:64] = True
        assert torch.equal(nan, want)


@pytest.mark.parametrize("n,budget", [(5000, 1111), (9000, 100), (20000, 19000), (70000, 30000), (140000, 700)])
def test_evict_equal_weights_over_several_ctas(cuda, n, budget):
    """All keys equal, and a few distinct values: thresholds that many rows share."""
    c = filled(1, 2, n, 64, 17)
    c.weights[0, 0] = 0.25
    c.weights[0, 1] = torch.arange(n, device="cuda").remainder(5).float() * 1e-3
    out = ops.kv4_cache(1, 2, budget, 64, track=True)
    check_evict(c, n, budget, n - 10, out, host=True)
    check_evict(c, n, budget, n - 10, host=True)

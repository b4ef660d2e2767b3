"""The 4-bit KV cache's operators, as cases to measure: the write (attention
prologue into the cache), the attention that reads it, and the eviction by
accumulated attention weight.

Each case runs either in plain form (elementary torch operations in fp32) or,
with `own` set, through the framework's calls.  `exact` restates each operator
in 64 bits, apart from the plain form.

The cache, per (batch, kv head, row):
  codes   [B, Hk, L, D/2]      uint8: byte i holds element 2i (low nibble) and 2i+1
  scales  [B, Hk, L, D/32, 2]  bf16: (scale, base) of each group of 32 elements
  value = bf16(scale * (1 + code / 16) + base)
  weights [B, Hk, L] fp32, positions [B, Hk, L] int32   (tracked caches)
"""

import math

import torch

own = False

GROUP = 32
THETA = 10000.0


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # One token for each of 64 streams, the smallest write: a decode step of a served batch.
        dict(name="write decode 64x1", op="write", batch=64, seq=1, heads=16, dim=128, cache=1024, ragged=True),
        # A prompt of odd length at the model's own width (12 heads of 128).
        dict(name="write prompt 1x1001", op="write", batch=1, seq=1001, heads=12, dim=128, cache=1536, ragged=False),
        # The prefill of 8 sequences of 4096 tokens, 16 heads: the framework's RoPE workload.
        dict(name="write prefill 8x4096", op="write", batch=8, seq=4096, heads=16, dim=128, cache=4096, ragged=False),
        # The decode step of one chat at the model's longest context (4096 rows, 12 heads).
        dict(name="decode 1x4096", op="attend", batch=1, seq=1, heads=12, kv=12, dim=128, rows=4096, ragged=False,
             gate=True, track=False, prefix=0),
        # One stream over a long document.
        dict(name="decode 1x65536", op="attend", batch=1, seq=1, heads=12, kv=12, dim=128, rows=65536, ragged=False,
             gate=False, track=False, prefix=0),
        # A served batch of mixed lengths, weights accumulated for the eviction.
        dict(name="decode 32x8191 tracked", op="attend", batch=32, seq=1, heads=16, kv=16, dim=128, rows=8191,
             ragged=True, gate=True, track=True, prefix=0),
        # Shared kv heads, narrow heads, three drafted tokens checked at once.
        dict(name="verify 16x2500 shared", op="attend", batch=16, seq=3, heads=16, kv=8, dim=64, rows=2500,
             ragged=True, gate=False, track=False, prefix=0),
        # A further turn of a chat: 512 new tokens over 8192 cached rows.
        dict(name="chunk 512 over 8192", op="attend", batch=1, seq=512, heads=16, kv=16, dim=128, rows=8704,
             ragged=False, gate=False, track=False, prefix=0),
        # A prompt of 4096 tokens per sequence with a bidirectional prefix, weights accumulated.
        dict(name="prompt 2x4096 tracked", op="attend", batch=2, seq=4096, heads=12, kv=12, dim=128, rows=4096,
             ragged=False, gate=True, track=True, prefix=1000),
        # The smallest eviction: each stream's new row replaces its lightest one, in place.
        dict(name="evict step 64x1024", op="evict", batch=64, heads=16, dim=128, rows=1025, budget=1024, recent=64,
             ragged=False, step=True),
        # A long prompt's cache cut to 4096 rows for decoding, into a cache of that size.
        dict(name="evict prompt 1x32768", op="evict", batch=1, heads=12, dim=128, rows=32768, budget=4096, recent=256,
             ragged=False, step=False),
        # A batch of prompts of mixed lengths, cut to an odd budget.
        dict(name="evict prompts 16x5000", op="evict", batch=16, heads=16, dim=64, rows=5000, budget=1111, recent=100,
             ragged=True, step=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "attend", "evict"])
    dim = rng.choice([64, 128, 128, 128, 256])
    if op == "write":
        heads = rng.choice([1, 4, 12, 16])
        seq = _log(rng, 1, 4096)
        batch = _log(rng, 1, max(1, min(64, 3_000_000 * 16 // (seq * heads * dim))))
        return dict(op=op, batch=batch, seq=seq, heads=heads, dim=dim, cache=seq + _log(rng, 1, 2000),
                    ragged=rng.random() < 0.5)
    if op == "evict":
        rows = _log(rng, 200, 32768)
        heads = rng.choice([1, 8, 12, 16])
        batch = _log(rng, 1, max(1, min(64, 2_500_000 * 128 // (rows * heads * dim))))
        budget = max(1, int(rows * rng.uniform(0.05, 0.95)))
        step = rng.random() < 0.3
        return dict(op=op, batch=batch, heads=heads, dim=dim, rows=budget + 1 if step else rows, budget=budget,
                    recent=int(budget * rng.uniform(0.0, 0.5)), ragged=not step and rng.random() < 0.5, step=step)
    kv = rng.choice([1, 2, 8, 12, 16])
    group = rng.choice([1, 1, 1, 2, 4])
    seq = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 2048)])
    rows = seq + _log(rng, 1, max(2, min(65536, 100_000_000 // (seq * kv * group))))
    batch = _log(rng, 1, max(1, min(32, 4_000_000 * 128 // (rows * kv * dim), 100_000_000 // (rows * seq * kv * group))))
    return dict(op=op, batch=batch, seq=seq, heads=kv * group, kv=kv, dim=dim, rows=rows, ragged=rng.random() < 0.5,
                gate=rng.random() < 0.5, track=rng.random() < 0.4, prefix=rng.choice([0, 0, rows // 3]))


def _lengths(case, lowest):
    """Rows of each sequence: all `rows`, or spread evenly from `lowest` up to `rows`."""
    n, b = case["rows"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [lowest + (n - lowest) * (i + 1) // b for i in range(b)]


def _offsets(case):
    """Cache rows before a write case's tokens, per sequence."""
    room = case["cache"] - case["seq"]
    if not case["ragged"]:
        return [room // 2] * case["batch"]
    return [room * (i + 1) // case["batch"] for i in range(case["batch"])]


# ------------------------------------------------------------------ the inputs
def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _make_cache(case, g, rows):
    """A cache of `rows` rows as a decode loop leaves it: quantised keys and values, a few outlying
    channels among them as rotated keys have."""
    b, h, d = case["batch"], case["kv"] if "kv" in case else case["heads"], case["dim"]
    out = {}
    for name in ("k", "v"):
        x = _normal(g, b, h, rows, d)
        if name == "k":
            x[..., :: max(1, d // 4)] *= 4.0
        codes, scales = _quantise(x.bfloat16())
        out[name + "_codes"], out[name + "_scales"] = _pack(codes), scales
    out["weights"] = torch.rand((b, h, rows), generator=g, device="cuda").pow(4) * 3
    out["positions"] = torch.arange(rows, device="cuda", dtype=torch.int32).expand(b, h, rows).contiguous()
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, d = case["batch"], case["dim"]
    if case["op"] == "write":
        s, h, n = case["seq"], case["heads"], case["cache"]
        st = dict(op="write", heads=h, gqkv=torch.empty((b, s, 4 * h * d), dtype=torch.bfloat16, device="cuda"))
        st["gqkv"].normal_(generator=g)
        new = dict(device="cuda")
        st["cache"] = dict(
            k_codes=torch.zeros((b, h, n, d // 2), dtype=torch.uint8, **new),
            k_scales=torch.zeros((b, h, n, d // GROUP, 2), dtype=torch.bfloat16, **new),
            v_codes=torch.zeros((b, h, n, d // 2), dtype=torch.uint8, **new),
            v_scales=torch.zeros((b, h, n, d // GROUP, 2), dtype=torch.bfloat16, **new),
            weights=torch.ones((b, h, n), **new), positions=torch.zeros((b, h, n), dtype=torch.int32, **new))
        st["offset"] = torch.tensor(_offsets(case), dtype=torch.int32, device="cuda")
        # the fp32 cos/sin table that a program builds once
        inv = torch.exp(torch.arange(d // 2, device="cuda", dtype=torch.float64) * (-2.0 * math.log(THETA) / d))
        a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
        st["table"] = torch.cat([a.cos(), a.sin()], dim=1).float()
        return st
    if case["op"] == "attend":
        s, h, lens = case["seq"], case["heads"], _lengths(case, case["seq"])
        st = dict(op="attend", prefix=case["prefix"], track=case["track"], cache=_make_cache(case, g, case["rows"]))
        st["q"] = _normal(g, b, h, s, d).bfloat16()
        st["gate"] = _normal(g, b, s, h, d).bfloat16() if case["gate"] else None
        st["offset"] = torch.tensor([n - s for n in lens], dtype=torch.int32, device="cuda")
        return st
    lens = _lengths(case, max(1, case["budget"] // 2))
    st = dict(op="evict", budget=case["budget"], step=case["step"], cache=_make_cache(case, g, case["rows"]))
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["protect"] = st["lengths"] - case["recent"]
    if case["step"]:  # the new token's key and value, written to row `budget` before the eviction
        st["k"] = _normal(g, b, case["heads"], 1, d).bfloat16()
        st["v"] = _normal(g, b, case["heads"], 1, d).bfloat16()
    else:  # the decoding cache
        st["out"] = {k: torch.zeros((b, case["heads"], case["budget"], *v.shape[3:]), dtype=v.dtype, device="cuda")
                     for k, v in st["cache"].items()}
    return st


# -------------------------------------------------------------- the plain form
def _quantise(x):
    """codes (uint8, 0..15) and (scale, base) of bf16 x [..., D] in groups of 32."""
    xg = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = xg.amin(-1), xg.amax(-1)
    r = hi - lo
    scale = torch.where(r < 2.0 ** -100, torch.zeros_like(r), r * (16.0 / 15.0)).bfloat16().float()
    base = (lo - scale).bfloat16().float()
    inv = torch.where(scale > 0, 16.0 / scale, torch.zeros_like(scale))
    t = (xg - base[..., None]) * inv[..., None] - 16.0
    codes = torch.where(scale[..., None] > 0, t.round().clamp(0, 15), torch.zeros_like(t)).to(torch.uint8)
    return codes.flatten(-2), torch.stack([scale, base], -1).bfloat16()


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(codes, scales):
    """fp32 values that codes (one per element) and scales stand for."""
    s = scales.float().repeat_interleave(GROUP, dim=-2)
    m = 1.0 + codes.float() * 0.0625
    return (s[..., 0] * m + s[..., 1]).bfloat16().float()


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def _plain_store(c, offset, k, v):
    """Writes k, v [B, H, S, D] bf16 at rows offset[b] + s; returns the values stored."""
    b, h, s, d = k.shape
    rows = (offset.long()[:, None, None] + torch.arange(s, device=k.device)).expand(b, h, s)
    kept = []
    for name, x in (("k", k), ("v", v)):
        codes, scales = _quantise(x)
        c[name + "_codes"].scatter_(2, rows[..., None].expand(b, h, s, d // 2), _pack(codes))
        c[name + "_scales"].scatter_(2, rows[..., None, None].expand(b, h, s, d // GROUP, 2), scales)
        kept.append(_values(codes, scales).bfloat16())
    c["weights"].scatter_(2, rows, torch.zeros((b, h, s), device=k.device))
    c["positions"].scatter_(2, rows, rows.int())
    return kept


def _plain_write(st):
    b, s, _ = st["gqkv"].shape
    x = st["gqkv"].unflatten(-1, (4, st["heads"], -1))
    gate = x[:, :, 0].contiguous()
    q, k, v = (x[:, :, i].transpose(1, 2) for i in (1, 2, 3))
    pos = st["offset"].long()[:, None] + torch.arange(s, device=q.device)
    cs = st["table"][pos].double()[:, None]
    half = q.shape[-1] // 2
    cos, sin = cs[..., :half], cs[..., half:]

    def rotate(t):  # in 64 bits: the bf16 results feed the quantiser's borders
        t = t.double()
        a, e = t[..., :half], t[..., half:]
        return torch.cat([a * cos - e * sin, e * cos + a * sin], -1).bfloat16()

    kv, vv = _plain_store(st["cache"], st["offset"], rotate(k), v)
    return [gate, rotate(q), kv, vv, st["cache"]["weights"], st["cache"]["positions"]]


def _limits(st, s, device):
    """Rows that query s of each sequence sees: up to itself, or the prefix, within the rows written."""
    off = st["offset"].long()[:, None]
    lim = torch.maximum(off + 1 + torch.arange(s, device=device), torch.full_like(off, st["prefix"]))
    return torch.minimum(lim, off + s)


def _plain_attend(st):
    q, c = st["q"].float(), st["cache"]
    b, h, s, d = q.shape
    k = _values(_unpack(c["k_codes"]), c["k_scales"])
    v = _values(_unpack(c["v_codes"]), c["v_scales"])
    hk, n = k.shape[1], k.shape[2]
    q = q.reshape(b, hk, (h // hk) * s, d)
    p = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    seen = torch.arange(n, device=q.device) < _limits(st, s, q.device)[..., None]
    seen = seen[:, None, None].expand(b, hk, h // hk, s, n).reshape(b, hk, -1, n)
    p = p.masked_fill(~seen, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p, v).reshape(b, h, s, d).transpose(1, 2)
    if st["gate"] is not None:
        o = o / (1.0 + torch.exp(-st["gate"].float()))
    out = [o.bfloat16().contiguous()]
    if st["track"]:
        out.append(c["weights"].add_(p.sum(2)))
    return out


def _plain_evict(st):
    c, n, budget = st["cache"], st["lengths"].long(), st["budget"]
    if st["step"]:
        _plain_store(c, torch.full_like(n, budget), st["k"], st["v"])
    w = c["weights"]
    at = torch.arange(w.shape[2], device=w.device)
    live = (at < n[:, None])[:, None].expand_as(w)
    key = torch.where(c["positions"] >= st["protect"][:, None, None], torch.full_like(w, math.inf), w)
    key = torch.where(live, key, torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(live).scatter_(2, order[..., :budget], True) & live
    low = at < torch.minimum(n, torch.full_like(n, budget))[:, None, None]
    hole, move = low & ~keep, keep & (at >= budget)
    # the i-th row that moves goes to the i-th hole
    first = torch.sort((~move).to(torch.uint8), dim=-1, stable=True).indices
    src = torch.where(hole, first.gather(2, (hole.long().cumsum(-1) - 1).clamp(min=0)), at.expand_as(first))
    src = src[..., :budget]
    to = c if st["step"] else st["out"]
    done = {}
    for name, x in c.items():
        i = src[(...,) + (None,) * (x.dim() - 3)].expand(*src.shape, *x.shape[3:])
        got = x.gather(2, i)
        ok = low[..., :budget].expand_as(src)[(...,) + (None,) * (x.dim() - 3)]
        to[name][:, :, :budget] = torch.where(ok, got, to[name][:, :, :budget])
        done[name] = to[name][:, :, :budget]
    return [torch.minimum(n, torch.full_like(n, budget)).int(), done]


# ------------------------------------------------------------- the framework's
def _own(st):
    import sys

    if "hrm_layer_ops" not in sys.modules:
        sys.path.insert(0, "hrm-text-cuda_b200")
    import hrm_layer_ops as ops

    if "handle" not in st:  # a program wraps its buffers once
        st["handle"] = ops.Kv4Cache(**st["cache"])
        st["out_handle"] = ops.Kv4Cache(**st["out"]) if "out" in st else None
    c = st["handle"]
    if st["op"] == "write":
        gate, q, k, v = ops.split_gqkv_rope_kv4(st["gqkv"], st["heads"], c, st["offset"], THETA, st["table"],
                                                cache_offset=st["offset"])
        return [gate, q, k, v, c.weights, c.positions]
    if st["op"] == "attend":
        o = ops.kv4_attention(st["q"], c, st["offset"], gate=st["gate"], prefix_len=st["prefix"],
                              accumulate=st["track"])
        return [o, c.weights] if st["track"] else [o]
    if st["step"]:
        ops.kv4_update(c, st["k"], st["v"], position_offset=st["budget"], cache_offset=st["budget"])
    n = ops.kv4_evict(c, st["lengths"], st["budget"], st["protect"], out=st["out_handle"])
    to = c if st["step"] else st["out_handle"]
    # bytes that the eviction only moves: compared as they are
    return [n, {name: getattr(to, name)[:, :, : st["budget"]] for name in st["cache"]}]


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "attend": _plain_attend, "evict": _plain_evict}[state["op"]](state)


# ------------------------------------------------------------- what it must cost
def work(case):
    b, d = case["batch"], case["dim"]
    row = 2 * (d // 2 + d // GROUP * 4)  # a cached row of one head: codes and scales of k and v
    if case["op"] == "write":
        t = b * case["seq"] * case["heads"]
        places = b * case["seq"] if case["ragged"] else case["seq"]
        return {"bytes": t * (8 * d + 8 * d + row + 8) + min(places, case["cache"]) * 4 * d,
                "flops": t * d * 2 * 3 + t * d * 2 * 4}
    if case["op"] == "attend":
        s, lens = case["seq"], _lengths(case, case["seq"])
        q = b * s * case["heads"] * d * 2
        pairs = 0
        for n in lens:
            p = min(max(case["prefix"], 0), n)
            first = n - s
            low = min(max(p - first, 0), s)  # queries that see the whole prefix and no more
            pairs += low * p + (s - low) * (first + 1 + low + n) // 2
        return {"bytes": sum(lens) * case["kv"] * (row + (8 if case["track"] else 0)) + q * (3 if case["gate"] else 2),
                "flops": 4 * d * pairs * case["heads"]}
    lens = _lengths(case, max(1, case["budget"] // 2))
    h = case["heads"]
    if case["step"]:
        return {"bytes": b * h * (case["rows"] * 8 + 2 * (row + 8) + 4 * d + row + 8), "flops": b * h * case["rows"]}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": h * (sum(lens) * 8 + kept * (2 * row + 16)), "flops": h * sum(lens)}


# ------------------------------------------------------------ the same in 64 bits
def _exact_values(packed, scales):
    d = packed.shape[-1] * 2
    e = torch.arange(d, device=packed.device)
    code = (packed[..., e // 2].int() >> (4 * (e % 2)).int()) & 15
    sc = scales.double()[..., e // GROUP, :]
    return (sc[..., 0] * (16 + code) / 16 + sc[..., 1]).bfloat16().double()


def _exact_codes(x):
    """bf16 x as the cache would hold it, and the values that it stands for."""
    g = x.double().unflatten(-1, (-1, GROUP))
    span = g.amax(-1) - g.amin(-1)
    scale = (span * 16 / 15).bfloat16().double()
    base = (g.amin(-1) - scale).bfloat16().double()
    n = torch.round(((g - base[..., None]) / scale[..., None] - 1) * 16).clamp(0, 15).nan_to_num()
    return (scale[..., None] * (1 + n / 16) + base[..., None]).bfloat16().double().flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "write":
        b, s, h, d = case["batch"], case["seq"], case["heads"], case["dim"]
        x = st["gqkv"].view(b, s, 4, h, d).double()
        place = st["offset"].double()[:, None] + torch.arange(s, device="cuda", dtype=torch.float64)
        row = st["table"].double()[place.long()]
        z = torch.complex(row[..., : d // 2], row[..., d // 2:])[:, :, None]

        def turned(t):  # pairs (i, i + d/2) as complex numbers, turned by the table's angles
            w = torch.complex(t[..., : d // 2], t[..., d // 2:]) * z
            return torch.cat([w.real, w.imag], -1).permute(0, 2, 1, 3)

        k = _exact_codes(turned(x[:, :, 2]).bfloat16())
        v = _exact_codes(x[:, :, 3].permute(0, 2, 1, 3))
        return [x[:, :, 0], turned(x[:, :, 1]), k, v, None, None]
    if case["op"] == "attend":
        b, s, h, d, hk = case["batch"], case["seq"], case["heads"], case["dim"], case["kv"]
        c, off = st["cache"], st["offset"].tolist()
        o = torch.zeros((b, s, h, d), dtype=torch.float64, device="cuda")
        w = c["weights"].double()
        for i in range(b):
            k, v = (_exact_values(c[t + "_codes"][i], c[t + "_scales"][i]) for t in "kv")
            for j in range(h):
                m = off[i] + s
                x = st["q"][i, j].double() @ k[j * hk // h, :m].T / math.sqrt(d)
                q_at = off[i] + torch.arange(s, device="cuda")[:, None]
                k_at = torch.arange(m, device="cuda")[None]
                x = x.masked_fill((k_at > q_at) & (k_at >= case["prefix"]), -math.inf)
                p = torch.softmax(x, dim=-1)
                o[i, :, j] = p @ v[j * hk // h, :m]
                w[i, j * hk // h, :m] += p.sum(0)
        if st["gate"] is not None:
            o = o * torch.sigmoid(st["gate"].double())
        return [o, w] if case["track"] else [o]
    return None

"""GPU: the 4-bit cache's operators as a server uses them: a prompt, decoding steps and
evictions through the recurrent loop, on explicit and several streams, in captured
and replayed steps, with the caller's buffers; and long prompts' query tiles.

Tolerances as in tests/test_kv4_gpu.py (whose checks these use); where two runs of the
same calls are compared, bits are.
"""

import pytest
import torch

import hrm_layer_ops as ops
import kv4_reference as ref
from hrm_layer_ops import module
import test_kv4_gpu as base
from test_kv4_gpu import U, buffers, filled, rand, run_attention, same, snapshot

pytestmark = pytest.mark.gpu


def check_vectorised(c, q, off, gate, prefix, got, w0):
    """run_attention's bounds for many query rows: outputs and weights."""
    b, h, s, d = q.shape
    n, group = c.shape[2], h // c.shape[1]
    k, v = ref.values(c.k_codes, c.k_scales), ref.values(c.v_codes, c.v_scales)
    offs = off.cpu() if isinstance(off, torch.Tensor) else torch.full((b,), off)
    lim = ref.limits(offs, s, prefix, n).cuda()
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    x = torch.einsum("bhsd,bhld->bhsl", q.double(), k) * d**-0.5
    seen = torch.arange(n, device="cuda") < lim[:, None, :, None]
    p = torch.softmax(x.masked_fill(~seen, -float("inf")), -1).nan_to_num(0.0)
    sig = torch.sigmoid(gate.double())
    want, spread = torch.einsum("bhsl,bhld->bshd", p, v) * sig, torch.einsum("bhsl,bhld->bshd", p, v.abs()) * sig
    score = torch.einsum("bhsd,bhld->bhsl", q.double().abs(), k.abs()).amax() * d**-0.5
    rel = 2 * (d + 8) * 2.0**-23 * float(score) + (n + 64) * 2.0**-23 + 2.0**-20 + 2.0**-18
    assert bool(((got.double() - want).abs() <= U * want.abs() + (rel + U) * spread + 1e-37).all())
    w = p.unflatten(1, (c.shape[1], group)).sum((2, 3))
    err = (c.weights.double() - w0 - w).abs()
    assert bool((err <= rel * w + (group * s + 2) * 2.0**-23 * (w0 + w)).all()), float(err.max())


@pytest.mark.parametrize("b,hk,group,s,n,d,prefix,ragged", [
    (1, 2, 1, 700, 900, 128, 0, False), (2, 1, 3, 300, 900, 64, 0, False), (2, 1, 2, 517, 1030, 128, 400, False),
    (3, 1, 2, 400, 700, 192, 0, True), (3, 2, 1, 640, 640, 64, 129, True), (1, 1, 7, 100, 300, 128, 0, False),
    (2, 1, 1, 257, 1500, 256, 1300, True), (1, 1, 40, 5, 2000, 128, 0, False)])
def test_prompts_against_the_plain_form(cuda, b, hk, group, s, n, d, prefix, ragged):
    """Query tiles that cross heads, begin past rows that they do not see, or see all."""
    c = filled(b, hk, n, d, s)
    q, gate = rand((b, hk * group, s, d), 3), rand((b, s, hk * group, d), 4)
    off = torch.tensor([n - s, -s // 2, -s - 1][:b], dtype=torch.int32, device="cuda") if ragged else n - s
    w0 = c.weights.double()
    got = ops.kv4_attention(q, c, off, gate=gate, prefix_len=prefix, accumulate=True)
    check_vectorised(c, q, off, gate, prefix, got, w0)
    assert ops.wait_timeouts() == 0


@pytest.mark.parametrize("b,hk,group,s,n,d,ragged", [
    (1, 2, 1, 4, 13000, 128, False), (3, 1, 4, 2, 12800, 256, True), (2, 1, 2, 9, 14000, 64, False),
    (1, 1, 1, 3, 13000, 192, False), (5, 2, 1, 1, 15000, 128, True), (1, 1, 4, 8, 12289, 128, True),
    (80, 2, 1, 2, 4200, 64, True)])
def test_long_caches_in_equal_shares(cuda, b, hk, group, s, n, d, ragged):
    """Caches past what a cluster serves, with one and several query rows per item."""
    base.test_attention_long_caches(cuda, b, hk, group, s, n, d, ragged)


def test_equal_shares_nan_rows(cuda):
    """As test_long_caches_nan_rows_and_lse_order, in the equal shares."""
    n, d, s = 14000, 128, 4
    c = filled(1, 2, n, d, 33)
    q = rand((1, 2, s, d), 34)
    clean = ops.kv4_attention(q, c, n - s)
    c.v_scales[:, :, n - 1, 1, 0] = float("nan")
    got = ops.kv4_attention(q, c, n - s)
    same(got[:, :-1], clean[:, :-1])
    nan = torch.isnan(got[0, -1])
    want = torch.zeros_like(nan)
    want[:, 32:64] = True
    assert torch.equal(nan, want)


def test_prompt_and_eviction_past_four_gigabytes(cuda):
    """Offsets past 2^32 bytes in the prompt's kernels and in the eviction: the last head
    of a large cache."""
    b, h, n, d, s = 3, 12, 1 << 20, 256, 70
    c = ops.kv4_cache(b, h, n, d, track=True)
    assert c.k_codes.numel() > 1 << 32
    small = filled(1, 1, 4096, d, 95)
    for name, t in buffers(c).items():
        t[-1, -1, -4096:] = buffers(small)[name][0, 0]
        t[-1, -1, :4096] = buffers(small)[name][0, 0]
    c.weights[-1, -1, 4096:].zero_()
    q = rand((b, h, s, d), 97)
    off = torch.tensor([-s, -s, n - s], dtype=torch.int32, device="cuda")
    w0 = c.weights[-1, -1].double()
    got = ops.kv4_attention(q, c, off, accumulate=True)
    assert not bool(got[:2].any()) and ops.wait_timeouts() == 0
    kk, vv = ref.values(c.k_codes[-1, -1], c.k_scales[-1, -1]), ref.values(c.v_codes[-1, -1], c.v_scales[-1, -1])
    x = q[-1, -1].double() @ kk.T / 16
    seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - s, n, device="cuda")[:, None]
    p = torch.softmax(x.masked_fill(~seen, -float("inf")), 1)
    want, spread = p @ vv, p @ vv.abs()
    # fp32 sums of 2^20 rows, 16 to an addition, at most 2^-23 each: 2^-7; of 128 to an addition in l: 2^-10
    assert bool(((got[-1, :, -1].double() - want).abs() <= U * want.abs() + spread * (2.0**-6 + U)).all())
    err, w = (c.weights[-1, -1].double() - w0 - p.sum(0)).abs(), p.sum(0)
    assert bool((err <= 2.0**-9 * w + 100 * 2.0**-23 * (w0 + w)).all())
    del kk, vv, x, seen, p
    # the first 4096 rows of each head, of which the last head's have weights
    want = ref.evict(c.weights[-1, -1, :4096].cpu().numpy(), c.positions[-1, -1, :4096].cpu().numpy(), 4096, 1000, 4090)
    before = {name: t[-1, -1, :4096].clone() for name, t in buffers(c).items()}
    lengths = ops.kv4_evict(c, 4096, 1000, 4090)
    assert lengths.tolist() == [1000] * b
    for name, t in buffers(c).items():
        same(t[-1, -1, :1000], before[name][want], name)
    del c, before
    torch.cuda.empty_cache()
    with pytest.raises(ops.HrmError):  # more rows than an eviction takes
        ops.kv4_evict(ops.kv4_cache(1, 1, 500000, 64, track=True), 500000, 100, 0)


@pytest.mark.parametrize("s", [1, 40])
def test_gate_extremes(cuda, s):
    """sigmoid(gate) at its ends; what it makes smaller than 2^-126 may be 0."""
    c = filled(1, 1, 50, 64, 1)
    q = rand((1, 1, s, 64), 2)
    plain = ops.kv4_attention(q, c, 50 - s).double()
    gate = torch.zeros((1, s, 1, 64), dtype=torch.bfloat16, device="cuda")
    values = torch.tensor([float("inf"), 200.0, 88.0, 20.0, 0.0, -20.0, -86.0, -88.0, -100.0, -float("inf")])
    gate[..., :10] = values.bfloat16().cuda()
    gate[..., 10] = float("nan")
    got = ops.kv4_attention(q, c, 50 - s, gate=gate).double()
    want = plain * torch.sigmoid(gate.double())
    # plain has its own rounding, the result another
    near = (got - want).abs() <= 2.01 * U * want.abs() + 2.0**-126 * (1 + plain.abs())
    assert bool(near[..., :10].all()) and bool(near[..., 11:].all()) and bool(torch.isnan(got[..., 10]).all())


@pytest.mark.parametrize("s", [0, 1, 3, 33])
def test_empty_sizes(cuda, s):
    """No queries: nothing is written.  No rows: a query sees none and gives 0."""
    c = filled(2, 2, 8, 64, 3)
    before = snapshot(c)
    if s == 0:
        assert ops.kv4_attention(rand((2, 2, 0, 64), 1), c, 3, accumulate=True).shape == (2, 0, 2, 64)
        ops.kv4_update(c, rand((2, 2, 0, 64), 1), rand((2, 2, 0, 64), 1), 0, 0)
        for n, t in buffers(c).items():
            same(t, before[n], n)
    else:
        idle = torch.full((2,), -s, dtype=torch.int32, device="cuda")
        got = ops.kv4_attention(rand((2, 2, s, 64), 1), c, idle, accumulate=True)
        assert not bool(got.any())
        for n, t in buffers(c).items():
            same(t, before[n], n)


@pytest.mark.parametrize("b,s,n", [(2, 1, 3000), (3, 1, 6000), (2, 12, 5000), (1, 300, 2000)])
def test_callers_buffers_and_guards(cuda, b, s, n):
    """out and workspace of the caller's, in the middle of a larger buffer that stays as it was."""
    h, d = 2, 128
    c = filled(b, h, n, d, n)
    q, gate = rand((b, h, s, d), 5), rand((b, s, h, d), 6)
    w0 = c.weights.clone()
    want = ops.kv4_attention(q, c, n - s, gate=gate, accumulate=True)
    w1 = c.weights.clone()
    c.weights.copy_(w0)
    need = ops.kv4_attention_workspace(c, h, s, True)
    space = torch.full((need + 8192,), 0xA5, dtype=torch.uint8, device="cuda")
    whole = torch.full((want.numel() + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = whole[2048:2048 + want.numel()].view_as(want)
    got = ops.kv4_attention(q, c, n - s, gate=gate, accumulate=True, out=out, workspace=space[4096:4096 + need])
    assert got.data_ptr() == out.data_ptr()
    same(got, want, "out")
    same(c.weights, w1, "weights")
    assert bool((space[:4096] == 0xA5).all()) and bool((space[4096 + need:] == 0xA5).all())
    assert bool((whole[:2048] == 7).all()) and bool((whole[2048 + want.numel():] == 7).all())


def step(c, gqkv, heads, rows, position, budget, protect, theta=10000.0):
    gate, q, _, _ = ops.split_gqkv_rope_kv4(gqkv, heads, c, position, theta, cache_offset=rows, keep_kv=False)
    return ops.kv4_attention(q, c, rows, gate=gate, accumulate=True)


@pytest.mark.parametrize("place", ["in place", "out"])
def test_evict_long_rows_of_many_heads(cuda, place):
    """More clusters than the GPU holds at once."""
    c = filled(19, 8, 8500, 64, 70)
    lengths = [8500 - 400 * i for i in range(19)]
    out = ops.kv4_cache(19, 8, 3000, 64, track=True) if place == "out" else None
    base.check_evict(c, lengths, 3000, 8000, out)


def test_two_streams_at_once(cuda):
    """Two servers' steps side by side: each as if it ran alone."""
    h, d, b = 4, 128, 3
    xs = [rand((b, s, 4 * h * d), 10 + i) for i, s in enumerate((200, 1, 1, 5, 1))]

    def serve(c, stream):
        outs, rows = [], 0
        with torch.cuda.stream(stream):
            for i, x in enumerate(xs):
                outs.append(step(c, x, h, rows, rows, 0, 0))
                rows += x.shape[1]
                if i == 0:
                    lengths = ops.kv4_evict(c, rows, 150, rows - 10)
                    assert lengths.tolist() == [150] * b
                    rows = 150
        return outs

    alone = ops.kv4_cache(b, h, 5000, d, track=True)
    want = serve(alone, torch.cuda.current_stream())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        caches = [ops.kv4_cache(b, h, 5000, d, track=True) for _ in streams]
        torch.cuda.synchronize()
        got = [serve(c, st) for c, st in zip(caches, streams)]
        torch.cuda.synchronize()
        for c, outs in zip(caches, got):
            for a, w in zip(outs, want):
                same(a, w, "out")
            for n, t in buffers(alone).items():
                same(buffers(c)[n], t, n)


def test_explicit_stream_argument(cuda):
    """stream=: inputs made on that stream, while the current one does other work."""
    c, c2 = filled(2, 2, 4200, 128, 1), filled(2, 2, 4200, 128, 1)
    x, big = rand((2, 2, 9, 128), 2), rand((4096, 4096), 3)
    want = ops.kv4_attention(x * 2, c, 4000, accumulate=True)
    wl = ops.kv4_evict(c, 4009, 1000, 4000)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for _ in range(4):
            big @ big
        q = x * 2
    got = ops.kv4_attention(q, c2, 4000, accumulate=True, stream=st)
    lengths = ops.kv4_evict(c2, 4009, 1000, 4000, stream=st)
    st.synchronize()
    same(got, want, "out")
    same(lengths, wl, "lengths")
    for n, t in buffers(c).items():
        same(buffers(c2)[n], t, n)


@pytest.mark.parametrize("cache_len,budget", [(300, 64), (9000, 5000)])
def test_captured_decode_step_replays(cuda, cache_len, budget):
    """A step with device offsets, captured once and replayed as they advance, against
    the same steps run one by one."""
    b, h, d, steps = 2, 3, 128, 6
    first = filled(b, h, cache_len, d, 40)
    table = ops.rope_table(cache_len + 64, d, 10000.0)
    xs = [rand((b, 1, 4 * h * d), 60 + i) for i in range(steps)]
    state = {}

    def make():
        c = ops.kv4_cache(b, h, cache_len, d, track=True)
        for n, t in buffers(first).items():
            buffers(c)[n].copy_(t)
        rows = torch.tensor([budget, budget - 7], dtype=torch.int32, device="cuda")
        pos = torch.tensor([cache_len, cache_len - 5], dtype=torch.int32, device="cuda")
        return c, rows, pos, torch.empty((b, 1, 4 * h * d), dtype=torch.bfloat16, device="cuda")

    def one(c, rows, pos, x):
        gate, q, _, _ = ops.split_gqkv_rope_kv4(x, h, c, pos, 10000.0, table, rows, keep_kv=False)
        o = ops.kv4_attention(q, c, rows, gate=gate, accumulate=True)
        lengths = ops.kv4_evict(c, rows + 1, budget, pos - 8)
        rows.copy_(lengths)
        pos.add_(1)
        return o

    c, rows, pos, x = make()
    want = []
    for t in xs:
        x.copy_(t)
        want.append(one(c, rows, pos, x).clone())
    c2, rows2, pos2, x2 = make()
    one(*make())  # warm
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            state["o"] = one(c2, rows2, pos2, x2)
    torch.cuda.current_stream().wait_stream(side)
    for t, w in zip(xs, want):
        x2.copy_(t)
        g.replay()
        same(state["o"], w, "out")
    same(rows2, rows, "rows")
    for n, t in buffers(c).items():
        same(buffers(c2)[n], t, n)


def test_recurrent_loop_over_caches(cuda):
    """The recurrent forward with this attention in every KV slot: a prompt, then tokens
    one by one with an eviction before each; every attention against the plain form
    over the values that its cache holds."""
    B, H, D, I, layers, hc, lc = 2, 2, 64, 256, 2, 2, 1
    hidden, vocab = H * D, 50
    slots = layers * hc * (lc + 1)
    caches = [ops.kv4_cache(B, H, 64, D, track=True) for _ in range(slots)]
    w = {n: rand(shape, 90 + i, 0.05) for i, (n, shape) in enumerate(
        (("gqkv", (4 * hidden, hidden)), ("o", (hidden, hidden)), ("g", (I, hidden)), ("u", (I, hidden)),
         ("d", (hidden, I))))}
    at = {"rows": 0, "position": 0, "s": 0}
    calls = []

    def attention(layer, slot, normed, out):
        s, c = at["s"], caches[slot]
        gqkv = (normed @ w["gqkv"].T).view(B, s, 4 * hidden)
        gate, q, _, _ = ops.split_gqkv_rope_kv4(gqkv, H, c, at["position"], 10000.0, cache_offset=at["rows"],
                                                keep_kv=False)
        w0 = c.weights.clone()
        o = run_attention(c, q, at["rows"], gate=gate, accumulate=True)
        assert bool((c.weights >= w0).all())
        torch.matmul(o.reshape(B * s, hidden), w["o"].T, out=out)
        calls.append(slot)

    def gate_up(layer, n, g, u):
        torch.matmul(n, w["g"].T, out=g)
        torch.matmul(n, w["u"].T, out=u)

    def down(layer, a, o):
        torch.matmul(a, w["d"].T, out=o)

    fns = module.ModuleFns(layers, attention, gate_up, down)
    table, init = rand((vocab, hidden), 80, 0.02), rand((hidden,), 81)

    def forward(s):
        at["s"] = s
        scratch = module.ModuleScratch(B * s, hidden, I, "cuda")
        ids = torch.arange(B * s, dtype=torch.int32, device="cuda") % vocab
        return module.recurrent_forward(ids, table, 1.0, init, hc, lc, fns, fns, scratch)

    forward(40)
    assert calls == list(range(slots))
    at["rows"] = at["position"] = 40
    for _ in range(3):
        for c in caches:
            lengths = ops.kv4_evict(c, at["rows"], 24, at["position"] - 4)
            assert lengths.tolist() == [24] * B
            assert bool((c.positions[:, :, :24] >= at["position"] - 4).sum(-1).eq(4).all())
        at["rows"] = 24
        z_h, z_l = forward(1)
        assert bool(torch.isfinite(z_h).all()) and bool(torch.isfinite(z_l).all())
        at["rows"] += 1
        at["position"] += 1
    assert len(calls) == 4 * slots and ops.wait_timeouts() == 0


def test_front_end_refusals(cuda):
    c = ops.kv4_cache(2, 2, 16, 128, track=True)
    plain = ops.kv4_cache(2, 2, 16, 128)
    q = rand((2, 4, 3, 128), 1)
    ints = torch.zeros(2, dtype=torch.int32, device="cuda")
    cases = [
        lambda: ops.kv4_cache(1, 1, 4, 96),
        lambda: ops.kv4_attention(q[:, :3].contiguous(), c, 0),                     # 3 heads over 2
        lambda: ops.kv4_attention(q[..., :64].contiguous(), c, 0),                  # another head_dim
        lambda: ops.kv4_attention(q.transpose(1, 2), c, 0),                         # not contiguous
        lambda: ops.kv4_attention(q.float(), c, 0),
        lambda: ops.kv4_attention(q, plain, 0, accumulate=True),
        lambda: ops.kv4_attention(q, c, ints.long()),
        lambda: ops.kv4_attention(q, c, ints[:1]),
        lambda: ops.kv4_attention(q, c, 14),                                        # rows past the cache
        lambda: ops.kv4_attention(q, c, -1),
        lambda: ops.kv4_attention(q, c, 0, prefix_len=-1),
        lambda: ops.kv4_attention(q, c, 0, out=q[:1].contiguous()),
        lambda: ops.kv4_attention(q, c, 0, gate=q[:1].contiguous()),
        lambda: ops.kv4_attention(rand((2, 2, 1, 128), 1), c, 0, accumulate=True,
                                  workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
        lambda: ops.kv4_update(c, q, q),
        lambda: ops.kv4_update(c, q[:, :2].contiguous(), q[:, :2].contiguous(), 0, 14),
        lambda: ops.split_gqkv_rope_kv4(rand((2, 1, 2 * 2 * 128), 1), 2, c),
        lambda: ops.kv4_evict(plain, 8, 4, 0),
        lambda: ops.kv4_evict(c, 17, 4, 0),
        lambda: ops.kv4_evict(c, 8, 4, 0, out=ops.kv4_cache(2, 2, 3, 128, track=True)),
        lambda: ops.kv4_evict(c, 8, 4, 0, out=ops.kv4_cache(2, 1, 8, 128, track=True)),
        lambda: ops.kv4_evict(c, ints, 4, 0, new_lengths=ints),                     # lengths in place
    ]
    before = snapshot(c)
    for i, f in enumerate(cases):
        with pytest.raises((ValueError, TypeError, ops.HrmError)):
            f()
            pytest.fail(f"case {i} was accepted")
    torch.cuda.synchronize()
    for n, t in buffers(c).items():
        same(t, before[n], n)

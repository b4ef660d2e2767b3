"""CPU: with an explicit `stream`, what a call allocates comes from that stream.

A block from the current stream's pool may still be in use by kernels queued there,
and a dropped result goes back to that pool while the launch's stream writes it.  The
calls run here up to the launch, which is recorded instead; no memory is raced for.
"""

import contextlib
from types import SimpleNamespace

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from hrm_layer_ops import kv4

B, H, N, D = 2, 3, 16, 64
MADE = {"empty", "new_empty", "empty_like", "empty_strided", "zeros", "new_zeros"}


class Made(TorchDispatchMode):
    """Records, of each tensor made, whether the launch's stream was current."""

    def __init__(self, now):
        super().__init__()
        self.now, self.on = now, []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.overloadpacket.__name__ in MADE:
            self.on.append(self.now["stream"])
        return func(*args, **(kwargs or {}))


@pytest.fixture
def now(monkeypatch):
    """The current stream, as the calls under test set it."""
    state = {"stream": None, "launches": []}

    @contextlib.contextmanager
    def stream(s):
        state["stream"], before = s, state["stream"]
        yield
        state["stream"] = before

    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(kv4, "_need", lambda *a: None)
    monkeypatch.setattr(kv4, "_launch", lambda name, device, tensors, s, *a: state["launches"].append((name, s)))
    monkeypatch.setattr(kv4, "kv4_attention_workspace", lambda *a: 64)
    return state


def fake_cache():
    z = torch.zeros((B, H, N), dtype=torch.int32)
    return SimpleNamespace(shape=(B, H, N, D), device=z.device, weights=z.float(), positions=z, k_codes=z, _ref=None)


def split(**kw):
    x, c = torch.zeros((B, 2, 4 * H * D), dtype=torch.bfloat16), fake_cache()
    return lambda s: kv4.split_gqkv_rope_kv4(x, H, c, stream=s, **kw)


def attention(**kw):
    q, c = torch.zeros((B, H, 2, D), dtype=torch.bfloat16), fake_cache()
    return lambda s: kv4.kv4_attention(q, c, 4, stream=s, **kw)


def evict():
    c = fake_cache()
    return lambda s: kv4.kv4_evict(c, 8, 4, 0, stream=s)


# the call, and how many tensors it makes: results and, of the attention, the workspace
CALLS = [(split, {}, 4), (split, {"keep_kv": False}, 2), (attention, {}, 2), (evict, {}, 1)]


@pytest.mark.parametrize("make,kw,tensors", CALLS)
def test_results_are_allocated_on_the_launch_stream(now, make, kw, tensors):
    call, st = make(**kw), object()
    with Made(now) as made:
        call(st)
    assert [s for _, s in now["launches"]] == [st]
    assert made.on == [st] * tensors


@pytest.mark.parametrize("make,kw,tensors", CALLS)
def test_without_a_stream_the_current_one_is_used(now, make, kw, tensors):
    call = make(**kw)
    with Made(now) as made:
        call(None)
    assert [s for _, s in now["launches"]] == [None]
    assert made.on == [None] * tensors

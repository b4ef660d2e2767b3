"""CPU: with an explicit `stream`, what a layer operator's call allocates comes from that stream.

A block from the current stream's pool may still be in use by kernels queued there,
and a dropped result goes back to that pool while the launch's stream writes it.  The
calls run here up to the launch, which is recorded instead; no memory is raced for.
"""

import contextlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from hrm_layer_ops import ops

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
    monkeypatch.setattr(ops, "_need", lambda *a: None)
    monkeypatch.setattr(ops, "_launch", lambda name, tensors, s, *a: state["launches"].append(s))
    return state


x = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
table, ids, raw = torch.zeros((7, 64), dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32), torch.zeros(8).byte()
CALLS = {
    "additive_inject": (lambda s: ops.additive_inject(x, x, stream=s), 1),
    "swiglu_ffn": (lambda s: ops.swiglu_ffn(x, x, stream=s), 1),
    "rms_norm": (lambda s: ops.rms_norm(x, stream=s), 1),
    "add_rms_norm": (lambda s: ops.add_rms_norm(x, x, stream=s), 2),
    "rope_table": (lambda s: ops.rope_table(4, 64, device="cpu", stream=s), 1),
    "embedding_lookup": (lambda s: ops.embedding_lookup(ids, table, 1.0, stream=s), 1),
    "embed_rms_norm": (lambda s: ops.embed_rms_norm(ids, table, 1.0, stream=s), 2),
    "embed_rms_norm, normed only": (lambda s: ops.embed_rms_norm(ids, table, 1.0, keep_hidden=False, stream=s), 1),
    "split_gqkv_rope": (lambda s: ops.split_gqkv_rope(x, 2, stream=s), 4),
    "gated_attn_output": (lambda s: ops.gated_attn_output(x, x, stream=s), 1),
    "broadcast_vec": (lambda s: ops.broadcast_vec(x, 3, stream=s), 1),
    "convert_to_bf16": (lambda s: ops.convert_to_bf16(raw, "f32", stream=s), 1),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_results_are_allocated_on_the_launch_stream(now, name):
    call, tensors = CALLS[name]
    for st in (object(), None):
        now["launches"].clear()
        with Made(now) as made:
            call(st)
        assert now["launches"] == [st]
        assert made.on == [st] * tensors

"""CPU: a caller's output buffer, table or cache of another size is refused before anything is queued
(the library is given addresses only: a short one would be read or written past its end)."""

import pytest
import torch

from hrm_layer_ops import ops

BF = dict(dtype=torch.bfloat16)


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    def launch(*a):
        pytest.fail("a launch was reached")

    monkeypatch.setattr(ops, "_need", lambda *a: None)
    monkeypatch.setattr(ops, "_launch", launch)


x, table, ids = torch.zeros((2, 4, 64), **BF), torch.zeros((7, 64), **BF), torch.zeros(5, dtype=torch.int32)
short = torch.zeros(64, **BF)
CALLS = {
    "additive_inject": lambda: ops.additive_inject(x, x, out=short),
    "swiglu_ffn": lambda: ops.swiglu_ffn(x, x, out=short),
    "rms_norm": lambda: ops.rms_norm(x, out=short),
    "add_rms_norm": lambda: ops.add_rms_norm(x, x, residual_out=short, normed_out=x.clone()),
    "add_rms_norm normed": lambda: ops.add_rms_norm(x, x, residual_out=x.clone(), normed_out=short),
    "rope_table": lambda: ops.rope_table(4, 64, out=short),
    "embedding_lookup": lambda: ops.embedding_lookup(ids, table, 1.0, out=short),
    "embed_rms_norm": lambda: ops.embed_rms_norm(ids, table, 1.0, normed_out=short),
    "embed_rms_norm hidden": lambda: ops.embed_rms_norm(ids, table, 1.0, hidden_out=short),
    "split_gqkv_rope": lambda: ops.split_gqkv_rope(x, 2, out=(short, *(x[..., :16].clone() for _ in range(3)))),
    "split_gqkv_rope v": lambda: ops.split_gqkv_rope(x, 2, out=(*(x[..., :16].clone() for _ in range(3)), short)),
    "split_gqkv_rope caches": lambda: ops.split_gqkv_rope(x, 2, k_cache=torch.zeros((2, 2, 9, 4), **BF),
                                                          v_cache=torch.zeros((2, 2, 9, 4), **BF)),
    "split_gqkv_rope table": lambda: ops.split_gqkv_rope(x, 2, table=torch.zeros((9, 4))),
    "gated_attn_output": lambda: ops.gated_attn_output(x, x, out=short),
    "broadcast_vec": lambda: ops.broadcast_vec(short, 3, out=short),
    "convert_to_bf16": lambda: ops.convert_to_bf16(torch.zeros(8).byte(), "f32", out=short),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_a_buffer_of_another_size_is_refused(name):
    with pytest.raises(ValueError):
        CALLS[name]()

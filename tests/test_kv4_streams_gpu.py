"""GPU: with an explicit `stream`, a call's results lie in that stream's pool (the
allocator's own record), not in the current stream's."""

import pytest
import torch

import hrm_layer_ops as ops

pytestmark = pytest.mark.gpu


def pool_of(t):
    """The stream whose pool a tensor's block is from."""
    for seg in torch.cuda.memory_snapshot():
        if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"]:
            return seg["stream"]
    raise AssertionError("not the allocator's")


def test_results_lie_in_the_launch_streams_pool(cuda):
    c = ops.kv4_cache(2, 3, 64, 128, track=True)
    x = torch.zeros((2, 5, 4 * 3 * 128), dtype=torch.bfloat16, device=cuda)
    # freed blocks of the results' sizes in the current stream's pool, which must not be taken
    del_me = [torch.empty((2, 5, 3, 128), dtype=torch.bfloat16, device=cuda) for _ in range(8)]
    here = pool_of(del_me[0])
    del del_me
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    got = list(ops.split_gqkv_rope_kv4(x, 3, c, stream=st))
    got.append(ops.kv4_attention(got[1], c, 0, gate=got[0], accumulate=True, stream=st))
    got.append(ops.kv4_evict(c, 5, 3, 4, stream=st))
    st.synchronize()
    assert here != st.cuda_stream and [pool_of(t) for t in got] == [st.cuda_stream] * 6
    assert got[-1].tolist() == [3, 3]
    q = ops.split_gqkv_rope_kv4(x, 3, c)[1]
    assert pool_of(q) == here and pool_of(ops.kv4_attention(q, c, 0)) == here

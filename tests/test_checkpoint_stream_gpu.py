"""GPU: a load on another stream begins after what the current stream has queued,
which may still use the blocks that the weights are given."""

import os

import pytest
import torch

from conftest import GOLDEN
from hrm_layer_ops import checkpoint as ck

pytestmark = pytest.mark.gpu


class Recorded(torch.cuda.Stream):
    waits = ()

    def wait_stream(self, other):
        self.waits = (*self.waits, other)
        super().wait_stream(other)


def test_load_waits_for_the_current_stream(cuda):
    path = os.path.join(GOLDEN, "ckpt_tiny_attn.safetensors")
    want = ck.load_safetensors(path, 2, 32, 48, device=cuda)
    st = Recorded()
    got = ck.load_safetensors(path, 2, 32, 48, device=cuda, stream=st)
    assert st.waits == (torch.cuda.current_stream(),)
    for a, b in ((got.embed_tokens, want.embed_tokens), (got.h_module[1].up_proj, want.h_module[1].up_proj)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))

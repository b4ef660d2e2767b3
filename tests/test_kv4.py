"""CPU: what the 4-bit KV cache's calls refuse (no kernel is launched: every case
returns before anything is queued), and the restatement that the GPU tests use."""

import ctypes

import numpy as np
import pytest
import torch

import kv4_reference as ref
from hrm_layer_ops import _lib, kv4

vp = ctypes.c_void_p
BASE, STEP = 0x10000000, 0x10000000
PTR = [BASE + i * STEP for i in range(16)]


@pytest.fixture(scope="module")
def lib():
    return _lib.LIB


def cache(at=0, batch=2, heads=3, rows=8, dim=128, **change):
    """Fake device addresses, 256 MB apart from PTR[at] on."""
    f = dict(k_codes=PTR[at], k_scales=PTR[at + 1], v_codes=PTR[at + 2], v_scales=PTR[at + 3], weights=PTR[at + 4],
             positions=PTR[at + 5], batch=batch, kv_heads=heads, cache_len=rows, head_dim=dim)
    f.update(change)
    return ctypes.byref(_lib.Kv4CacheStruct(**f))


SHAPES = [(dict(batch=-1), "INVALID_SHAPE"), (dict(heads=0), "INVALID_SHAPE"), (dict(rows=-1), "INVALID_SHAPE"),
          (dict(dim=0), "INVALID_SHAPE"), (dict(dim=96), "INVALID_SHAPE"), (dict(dim=320), "INVALID_SHAPE"),
          (dict(rows=2**31), "SIZE_OVERFLOW"), (dict(batch=2**40, rows=2**30), "SIZE_OVERFLOW")]
POINTERS = [(dict(k_codes=None), "NULL_POINTER"), (dict(v_scales=None), "NULL_POINTER"),
            (dict(k_codes=PTR[0] + 8), "ALIGNMENT"), (dict(v_scales=PTR[3] + 4), "ALIGNMENT"),
            (dict(weights=PTR[4] + 2), "ALIGNMENT")]


def code(name):
    return getattr(_lib, "HRM_ERR_" + name)


def update(lib, c, k=PTR[6], v=PTR[7], seq=2, pos=0, off=0, poss=None, offs=None):
    return lib.hrm_kv4_update(c, vp(k), vp(v), seq, pos, vp(poss), off, vp(offs), None)


def split(lib, c, gqkv=PTR[6], gate=PTR[10], q=PTR[11], k=PTR[12], v=PTR[13], seq=2, pos=0, poss=None, table=None,
          tp=0, off=0, offs=None):
    return lib.hrm_split_gqkv_rope_kv4(vp(gqkv), vp(gate), vp(q), vp(k), vp(v), c, seq, pos, vp(poss), 1e4, vp(table),
                                       tp, off, vp(offs), None)


def attend(lib, c, q=PTR[6], gate=None, out=PTR[7], heads=3, seq=2, off=0, offs=None, prefix=0, scale=0.1, acc=0,
           ws=None, nbytes=0):
    return lib.hrm_kv4_attention(vp(q), c, vp(gate), vp(out), heads, seq, off, vp(offs), prefix, scale, acc, vp(ws),
                                 nbytes, None)


def evict(lib, c, out, length=8, lengths=None, budget=4, protect=0, protects=None, new=PTR[14]):
    return lib.hrm_kv4_evict(c, out, length, vp(lengths), budget, protect, vp(protects), vp(new), None)


@pytest.mark.parametrize("change,status", SHAPES + POINTERS)
def test_cache_refusals(lib, change, status):
    for got in (update(lib, cache(**change)), split(lib, cache(**change)), attend(lib, cache(**change)),
                evict(lib, cache(**change), cache(**change))):
        assert got == code(status)


def test_write_refusals(lib):
    c = cache()
    for call in (update, split):
        assert call(lib, c, seq=-1) == code("INVALID_SHAPE")
        assert call(lib, c, off=-1) == code("INVALID_SHAPE")
        assert call(lib, c, off=7) == code("INVALID_SHAPE")
        assert call(lib, c, seq=9) == code("INVALID_SHAPE")
        assert call(lib, c, pos=-1) == code("INVALID_SHAPE")
        assert call(lib, c, pos=2**31 - 1) == code("SIZE_OVERFLOW")
        assert call(lib, c, offs=PTR[15] + 2) == code("ALIGNMENT")
        assert call(lib, c, offs=PTR[0]) == code("ALIASING")
        assert call(lib, None) == code("NULL_POINTER")
        assert call(lib, cache(batch=0)) == 0 and call(lib, c, seq=0) == 0
    assert update(lib, c, k=None) == code("NULL_POINTER")
    assert update(lib, c, v=PTR[7] + 2) == code("ALIGNMENT")
    assert update(lib, c, k=PTR[2]) == code("ALIASING")
    assert update(lib, cache(v_codes=PTR[0])) == code("ALIASING")
    assert split(lib, c, gqkv=None) == code("NULL_POINTER")
    assert split(lib, c, k=None) == code("NULL_POINTER")
    assert split(lib, c, gate=PTR[11] + 16) == code("ALIASING")
    assert split(lib, c, q=PTR[11] + 2) == code("ALIGNMENT")
    assert split(lib, c, table=PTR[15], tp=1) == code("TABLE_RANGE")
    assert split(lib, c, table=PTR[10], tp=2) == code("ALIASING")


def test_attention_refusals(lib):
    c = cache()
    assert attend(lib, None) == code("NULL_POINTER")
    assert attend(lib, c, q=None) == code("NULL_POINTER")
    assert attend(lib, c, heads=4) == code("INVALID_SHAPE")
    assert attend(lib, c, heads=0) == code("INVALID_SHAPE")
    assert attend(lib, c, seq=-1) == code("INVALID_SHAPE")
    assert attend(lib, c, off=7) == code("INVALID_SHAPE")
    assert attend(lib, c, off=-1) == code("INVALID_SHAPE")
    assert attend(lib, c, prefix=-1) == code("INVALID_SHAPE")
    assert attend(lib, c, scale=float("nan")) == code("INVALID_SHAPE")
    assert attend(lib, c, nbytes=-1) == code("INVALID_SHAPE")
    assert attend(lib, c, out=PTR[7] + 4) == code("ALIGNMENT")
    assert attend(lib, c, out=PTR[6]) == code("ALIASING")
    assert attend(lib, c, out=PTR[0]) == code("ALIASING")
    assert attend(lib, c, acc=1) == code("NULL_POINTER")  # no workspace
    assert attend(lib, cache(weights=None), acc=1, ws=PTR[8], nbytes=1 << 20) == code("NULL_POINTER")
    assert attend(lib, c, acc=1, ws=PTR[8], nbytes=8) == code("SCRATCH_LIMIT")
    assert attend(lib, c, acc=1, ws=PTR[4], nbytes=1 << 20) == code("ALIASING")
    assert attend(lib, cache(rows=2**20), heads=3 * 2**10, seq=2**20 - 1) == code("SIZE_OVERFLOW")
    assert attend(lib, c, seq=0) == 0 and attend(lib, cache(batch=0)) == 0


def test_attention_workspace_sizes(lib):
    def size(heads, seq, acc, **kw):
        n = ctypes.c_int64(-1)
        assert lib.hrm_kv4_attention_workspace(cache(**kw), heads, seq, acc, ctypes.byref(n)) == 0
        return n.value

    assert size(3, 2, 0) == 0
    assert size(3, 2, 1) == 4 * 2 * 3 * 2 * 8       # scores of every query and cache row
    assert size(6, 5, 1) == 4 * 2 * 6 * 5 * (8 + 1)  # and one number per query
    assert size(6, 9, 1) == 4 * 2 * 6 * 9           # that alone
    assert size(3, 1, 0, rows=4096) == 0
    assert size(3, 1, 0, rows=65536) > 0            # partial results of a split decode
    assert size(3, 33, 0, rows=65536, batch=200) == 0
    assert lib.hrm_kv4_attention_workspace(cache(), 3, 2, 1, None) == code("NULL_POINTER")


def test_evict_refusals(lib):
    c = cache()
    assert evict(lib, None, c) == code("NULL_POINTER")
    assert evict(lib, c, None) == code("NULL_POINTER")
    assert evict(lib, c, c, budget=0) == code("INVALID_SHAPE")
    assert evict(lib, c, c, length=9) == code("INVALID_SHAPE")
    assert evict(lib, c, c, length=-1) == code("INVALID_SHAPE")
    assert evict(lib, c, c, new=None) == code("NULL_POINTER")
    assert evict(lib, c, c, lengths=PTR[14]) == code("ALIASING")
    assert evict(lib, c, c, protects=PTR[14] + 1) == code("ALIGNMENT")
    assert evict(lib, c, cache(6, rows=3)) == code("INVALID_SHAPE")
    assert evict(lib, c, cache(6, heads=2)) == code("INVALID_SHAPE")
    assert evict(lib, c, cache(6, v_codes=PTR[2])) == code("ALIASING")  # shares one buffer
    assert evict(lib, cache(weights=None), cache(6)) == code("NULL_POINTER")
    assert evict(lib, c, cache(6, positions=None)) == code("NULL_POINTER")
    big = cache(rows=200_000, heads=1, batch=1)
    assert evict(lib, big, big, length=200_000, budget=100_000) == code("SCRATCH_LIMIT")
    assert evict(lib, cache(batch=0), cache(6, batch=0)) == 0


def test_status_string(lib):
    assert "aligned" in lib.hrm_status_string(_lib.HRM_ERR_ALIGNMENT).decode()


def test_front_end_refuses_cpu_tensors():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        kv4.Kv4Cache(z((1, 1, 4, 64), dtype=torch.uint8), z((1, 1, 4, 4, 2), dtype=torch.bfloat16),
                     z((1, 1, 4, 64), dtype=torch.uint8), z((1, 1, 4, 4, 2), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="head_dim"):
        kv4.kv4_cache(1, 1, 4, 80, device="cpu")


def test_restatement_round_trip():
    """Codes survive packing; the extremes of a group come back within the grid's roundings."""
    x = torch.randn((3, 5, 128), generator=torch.Generator().manual_seed(0)).bfloat16()
    codes, scales = ref.quantise(x)
    assert torch.equal(ref.unpack(ref.pack(codes)), codes)
    assert int(codes.max()) == 15 and int(codes.min()) == 0
    err = (ref.values(ref.pack(codes), scales) - x.double()).abs()
    step = scales[..., 0].double().repeat_interleave(32, -1) / 16
    assert bool((err <= step).all())


def test_restated_eviction():
    w = np.array([1.0, 3.0, 2.0, 2.0, np.nan, 5.0], np.float32)
    p = np.arange(6)
    assert ref.evict(w, p, 6, 3, 100) == [5, 1, 2]   # row 2 wins the tie with row 3; 5 takes 0's place
    assert ref.evict(w, p, 6, 3, 4) == [4, 1, 5]     # 4 and 5 are protected
    assert ref.evict(w, p, 2, 3, 0) == [0, 1]

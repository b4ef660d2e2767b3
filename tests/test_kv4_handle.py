"""CPU: a Kv4Cache's C struct holds its tensors' addresses, so its tensors stay."""

import dataclasses

import pytest
import torch

from hrm_layer_ops import kv4


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(kv4, "_need", lambda *a: None)  # CPU tensors; nothing is launched
    return kv4.kv4_cache(2, 3, 8, 128, device="cpu", track=True)


def test_tensors_of_a_cache_are_not_replaced(cache):
    old = cache.weights
    for name in ("k_codes", "k_scales", "v_codes", "v_scales", "weights", "positions"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros_like(getattr(cache, name)))
        assert getattr(cache._struct, name) == getattr(cache, name).data_ptr()
    with pytest.raises(AttributeError):
        cache.weights = None
    assert cache.weights is old
    cache.weights.zero_()


def test_replace_makes_another_struct(cache):
    other = dataclasses.replace(cache, weights=torch.ones_like(cache.weights))
    assert other._struct.weights == other.weights.data_ptr() != cache._struct.weights == cache.weights.data_ptr()
    assert other._struct.k_codes == cache._struct.k_codes and other.shape == cache.shape
    assert other != cache and len({other, cache}) == 2

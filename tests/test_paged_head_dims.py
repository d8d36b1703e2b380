"""Paged caches of head dims that no kernel has are refused, whatever their pages hold."""
import pytest

from opendecider_amd import PagedKVCache, PagedStates


@pytest.mark.parametrize("quantized", [True, False, "int8", "int4"])
def test_head_dims(quantized):
    for d in (64, 128, 256):
        assert PagedKVCache(2, 1, d, 16, "cpu", quantized=quantized).head_dim == d
    for d in (0, 1, 32, 63, 65, 127, 129, 192, 255, 257, 512):
        with pytest.raises(ValueError, match="head_dim"):
            PagedKVCache(2, 1, d, 16, "cpu", quantized=quantized)
        with pytest.raises(ValueError, match="head_dim"):
            PagedStates(1, 1, 1, d, 2, 32, 16, "cpu", quantized)

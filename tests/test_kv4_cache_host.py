"""Shapes that the 4-bit cache refuses, beyond those of test_kv4_host.py: no GPU needed."""

from __future__ import annotations

import pytest

from qtts_b200 import kv4


def test_a_cache_without_heads_is_refused():
    with pytest.raises(ValueError, match="kv_heads"):
        kv4.Kv4Cache.empty(2, 0, 16, 64, device="cpu")


def test_a_cache_without_pages_is_one():
    cache = kv4.Kv4Cache.empty(0, 2, 16, 64, device="cpu")
    assert cache.pages == 0 and cache.nbytes == 0

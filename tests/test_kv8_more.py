"""The 8-bit cache's cross, shared-prefix and weighing attention and its eviction without a
GPU: what the calls refuse before they look at a device."""
from __future__ import annotations

import ctypes

import pytest


def test_null_handles_are_refused(dsd):
    lib = dsd.load_library()
    batch, prefix = dsd.Kv8Batch(1), dsd.Kv8Prefix(1)
    size = ctypes.c_size_t()
    assert lib.dsd_kv8_attend_cross(None, batch.pointer, 0, 1, None, 0, None, 0, 0.0, None, 0, None,
                                    None) == 1
    assert lib.dsd_kv8_attend_shared(None, batch.pointer, prefix.pointer, 0, 1, None, 0, None, 0, 0.0,
                                     None, 0, None, None) == 1
    assert lib.dsd_kv8_attend_weigh(None, batch.pointer, 0, 1, None, 0, None, 0, 0.0, None, None, 0,
                                    None, None) == 1
    assert lib.dsd_kv8_evict(None, batch.pointer, 1, 0, 0, None, None, 1, None, None, None, 0, None,
                             None) == 1
    for call in (lib.dsd_kv8_weigh_workspace_bytes, lib.dsd_kv8_evict_workspace_bytes):
        assert call(None, batch.pointer, 1, ctypes.byref(size)) == 1
        assert b"non-null" in lib.dsd_last_error()
    assert lib.dsd_kv8_shared_workspace_bytes(None, batch.pointer, prefix.pointer, 1,
                                              ctypes.byref(size)) == 1


@pytest.mark.parametrize("bad,what", [
    (dict(groups=-1), "non-negative"), (dict(max_requests=-1), "non-negative"),
    (dict(max_pages=-1), "non-negative"), (dict(total_pages=-1), "non-negative"),
    (dict(groups=65536), "65535"),
])
def test_prefix_is_checked_first(dsd, bad, what):
    lib = dsd.load_library()
    prefix = dsd.Kv8Prefix(**{**dict(groups=1), **bad})
    assert lib.dsd_kv8_attend_shared(None, dsd.Kv8Batch(1).pointer, prefix.pointer, 0, 1, None, 0, None,
                                     0, 0.0, None, 0, None, None) == 1
    assert what in lib.dsd_last_error().decode()
    assert lib.dsd_kv8_attend_shared(None, dsd.Kv8Batch(1).pointer, None, 0, 1, None, 0, None, 0, 0.0,
                                     None, 0, None, None) == 1
    assert "prefix" in lib.dsd_last_error().decode()

"""Sizes at the edge of the paged operators' 32-bit counts are refused before a device is touched (no GPU here)."""

import ctypes
import importlib

import pytest

FAKE = 1 << 20  # never dereferenced


def _kv(mod, **kw):
    f = dict(k=FAKE, v=FAKE, block_table=FAKE, table_stride=4, page_stride=1024 * 128 * 2, head_stride=1024 * 128,
             slot_stride=128, dtype=1, pages=8, page_size=1024, kv_heads=2, head_dim=128, table_width=4)
    return mod.PagedKV(*[{**f, **kw}[n] for n, _ in mod.PagedKV._fields_])


@pytest.mark.parametrize("pages,length", [
    (1 << 20, (1 << 30) + 1), (1 << 21, 1 << 31), (1 << 22, (1 << 32) + 5), (1 << 62, 1 << 33), (1, 1025)])
def test_a_prefix_beyond_its_counts_is_refused(b200, pages, length):
    """(A length of 2^31 or more would wrap into a negative 32-bit one, which says that the lengths are on the device.)"""
    mod = importlib.import_module(b200.__name__ + "._lib")
    lib, kv = mod.load(), _kv(mod)
    assert lib.qi4_shared_prefix_attention(ctypes.byref(kv), FAKE, 1536, 128, FAKE, 4, 4, 12, FAKE, pages, length, None,
                                           FAKE, 1, 0.1, None, 0, None) == -3
    assert "prefix" in mod.last_error()


@pytest.mark.parametrize("change", [dict(page_stride=0), dict(head_stride=0)])
def test_pages_and_heads_that_share_their_memory_are_refused(b200, change):
    mod = importlib.import_module(b200.__name__ + "._lib")
    lib, kv = mod.load(), _kv(mod, **change)
    assert lib.qi4_paged_attention(ctypes.byref(kv), FAKE, 1536, 128, FAKE, 4, 4, 12, None, FAKE, 1, 0.1, 1, None, 0,
                                   None) == -4
    assert lib.qi4_rope_paged_append(ctypes.byref(kv), FAKE, 1536, 128, FAKE, 256, 128, FAKE, 256, 128, FAKE, 1536, 128,
                                     4, 4, 12, None, FAKE, None, FAKE, FAKE, 64, 128, 0, None) == -4


@pytest.mark.parametrize("token_stride,head_stride", [(0, 128), (1536, 0)])
def test_rotated_queries_that_share_their_memory_are_refused(b200, token_stride, head_stride):
    mod = importlib.import_module(b200.__name__ + "._lib")
    lib, kv = mod.load(), _kv(mod)
    assert lib.qi4_rope_paged_append(ctypes.byref(kv), FAKE, 1536, 128, FAKE, 256, 128, FAKE, 256, 128, FAKE,
                                     token_stride, head_stride, 4, 4, 12, None, FAKE, None, FAKE, FAKE, 64, 128, 0,
                                     None) == -4

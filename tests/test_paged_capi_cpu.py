"""Paged-cache operators at the C ABI: arguments are refused before a device is touched (no GPU here)."""

import ctypes
import importlib

import pytest
import torch

FAKE = 1 << 20  # never dereferenced


def _mod(b200):
    return importlib.import_module(b200.__name__ + "._lib")


def _kv(mod, **kw):
    f = dict(k=FAKE, v=FAKE, block_table=FAKE, table_stride=4, page_stride=16 * 128 * 2, head_stride=16 * 128,
             slot_stride=128, dtype=1, pages=8, page_size=16, kv_heads=2, head_dim=128, table_width=4)
    return mod.PagedKV(*[{**f, **kw}[n] for n, _ in mod.PagedKV._fields_])


@pytest.mark.parametrize("change,code", [
    (dict(k=None), -1), (dict(block_table=None), -1), (dict(dtype=2), -2), (dict(pages=0), -1),
    (dict(page_size=12), -3), (dict(page_size=4), -3), (dict(page_size=2048), -3), (dict(k=FAKE + 8), -4),
    (dict(page_stride=100), -4), (dict(slot_stride=64), -4), (dict(table_width=0), -1),
    (dict(table_width=1 << 30), -3)])
def test_cache_descriptor_is_checked(b200, change, code):
    mod = _mod(b200)
    lib, kv = mod.load(), _kv(mod, **change)
    assert lib.qi4_paged_attention(ctypes.byref(kv), FAKE, 1536, 128, FAKE, 4, 4, 12, None, FAKE, 1, 0.1, 1, None, 0,
                                   None) == code
    assert lib.qi4_rope_paged_append(ctypes.byref(kv), FAKE, 1536, 128, FAKE, 256, 128, FAKE, 256, 128, FAKE, 1536, 128,
                                     4, 4, 12, None, FAKE, None, FAKE, FAKE, 64, 128, 0, None) == code
    assert mod.last_error()


@pytest.mark.parametrize("change,code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(lengths=None), -1), (dict(T=5), -3), (dict(T=-1), -1),
    (dict(B=0), -1), (dict(Hq=13), -3), (dict(q=FAKE + 2), -4), (dict(q_tok=7), -4), (dict(most=-1), -1),
    (dict(T=1 << 29, cu=FAKE), -3)])
def test_attention_arguments_are_checked(b200, change, code):
    mod = _mod(b200)
    lib, kv = mod.load(), _kv(mod)
    a = {**dict(q=FAKE, q_tok=1536, out=FAKE, T=4, B=4, Hq=12, cu=None, lengths=FAKE, most=1), **change}
    assert lib.qi4_paged_attention(ctypes.byref(kv), a["q"], a["q_tok"], 128, a["out"], a["T"], a["B"], a["Hq"], a["cu"],
                                   a["lengths"], a["most"], 0.1, 1, None, 0, None) == code


def test_prefix_and_head_dim_are_checked(b200):
    mod = _mod(b200)
    lib = mod.load()

    def call(kv, table, pages, length):
        return lib.qi4_shared_prefix_attention(ctypes.byref(kv), FAKE, 1536, 128, FAKE, 4, 4, 12, table, pages, length,
                                               None, FAKE, 1, 0.1, None, 0, None)

    assert call(_kv(mod), None, 2, 5) == -1
    assert call(_kv(mod), FAKE, 2, -5) == -1
    assert call(_kv(mod), FAKE, 2, 33) == -3
    assert call(_kv(mod, head_dim=96, slot_stride=96), FAKE, 2, 5) == -3
    none = _kv(mod)
    assert lib.qi4_paged_attention(ctypes.byref(none), None, 0, 0, None, 0, 4, 12, None, None, 0, 0.1, 1, None, 0,
                                   None) == 0  # no tokens, nothing to do


@pytest.mark.parametrize("change,code", [
    (dict(k=None), -1), (dict(lengths=None), -1), (dict(T=6), -3), (dict(rot=24), -3), (dict(rot=144), -3),
    (dict(cos=None), -1), (dict(rows=0), -1), (dict(stride=100), -4), (dict(cos=FAKE + 4), -4), (dict(q=None), -1)])
def test_append_arguments_are_checked(b200, change, code):
    mod = _mod(b200)
    lib, kv = mod.load(), _kv(mod)
    a = {**dict(q=FAKE, k=FAKE, T=4, lengths=FAKE, cos=FAKE, rows=64, rot=128, stride=256), **change}
    assert lib.qi4_rope_paged_append(ctypes.byref(kv), a["q"], 1536, 128, a["k"], a["stride"], 128, FAKE, 256, 128, FAKE,
                                     1536, 128, a["T"], 4, 12, None, a["lengths"], None, a["cos"], FAKE, a["rows"],
                                     a["rot"], 0, None) == code


@pytest.mark.parametrize("change,code", [
    (dict(target=None), -1), (dict(tokens=None), -1), (dict(dtype=5), -2), (dict(B=0), -3), (dict(K=-1), -3),
    (dict(V=0), -3), (dict(V=1 << 23), -3), (dict(stride=-1), -1)])
def test_verify_arguments_are_checked(b200, change, code):
    mod = _mod(b200)
    a = {**dict(tokens=FAKE, target=FAKE, dtype=2, B=2, K=3, V=100, stride=100), **change}
    assert mod.load().qi4_verify_draft(a["tokens"], a["target"], 400, a["stride"], FAKE, 300, 100, a["dtype"], FAKE, None,
                                       a["B"], a["K"], a["V"], FAKE, FAKE, None) == code


def test_rope_table_follows_the_formula(b200):
    cos, sin = b200.rope_table(50, 32, base=1e6, scaling=4.0, attention_scaling=1.25)
    assert cos.shape == sin.shape == (50, 16) and cos.dtype == torch.float32
    for p, m in ((0, 0), (7, 3), (49, 15)):
        angle = torch.tensor(p / 4.0 * 1e6 ** (-2 * m / 32), dtype=torch.float64)
        assert abs(float(cos[p, m]) - 1.25 * float(angle.cos())) < 1e-6
        assert abs(float(sin[p, m]) - 1.25 * float(angle.sin())) < 1e-6
    for bad in ((0, 32), (5, 24)):
        with pytest.raises(ValueError):
            b200.rope_table(*bad)


def test_operators_need_a_gpu(b200):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(RuntimeError, match="CUDA device"):
        b200.b200_verify_draft(torch.zeros(1, 1, dtype=torch.int64), torch.ones(1, 2, 4), torch.zeros(1, 2))


@pytest.mark.parametrize("token_stride,head_stride", [(0, 128), (1536, 0), (-1536, 128), (1540, 128)])
def test_attention_refuses_strides_it_cannot_read(b200, token_stride, head_stride):
    mod = _mod(b200)
    kv = _kv(mod)
    assert mod.load().qi4_paged_attention(ctypes.byref(kv), FAKE, token_stride, head_stride, FAKE, 4, 4, 12, None, FAKE,
                                          0, 0.1, 1, None, 0, None) == -4

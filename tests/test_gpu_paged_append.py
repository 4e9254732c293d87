"""b200_rope_paged_append on a GPU, against the rotation in 64 bits.

Rotated values: FP32 products and one sum, |error| <= 3 * 2^-24 (|a| + |b|),
then one rounding to the type. Values, dimensions past the rotary part and
every slot that no new token owns are equal bit for bit.
"""

import importlib

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu


def _setup(dev, news, olds, *, Hq, Hkv, D, page, dtype, rot, seed=0, slots_first=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    B, T = len(news), sum(news)
    width = max(-(-(n + o) // page) for n, o in zip(news, olds)) + 1
    pages = B * width + 2
    table = torch.randperm(pages, generator=g, device=dev)[:B * width].view(B, width).int()
    shape = (pages, page, Hkv, D) if slots_first else (pages, Hkv, page, D)
    kc, vc = (torch.randn(shape, generator=g, device=dev).to(dtype) for _ in range(2))
    if slots_first:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device=dev).to(dtype)
    cu = torch.tensor([0] + [sum(news[:i + 1]) for i in range(B)], dtype=torch.int32, device=dev)
    lengths = torch.tensor(olds, dtype=torch.int32, device=dev)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], kc, vc, table, cu, lengths


def _places(news, olds, table, page):
    at = torch.cat([torch.arange(o, o + n) for n, o in zip(news, olds)]).to(table.device)
    b = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).to(table.device)
    return at, table.long()[b, at // page], at % page


def _near(got, want, x, dtype):
    slack = pg.ROUND[dtype] * want.abs() + 3 * 2.0 ** -23 * x + 1e-7 * (dtype == torch.float16)
    assert bool(((got.double() - want).abs() <= slack).all())


CASES = [
    # news, olds, Hq, Hkv, D, page, rot, interleaved, slots first
    ([1], [0], 12, 2, 128, 16, 128, False, False),
    ([1] * 5, [0, 15, 16, 31, 700], 12, 2, 128, 16, 128, False, False),
    ([7, 0, 33, 1], [5, 9, 0, 64], 8, 8, 64, 32, 64, True, True),
    ([130, 3], [0, 1000], 16, 4, 128, 8, 64, True, False),
    ([65], [77], 4, 1, 80, 64, 32, False, False),
    ([3, 2], [1, 0], 6, 3, 256, 128, 256, True, True),
    ([5, 6], [3, 4], 2, 2, 96, 16, 16, False, False),
    ([1] * 300, list(range(300)), 2, 1, 64, 16, 64, False, False),
    ([2500, 1700], [10, 0], 12, 2, 128, 16, 128, False, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news,olds,Hq,Hkv,D,page,rot,inter,slots", CASES)
def test_append_rotates_and_places(b200, cuda_device, dtype, news, olds, Hq, Hkv, D, page, rot, inter, slots):
    q, k, v, kc, vc, table, cu, lengths = _setup(cuda_device, news, olds, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype,
                                                 rot=rot, slots_first=slots)
    cos, sin = b200.rope_table(max(n + o for n, o in zip(news, olds)), rot, base=1e4, device=cuda_device)
    at, pages, slot = _places(news, olds, table, page)
    k0, v0 = kc.clone(), vc.clone()
    out = b200.b200_rope_paged_append(q, k, v, kc, vc, table, lengths, cos, sin, cu_tokens=cu, interleaved=inter)
    h = rot // 2
    for x, got in ((q, out), (k, kc[pages, :, slot])):
        want = pg.rotate64(x, cos[at], sin[at], inter)
        size = x.double().abs()
        i, j = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, h), slice(h, rot))
        both = size[..., i] + size[..., j]
        size[..., i], size[..., j] = both, both
        _near(got, want, size, dtype)
        assert torch.equal(got[..., rot:], x[..., rot:])
    assert torch.equal(vc[pages, :, slot], v)
    k0[pages, :, slot], v0[pages, :, slot] = kc[pages, :, slot], v
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # nothing else was written
    lib = importlib.import_module(b200.__name__ + "._lib").load()
    assert lib.qi4_device_status(torch.cuda.current_stream().cuda_stream) == 0


def test_append_forms(b200, cuda_device):
    """Equal counts need no cu_tokens; positions choose the rotary row; q_out may be q; without a table nothing turns;
    the rotation is the dense decode path's (half layout)."""
    news, olds = [3] * 4, [9, 0, 40, 2]
    q, k, v, kc, vc, table, cu, lengths = _setup(cuda_device, news, olds, Hq=4, Hkv=2, D=128, page=16,
                                                 dtype=torch.bfloat16, rot=128)
    cos, sin = b200.rope_table(64, 128, device=cuda_device)
    at, pages, slot = _places(news, olds, table, 16)
    caches = [(kc.clone(), vc.clone()) for _ in range(4)]
    one = b200.b200_rope_paged_append(q, k, v, *caches[0], table, lengths, cos, sin, cu_tokens=cu)
    two = b200.b200_rope_paged_append(q, k, v, *caches[1], table, lengths, cos, sin, positions=at.int())
    assert torch.equal(one, two) and all(torch.equal(a, b) for a, b in zip(caches[0], caches[1]))
    shifted = (63 - at).int()
    three = b200.b200_rope_paged_append(q, k, v, *caches[2], table, lengths, cos, sin, positions=shifted)
    _near(three, pg.rotate64(q, cos[shifted.long()], sin[shifted.long()], False), 4 * q.double().abs().amax(), q.dtype)
    plain = b200.b200_rope_paged_append(q, k, v, *caches[3], table, lengths)
    assert torch.equal(plain, q) and torch.equal(caches[3][0][pages, :, slot], k)
    own = q.clone()
    back = b200.b200_rope_paged_append(own, k, v, kc, vc, table, lengths, cos, sin, q_out=own)
    assert back.data_ptr() == own.data_ptr() and torch.equal(own, one)
    # A last dimension with gaps and an unaligned start are copied.
    gaps = torch.empty(*q.shape[:2], 256, dtype=q.dtype, device=q.device)[..., ::2]
    gaps.copy_(q)
    odd = torch.empty(k.numel() + 1, dtype=k.dtype, device=k.device)[1:].view(k.shape).copy_(k)
    assert torch.equal(b200.b200_rope_paged_append(gaps, odd, v, kc, vc, table, lengths, cos, sin), one)
    assert torch.equal(kc, caches[0][0])


def test_append_reports_what_it_cannot_place(b200, cuda_device):
    """No page, a page outside the pool, a position beyond the table of angles: nothing is written, the status says so."""
    q, k, v, kc, vc, table, cu, lengths = _setup(cuda_device, [2, 1, 1], [0, 3, 5], Hq=2, Hkv=1, D=64, page=8,
                                                 dtype=torch.bfloat16, rot=64)
    lib = importlib.import_module(b200.__name__ + "._lib").load()
    status = lambda: lib.qi4_device_status(torch.cuda.current_stream().cuda_stream)  # noqa: E731
    cos, sin = b200.rope_table(64, 64, device=cuda_device)
    k0, v0 = kc.clone(), vc.clone()
    far = torch.full_like(lengths, 10 ** 9)
    b200.b200_rope_paged_append(q, k, v, kc, vc, table, far, cos, sin, cu_tokens=cu)
    assert status() == 2 | 8 and torch.equal(kc, k0) and torch.equal(vc, v0)
    for bad in (-1, kc.shape[0], 2 ** 31 - 1):
        b200.b200_rope_paged_append(q, k, v, kc, vc, torch.full_like(table, bad), lengths, cos, sin, cu_tokens=cu)
        assert status() == 4 and torch.equal(kc, k0) and torch.equal(vc, v0)
    b200.b200_rope_paged_append(q, k, v, kc, vc, table, torch.full_like(lengths, -5), cos, sin, cu_tokens=cu)
    assert status() == 2 | 8 and torch.equal(kc, k0)
    b200.b200_rope_paged_append(q, k, v, kc, vc, table, lengths, cos[:4], sin[:4], cu_tokens=cu)
    assert status() == 8
    # Boundaries that leave the tokens are clipped to them.
    wild = torch.tensor([0, 10 ** 6, -3, 10 ** 6], dtype=torch.int32, device=cuda_device)
    b200.b200_rope_paged_append(q, k, v, kc, vc, table, lengths, cos, sin, cu_tokens=wild)
    assert status() & ~(2 | 8) == 0
    none = b200.b200_rope_paged_append(q[:0], k[:0], v[:0], kc, vc, table, lengths, cos, sin)
    assert none.shape == (0, 2, 64) and status() == 0


def test_append_refuses(b200, cuda_device):
    q, k, v, kc, vc, table, cu, lengths = _setup(cuda_device, [2, 2], [0, 3], Hq=4, Hkv=2, D=64, page=8,
                                                 dtype=torch.bfloat16, rot=64)
    cos, sin = b200.rope_table(16, 64, device=cuda_device)
    good = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, block_table=table, lengths=lengths, cos=cos, sin=sin)

    def call(**kw):
        return b200.b200_rope_paged_append(**{**good, **kw})

    call()
    for error, kw in [
        (TypeError, dict(q=q.float())), (TypeError, dict(lengths=lengths.long())), (TypeError, dict(cos=cos.half())),
        (TypeError, dict(k_cache=kc.float(), v_cache=vc.float())), (TypeError, dict(v=v.half())),
        (ValueError, dict(k=k[:, :1])), (ValueError, dict(q=q[:3])), (ValueError, dict(lengths=lengths[:1])),
        (ValueError, dict(cos=None)), (ValueError, dict(cos=cos[:, :4], sin=sin[:, :4])),
        (ValueError, dict(cu_tokens=cu[:2])), (ValueError, dict(positions=lengths)),
        (ValueError, dict(block_table=table[0])), (ValueError, dict(k_cache=kc[:, :, :6], v_cache=vc[:, :, :6])),
        (ValueError, dict(k_cache=kc.cpu())), (ValueError, dict(lengths=lengths.cpu())),
        (ValueError, dict(v_cache=vc.transpose(1, 2).contiguous().transpose(1, 2))),
        (ValueError, dict(q=q[:3], k=k[:3], v=v[:3])),  # 3 tokens for 2 sequences, without cu_tokens
        (ValueError, dict(q_out=torch.empty_like(q)[:, :3])),
    ]:
        with pytest.raises(error):
            call(**kw)

"""Paged attention where the tiles of few rows must do for many: more query heads per KV head than a tensor-core tile
has rows for, and scales below zero."""

import math

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
SEQS = [(1, 700), (3, 40), (0, 5), (2, 0), (50, 300), (1, 1), (9, 4)]
CASES = [
    # sequences, query heads, KV heads, dims, type, scale, prefix
    (SEQS, 144, 1, 128, BF16, None, 0),
    (SEQS, 260, 2, 64, F16, None, 0),
    ([(1, 3000)], 200, 1, 128, F16, None, 0),
    ([(1, 30 + 5 * i) for i in range(40)], 129, 1, 64, BF16, None, 0),
    ([(2, 90), (1, 300), (0, 0)], 144, 1, 128, BF16, None, 500),
    (SEQS, 12, 2, 128, BF16, -0.1, 0),
    (SEQS, 40, 1, 128, F16, -0.05, 0),
    (SEQS, 8, 8, 64, BF16, -0.125, 0),
    ([(4, 700), (90, 1500)], 16, 2, 128, F16, -0.1, 0),
    ([(5, 700), (4, 30)], 12, 2, 128, BF16, -0.1, 0),  # one tile of 30 rows each, in clusters
    ([(5, 700)] * 90, 12, 2, 128, F16, -0.1, 0),
    ([(4, 90), (2, 300), (9, 40)], 12, 2, 128, BF16, -0.1, 600),
]


def _run(b200, x, scale):
    how = dict(cu_tokens=x["cu"], max_tokens=x["most"], scale=scale)
    if x["prefix"]:
        return b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], x["prefix_table"], x["prefix"], x["table"],
                                                 x["lengths"], **how)
    return b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], **how)


@pytest.mark.parametrize("seqs,Hq,Hkv,D,dtype,scale,prefix", CASES)
def test_many_heads_and_negative_scales(b200, cuda_device, seqs, Hq, Hkv, D, dtype, scale, prefix):
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=16, dtype=dtype, device=cuda_device, prefix=prefix)
    for table in (x["table"], torch.nn.functional.pad(x["table"], (0, 300), value=-1)):
        y = dict(x, table=table)
        out = _run(b200, y, scale)
        pg.check_attention(out, y, scale=scale)
        assert torch.equal(out, _run(b200, y, scale))


@pytest.mark.parametrize("seqs,Hq,Hkv,D,dtype,scale,prefix", CASES)
def test_values_that_are_nan_reach_the_tokens_that_see_them(b200, cuda_device, seqs, Hq, Hkv, D, dtype, scale, prefix):
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=16, dtype=dtype, device=cuda_device, prefix=prefix)
    v = x["v"].clone()
    used = torch.zeros(*x["q"].shape[:2], D, dtype=torch.bool, device=cuda_device)
    for b, (n, length) in enumerate(seqs):
        i = n // 2
        p = length - n + i
        if n > 1 and p >= 0:
            v[int(x["table"][b, p // 16]), 0, p % 16, 5] = math.nan
            used[int(x["cu"][b]) + i:int(x["cu"][b + 1]), :Hq // Hkv, 5] = True
    got = _run(b200, dict(x, v=v), scale)
    assert bool(got[used].isnan().all())
    ref, _ = pg.attention64(x, scale=scale)
    pg.check_attention(torch.where(used, ref.to(got.dtype), got), x, scale=scale)

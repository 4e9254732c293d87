"""Paged attention where one key takes nearly all and the output is the others': small weights must keep their bits.

The scores are exact: `gap` for the first key, whose value is zero, and 0 for all others, whose values are 1024 (in the
first 16 keys of every 128 alone, where the kernel for few rows takes each group of 16 relative to its own maximum).
"""

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _batch(device, seqs, gap, *, D, dtype, prefix=0, groups=True, Hq=12, Hkv=2):
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=16, dtype=dtype, device=device, prefix=prefix, wide=0)
    x["q"].zero_()
    x["q"][..., 0] = 1
    x["k"].masked_fill_(~x["k"].isnan(), 0)
    x["v"].masked_fill_(~x["v"].isnan(), 0)
    first = [x["prefix_table"]] if prefix else x["table"]
    for row in first:
        x["k"][int(row[0]), :, 0, 0] = gap
    for row in [*x["table"], x["prefix_table"]]:
        for j, page in enumerate(row.tolist()):
            if page >= 0 and (j % 8 == 0 or not groups):
                at = x["v"][page]
                at.masked_fill_(~at.isnan(), 1024)
    for row in first:
        x["v"][int(row[0]), :, 0] = 0
    return x


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gap", [4, 14, 16, 20])
@pytest.mark.parametrize("seqs,prefix,D,groups", [
    ([(1, 480)] * 80, 0, 128, True),     # one CTA per item
    ([(1, 300), (4, 500)], 0, 64, True),  # clusters
    ([(4, 6000)] * 20, 0, 64, True),      # dealt to all SMs
    ([(300, 300)], 0, 128, False),        # tensor cores
    ([(200, 500), (90, 400)], 0, 64, False),
    ([(1, 20)] * 40, 400, 128, False),    # a prefix
])
def test_small_weights_count(b200, cuda_device, seqs, prefix, D, groups, gap, dtype):
    x = _batch(cuda_device, seqs, gap, D=D, dtype=dtype, prefix=prefix, groups=groups)
    how = dict(cu_tokens=x["cu"], max_tokens=x["most"], scale=1.0)
    if prefix:
        got = b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], x["prefix_table"], prefix, x["table"],
                                                x["lengths"], **how)
    else:
        got = b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], **how)
    ref, size = pg.attention64(x, scale=1.0)
    # The result's rounding, the weights' (u at most) and that of the FP32 sums. FP16 weights stand relative to at
    # least 2^7 for the largest one and are whole multiples of 2^-24, so that each is off by up to 2^-32 of it besides.
    u = pg.ROUND[dtype]
    bound = u * ref.abs() + (u + 2.0 ** -13) * size
    if dtype == F16:
        bound += 2.0 ** -32 * 1024 * (prefix + max(n for _, n in seqs))
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"worst {(err / bound.clamp_min(1e-30)).max():.3f} of the bound"
    assert bool((ref > 0).any())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("seqs,prefix,D,Hq,Hkv", [
    ([(1, 480)] * 80, 0, 128, 12, 2),
    ([(1, 300), (4, 700)], 0, 128, 12, 2),
    ([(1, 1151)] * 64, 0, 128, 12, 2),
    ([(5, 3000 + 100 * i) for i in range(12)], 0, 64, 16, 4),
    ([(1, 9000)], 0, 128, 12, 2),
    ([(1, 40), (2, 90)], 900, 128, 12, 2),
])
def test_few_rows_keep_more_of_a_weight_than_the_type_has(b200, cuda_device, seqs, prefix, D, Hq, Hkv, dtype):
    """Few rows per key: a weight is a value and its remainder, 2^-16 of it lost at most, which is within the 2^-13 of
    FP32 scores and sums (_paged.check_attention); only the result is rounded to the type."""
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=16, dtype=dtype, device=cuda_device, prefix=prefix)
    how = dict(cu_tokens=x["cu"], max_tokens=x["most"])
    if prefix:
        got = b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], x["prefix_table"], prefix, x["table"],
                                                x["lengths"], **how)
    else:
        got = b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], **how)
    ref, size = pg.attention64(x)
    bound = pg.ROUND[dtype] * ref.abs() + (2.0 ** -16 + 2.0 ** -13) * size
    if dtype == F16:
        bound += 2.0 ** -24  # (results below FP16's normal numbers)
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"worst {(err / bound).max():.3f} of the bound"

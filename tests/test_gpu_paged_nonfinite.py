"""Queries, keys and values that are not finite: they reach the tokens that use them, all of those and no other."""

import math

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16

# Every way the work is done: a cluster per item, items dealt to all SMs, items of one CTA each, tensor cores split
# and whole, a shared prefix before either. (sequences, prefix, pages the table is widened by, Hq, Hkv, D, dtype)
WAYS = [
    ([(4, 641), (1, 300)], 0, 0, 12, 2, 128, BF16),
    ([(5, 2000), (3, 129), (4, 3900)], 0, 0, 16, 4, 64, F16),
    ([(1, 900 + 7 * i) for i in range(70)], 0, 600, 12, 2, 128, F16),
    ([(4, 700 + 9 * i) for i in range(20)], 0, 600, 12, 2, 128, BF16),
    ([(3, 100 + 5 * i) for i in range(80)], 0, 0, 8, 2, 64, BF16),
    ([(1, 40000)], 0, 0, 12, 2, 128, BF16),
    ([(300, 1500), (90, 90)], 0, 600, 12, 2, 128, BF16),
    ([(100, 400), (60, 61)], 0, 0, 8, 8, 64, F16),
    ([(4, 90), (2, 700)], 500, 0, 12, 2, 128, BF16),
    ([(3, 30 + i) for i in range(40)], 3000, 0, 16, 4, 64, F16),
]


def _build(device, way):
    seqs, prefix, wide, Hq, Hkv, D, dtype = way
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=16, dtype=dtype, device=device, prefix=prefix, wide=0)
    if wide:
        table = torch.full((len(seqs), x["table"].shape[1] + wide), -1, dtype=torch.int32, device=device)
        table[:, :x["table"].shape[1]] = x["table"]
        x["table"] = table
    return x


def _run(b200, x):
    if x["prefix"]:
        return b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], x["prefix_table"], x["prefix"], x["table"],
                                                 x["lengths"], cu_tokens=x["cu"], max_tokens=x["most"])
    return b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], cu_tokens=x["cu"],
                                     max_tokens=x["most"])


def _slot(x, b, p):
    """Page and slot of position p of sequence b."""
    return int(x["table"][b, p // x["page"]]), p % x["page"]


def _rows(x, b, first=0):
    """Mask [T] of sequence b's tokens from its `first` on."""
    at = torch.zeros(x["q"].shape[0], dtype=torch.bool, device=x["q"].device)
    at[int(x["cu"][b]) + first:int(x["cu"][b + 1])] = True
    return at


def _check_but(got, x, rows):
    """The bound of _paged.check_attention for all tokens but `rows` (whose elements are replaced by a right answer)."""
    ref, _ = pg.attention64(x)
    pg.check_attention(torch.where(rows[:, None, None], ref.to(got.dtype), got), x)


@pytest.mark.parametrize("way", WAYS)
def test_a_query_that_is_nan_makes_its_own_output_nan(b200, cuda_device, way):
    x = _build(cuda_device, way)
    q = x["q"].clone()
    rows = torch.zeros(q.shape[0], dtype=torch.bool, device=cuda_device)
    for t in {0, q.shape[0] // 2, q.shape[0] - 1}:
        q[t, 1, 7] = math.nan
        rows[t] = True
    got = _run(b200, dict(x, q=q))
    assert bool(got[rows, 1].isnan().all())
    got[rows, 1] = 0
    want = _run(b200, x)
    want[rows, 1] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("way", WAYS)
def test_a_key_that_is_nan_reaches_the_tokens_that_see_it(b200, cuda_device, way):
    x = _build(cuda_device, way)
    k = x["k"].clone()
    b = len(x["seqs"]) - 1
    n, length = x["seqs"][b]
    page, slot = _slot(x, b, length - n + n // 2)  # the middle one of the new tokens
    k[page, 0, slot, 3] = math.nan
    got = _run(b200, dict(x, k=k))
    rows = _rows(x, b, n // 2)
    G = got.shape[1] // x["Hkv"]
    assert bool(got[rows, :G].isnan().all())
    assert bool(torch.isfinite(got[rows, G:]).all())
    _check_but(got, x, rows)


@pytest.mark.parametrize("way", WAYS)
def test_keys_that_are_all_nan(b200, cuda_device, way):
    """No score of a sequence is a number: its outputs are NaN, not zeros."""
    x = _build(cuda_device, way)
    k = x["k"].clone()
    k[x["table"][0][x["table"][0] >= 0].long()] = math.nan
    got = _run(b200, dict(x, k=k))
    rows = _rows(x, 0)
    assert bool(got[rows].isnan().all())
    _check_but(got, x, rows)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("way", WAYS)
def test_a_value_reaches_no_token_that_does_not_see_its_key(b200, cuda_device, way, value):
    """Values of new tokens, hidden from the tokens before them though in the same tile: w V with no weight for V is
    not 0 x V. Those that see the key have the value's infinity, or NaN, in its dimension."""
    x = _build(cuda_device, way)
    v = x["v"].clone()
    T, D = x["q"].shape[0], x["D"]
    G = x["q"].shape[1] // x["Hkv"]
    used = torch.zeros(T, x["q"].shape[1], D, dtype=torch.bool, device=cuda_device)
    for b, (n, length) in enumerate(x["seqs"]):
        for j, (i, d) in enumerate(((n - 1, 0), (n // 2, D - 1), (n // 2, 17), (1, 40))):
            if 0 < i < n and length - n + i >= 0:
                page, slot = _slot(x, b, length - n + i)
                v[page, j % x["Hkv"], slot, d] = value
                used[_rows(x, b, i), (j % x["Hkv"]) * G:(j % x["Hkv"] + 1) * G, d] = True
    got = _run(b200, dict(x, v=v))
    assert bool((got[used].isnan() if math.isnan(value) else got[used] == value).all())
    assert bool(torch.isfinite(got[~used]).all())
    ref, _ = pg.attention64(x)
    pg.check_attention(torch.where(used, ref.to(got.dtype), got), x)

"""b200_paged_attention and b200_shared_prefix_attention on a GPU, against 64 bits (bounds: _paged.check_attention)."""

import importlib

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _run(b200, x, **kw):
    return b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], cu_tokens=x["cu"], **kw)


def _status(b200):
    lib = importlib.import_module(b200.__name__ + "._lib").load()
    return lib.qi4_device_status(torch.cuda.current_stream().cuda_stream)


ONE = [(1, n) for n in (1, 2, 15, 16, 17, 63, 64, 127, 128, 129, 255, 257, 1000)]
MIXED = [(1, 700), (0, 50), (5, 5), (2, 1), (3, 0), (130, 131), (1, 1), (64, 300), (0, 0), (17, 2000)]
CASES = [
    # sequences, Hq, Hkv, D, page, dtype, pool with slots first
    ([(1, 1)], 12, 2, 128, 16, BF16, False),
    (ONE, 12, 2, 128, 16, BF16, False),
    (ONE, 16, 4, 64, 32, F16, True),
    ([(5, n + 5) for n in (0, 3, 120, 124, 500)], 12, 2, 128, 8, BF16, True),
    ([(2, n + 2) for n in (0, 126, 700)], 8, 1, 128, 64, F16, False),
    (MIXED, 12, 2, 128, 16, BF16, False),
    (MIXED, 14, 2, 64, 128, BF16, True),
    (MIXED, 4, 4, 128, 256, F16, False),
    ([(300, 300)], 12, 2, 128, 16, BF16, False),
    ([(700, 1500), (1, 4000)], 8, 8, 64, 16, F16, False),
    ([(1, 40000)], 12, 2, 128, 64, BF16, False),
    ([(4, 9001), (4, 20)], 16, 4, 64, 16, BF16, False),
    ([(1, 1 + 7 * (i % 50)) for i in range(400)], 6, 1, 128, 16, BF16, False),
    ([(1, 513)] * 3, 40, 1, 128, 16, F16, False),
]


@pytest.mark.parametrize("hint", [True, False])
@pytest.mark.parametrize("seqs,Hq,Hkv,D,page,dtype,slots", CASES)
def test_attention_matches_64_bits(b200, cuda_device, seqs, Hq, Hkv, D, page, dtype, slots, hint):
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=cuda_device, slots_first=slots)
    out = _run(b200, x, max_tokens=x["most"] if hint else None)
    pg.check_attention(out, x)
    assert _status(b200) == 0
    again = _run(b200, x, max_tokens=x["most"] if hint else None)
    assert torch.equal(out, again)  # the order in which the pieces arrive does not matter


@pytest.mark.parametrize("seqs", [[(1, 700), (5, 40), (0, 3), (2, 0)], [(200, 1000), (1, 1)]])
def test_attention_without_causality_and_with_a_scale(b200, cuda_device, seqs):
    x = pg.build(seqs, Hq=12, Hkv=2, D=128, page=16, dtype=BF16, device=cuda_device)
    pg.check_attention(_run(b200, x, causal=False, scale=0.2), x, causal=False, scale=0.2)


def test_rows_that_see_nothing_are_zero(b200, cuda_device):
    x = pg.build([(4, 2), (3, 0), (1, 5), (200, 30)], Hq=4, Hkv=2, D=64, page=8, dtype=BF16, device=cuda_device)
    out = _run(b200, x)
    pg.check_attention(out, x)
    assert torch.count_nonzero(out[:2]) == 0 and torch.count_nonzero(out[4:7]) == 0
    assert torch.count_nonzero(out[8:8 + 170]) == 0 and bool((out[8 + 170:] != 0).any())


@pytest.mark.parametrize("tokens", [1, 6, 100])
def test_uniform_batch_needs_no_boundaries(b200, cuda_device, tokens):
    x = pg.build([(tokens, tokens + 37 * i) for i in range(5)], Hq=12, Hkv=2, D=128, page=16, dtype=BF16,
                 device=cuda_device)
    out = b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"])
    pg.check_attention(out, x)
    assert torch.equal(out, _run(b200, x, max_tokens=tokens))


@pytest.mark.parametrize("tokens", [1, 150])
def test_strided_queries_own_memory_and_streams(b200, cuda_device, tokens):
    """Queries inside a joint projection, a caller's output and workspace, a side stream, a captured graph."""
    x = pg.build([(tokens, tokens + 300), (tokens, tokens + 5)], Hq=8, Hkv=2, D=128, page=16, dtype=BF16,
                 device=cuda_device)
    want = _run(b200, x)
    joint = torch.randn(x["q"].shape[0], 12, 128, device=cuda_device).to(BF16)
    joint[:, :8] = x["q"]
    lib = importlib.import_module(b200.__name__ + "._lib").load()
    n = lib.qi4_paged_attention_workspace(x["q"].shape[0], 8, 2, 128, 0, 0)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=cuda_device)
    out = torch.empty_like(x["q"])
    args = dict(cu_tokens=x["cu"], out=out, workspace=ws)
    assert b200.b200_paged_attention(joint[:, :8], x["k"], x["v"], x["table"], x["lengths"], **args) is not None
    assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = b200.b200_paged_attention(joint[:, :8], x["k"], x["v"], x["table"], x["lengths"], cu_tokens=x["cu"])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b200.b200_paged_attention(joint[:, :8], x["k"], x["v"], x["table"], x["lengths"], **args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    for length in (x["lengths"] - 3, x["lengths"]):
        lengths = x["lengths"].clone()
        x["lengths"].copy_(length)  # the graph reads the lengths of the moment
        out.fill_(7)
        for _ in range(3):
            graph.replay()
        assert torch.equal(out, _run(b200, x))
        x["lengths"].copy_(lengths)
    with pytest.raises(ValueError):
        b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], cu_tokens=x["cu"],
                                  workspace=ws[:64])


def test_extreme_scores(b200, cuda_device):
    """Scores far apart (one key takes all), and far below zero (the running maximum starts there)."""
    for factor, sign in ((60.0, 1.0), (200.0, -1.0)):
        x = pg.build([(1, 300), (9, 520), (140, 200)], Hq=4, Hkv=1, D=64, page=16, dtype=F16, device=cuda_device,
                     scale=1.0)
        x["q"] = (x["q"].sign() * 0.5).to(F16)
        x["k"].copy_(torch.where(x["k"].isnan(), x["k"], (x["k"].sign() * sign).to(F16)))
        # Scores are whole multiples of scale: exact in FP32, so the bound needs no more room than elsewhere.
        out = _run(b200, x, scale=factor / 64)
        pg.check_attention(out, x, scale=factor / 64)


def test_offsets_beyond_32_bits(b200, cuda_device):
    """Pages whose elements lie beyond 2^31 of the pool's start."""
    page, Hkv, D = 64, 2, 128
    pages = 2 ** 31 // (page * Hkv * D) + 40
    kc = torch.zeros(pages, Hkv, page, D, dtype=BF16, device=cuda_device)
    vc = torch.zeros_like(kc)
    x = pg.build([(1, 500), (3, 130), (150, 150)], Hq=4, Hkv=Hkv, D=D, page=page, dtype=BF16, device=cuda_device)
    n = x["k"].shape[0]
    kc[-n:], vc[-n:] = x["k"], x["v"]
    far = torch.where(x["table"] >= 0, x["table"] + (pages - n), x["table"])
    out = b200.b200_paged_attention(x["q"], kc, vc, far, x["lengths"], cu_tokens=x["cu"])
    assert torch.equal(out, _run(b200, x))
    pg.check_attention(out, x)
    k, v = (torch.randn(4, Hkv, D, device=cuda_device).to(BF16) for _ in range(2))
    cu = torch.tensor([0, 4, 4, 4], dtype=torch.int32, device=cuda_device)
    b200.b200_rope_paged_append(k[:, :0], k, v, kc, vc, far, x["lengths"] - 4, cu_tokens=cu)
    p = far[0].long()
    at = torch.arange(496, 500, device=cuda_device)
    assert torch.equal(kc[p[at // page], :, at % page], k) and torch.equal(vc[p[at // page], :, at % page], v)


def test_lengths_and_pages_that_do_not_fit_are_reported(b200, cuda_device):
    x = pg.build([(1, 100), (1, 30)], Hq=4, Hkv=2, D=64, page=16, dtype=BF16, device=cuda_device, wide=0)
    far = b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"] + 10 ** 9)
    assert far.shape == x["q"].shape and _status(b200) & 2
    bad = x["table"].clone()
    bad[0, 0] = x["k"].shape[0] + 5
    b200.b200_paged_attention(x["q"], x["k"], x["v"], bad, x["lengths"])
    assert _status(b200) == 4
    none = b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], torch.full_like(x["lengths"], -7))
    assert torch.count_nonzero(none) == 0 and _status(b200) == 0
    wild = torch.tensor([-4, 10 ** 8, 10 ** 9], dtype=torch.int32, device=cuda_device)
    b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], cu_tokens=wild)
    y = pg.build([(9, 100), (12, 30)], Hq=4, Hkv=2, D=64, page=16, dtype=BF16, device=cuda_device)
    _run(b200, y, max_tokens=4)
    assert _status(b200) == 32
    empty = b200.b200_paged_attention(x["q"][:0], x["k"], x["v"], x["table"], x["lengths"])
    assert empty.shape == (0, 4, 64) and _status(b200) == 0


PREFIX = [
    # sequences (own keys), prefix, Hq, Hkv, D, page, dtype
    ([(1, n) for n in (1, 16, 17, 90)], 100, 12, 2, 128, 16, BF16),
    ([(1, 1)], 1, 12, 2, 128, 16, BF16),
    ([(1, n + 1) for n in range(64)], 3001, 12, 2, 128, 64, BF16),
    ([(4, n + 4) for n in (0, 5, 700)], 1024, 16, 4, 64, 32, F16),
    ([(1, 5), (0, 9), (3, 3), (2, 0), (70, 71)], 260, 8, 8, 128, 16, F16),
    ([(40, 45)] * 3, 777, 14, 2, 64, 16, BF16),
]


@pytest.mark.parametrize("seqs,prefix,Hq,Hkv,D,page,dtype", PREFIX)
def test_shared_prefix_matches_64_bits(b200, cuda_device, seqs, prefix, Hq, Hkv, D, page, dtype):
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=cuda_device, prefix=prefix)

    def run(**kw):
        return b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], x["prefix_table"], prefix, x["table"],
                                                 x["lengths"], cu_tokens=x["cu"], **kw)

    out = run(max_tokens=x["most"])
    pg.check_attention(out, x)
    assert torch.equal(out, run(max_tokens=x["most"])) and _status(b200) == 0
    pg.check_attention(run(), x)


def test_an_empty_prefix_is_none(b200, cuda_device):
    x = pg.build([(1, 70), (3, 40)], Hq=12, Hkv=2, D=128, page=16, dtype=BF16, device=cuda_device)
    pre = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], pre, 0, x["table"], x["lengths"],
                                            cu_tokens=x["cu"])
    assert torch.equal(out, _run(b200, x))


def test_attention_refuses(b200, cuda_device):
    x = pg.build([(2, 70), (2, 40)], Hq=12, Hkv=2, D=128, page=16, dtype=BF16, device=cuda_device)
    good = dict(q=x["q"], k_cache=x["k"], v_cache=x["v"], block_table=x["table"], lengths=x["lengths"])

    def call(**kw):
        return b200.b200_paged_attention(**{**good, **kw})

    call()
    for error, kw in [
        (TypeError, dict(q=x["q"].half())), (TypeError, dict(lengths=x["lengths"].long())),
        (TypeError, dict(block_table=x["table"].long())), (TypeError, dict(workspace=torch.empty(8, device=cuda_device))),
        (ValueError, dict(q=x["q"][:, :5])), (ValueError, dict(q=x["q"][..., :64])), (ValueError, dict(q=x["q"][:3])),
        (ValueError, dict(lengths=x["lengths"][:1])), (ValueError, dict(cu_tokens=x["cu"][1:])),
        (ValueError, dict(max_tokens=-1)), (ValueError, dict(out=torch.empty_like(x["q"][:1]))),
        (ValueError, dict(k_cache=x["k"][:, :, :12], v_cache=x["v"][:, :, :12])),
        (ValueError, dict(k_cache=x["k"][..., :96], v_cache=x["v"][..., :96], q=x["q"][..., :96])),
        (ValueError, dict(q=x["q"].cpu())), (ValueError, dict(k_cache=x["k"][1:])),
    ]:
        with pytest.raises(error):
            call(**kw)
    pre = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    for length, table, error in ((33, pre, ValueError), (-1, pre, ValueError), (5, pre.long(), TypeError),
                                 (5, pre[None], ValueError)):
        with pytest.raises(error):
            b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], table, length, x["table"], x["lengths"])


MANY = [(1, 1 + 7 * i) for i in range(70)]


@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("seqs,Hq,Hkv,D,dtype", [
    (MANY, 12, 2, 128, BF16),                                                    # one row tile each, many of them
    ([(n % 6, 500 - 9 * n) for n in range(40)], 16, 4, 64, F16),                 # some without tokens
    ([(3, 255)], 12, 2, 128, BF16),                                              # few
    ([(1, 0), (4, 2), (2, 250)], 8, 8, 64, BF16),                                # rows that see nothing
    ([(300, 512), (0, 40), (1, 77), (130, 130), (60, 0)], 12, 2, 128, F16),      # several row tiles
    ([(40 + i, 40 + 11 * i) for i in range(37)], 4, 1, 64, BF16),
])
def test_short_tables_and_wide_ones(b200, cuda_device, seqs, Hq, Hkv, D, dtype, prefix):
    """The width of the table decides whether the work on a sequence is split: both ways give the attention."""
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=8, dtype=dtype, device=cuda_device, prefix=prefix, wide=0)
    assert x["table"].shape[1] * 8 <= 512
    wide = torch.full((len(seqs), 400), -1, dtype=torch.int32, device=cuda_device)
    wide[:, :x["table"].shape[1]] = x["table"]
    for table in (x["table"], wide):
        y = dict(x, table=table)

        def run():
            if not prefix:
                return _run(b200, y, max_tokens=y["most"])
            return b200.b200_shared_prefix_attention(y["q"], y["k"], y["v"], y["prefix_table"], prefix, table,
                                                     y["lengths"], cu_tokens=y["cu"], max_tokens=y["most"])

        out = run()
        pg.check_attention(out, y)
        assert torch.equal(out, run())
    assert _status(b200) == 0


@pytest.mark.parametrize("tokens", [1, 3, 90])
def test_queries_in_other_orders(b200, cuda_device, tokens):
    """Heads major in memory, one row expanded to all tokens, one head expanded to all heads."""
    x = pg.build([(tokens, tokens + 200), (tokens, tokens + 31)], Hq=8, Hkv=2, D=128, page=16, dtype=BF16,
                 device=cuda_device)
    T, H, D = x["q"].shape
    major = torch.empty(H, T, D, dtype=BF16, device=cuda_device).transpose(0, 1)
    major.copy_(x["q"])
    for q in (major, x["q"][:1].expand(T, H, D), x["q"][:, 1:2].expand(T, H, D), x["q"][:1, :1].expand(T, H, D)):
        out = b200.b200_paged_attention(q, x["k"], x["v"], x["table"], x["lengths"], cu_tokens=x["cu"])
        assert torch.equal(out, _run(b200, dict(x, q=q.contiguous())))
    pg.check_attention(out, dict(x, q=q))


@pytest.mark.parametrize("prefix", [0, 700])
@pytest.mark.parametrize("seqs,Hq,Hkv,D,dtype", [
    ([(1, 641)], 12, 2, 128, BF16),
    ([(1, 1), (1, 0), (1, 3900), (0, 9), (1, 128)], 12, 2, 128, F16),  # one key, none, no tokens
    ([(5, 2000), (4, 2), (3, 129), (5, 4000)], 16, 4, 64, F16),       # rows that see nothing; 20 rows
    ([(4, 3000), (1, 257)], 8, 1, 128, BF16),                         # 32 rows
    ([(2, 1025)], 8, 8, 64, BF16),
    ([(1, 300 + 7 * i) for i in range(9)], 16, 2, 128, BF16),         # 18 items
])
def test_few_sequences_however_wide_the_table(b200, cuda_device, seqs, Hq, Hkv, D, dtype, prefix):
    """Tables that cover 4096 keys and more of them: an item as one cluster's work, and dealt to all SMs."""
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=16, dtype=dtype, device=cuda_device, prefix=prefix, wide=0)
    for pages in (x["table"].shape[1], 256, 257):
        table = torch.full((len(seqs), pages), -1, dtype=torch.int32, device=cuda_device)
        table[:, :x["table"].shape[1]] = x["table"]
        y = dict(x, table=table)

        def run():
            if not prefix:
                return _run(b200, y, max_tokens=y["most"])
            return b200.b200_shared_prefix_attention(y["q"], y["k"], y["v"], y["prefix_table"], prefix, table,
                                                     y["lengths"], cu_tokens=y["cu"], max_tokens=y["most"])

        out = run()
        pg.check_attention(out, y)
        assert torch.equal(out, run())
    assert _status(b200) == 0


@pytest.mark.parametrize("seqs,Hq,Hkv,D,page,pages,dtype", [
    ([(1, 1 + 130 * i) for i in range(15)], 12, 2, 128, 16, 128, BF16),
    ([(1 + i % 5, 1000 - 31 * i) for i in range(9)], 16, 4, 64, 8, 200, F16),
    ([(i % 4, 11 * i) for i in range(31)], 8, 2, 128, 32, 32, F16),
])
def test_sequences_that_share_the_gpu_in_small_clusters(b200, cuda_device, seqs, Hq, Hkv, D, page, pages, dtype):
    x = pg.build(seqs, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, device=cuda_device, wide=0)
    table = torch.full((len(seqs), pages), -1, dtype=torch.int32, device=cuda_device)
    table[:, :x["table"].shape[1]] = x["table"]
    y = dict(x, table=table)
    out = _run(b200, y, max_tokens=y["most"])
    pg.check_attention(out, y)
    assert torch.equal(out, _run(b200, y, max_tokens=y["most"]))
    assert _status(b200) == 0

"""A report of one call's inputs (a page outside the pool, a length beyond the table, more tokens than announced)
concerns what it names alone: the call's other sequences, and every later call while the report has not been read,
give the attention. The batches are long enough for the kernels' producers and consumers to wait for one another."""

import importlib

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
FULL, PAGE, MANY = 2, 4, 32


@pytest.fixture
def status(b200):
    lib = importlib.import_module(b200.__name__ + "._lib").load()

    def read():
        return lib.qi4_device_status(torch.cuda.current_stream().cuda_stream)

    assert read() == 0
    yield read
    read()  # the next test starts without reports


def _run(b200, x, **kw):
    if x["prefix"]:
        return b200.b200_shared_prefix_attention(x["q"], x["k"], x["v"], x["prefix_table"], x["prefix"], x["table"],
                                                 x["lengths"], cu_tokens=x["cu"], max_tokens=x["most"], **kw)
    return b200.b200_paged_attention(x["q"], x["k"], x["v"], x["table"], x["lengths"], cu_tokens=x["cu"],
                                     max_tokens=x["most"], **kw)


def _batch(device, seqs, prefix=0, seed=0, **kw):
    how = dict(Hq=12, Hkv=2, D=128, page=16, dtype=BF16, **kw)
    return pg.build(seqs, device=device, prefix=prefix, seed=seed, **how)


# Decode steps (one launch and its join), prompts on the tensor cores, both behind a prefix.
LONG = [([(1, 30000), (1, 9000), (1, 1)], 0), ([(1, 1151)] * 64, 0), ([(3, 5000)] * 8, 0),
        ([(1500, 4000), (0, 3), (700, 700)], 0), ([(1, 90 + i) for i in range(64)], 8000), ([(60, 700)] * 4, 3000),
        ([(1, 40)] * 2, 900)]


def _leave_reports(b200, device, status):
    """Every kind of report, from both kernels; none is read."""
    for tokens in (1, 40):  # mma.sync, tcgen05
        x = _batch(device, [(tokens, 700), (tokens, 300)])
        bad = x["table"].clone()
        bad[0, 3] = x["k"].shape[0] + 5
        _run(b200, dict(x, table=bad))
        _run(b200, dict(x, table=x["table"][:, :20].contiguous()))
    for tokens, announced in ((9, 4), (100, 42)):
        x = _batch(device, [(tokens, 200), (1, 30)])
        _run(b200, dict(x, most=announced))


def test_later_calls_do_not_notice(b200, cuda_device, status):
    batches = [_batch(cuda_device, seqs, prefix, seed=i) for i, (seqs, prefix) in enumerate(LONG)]
    clean = [_run(b200, x) for x in batches]
    assert status() == 0
    _leave_reports(b200, cuda_device, status)
    for _ in range(5):
        for x, want in zip(batches, clean):
            assert torch.equal(_run(b200, x), want)
    for x in batches:
        pg.check_attention(_run(b200, x), x)
    assert status() == FULL | PAGE | MANY


@pytest.mark.parametrize("tokens", [1, 4, 90])
@pytest.mark.parametrize("prefix", [0, 2000])
def test_a_page_outside_the_pool_reads_as_zeros_and_no_other_does(b200, cuda_device, status, tokens, prefix):
    x = _batch(cuda_device, [(tokens, 2000 + 300 * i) for i in range(12)], prefix)
    spare = sorted(set(range(x["k"].shape[0])) - set(x["table"].flatten().tolist()) - set(x["prefix_table"].tolist()))
    x["k"][spare[0]], x["v"][spare[0]] = 0, 0
    zeros, bad = x["table"].clone(), x["table"].clone()
    for b, j in ((0, 0), (3, 77), (3, 78), (11, 300)):
        zeros[b, j], bad[b, j] = spare[0], x["k"].shape[0] + b
    for _ in range(5):
        out = _run(b200, dict(x, table=bad))
        assert torch.equal(out, _run(b200, dict(x, table=zeros)))
    pg.check_attention(out, dict(x, table=zeros))
    assert status() == PAGE


@pytest.mark.parametrize("tokens", [1, 90])
def test_a_length_beyond_the_table_spoils_no_other_sequence(b200, cuda_device, status, tokens):
    seqs = [(tokens, 3000 - 100 * i) for i in range(10)]
    x = _batch(cuda_device, seqs)
    far = x["lengths"].clone()
    far[4] = 10 ** 9
    x["table"][4] = x["table"][3]
    clean = _run(b200, x)
    others = torch.ones(clean.shape[0], dtype=torch.bool, device=cuda_device)
    others[4 * tokens:5 * tokens] = False
    for _ in range(5):
        out = _run(b200, dict(x, lengths=far))
        pg.check_attention(torch.where(others[:, None, None], out, clean), x)
    assert status() & FULL

"""Layers in a row, each launched before the one before it has ended: the queries of a layer are the ones that its
append has just written, although every layer's are in the same memory."""

import pytest
import torch

import _paged as pg

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("seqs,prefix", [
    ([(1, 40)], 900), ([(1, 40 + i) for i in range(4)], 3000), ([(2, 30), (2, 90)], 200),  # few rows behind the prefix
    ([(1, 40 + i) for i in range(64)], 2000), ([(30, 60)] * 4, 700),                       # many
    ([(1, 600)], 0), ([(1, 900)] * 64, 0), ([(200, 300)], 0)])
def test_queries_are_the_layers_own(b200, cuda_device, seqs, prefix):
    layers = 60
    x = pg.build(seqs, Hq=12, Hkv=2, D=128, page=16, dtype=BF16, device=cuda_device, prefix=prefix)
    T = x["q"].shape[0]
    g = torch.Generator(device=cuda_device).manual_seed(1)
    new = torch.randn(layers, T, 16, 128, generator=g, device=cuda_device).to(BF16)
    cos, sin = b200.rope_table(4096, 128, device=cuda_device)
    count = torch.tensor([n for n, _ in seqs], dtype=torch.int32, device=cuda_device)
    before = x["lengths"] - count
    joint = torch.empty_like(new[0])

    def layer(i, out):
        joint.copy_(new[i])
        q = joint[:, :12]
        b200.b200_rope_paged_append(q, joint[:, 12:14], joint[:, 14:], x["k"], x["v"], x["table"], before, cos, sin,
                                    cu_tokens=x["cu"], q_out=q)
        how = dict(cu_tokens=x["cu"], max_tokens=x["most"], out=out)
        if prefix:
            b200.b200_shared_prefix_attention(q, x["k"], x["v"], x["prefix_table"], prefix, x["table"], x["lengths"],
                                              **how)
        else:
            b200.b200_paged_attention(q, x["k"], x["v"], x["table"], x["lengths"], **how)

    outs = torch.empty(2, layers, T, 12, 128, dtype=BF16, device=cuda_device)
    for i in range(layers):  # each alone
        torch.cuda.synchronize()
        layer(i, outs[0, i])
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(layers):
            layer(i, outs[1, i])
        assert torch.equal(outs[0], outs[1])
    # And from a graph, without the host between the launches.
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        for i in range(layers):
            layer(i, outs[1, i])
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(5):
        outs[1].zero_()
        graph.replay()
        assert torch.equal(outs[0], outs[1])

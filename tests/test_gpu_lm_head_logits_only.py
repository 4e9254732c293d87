"""b200_lm_head for the logits alone (no argmax, so no key words to merge into)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,d", [(1, 512, 256), (3, 1000, 1536), (8, 7, 64)])
def test_logits_without_argmax_equal_those_with_it(b200, cuda_device, m, n, d):
    g = torch.Generator().manual_seed(m)
    w = (torch.randn(n, d, generator=g) * 0.02).to(torch.bfloat16).to(cuda_device)
    x = torch.randn(m, d, generator=g).to(torch.bfloat16).to(cuda_device)
    logits, none = b200.b200_lm_head(x, w, return_argmax=False)
    torch.cuda.synchronize()
    assert none is None
    assert torch.equal(logits, b200.b200_lm_head(x, w)[0])

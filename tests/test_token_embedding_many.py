"""The table's gradient from more tokens than one CTA's counting holds: blocks that are
sorted each and merged by searches in all the others."""
import pytest
import torch

from metallora_b200 import _lib, kernels


@pytest.mark.gpu
@pytest.mark.parametrize("t", [16385, 70_001, 200_000])
@pytest.mark.parametrize("v,padding", [(50_000, None), (300, 7), (3, 1)])
def test_gradient_of_many_tokens(cuda, t, v, padding):
    """Whole numbers whose sums are exact in fp32 (below 2^24): equal to 64 bits'."""
    gen = torch.Generator(device=cuda).manual_seed(t + v)
    idx = (v * torch.rand(t, device=cuda, generator=gen).double() ** 3).long().clamp(max=v - 1)
    dy = torch.randint(-20, 21, (t, 12), device=cuda, generator=gen).float()
    keep = idx != (-1 if padding is None else padding)
    want = torch.zeros(v, 12, dtype=torch.float64, device=cuda)
    want.index_add_(0, idx[keep], dy[keep].double())
    got = kernels.embedding_bwd(dy, idx, v, padding_idx=padding)
    assert torch.equal(got.double(), want)
    assert torch.equal(got, kernels.embedding_bwd(dy, idx, v, padding_idx=padding))
    assert _lib.device_status(reset=True) == 0

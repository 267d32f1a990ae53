"""Calls of rotate and of the 8-bit cache that are all edge, vs 64 bits or the ordinary call."""

import pytest
import torch

from lsa_rocm_lab.port import pipeline

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate_of_keys_alone(interleaved):
    """No query heads: the keys come out as they do beside some."""
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(2, 5, n, 64, generator=g).to(torch.bfloat16).to(DEV) for n in (4, 2))
    w = torch.rand(2, 64, generator=g).add(0.5).to(DEV)
    rest = torch.arange(7, 12, device=DEV), pipeline.rotary_frequencies(64, device=DEV), w[0], w[1]
    want = pipeline.rotate(q, k, *rest, interleaved=interleaved)[1]
    none, got = pipeline.rotate(q[:, :, :0], k, *rest, interleaved=interleaved)
    assert none.shape == (2, 5, 0, 64) and torch.equal(got, want)

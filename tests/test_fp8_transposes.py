"""Weights whose transpose is not theirs, refused before anything runs."""
from __future__ import annotations

import pytest
import torch


def _blocks(rows, k, block_rows=128):
    return (torch.zeros((rows, -(-k // 128) * 128), dtype=torch.uint8).view(torch.float8_e4m3fn),
            torch.zeros((-(-rows // block_rows), -(-k // 512) * 4), dtype=torch.uint8).view(torch.float8_e8m0fnu))


@pytest.mark.parametrize("rows", [129, 255, 257, 300])
def test_a_transpose_of_another_k(rows):
    """The gradient would have as many columns as the transpose has rows."""
    from engraft_ngram_amd import fp8, norm
    q, scales = _blocks(140, 256)
    w = fp8.Fp8Weight(q, scales, 256, *_blocks(rows, 140))
    x = torch.zeros((3, 256)).requires_grad_()
    for call in (lambda: fp8.product_grad(torch.zeros((3, 140)), w), lambda: fp8.product(x, w), lambda: fp8.product(x[None], w, split=128),
                 lambda: norm.normed_product(x, None, None, w)):
        with pytest.raises(ValueError, match="transpose"):
            call()


def test_a_transpose_without_scales():
    from engraft_ngram_amd import fp8
    q, scales = _blocks(140, 256)
    w = fp8.Fp8Weight(q, scales, 256, _blocks(256, 140)[0])
    for call in (lambda: fp8.product_grad(torch.zeros((3, 140)), w), lambda: fp8.product(torch.zeros((3, 256)).requires_grad_(), w)):
        with pytest.raises(ValueError, match="transpose"):
            call()


def test_gradients_of_other_shapes():
    from engraft_ngram_amd import fp8
    q, scales = _blocks(140, 256)
    w = fp8.Fp8Weight(q, scales, 256, *_blocks(256, 140))
    with pytest.raises(ValueError, match="n"):
        fp8.product_grad(torch.zeros(()), w)

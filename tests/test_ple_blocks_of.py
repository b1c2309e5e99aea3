"""What kept 8-bit blocks take for the weights that they were made of, on the host."""
from __future__ import annotations

import weakref

import pytest
import torch


def _blocks(key, value):
    from engraft_ngram_amd import ple
    return ple.PleBlocks((), key.shape[0], value.shape[0], tuple((weakref.ref(x), ple._place(x)) for x in (key, value)))


def _refused(blocks, *ws):
    with pytest.raises(ValueError, match="quantize_projections"):
        blocks.check_weights(*ws)


def test_the_weights_and_views_of_all_of_them_are_known():
    key, value = torch.randn(8, 4), torch.randn(4, 4)
    blocks = _blocks(key, value)
    for ws in ((key, value), (key, None), (None, value), (None, None), (key.detach(), value.view(4, 4)), (torch.nn.Parameter(key), value)):
        blocks.check_weights(*ws)
    _refused(blocks, key.clone(), value)
    _refused(blocks, key[:4], value)
    _refused(blocks, key, value.T)
    _refused(blocks, value, key)


def test_weights_that_were_written_are_not():
    for write in (lambda x: x.mul_(2.0), lambda x: x[0].zero_(), lambda x: x.detach().add_(1.0)):
        key, value = torch.randn(8, 4), torch.randn(4, 4)
        blocks = _blocks(key, value)
        write(value)
        _refused(blocks, key, value)
        blocks.check_weights(key, None)


def test_weights_that_are_gone_or_moved_are_not():
    key, value = torch.randn(8, 4), torch.randn(4, 4)
    blocks, alias = _blocks(key, value), value.detach()
    blocks.check_weights(key, alias)
    value.data = torch.randn(4, 4)
    _refused(blocks, key, value)
    _refused(blocks, key, alias)
    blocks = _blocks(key, alias)
    del alias
    _refused(blocks, key, value)


def test_blocks_that_a_call_takes_itself_know_none():
    from engraft_ngram_amd import ple
    ple.PleBlocks((), 8, 4).check_weights(torch.zeros(8, 4), torch.zeros(4, 4))

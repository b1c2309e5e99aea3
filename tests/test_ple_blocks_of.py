"""What kept 8-bit blocks take for the weights that they were made of, on the host."""
from __future__ import annotations

import copy
import pickle
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


@pytest.mark.parametrize("copied", [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
def test_copied_blocks_know_none(copied):
    """Their values are the same; which weights they were made of is not known any more, and none has to be given."""
    from engraft_ngram_amd import fp8, ple
    key, value = torch.randn(8, 4), torch.randn(4, 4)
    blocks = _blocks(key, value)
    blocks.parts = (fp8.Fp8Weight(torch.arange(128, dtype=torch.uint8)[None], torch.full((1, 4), 127, dtype=torch.uint8), 4),)
    other = copied(blocks)
    assert (other.n_key, other.n_value, other.parts[0].k) == (8, 4, 4) and torch.equal(other.parts[0].q, blocks.parts[0].q)
    other.check_weights(None, None)
    _refused(other, key, None)
    _refused(other, None, value)
    _refused(ple.PleBlocks(blocks.parts, 8, 4), key, value)
    blocks.check_weights(key, value)

"""What the decoder block refuses of a cache, before it computes or stores anything."""
import pytest
import torch

import flashoverlap_b200  # noqa: F401
from flashoverlap_b200.models.decoder_block import TPDecoderBlock


class Cache:
    """Nothing but lengths; what would store or attend is not reached."""

    def __init__(self, *lengths):
        self.lengths = lengths

    def length(self, seq):
        return self.lengths[seq]


def block(hidden=256, heads=4, kv_heads=2):
    return TPDecoderBlock(None, hidden, 64, heads, kv_heads, device="cpu")   # no GEMMs either


def test_prompts_with_a_cache():
    x = torch.zeros(8, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="needs the sequences"):
        block()(x, x, 2, 4, cache=Cache())
    with pytest.raises(ValueError, match="empty"):
        block()(x, x, 2, 4, cache=Cache(0, 1), seqs=[0, 1])
    with pytest.raises(ValueError, match="heads of 64 or 128"):
        block(heads=8, kv_heads=8)(x, x, 2, 4, cache=Cache(0, 0), seqs=[0, 1])


def test_single_tokens():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    for h, r in ((x[:1], x), (x, x[:1]), (x.repeat(2, 1), x), (x.repeat(2, 1), x.repeat(2, 1))):
        with pytest.raises(ValueError, match="one row for each of the 2"):
            block().decode(h, r, Cache(3, 4), [0, 1])
    with pytest.raises(ValueError, match="heads of 64 or 128"):
        block(heads=8, kv_heads=8).decode(x, x, Cache(3, 4), [0, 1])
    many = block()
    many.heads, many.kv_heads = 258, 2
    for call in (lambda: many.decode(x, x, Cache(3, 4), [0, 1]), lambda: many(x, x, 2, 1, cache=Cache(0, 0), seqs=[0, 1])):
        with pytest.raises(ValueError, match="up to 128 query heads"):
            call()

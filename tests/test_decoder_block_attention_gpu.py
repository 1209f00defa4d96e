"""The attention inside the decoder block against 64 bits: what it gets from the projection, what it hands to the products
behind it.  (Whole steps can only be compared up to the roundings of five products.)"""
import pytest
import torch

import flashoverlap_b200  # noqa: F401
from attention_oracle import attend, check
from flashoverlap_b200.models import PagedKVCache
from flashoverlap_b200.models.decoder_block import TPDecoderBlock
from test_attention_gpu import BF16, FP16, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("heads,kv,dim,window,sinks", [(8, 2, 64, 0, 0), (8, 2, 64, 1, 0), (8, 8, 128, 50, 3), (4, 1, 128, 100, 1)])
def test_attention_of_a_block(dtype, heads, kv, dim, window, sinks):
    block = TPDecoderBlock(None, heads * dim, 64, heads, kv, dtype=dtype, window=window, sinks=sinks)
    block._project = lambda h: h @ block.w_qkv.t()
    seen = {}

    def after(attn, resid):
        seen["attn"] = attn.clone()
        return attn, resid

    block._after = after
    batch, first, steps = 3, 150, 5
    cache = PagedKVCache(40, 16, kv, dim, dtype=dtype)
    seqs = [cache.add() for _ in range(batch)]
    x = randn(batch, first + steps, heads * dim, dtype=dtype, seed=3)
    qkv = [(block._project(x[:, :first].reshape(batch * first, -1)).view(batch, first, -1, dim))]

    def compare(got, at, rows):
        """got [batch, rows, heads, dim]: of the tokens from position `at` on."""
        q, k, v = torch.cat(qkv, 1).split([heads, kv, kv], dim=2)
        for b in range(batch):
            for h in range(heads):
                want, tol = attend(q[b, at:at + rows, h], k[b, :, h * kv // heads], v[b, :, h * kv // heads], at, at + rows, window, sinks)
                check(got[b, :, h], want, tol, f"sequence {b}, head {h}, from {at} on")

    block(x[:, :first].reshape(batch * first, -1), x[:, :first].reshape(batch * first, -1), batch, first, cache=cache, seqs=seqs)
    if window:        # without one the block's prompts are the library's
        compare(seen["attn"].view(batch, first, heads, dim), 0, first)
    for t in range(first, first + steps):
        h = x[:, t]
        # the projection as decode computes it: rows of zeros behind the sequences'
        padded = torch.zeros(128, heads * dim, dtype=dtype, device="cuda")
        padded[:batch] = h
        qkv.append(block._project(padded)[:batch].view(batch, 1, -1, dim))
        block.decode(h, h, cache, seqs)
        assert seen["attn"].shape[0] == 128 and not seen["attn"][batch:].any()
        compare(seen["attn"][:batch].view(batch, 1, heads, dim), t, 1)

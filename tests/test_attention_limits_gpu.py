"""Attention at the borders of what it accepts: scales and scores near the ends of fp32, weights near the ends of fp16."""
import pytest
import torch

import flashoverlap_b200  # noqa: F401
from attention_oracle import attend, check  # noqa: F401
from flashoverlap_b200 import ops
from test_attention_gpu import BF16, FP16, Paged, check_prompt, ints, randn  # noqa: F401

pytestmark = pytest.mark.gpu

# (batch, sq, sk, heads, kv): so few pairs of tiles that their keys are divided over CTAs, and as many as need no division
SHAPES = [(1, 20, 3000, 8, 1), (2, 300, 300, 4, 2)]


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [1e-30, 1.5e-38, 1e-40])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 3)])
def test_scales_of_almost_nothing(dtype, dim, scale, window, sinks):
    # all scores are nearly zero: a row is the mean of the values it sees, however its keys are divided
    for batch, sq, sk, heads, kv in SHAPES:
        q = randn(batch, sq, heads, dim, dtype=dtype, seed=1)
        k, v = randn(batch, sk, kv, dim, dtype=dtype, seed=2), randn(batch, sk, kv, dim, dtype=dtype, seed=3)
        got = ops.prompt_attention(q, k, v, window=window, sinks=sinks, scale=scale)
        check_prompt(q, k, v, got, window, sinks, scale=scale)
    for lengths in ([40, 300], [9000, 33]):
        p = Paged(lengths, 1, dim, 16, dtype)
        q = randn(len(lengths), 5, dim, dtype=dtype)
        p.check(q, ops.paged_attention(q, p.cache, p.table, p.lengths, window=window, sinks=sinks, scale=scale), window, sinks, scale=scale)


def test_scores_near_the_lowest_number():
    # all scores within 0.8 % of the lowest number of fp32; scaled, they lie between -1357 and -1351
    scale, steps = 4e-36, torch.tensor([2.0 ** 63, 2.0 ** 63 * 255 / 256])
    for batch, sq, sk, heads, kv in SHAPES:
        q = torch.zeros(batch, sq, heads, 64, dtype=BF16, device="cuda")
        k, v = torch.zeros(batch, sk, kv, 64, dtype=BF16, device="cuda"), randn(batch, sk, kv, 64, dtype=BF16, seed=3)
        q[..., 0] = -255 / 128 * 2.0 ** 64
        k[..., 0] = steps[torch.arange(sk) % 7 // 3 % 2].cuda()[None, :, None]
        check_prompt(q, k, v, ops.prompt_attention(q, k, v, scale=scale), scale=scale)
